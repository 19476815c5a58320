// Per-head RMS norm of queries and keys, position rotation and (optionally) the Hadamard rotation of
// the head, in one pass over the data (mi_qk_norm_rope), and its gradients (mi_qk_norm_rope_backward).
//
//   n_i = x_i * rho * w_i,  rho = (mean x^2 + eps)^-1/2
//   pair (a, b), frequency f:  (a cos - b sin, b cos + a sin),  angle = position[axis(f)] * inv_freq[f]
//   y   = H_D / sqrt(D) * rotated           (with the Hadamard flag)
// and backwards, with g the gradient brought back through the two orthogonal maps (their transposes):
//   dw_i = sum over tokens and heads of g_i x_i rho
//   dx_i = rho (w_i g_i - x_i rho^2 mean(w g x))
//
// Layout.  A head of D values lies on D/16 lanes (a power of two of them, 2^lg, the rest idle), two
// runs of eight consecutive values ("units") per lane, chosen so that both members of every rotated
// pair are in one lane: units j and j + R/16 where the pairs are i, i + R/2; units 2j and 2j + 1 where
// they are neighbours, and in the part of the head that is not rotated.  Lane l holds j = l ^ (l >> 1)
// (Gray code): the lanes whose j differ in bit b alone are then l and l ^ (2^(b+1) - 1), which are
// row mirrors and quad permutes, so the sums and the Hadamard butterflies across lanes cost no LDS.
// Everything between the load and the one rounding at the store is fp32; angles are reduced in fp64.
#include <type_traits>

#include "common.hpp"

namespace mi {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxHalfRotary = 256;  // head_dim <= 512
constexpr uint32_t kMaxPartials = 1024;   // workgroups of the backward pass, each with a row of partial sums

struct HeadsArgs {
    const void* x[2];     // queries, keys
    const void* g[2];     // gradients of the outputs (backward)
    void* y[2];           // outputs; gradients of x (backward)
    const void* w[2];
    const void* positions;
    const void* freq;
    float* partials;      // [workgroups][2][D] (backward)
    uint64_t tokens;
    uint64_t x_ts[2], x_hs[2], g_ts[2], g_hs[2], y_ts[2], y_hs[2];  // token and head strides, elements
    uint32_t heads[2];
    uint32_t D, R, lg;
    uint32_t section_end[3];
    float eps, out_scale;
    bool w_f32, pos64, freq64, neighbours, hadamard, mixed;
    uint32_t tokens_per_block;  // 4: a wavefront per token; 1: the wavefronts share a token's heads
};

template <class E>
__device__ __forceinline__ void load_unit(const E* p, float (&v)[8])
{
    if constexpr (std::is_same<E, float>::value) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    } else {
        typedef E V8 __attribute__((ext_vector_type(8)));
        const V8 a = *reinterpret_cast<const V8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
    }
}

template <class E>
__device__ __forceinline__ void store_unit(E* p, const float (&v)[8])
{
    if constexpr (std::is_same<E, float>::value) {
        f32x4 a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) { a[i] = v[i]; b[i] = v[4 + i]; }
        *reinterpret_cast<f32x4*>(p) = a;
        *reinterpret_cast<f32x4*>(p + 4) = b;
    } else {
        typedef E V8 __attribute__((ext_vector_type(8)));
        V8 a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = (E)v[i];
        *reinterpret_cast<V8*>(p) = a;
    }
}

// The value of lane l ^ (2^(STEP+1) - 1).
template <int STEP>
__device__ __forceinline__ float mirror_lane(float v)
{
    if constexpr (STEP < 4) {
        constexpr int ctrl[4] = {0xB1, 0x1B, 0x141, 0x140};  // quad_perm 1,0,3,2 / 3,2,1,0; half row; row
        return __builtin_bit_cast(
            float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl[STEP], 0xf, 0xf, false));
    } else {
        return __shfl_xor(v, 31);
    }
}

__device__ __forceinline__ float lane_group_sum(float v, uint32_t lg)
{
    if (lg > 0) v += mirror_lane<0>(v);
    if (lg > 1) v += mirror_lane<1>(v);
    if (lg > 2) v += mirror_lane<2>(v);
    if (lg > 3) v += mirror_lane<3>(v);
    if (lg > 4) v += mirror_lane<4>(v);
    return v;
}

template <int STEP>
__device__ __forceinline__ void lane_butterfly(float (&v)[2][8], uint32_t j)
{
    const float s = (j >> STEP & 1u) ? -1.0f : 1.0f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = mirror_lane<STEP>(v[u][i]) + s * v[u][i];
}

// Unnormalised H_D over the head: the index bits are 3 in a unit, 1 between the lane's units and lg
// across lanes, and the stages commute.
__device__ __forceinline__ void head_butterflies(float (&v)[2][8], uint32_t j, uint32_t lg)
{
#pragma unroll
    for (int b = 1; b < 8; b <<= 1)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!(i & b)) {
                    const float p = v[u][i], q = v[u][i | b];
                    v[u][i] = p + q;
                    v[u][i | b] = p - q;
                }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float p = v[0][i], q = v[1][i];
        v[0][i] = p + q;
        v[1][i] = p - q;
    }
    if (lg > 0) lane_butterfly<0>(v, j);
    if (lg > 1) lane_butterfly<1>(v, j);
    if (lg > 2) lane_butterfly<2>(v, j);
    if (lg > 3) lane_butterfly<3>(v, j);
    if (lg > 4) lane_butterfly<4>(v, j);
}

// Where unit u of a head is while it is laid out for a partial rotation of halves (0 < R < D).
__device__ __forceinline__ void rotary_place(uint32_t u, uint32_t rl, uint32_t& j, uint32_t& slot)
{
    slot = u < rl ? 0u : u < 2u * rl ? 1u : u & 1u;
    j = u < rl ? u : u < 2u * rl ? u - rl : u >> 1;
}

// From the layout for a partial rotation of halves to units 2j, 2j + 1 in lane j (and back, BACK).
template <bool BACK>
__device__ __forceinline__ void relayout(float (&v)[2][8], uint32_t lane, uint32_t j, uint32_t lg, uint32_t rl)
{
    const uint32_t base = lane >> lg << lg;
    float out[2][8];
#pragma unroll
    for (uint32_t s = 0; s < 2; ++s) {
        uint32_t from_j, from_slot;
        if (BACK) {  // unit that this lane's slot s holds in the rotary layout, found in the plain one
            const uint32_t u = j < rl ? j + s * rl : 2u * j + s;
            from_j = u >> 1;
            from_slot = u & 1u;
        } else {
            rotary_place(2u * j + s, rl, from_j, from_slot);
        }
        // lane of a unit: the inverse of the Gray code
        uint32_t l = from_j;
        l ^= l >> 1;
        l ^= l >> 2;
        l ^= l >> 4;
        const int from = (int)(base | l);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = __shfl(v[0][i], from), q = __shfl(v[1][i], from);
            out[s][i] = from_slot ? q : p;
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = out[u][i];
}

// Rotation of a lane's eight pairs by its eight angles; DIR = -1 turns back.
template <int DIR>
__device__ __forceinline__ void rotate_pairs(float (&v)[2][8], const float (&c)[8], const float (&s)[8], bool neighbours)
{
    if (neighbours) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = v[u][2 * i], b = v[u][2 * i + 1], cc = c[4 * u + i], ss = DIR * s[4 * u + i];
                v[u][2 * i] = __builtin_fmaf(-b, ss, a * cc);
                v[u][2 * i + 1] = __builtin_fmaf(a, ss, b * cc);
            }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = v[0][i], b = v[1][i], cc = c[i], ss = DIR * s[i];
            v[0][i] = __builtin_fmaf(-b, ss, a * cc);
            v[1][i] = __builtin_fmaf(a, ss, b * cc);
        }
    }
}

// cos and sin of position * inv_freq.  The product and its reduction to a part of a turn are fp64: an
// fp32 angle of position 10^5 would be off by 4e-3.
__device__ __forceinline__ float2 turn(const HeadsArgs& a, uint64_t token, uint32_t f)
{
    const uint32_t axis = (f >= a.section_end[0]) + (f >= a.section_end[1]) + (f >= a.section_end[2]);
    const uint64_t at = axis * a.tokens + token;
    const double pos = a.pos64 ? (double)static_cast<const int64_t*>(a.positions)[at]
                               : (double)static_cast<const int32_t*>(a.positions)[at];
    const double freq = a.freq64 ? static_cast<const double*>(a.freq)[f] : (double)static_cast<const float*>(a.freq)[f];
    const double turns = pos * freq * 0.15915494309189533577;
    const float r = (float)(turns - __builtin_rint(turns));
    float2 cs;
    sincospif(2.0f * r, &cs.y, &cs.x);
    return cs;
}

// The lane's place in its head and in the wavefront.
struct LanePlace {
    uint32_t lane, group, groups, j, unit[2], plain[2];
    bool active, rotated;
    __device__ __forceinline__ explicit LanePlace(const HeadsArgs& a)
    {
        lane = threadIdx.x & 63u;
        const uint32_t l = lane & ((1u << a.lg) - 1u);
        group = lane >> a.lg;
        groups = 64u >> a.lg;
        j = l ^ (l >> 1);
        active = j < a.D / 16u;
        const uint32_t rl = a.R / 16u;
        rotated = j < rl;
        plain[0] = 16u * j;
        plain[1] = 16u * j + 8u;
        const bool halves = rotated && !a.neighbours;
        unit[0] = halves ? 8u * j : plain[0];
        unit[1] = halves ? 8u * (j + rl) : plain[1];
    }
};

__device__ __forceinline__ void load_weight(const HeadsArgs& a, const LanePlace& p, int kind, float (&w)[2][8], int dtype)
{
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) w[u][i] = 1.0f;
    if (!a.w[kind] || !p.active) return;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (dtype == MI_F32) load_unit(static_cast<const float*>(a.w[kind]) + p.unit[u], w[u]);
        else if (dtype == MI_BF16) load_unit(static_cast<const __bf16*>(a.w[kind]) + p.unit[u], w[u]);
        else load_unit(static_cast<const _Float16*>(a.w[kind]) + p.unit[u], w[u]);
    }
}

template <class E> constexpr int dtype_of = MI_F32;
template <> constexpr int dtype_of<__bf16> = MI_BF16;
template <> constexpr int dtype_of<_Float16> = MI_F16;

// Fills the cosine / sine table of the block's tokens.
__device__ __forceinline__ void fill_turns(const HeadsArgs& a, uint64_t first, float2 (*table)[kMaxHalfRotary])
{
    const uint32_t half = a.R / 2u;
    for (uint32_t i = threadIdx.x; i < a.tokens_per_block * half; i += kThreads) {
        const uint32_t t = i / half, f = i - t * half;
        if (first + t < a.tokens) table[t][f] = turn(a, first + t, f);
    }
}

template <class E>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(HeadsArgs a)
{
    __shared__ float2 table[4][kMaxHalfRotary];
    const LanePlace p(a);
    const uint32_t wave = threadIdx.x >> 6;
    const bool share = a.tokens_per_block == 1u;
    const uint32_t rl = a.R / 16u;
    const float inv_d = 1.0f / (float)a.D;
    const int wdt = a.w_f32 ? MI_F32 : dtype_of<E>;
    float w[2][2][8];
    load_weight(a, p, 0, w[0], wdt);
    load_weight(a, p, 1, w[1], wdt);

    for (uint64_t first = (uint64_t)blockIdx.x * a.tokens_per_block; first < a.tokens;
         first += (uint64_t)gridDim.x * a.tokens_per_block) {
        __syncthreads();  // the table is still being read for the previous tokens
        fill_turns(a, first, table);
        __syncthreads();
        const uint64_t token = first + (share ? 0u : wave);
        if (token >= a.tokens) continue;  // no wavefront leaves: every one meets the barriers above
        float c[8], s[8];
        if (p.rotated) {
            const float2* row = &table[share ? 0 : wave][8u * p.j];
#pragma unroll
            for (int i = 0; i < 8; ++i) { c[i] = row[i].x; s[i] = row[i].y; }
        }
        uint32_t pass = 0;
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
            const E* x = static_cast<const E*>(a.x[kind]) + token * a.x_ts[kind];
            E* y = static_cast<E*>(a.y[kind]) + token * a.y_ts[kind];
            for (uint32_t h0 = 0; h0 < a.heads[kind]; h0 += p.groups, ++pass) {
                if (share && (pass & 3u) != wave) continue;
                const uint32_t h = h0 + p.group;
                const bool here = p.active && h < a.heads[kind];
                float v[2][8] = {};
                if (here) {
                    load_unit(x + h * a.x_hs[kind] + p.unit[0], v[0]);
                    load_unit(x + h * a.x_hs[kind] + p.unit[1], v[1]);
                }
                float ss = 0.0f;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(v[u][i], v[u][i], ss);
                ss = lane_group_sum(ss, a.lg);
                const float rho = 1.0f / __builtin_sqrtf(__builtin_fmaf(ss, inv_d, a.eps)) * a.out_scale;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[u][i] = v[u][i] * rho * w[kind][u][i];
                if (p.rotated) rotate_pairs<1>(v, c, s, a.neighbours);
                if (a.hadamard) {
                    if (a.mixed) relayout<false>(v, p.lane, p.j, a.lg, rl);
                    head_butterflies(v, p.j, a.lg);
                }
                if (here) {
                    const bool moved = a.hadamard && a.mixed;
                    E* row = y + h * a.y_hs[kind];
                    store_unit(row + (moved ? p.plain[0] : p.unit[0]), v[0]);
                    store_unit(row + (moved ? p.plain[1] : p.unit[1]), v[1]);
                }
            }
        }
    }
}

template <class E>
__global__ void __launch_bounds__(256) qk_norm_rope_backward_kernel(HeadsArgs a)
{
    __shared__ float2 table[4][kMaxHalfRotary];
    const LanePlace p(a);
    const uint32_t wave = threadIdx.x >> 6;
    const bool share = a.tokens_per_block == 1u;
    const uint32_t rl = a.R / 16u;
    const float inv_d = 1.0f / (float)a.D;
    const int wdt = a.w_f32 ? MI_F32 : dtype_of<E>;
    float w[2][2][8], dw[2][2][8] = {};
    load_weight(a, p, 0, w[0], wdt);
    load_weight(a, p, 1, w[1], wdt);
    const bool moved = a.hadamard && a.mixed;
    const uint32_t g_unit[2] = {moved ? p.plain[0] : p.unit[0], moved ? p.plain[1] : p.unit[1]};

    for (uint64_t first = (uint64_t)blockIdx.x * a.tokens_per_block; first < a.tokens;
         first += (uint64_t)gridDim.x * a.tokens_per_block) {
        __syncthreads();
        fill_turns(a, first, table);
        __syncthreads();
        const uint64_t token = first + (share ? 0u : wave);
        if (token >= a.tokens) continue;
        float c[8], s[8];
        if (p.rotated) {
            const float2* row = &table[share ? 0 : wave][8u * p.j];
#pragma unroll
            for (int i = 0; i < 8; ++i) { c[i] = row[i].x; s[i] = row[i].y; }
        }
        uint32_t pass = 0;
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
            const E* x = static_cast<const E*>(a.x[kind]) + token * a.x_ts[kind];
            const E* g = static_cast<const E*>(a.g[kind]) + token * a.g_ts[kind];
            E* y = static_cast<E*>(a.y[kind]) + token * a.y_ts[kind];
            for (uint32_t h0 = 0; h0 < a.heads[kind]; h0 += p.groups, ++pass) {
                if (share && (pass & 3u) != wave) continue;
                const uint32_t h = h0 + p.group;
                const bool here = p.active && h < a.heads[kind];
                float v[2][8] = {}, d[2][8] = {};
                if (here) {
                    load_unit(x + h * a.x_hs[kind] + p.unit[0], v[0]);
                    load_unit(x + h * a.x_hs[kind] + p.unit[1], v[1]);
                    load_unit(g + h * a.g_hs[kind] + g_unit[0], d[0]);
                    load_unit(g + h * a.g_hs[kind] + g_unit[1], d[1]);
                }
                if (a.hadamard) {
                    head_butterflies(d, p.j, a.lg);
                    if (a.mixed) relayout<true>(d, p.lane, p.j, a.lg, rl);
                }
                if (p.rotated) rotate_pairs<-1>(d, c, s, a.neighbours);
                float ss = 0.0f, dot = 0.0f;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        d[u][i] *= a.out_scale;
                        ss = __builtin_fmaf(v[u][i], v[u][i], ss);
                        dot = __builtin_fmaf(d[u][i] * w[kind][u][i], v[u][i], dot);
                    }
                ss = lane_group_sum(ss, a.lg);
                dot = lane_group_sum(dot, a.lg);
                const float rho = 1.0f / __builtin_sqrtf(__builtin_fmaf(ss, inv_d, a.eps));
                const float back = rho * rho * dot * inv_d;
                float out[2][8];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        out[u][i] = rho * __builtin_fmaf(-back, v[u][i], d[u][i] * w[kind][u][i]);
                        dw[kind][u][i] = __builtin_fmaf(d[u][i] * rho, v[u][i], dw[kind][u][i]);
                    }
                if (here) {
                    E* row = y + h * a.y_hs[kind];
                    store_unit(row + p.unit[0], out[0]);
                    store_unit(row + p.unit[1], out[1]);
                }
            }
        }
    }

    // Weight gradients of the workgroup: over the lane groups, then over the wavefronts, always in the
    // same order.  Lanes without a head, or without a place in it, hold zeros.
    __shared__ float sums[4][2][512];
    if (!a.partials) return;
#pragma unroll
    for (int kind = 0; kind < 2; ++kind)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float t = dw[kind][u][i];
                for (uint32_t step = 1u << a.lg; step < 64u; step <<= 1) t += __shfl_xor(t, (int)step);
                if (p.active && p.group == 0) sums[wave][kind][p.unit[u] + i] = t;
            }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 2u * a.D; i += kThreads) {
        const uint32_t kind = i >= a.D, e = i - kind * a.D;
        a.partials[(uint64_t)blockIdx.x * 2u * a.D + i] =
            (sums[0][kind][e] + sums[1][kind][e]) + (sums[2][kind][e] + sums[3][kind][e]);
    }
}

// Weight gradients: sums of the workgroups' rows, four columns per workgroup.
__global__ void __launch_bounds__(256) weight_gradient_kernel(const float* partials, uint32_t rows, uint32_t D, void* dqw, void* dkw,
                                                              int dtype)
{
    __shared__ f32x4 part[256];
    const uint32_t col = blockIdx.x * 4u;
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t r = threadIdx.x; r < rows; r += 256u) t += *reinterpret_cast<const f32x4*>(partials + (uint64_t)r * 2u * D + col);
    part[threadIdx.x] = t;
    __syncthreads();
    for (uint32_t half = 128u; half; half >>= 1) {
        if (threadIdx.x < half) part[threadIdx.x] += part[threadIdx.x + half];
        __syncthreads();
    }
    if (threadIdx.x >= 4u) return;
    const uint32_t i = col + threadIdx.x;
    void* out = i >= D ? dkw : dqw;
    const uint32_t e = i >= D ? i - D : i;
    const float v = part[0][threadIdx.x];
    if (!out) return;
    if (dtype == MI_F32) static_cast<float*>(out)[e] = v;
    else if (dtype == MI_BF16) static_cast<__bf16*>(out)[e] = (__bf16)v;
    else static_cast<_Float16*>(out)[e] = (_Float16)v;
}

// Checks a call and fills the kernel's arguments; `tensors` is 4 forward (x, y) and 6 backward (x, g, y).
int make_args(const mi_heads* d, const void* const* tensors, int count, const void* positions, const void* inv_freq, HeadsArgs& a)
{
    if (!d) return MI_ERR_NULL;
    if (d->dtype != MI_F32 && d->dtype != MI_BF16 && d->dtype != MI_F16) return MI_ERR_DTYPE;
    if (d->weight_dtype != d->dtype && d->weight_dtype != MI_F32) return MI_ERR_DTYPE;
    if ((d->position_bits != 32u && d->position_bits != 64u) || (d->freq_bits != 32u && d->freq_bits != 64u))
        return MI_ERR_DTYPE;
    if (d->head_dim < 16u || d->head_dim > 512u || d->head_dim % 16u) return MI_ERR_SIZE;
    if (d->rotary_dim > d->head_dim || d->rotary_dim % 16u) return MI_ERR_SIZE;
    if ((d->flags & MI_HEADS_HADAMARD) && !is_pow2(d->head_dim)) return MI_ERR_SIZE;
    if (d->flags & ~(uint32_t)(MI_HEADS_HADAMARD | MI_HEADS_NEIGHBOURS)) return MI_ERR_SHAPE;
    if (d->axes < 1u || d->axes > 4u) return MI_ERR_SHAPE;
    uint32_t at = 0;
    for (uint32_t i = 0; i < d->axes; ++i) {
        if (d->section_end[i] < at) return MI_ERR_SHAPE;
        at = d->section_end[i];
    }
    if (at != d->rotary_dim / 2u) return MI_ERR_SHAPE;
    if (d->q_heads > 65536u || d->k_heads > 65536u || d->tokens >> 40) return MI_ERR_SHAPE;
    if (!(d->eps >= 0.0f)) return MI_ERR_SHAPE;
    a.tokens = d->tokens;
    a.heads[0] = d->q_heads;
    a.heads[1] = d->k_heads;
    a.D = d->head_dim;
    a.R = d->rotary_dim;
    a.lg = 0;
    while ((16u << a.lg) < a.D) ++a.lg;
    for (uint32_t i = 0; i < 3; ++i) a.section_end[i] = i + 1u < d->axes ? d->section_end[i] : 0xffffffffu;
    a.eps = d->eps;
    a.hadamard = d->flags & MI_HEADS_HADAMARD;
    a.neighbours = d->flags & MI_HEADS_NEIGHBOURS;
    a.mixed = !a.neighbours && a.R > 0 && a.R < a.D;
    a.out_scale = a.hadamard ? 1.0f / sqrtf((float)a.D) : 1.0f;
    a.w_f32 = d->weight_dtype == MI_F32;
    a.pos64 = d->position_bits == 64u;
    a.freq64 = d->freq_bits == 64u;
    a.positions = positions;
    a.freq = inv_freq;
    const uint64_t unit = d->dtype == MI_F32 ? 4u : 8u;  // elements of 16 bytes
    if (d->tokens == 0 || d->q_heads + d->k_heads == 0) return MI_OK;
    for (int i = 0; i < count; ++i) {
        if (a.heads[i & 1] == 0) continue;
        if (!tensors[i]) return MI_ERR_NULL;
        if (!aligned16(tensors[i]) || d->token_stride[i] % unit || d->head_stride[i] % unit) return MI_ERR_ALIGN;
    }
    if (a.R && (!positions || !inv_freq)) return MI_ERR_NULL;
    for (int kind = 0; kind < 2; ++kind) {
        const int out = count - 2 + kind;
        a.x[kind] = tensors[kind];
        a.x_ts[kind] = d->token_stride[kind];
        a.x_hs[kind] = d->head_stride[kind];
        a.g[kind] = count == 6 ? tensors[2 + kind] : nullptr;
        a.g_ts[kind] = d->token_stride[2 + kind];
        a.g_hs[kind] = d->head_stride[2 + kind];
        a.y[kind] = const_cast<void*>(tensors[out]);
        a.y_ts[kind] = d->token_stride[out];
        a.y_hs[kind] = d->head_stride[out];
    }
    return MI_OK;
}

// A wavefront per token once that gives every SIMD one (1024 tokens); fewer tokens than that are
// spread over four wavefronts each.
uint32_t tokens_per_block(uint64_t tokens) { return tokens >= 1024u ? 4u : 1u; }

}  // namespace
}  // namespace mi

extern "C" int mi_qk_norm_rope(const void* q, const void* k, const void* q_weight, const void* k_weight, const void* positions,
                               const void* inv_freq, void* q_out, void* k_out, const mi_heads* d, void* stream)
{
    using namespace mi;
    HeadsArgs a = {};
    const void* tensors[4] = {q, k, q_out, k_out};
    const int st = make_args(d, tensors, 4, positions, inv_freq, a);
    if (st != MI_OK) return st;
    if (d->tokens == 0 || d->q_heads + d->k_heads == 0) return MI_OK;
    a.w[0] = q_weight;
    a.w[1] = k_weight;
    if ((q_weight && !aligned16(q_weight)) || (k_weight && !aligned16(k_weight))) return MI_ERR_ALIGN;
    a.tokens_per_block = tokens_per_block(d->tokens);
    const uint64_t blocks = (d->tokens + a.tokens_per_block - 1u) / a.tokens_per_block;
    const dim3 grid((uint32_t)(blocks < 2048u ? blocks : 2048u));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (d->dtype == MI_F32) hipLaunchKernelGGL((qk_norm_rope_kernel<float>), grid, dim3(kThreads), 0, s, a);
    else if (d->dtype == MI_BF16) hipLaunchKernelGGL((qk_norm_rope_kernel<__bf16>), grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((qk_norm_rope_kernel<_Float16>), grid, dim3(kThreads), 0, s, a);
    return launch_status();
}

extern "C" uint64_t mi_qk_norm_rope_workspace(uint64_t tokens, uint32_t head_dim)
{
    using namespace mi;
    const uint32_t per = tokens_per_block(tokens);
    const uint64_t blocks = tokens / per + (tokens % per != 0);
    return (blocks < kMaxPartials ? blocks : kMaxPartials) * 2u * head_dim * sizeof(float);
}

extern "C" int mi_qk_norm_rope_backward(const void* q, const void* k, const void* q_grad, const void* k_grad, const void* q_weight,
                                        const void* k_weight, const void* positions, const void* inv_freq, void* dq, void* dk,
                                        void* dq_weight, void* dk_weight, void* workspace, const mi_heads* d, void* stream)
{
    using namespace mi;
    HeadsArgs a = {};
    const void* tensors[6] = {q, k, q_grad, k_grad, dq, dk};
    const int st = make_args(d, tensors, 6, positions, inv_freq, a);
    if (st != MI_OK) return st;
    a.w[0] = q_weight;
    a.w[1] = k_weight;
    if ((q_weight && !aligned16(q_weight)) || (k_weight && !aligned16(k_weight))) return MI_ERR_ALIGN;
    const bool any = d->tokens != 0 && d->q_heads + d->k_heads != 0;
    const bool weights = dq_weight || dk_weight;
    if (weights && any && !workspace) return MI_ERR_NULL;
    if (weights && any && !aligned16(workspace)) return MI_ERR_ALIGN;
    hipStream_t s = static_cast<hipStream_t>(stream);
    uint32_t grid = 0;
    if (any) {
        a.partials = weights ? static_cast<float*>(workspace) : nullptr;
        a.tokens_per_block = tokens_per_block(d->tokens);
        const uint64_t blocks = (d->tokens + a.tokens_per_block - 1u) / a.tokens_per_block;
        grid = (uint32_t)(blocks < kMaxPartials ? blocks : kMaxPartials);
        if (d->dtype == MI_F32) hipLaunchKernelGGL((qk_norm_rope_backward_kernel<float>), dim3(grid), dim3(kThreads), 0, s, a);
        else if (d->dtype == MI_BF16) hipLaunchKernelGGL((qk_norm_rope_backward_kernel<__bf16>), dim3(grid), dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((qk_norm_rope_backward_kernel<_Float16>), dim3(grid), dim3(kThreads), 0, s, a);
        const int launched = launch_status();
        if (launched != MI_OK) return launched;
    }
    if (weights) {
        hipLaunchKernelGGL(weight_gradient_kernel, dim3(a.D / 2u), dim3(256), 0, s, static_cast<const float*>(workspace), grid, a.D,
                           dq_weight, dk_weight, d->weight_dtype);
        return launch_status();
    }
    return MI_OK;
}
