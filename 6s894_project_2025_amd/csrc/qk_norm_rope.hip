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
//
// Work.  A wavefront takes 64 / 2^lg heads at a time (an item).  Workgroups are for the query heads or for
// the key heads, so that one set of weights stays in registers; a unit of work is a token's heads, or a part of
// them where there are few tokens.  A wavefront computes the sines and cosines of its token once (one angle
// per lane, exchanged through LDS that no other wavefront uses, so there is no barrier) and keeps requests
// for the next items, of its next tokens too, in flight.
//
// Bound: memory.  8192 tokens of 32 + 8 heads of 128 in bf16, out of packed rows, with the Hadamard rotation: 168 MB
// in 32.5 us (5.2 TB/s; a copy of 512 MB runs at 5.4), 2 us of it the rotation; the backward pass 252 MB in 54 us
// (4.7 TB/s), 4 us of it the sums of the weight gradients.  fp32: 4096 tokens in 33 and 51 us (5.1 and 4.9 TB/s).
#include <type_traits>

#include "common.hpp"

namespace mi {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxHalfRotary = 256;  // angles of a token, head_dim <= 512
constexpr uint32_t kMaxBlocks = 2048;     // eight workgroups per compute unit
constexpr uint32_t kMaxPartials = 512;    // of the backward pass: two per compute unit; each has a row of partial sums

struct Side {          // the queries, or the keys
    const void* x;
    const void* g;     // gradients of the outputs (backward)
    void* y;           // outputs; gradients of x (backward)
    const void* w;
    uint64_t x_ts, x_hs, g_ts, g_hs, y_ts, y_hs;  // token and head strides, elements
    uint32_t heads, lg_parts, blocks;             // wavefronts that share a token's heads; workgroups
};

struct HeadsArgs {
    Side q, k;
    const void* positions;
    const void* freq;
    float* partials;      // [workgroups][D] (backward)
    uint64_t tokens;
    uint32_t D, R, lg;
    uint32_t section_end[3];
    float eps, out_scale;
    bool w_f32, pos64, freq64, neighbours, hadamard, mixed;
};

// A lane's unit as it comes from memory.
template <class E> struct Raw { u32x4 v; };
template <> struct Raw<float> { u32x4 v, w; };

template <class E>
__device__ __forceinline__ void fetch(Raw<E>& r, const E* p)
{
    r.v = *reinterpret_cast<const u32x4*>(p);
    if constexpr (std::is_same<E, float>::value) r.w = *reinterpret_cast<const u32x4*>(p + 4);
}

template <class E>
__device__ __forceinline__ void unpack(const Raw<E>& r, float (&v)[8])
{
    if constexpr (std::is_same<E, float>::value) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = __builtin_bit_cast(float, (uint32_t)r.v[i]);
            v[4 + i] = __builtin_bit_cast(float, (uint32_t)r.w[i]);
        }
    } else {
        typedef E V8 __attribute__((ext_vector_type(8)));
        const V8 a = __builtin_bit_cast(V8, r.v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
    }
}

// Both units of a lane.  The values are pinned here, before the next request takes the registers they came in.
template <class E>
__device__ __forceinline__ void unpack_units(const Raw<E> (&r)[2], float (&v)[2][8])
{
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        unpack(r[u], v[u]);
        asm volatile("" : "+v"(v[u][0]), "+v"(v[u][1]), "+v"(v[u][2]), "+v"(v[u][3]), "+v"(v[u][4]), "+v"(v[u][5]), "+v"(v[u][6]), "+v"(v[u][7]));
    }
}

// Streaming stores: what a pass over a large batch writes is not read again before it would be evicted, and the
// heads of 8192 tokens took 34.5 us with them against 41.6.  Not for fp32, where one instruction writes every
// other 16 bytes of a line: 8192 tokens take 74 us with them against 66, the backward pass of 4096 tokens 58
// against 51 (4096 tokens forward 32 against 33).
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
        __builtin_nontemporal_store(a, reinterpret_cast<V8*>(p));
    }
}

// The value of lane l ^ (2^(STEP+1) - 1).
template <int STEP>
__device__ __forceinline__ float mirror_lane(float v)
{
    if constexpr (STEP < 4) {
        constexpr int ctrl[4] = {0xB1, 0x1B, 0x141, 0x140};  // quad_perm 1,0,3,2 / 3,2,1,0; half row; row
        return __builtin_bit_cast(
            float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl[STEP], 0xf, 0xf, true));
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

// One butterfly stage across lanes: with s = -1 in the lanes whose bit is set, the stage is
// partner + s own; s (partner + s own) = own + s partner is one instruction per value instead of two.
// The factor s stays in the lane and meets the partners' equal one in the other stages; what is left
// at the end is one sign per lane, lane_sign().
template <int STEP>
__device__ __forceinline__ void lane_butterfly(float (&v)[2][8], uint32_t j)
{
    const float s = (j >> STEP & 1u) ? -1.0f : 1.0f;
    if constexpr (STEP < 4) {
        // The compiler moves the partner's value into a register of its own first.  A register that a
        // vector instruction has just written may be read across lanes two issue slots later.
#define MI_STAGE8(u, CTRL)                                                                                            \
    asm("s_nop 1\n\t"                                                                                                \
        "v_fmac_f32_dpp %0, %0, %8 " CTRL " row_mask:0xf bank_mask:0xf\n\tv_fmac_f32_dpp %1, %1, %8 " CTRL          \
        " row_mask:0xf bank_mask:0xf\n\tv_fmac_f32_dpp %2, %2, %8 " CTRL                                             \
        " row_mask:0xf bank_mask:0xf\n\tv_fmac_f32_dpp %3, %3, %8 " CTRL                                             \
        " row_mask:0xf bank_mask:0xf\n\tv_fmac_f32_dpp %4, %4, %8 " CTRL                                             \
        " row_mask:0xf bank_mask:0xf\n\tv_fmac_f32_dpp %5, %5, %8 " CTRL                                             \
        " row_mask:0xf bank_mask:0xf\n\tv_fmac_f32_dpp %6, %6, %8 " CTRL                                             \
        " row_mask:0xf bank_mask:0xf\n\tv_fmac_f32_dpp %7, %7, %8 " CTRL " row_mask:0xf bank_mask:0xf"               \
        : "+v"(v[u][0]), "+v"(v[u][1]), "+v"(v[u][2]), "+v"(v[u][3]), "+v"(v[u][4]), "+v"(v[u][5]), "+v"(v[u][6]),     \
          "+v"(v[u][7])                                                                                               \
        : "v"(s))
        if constexpr (STEP == 0) { MI_STAGE8(0, "quad_perm:[1,0,3,2]"); MI_STAGE8(1, "quad_perm:[1,0,3,2]"); }
        if constexpr (STEP == 1) { MI_STAGE8(0, "quad_perm:[3,2,1,0]"); MI_STAGE8(1, "quad_perm:[3,2,1,0]"); }
        if constexpr (STEP == 2) { MI_STAGE8(0, "row_half_mirror"); MI_STAGE8(1, "row_half_mirror"); }
        if constexpr (STEP == 3) { MI_STAGE8(0, "row_mirror"); MI_STAGE8(1, "row_mirror"); }
#undef MI_STAGE8
    } else {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u][i] = __builtin_fmaf(mirror_lane<STEP>(v[u][i]), s, v[u][i]);
    }
}
__device__ __forceinline__ float lane_sign(uint32_t j) { return __popc(j) & 1 ? -1.0f : 1.0f; }

// lane_sign * unnormalised H_D over the head: the index bits are 3 in a unit, 1 between the lane's units
// and lg across lanes, and the stages commute.
__device__ __forceinline__ void head_butterflies(float (&v)[2][8], uint32_t j, uint32_t lg)
{
    if (lg > 0) lane_butterfly<0>(v, j);
    if (lg > 1) lane_butterfly<1>(v, j);
    if (lg > 2) lane_butterfly<2>(v, j);
    if (lg > 3) lane_butterfly<3>(v, j);
    if (lg > 4) lane_butterfly<4>(v, j);
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
}

// From the layout for a partial rotation of halves (0 < R < D) to units 2j, 2j + 1 in lane j, or back.
template <bool BACK>
__device__ __forceinline__ void relayout(float (&v)[2][8], uint32_t lane, uint32_t j, uint32_t lg, uint32_t rl)
{
    const uint32_t base = lane >> lg << lg;
    float out[2][8];
#pragma unroll
    for (uint32_t s = 0; s < 2; ++s) {
        uint32_t from_j, from_slot;
        if (BACK) {  // the unit of slot s in the rotary layout, found in the plain one
            const uint32_t u = j < rl ? j + s * rl : 2u * j + s;
            from_j = u >> 1;
            from_slot = u & 1u;
        } else {
            const uint32_t u = 2u * j + s;
            from_slot = u < rl ? 0u : u < 2u * rl ? 1u : s;
            from_j = u < rl ? u : u < 2u * rl ? u - rl : j;
        }
        uint32_t l = from_j;  // its lane: the inverse of the Gray code
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
template <int DIR, bool NEIGHBOURS>
__device__ __forceinline__ void rotate_pairs(float (&v)[2][8], const float2 (&cs)[8])
{
    if (NEIGHBOURS) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = v[u][2 * i], b = v[u][2 * i + 1], c = cs[4 * u + i].x, s = DIR * cs[4 * u + i].y;
                v[u][2 * i] = __builtin_fmaf(-b, s, a * c);
                v[u][2 * i + 1] = __builtin_fmaf(a, s, b * c);
            }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = v[0][i], b = v[1][i], c = cs[i].x, s = DIR * cs[i].y;
            v[0][i] = __builtin_fmaf(-b, s, a * c);
            v[1][i] = __builtin_fmaf(a, s, b * c);
        }
    }
}

// A lane's angles: frequencies lane, lane + 64, ... (FREQS of them) of the wavefront's token.  The product of position and
// frequency and its reduction to a part of a turn are fp64: an fp32 angle of position 10^5 would be
// off by 4e-3.
template <uint32_t FREQS, uint32_t I = 0>
struct Turns {
    double freq = 0.0;           // turns per position
    uint64_t at = 0;             // of the lane's axis in positions
    uint32_t low = 0, high = 0;  // the position as it comes from memory
    Turns<FREQS, I + 1> rest;

    __device__ __forceinline__ explicit Turns(const HeadsArgs& a) : rest(a)
    {
        const uint32_t f = (threadIdx.x & 63u) + 64u * I;
        if (f < a.R / 2u) {
            freq = a.freq64 ? static_cast<const double*>(a.freq)[f] : (double)static_cast<const float*>(a.freq)[f];
            freq *= 0.15915494309189533577;
            at = ((f >= a.section_end[0]) + (f >= a.section_end[1]) + (f >= a.section_end[2])) * a.tokens;
        }
    }
    __device__ __forceinline__ void request(const HeadsArgs& a, uint64_t token)  // not without frequencies
    {
        const uint32_t* words = static_cast<const uint32_t*>(a.positions) + ((at + token) << a.pos64);
        low = words[0];
        high = words[a.pos64];  // not used with 32 bits; no branch, so that the loads can be counted
        rest.request(a, token);
    }
    __device__ __forceinline__ void fill(const HeadsArgs& a, float2* table)
    {
        const uint32_t f = (threadIdx.x & 63u) + 64u * I;
        const double pos = a.pos64 ? (double)(int64_t)((uint64_t)high << 32 | low) : (double)(int32_t)low;
        const double turns = pos * freq;
        const float r = (float)(turns - __builtin_rint(turns));
        float2 cs;
        sincospif(2.0f * r, &cs.y, &cs.x);
        if (f < a.R / 2u) table[f] = cs;
        rest.fill(a, table);
    }
};
template <uint32_t FREQS>
struct Turns<FREQS, FREQS> {
    __device__ __forceinline__ explicit Turns(const HeadsArgs&) {}
    __device__ __forceinline__ void request(const HeadsArgs&, uint64_t) {}
    __device__ __forceinline__ void fill(const HeadsArgs&, float2*) {}
};

// The lane's place in its head and in the wavefront.  A lane without a part of the head (head_dim / 16 is not a
// power of two) does what the first lane does, and its sums count as zero; lanes behind the last head do
// what the last head's lanes do.  They store the same values to the same place, so every load and store is
// made by all lanes: behind a branch, a wait for one request would be a wait for all.
struct LanePlace {
    uint32_t lane, group, groups, j, unit[2], plain[2];
    bool active, rotated;
    __device__ __forceinline__ LanePlace(const HeadsArgs& a, uint32_t lg, bool neighbours)
    {
        lane = threadIdx.x & 63u;
        const uint32_t l = lane & ((1u << lg) - 1u);
        group = lane >> lg;
        groups = 64u >> lg;
        j = l ^ (l >> 1);
        active = j < a.D / 16u;
        if (!active) j = 0;
        const uint32_t rl = a.R / 16u;
        rotated = j < rl;
        plain[0] = 16u * j;
        plain[1] = 16u * j + 8u;
        const bool halves = rotated && !neighbours;
        unit[0] = halves ? 8u * j : plain[0];
        unit[1] = halves ? 8u * (j + rl) : plain[1];
    }
    __device__ __forceinline__ uint64_t head(uint32_t pass, uint32_t heads) const
    {
        const uint32_t h = pass * groups + group;
        return h < heads ? h : heads - 1u;
    }
};

template <class E>
__device__ __forceinline__ void load_weight(const HeadsArgs& a, const void* weight, const LanePlace& p, float (&w)[2][8])
{
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) w[u][i] = 1.0f;
    if (!weight) return;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (a.w_f32) {
            Raw<float> r;
            fetch(r, static_cast<const float*>(weight) + p.unit[u]);
            unpack(r, w[u]);
        } else {
            Raw<E> r;
            fetch(r, static_cast<const E*>(weight) + p.unit[u]);
            unpack(r, w[u]);
        }
    }
}

// Waits for every load so far (s_waitcnt vmcnt(0)).  Inside the loops each wait then stands behind the same
// loads and stores on every path, and the compiler lets the later ones stay in flight; without it the way
// in, which may have none behind it, would have every item wait for the item before it to be stored.
__device__ __forceinline__ void first_loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// A wavefront's way through its items: units (a token's heads, every 2^lg_parts-th group of them) in steps of
// all the side's wavefronts.
struct Cursor {
    uint64_t unit, stride;
    uint32_t lg_parts, per_token, pass;
    __device__ __forceinline__ Cursor(const Side& s, uint32_t groups, uint32_t wavefront)
        : unit(wavefront), stride(4u * s.blocks), lg_parts(s.lg_parts), per_token((s.heads + groups - 1u) / groups)
    {
        pass = (uint32_t)unit & ((1u << lg_parts) - 1u);
    }
    __device__ __forceinline__ uint64_t token() const { return unit >> lg_parts; }
    // true when the next item is another token's
    __device__ __forceinline__ bool next()
    {
        pass += 1u << lg_parts;
        if (pass < per_token) return false;
        unit += stride;
        pass = (uint32_t)unit & ((1u << lg_parts) - 1u);
        return true;
    }
};

// LG < 0: a.lg, any head size.  The common ones have kernels of their own (the branches on a run-time lg
// keep the stages from overlapping).
template <class E, int LG, bool NEIGHBOURS>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(HeadsArgs a)
{
    __shared__ float2 tables[4][kMaxHalfRotary];
    const uint32_t lg = LG < 0 ? a.lg : (uint32_t)LG;
    const LanePlace p(a, lg, NEIGHBOURS);
    const bool keys = blockIdx.x >= a.q.blocks;
    const Side side = keys ? a.k : a.q;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t heads = side.heads;
    const bool hadamard = a.hadamard, mixed = !NEIGHBOURS && hadamard && a.mixed;
    const E* x = static_cast<const E*>(side.x);
    E* y = static_cast<E*>(side.y);
    float2* table = tables[wave];

    Raw<E> raw[2];
    Cursor ahead(side, p.groups, 4u * (blockIdx.x - (keys ? a.q.blocks : 0u)) + wave), item = ahead;
    auto request = [&]() __attribute__((always_inline)) {
        // behind the last item: the first token's row, which the cache holds
        const uint64_t token = ahead.token() < a.tokens ? ahead.token() : 0u;
        const E* row = x + token * side.x_ts + p.head(ahead.pass, heads) * side.x_hs;
        fetch(raw[0], row + p.unit[0]);
        fetch(raw[1], row + p.unit[1]);
        ahead.next();
    };
    if (item.token() >= a.tokens) return;
    request();
    Turns<LG < 0 ? 4 : LG < 4 ? 1 : 2> turns(a);
    if (a.R) turns.request(a, item.token());
    float w[2][8];
    load_weight<E>(a, side.w, p, w);
    const float inv_d = 1.0f / (float)a.D;
    const float sign = hadamard ? lane_sign(p.j) * a.out_scale : 1.0f;
    float2 cs[8];
    first_loads_done();

    while (item.token() < a.tokens) {
        __builtin_amdgcn_wave_barrier();
        turns.fill(a, table);
        __builtin_amdgcn_wave_barrier();
        if (p.rotated)
#pragma unroll
            for (int i = 0; i < 8; ++i) cs[i] = table[8u * p.j + i];
        const uint64_t next = (item.unit + item.stride) >> item.lg_parts;
        if (a.R) turns.request(a, next < a.tokens ? next : 0u);
        do {
            float v[2][8];
            unpack_units(raw, v);
            request();
            float ss = 0.0f;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    ss = __builtin_fmaf(v[u][i], v[u][i], ss);
                    v[u][i] *= w[u][i];
                }
            if (p.rotated) rotate_pairs<1, NEIGHBOURS>(v, cs);
            ss = lane_group_sum(p.active ? ss : 0.0f, lg);
            const float rho = 1.0f / __builtin_sqrtf(__builtin_fmaf(ss, inv_d, a.eps)) * sign;
            if (hadamard) {
                if (mixed) relayout<false>(v, p.lane, p.j, lg, a.R / 16u);
                head_butterflies(v, p.j, lg);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[u][i] *= rho;
            E* row = y + item.token() * side.y_ts + p.head(item.pass, heads) * side.y_hs;
            store_unit(row + (mixed ? p.plain[0] : p.unit[0]), v[0]);
            store_unit(row + (mixed ? p.plain[1] : p.unit[1]), v[1]);
        } while (!item.next());
    }
}

template <class E, int LG, bool NEIGHBOURS>
__global__ void __launch_bounds__(256) qk_norm_rope_backward_kernel(HeadsArgs a)
{
    __shared__ float2 tables[4][kMaxHalfRotary];
    __shared__ float sums[4][512];
    const uint32_t lg = LG < 0 ? a.lg : (uint32_t)LG;
    const LanePlace p(a, lg, NEIGHBOURS);
    const bool keys = blockIdx.x >= a.q.blocks;
    const Side side = keys ? a.k : a.q;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t heads = side.heads;
    const bool hadamard = a.hadamard, mixed = !NEIGHBOURS && hadamard && a.mixed;
    const uint32_t g_unit[2] = {mixed ? p.plain[0] : p.unit[0], mixed ? p.plain[1] : p.unit[1]};
    const E* x = static_cast<const E*>(side.x);
    const E* g = static_cast<const E*>(side.g);
    E* y = static_cast<E*>(side.y);
    float2* table = tables[wave];
    const float inv_d = 1.0f / (float)a.D;
    const float sign = hadamard ? lane_sign(p.j) * a.out_scale : 1.0f;

    Raw<E> rx[2], rg[2];
    Cursor ahead(side, p.groups, 4u * (blockIdx.x - (keys ? a.q.blocks : 0u)) + wave), item = ahead;
    auto request = [&]() __attribute__((always_inline)) {
        const uint64_t token = ahead.token() < a.tokens ? ahead.token() : 0u, h = p.head(ahead.pass, heads);
        const E* row = x + token * side.x_ts + h * side.x_hs;
        const E* grad = g + token * side.g_ts + h * side.g_hs;
        fetch(rx[0], row + p.unit[0]);
        fetch(rx[1], row + p.unit[1]);
        fetch(rg[0], grad + g_unit[0]);
        fetch(rg[1], grad + g_unit[1]);
        ahead.next();
    };
    request();
    Turns<LG < 0 ? 4 : LG < 4 ? 1 : 2> turns(a);
    if (a.R) turns.request(a, item.token() < a.tokens ? item.token() : 0u);
    float w[2][8], dw[2][8] = {};
    load_weight<E>(a, side.w, p, w);
    float2 cs[8];
    first_loads_done();

    while (item.token() < a.tokens) {
        __builtin_amdgcn_wave_barrier();
        turns.fill(a, table);
        __builtin_amdgcn_wave_barrier();
        if (p.rotated)
#pragma unroll
            for (int i = 0; i < 8; ++i) cs[i] = table[8u * p.j + i];
        const uint64_t next = (item.unit + item.stride) >> item.lg_parts;
        if (a.R) turns.request(a, next < a.tokens ? next : 0u);
        do {
            float v[2][8], d[2][8];
            unpack_units(rx, v);
            unpack_units(rg, d);
            request();
            float ss = 0.0f;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(v[u][i], v[u][i], ss);
            ss = lane_group_sum(p.active ? ss : 0.0f, lg);
            const float rho = 1.0f / __builtin_sqrtf(__builtin_fmaf(ss, inv_d, a.eps));
            if (hadamard) {
                head_butterflies(d, p.j, lg);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[u][i] *= sign;
                if (mixed) relayout<true>(d, p.lane, p.j, lg, a.R / 16u);
            }
            if (p.rotated) rotate_pairs<-1, NEIGHBOURS>(d, cs);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[u][i] *= rho;  // the normed value
            if (p.active && item.pass * p.groups + p.group < heads) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 8; ++i) dw[u][i] = __builtin_fmaf(d[u][i], v[u][i], dw[u][i]);
            }
            float dot = 0.0f;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    d[u][i] *= w[u][i];
                    dot = __builtin_fmaf(d[u][i], v[u][i], dot);
                }
            const float mean = lane_group_sum(p.active ? dot : 0.0f, lg) * inv_d;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) d[u][i] = rho * __builtin_fmaf(-mean, v[u][i], d[u][i]);
            E* row = y + item.token() * side.y_ts + p.head(item.pass, heads) * side.y_hs;
            store_unit(row + p.unit[0], d[0]);
            store_unit(row + p.unit[1], d[1]);
        } while (!item.next());
    }

    // Weight gradients of the workgroup: over the lane groups, then over the wavefronts, always in the
    // same order.  Lanes without a head hold zeros.
    if (!a.partials) return;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float t = dw[u][i];
            for (uint32_t step = 1u << lg; step < 64u; step <<= 1) t += __shfl_xor(t, (int)step);
            if (p.active && p.group == 0) sums[wave][p.unit[u] + i] = t;
        }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.D; i += kThreads)
        a.partials[(uint64_t)blockIdx.x * a.D + i] = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
}

// Weight gradients: sums of the workgroups' rows, four columns per workgroup; blockIdx.y is the kind.
__global__ void __launch_bounds__(256) weight_gradient_kernel(const float* partials, uint32_t rows_q, uint32_t rows_k, uint32_t D,
                                                              void* dqw, void* dkw, int dtype)
{
    __shared__ f32x4 part[256];
    const uint32_t col = blockIdx.x * 4u, r0 = blockIdx.y ? rows_q : 0u, r1 = r0 + (blockIdx.y ? rows_k : rows_q);
    void* out = blockIdx.y ? dkw : dqw;
    if (!out) return;
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t r = r0 + threadIdx.x; r < r1; r += 256u) t += *reinterpret_cast<const f32x4*>(partials + (uint64_t)r * D + col);
    part[threadIdx.x] = t;
    __syncthreads();
    for (uint32_t half = 128u; half; half >>= 1) {
        if (threadIdx.x < half) part[threadIdx.x] += part[threadIdx.x + half];
        __syncthreads();
    }
    if (threadIdx.x >= 4u) return;
    const uint32_t i = col + threadIdx.x;
    const float v = part[0][threadIdx.x];
    if (dtype == MI_F32) static_cast<float*>(out)[i] = v;
    else if (dtype == MI_BF16) static_cast<__bf16*>(out)[i] = (__bf16)v;
    else static_cast<_Float16*>(out)[i] = (_Float16)v;
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
    a.q.heads = d->q_heads;
    a.k.heads = d->k_heads;
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
        if ((i & 1 ? d->k_heads : d->q_heads) == 0) continue;
        if (!tensors[i]) return MI_ERR_NULL;
        // outputs whose heads would overlap
        if (i >= count - 2 && ((d->tokens > 1u && d->token_stride[i] < a.D) || ((i & 1 ? d->k_heads : d->q_heads) > 1u && d->head_stride[i] < a.D)))
            return MI_ERR_SHAPE;
        if (!aligned16(tensors[i]) || d->token_stride[i] % unit || d->head_stride[i] % unit) return MI_ERR_ALIGN;
    }
    if (a.R && (!positions || !inv_freq)) return MI_ERR_NULL;
    if (a.R && (reinterpret_cast<uintptr_t>(positions) % (d->position_bits / 8u) || reinterpret_cast<uintptr_t>(inv_freq) % (d->freq_bits / 8u)))
        return MI_ERR_ALIGN;
    for (int kind = 0; kind < 2; ++kind) {
        const int out = count - 2 + kind;
        Side& side = kind ? a.k : a.q;
        side.x = tensors[kind];
        side.x_ts = d->token_stride[kind];
        side.x_hs = d->head_stride[kind];
        side.g = count == 6 ? tensors[2 + kind] : nullptr;
        side.g_ts = d->token_stride[2 + kind];
        side.g_hs = d->head_stride[2 + kind];
        side.y = const_cast<void*>(tensors[out]);
        side.y_ts = d->token_stride[out];
        side.y_hs = d->head_stride[out];
    }
    return MI_OK;
}

// Workgroups of each side, and how many wavefronts share a token.  At most `most` workgroups, which is what the
// chip holds at once, in proportion to the items; every wavefront of a side has the same number of units but for
// the last.  Where the tokens alone do not give that many wavefronts, their heads are shared out.
void cut_work(HeadsArgs& a, uint32_t most)
{
    const uint32_t groups = 64u >> a.lg;
    Side* const sides[2] = {&a.q, &a.k};
    uint64_t items[2];
    for (int i = 0; i < 2; ++i) items[i] = a.tokens * ((sides[i]->heads + groups - 1u) / groups);
    for (int i = 0; i < 2; ++i) {
        Side& s = *sides[i];
        s.lg_parts = s.blocks = 0;
        if (!items[i]) continue;
        const uint32_t per_token = (s.heads + groups - 1u) / groups;
        const uint64_t waves = 4u * (1u + items[i] * (most - 2u) / (items[0] + items[1]));
        while ((2u << s.lg_parts) <= per_token && a.tokens << s.lg_parts < waves) ++s.lg_parts;
        const uint64_t units = a.tokens << s.lg_parts, each = (units + waves - 1u) / waves;
        s.blocks = (uint32_t)(((units + each - 1u) / each + 3u) / 4u);
    }
}

template <bool BACKWARD, class E, int LG, bool NEIGHBOURS>
void launch(const HeadsArgs& a, hipStream_t s)
{
    const dim3 grid(a.q.blocks + a.k.blocks);
    if (BACKWARD) hipLaunchKernelGGL((qk_norm_rope_backward_kernel<E, LG, NEIGHBOURS>), grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((qk_norm_rope_kernel<E, LG, NEIGHBOURS>), grid, dim3(kThreads), 0, s, a);
}

template <bool BACKWARD, class E>
int launch_for(const HeadsArgs& a, hipStream_t s)
{
    auto pick = [&](auto lg) {
        constexpr int LG = decltype(lg)::value;
        if (a.neighbours) launch<BACKWARD, E, LG, true>(a, s);
        else launch<BACKWARD, E, LG, false>(a, s);
    };
    switch (a.lg) {
        case 2: pick(std::integral_constant<int, 2>{}); break;   // heads of 48, 64
        case 3: pick(std::integral_constant<int, 3>{}); break;   // 80 ... 128
        case 4: pick(std::integral_constant<int, 4>{}); break;   // 144 ... 256
        default: pick(std::integral_constant<int, -1>{}); break;
    }
    return launch_status();
}

template <bool BACKWARD>
int launch_heads(const HeadsArgs& a, int dtype, hipStream_t s)
{
    if (dtype == MI_F32) return launch_for<BACKWARD, float>(a, s);
    if (dtype == MI_BF16) return launch_for<BACKWARD, __bf16>(a, s);
    return launch_for<BACKWARD, _Float16>(a, s);
}

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
    a.q.w = q_weight;
    a.k.w = k_weight;
    if ((q_weight && !aligned16(q_weight)) || (k_weight && !aligned16(k_weight))) return MI_ERR_ALIGN;
    cut_work(a, kMaxBlocks);
    return launch_heads<false>(a, d->dtype, static_cast<hipStream_t>(stream));
}

extern "C" uint64_t mi_qk_norm_rope_workspace(uint64_t tokens, uint32_t head_dim)
{
    using namespace mi;
    return tokens ? (uint64_t)kMaxPartials * head_dim * sizeof(float) : 0u;
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
    a.q.w = q_weight;
    a.k.w = k_weight;
    if ((q_weight && !aligned16(q_weight)) || (k_weight && !aligned16(k_weight))) return MI_ERR_ALIGN;
    const bool any = d->tokens != 0 && d->q_heads + d->k_heads != 0;
    const bool weights = dq_weight || dk_weight;
    if (weights && any && !workspace) return MI_ERR_NULL;
    if (weights && any && !aligned16(workspace)) return MI_ERR_ALIGN;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (any) {
        a.partials = weights ? static_cast<float*>(workspace) : nullptr;
        cut_work(a, kMaxPartials);
        const int launched = launch_heads<true>(a, d->dtype, s);
        if (launched != MI_OK) return launched;
    }
    if (weights) {
        hipLaunchKernelGGL(weight_gradient_kernel, dim3(a.D / 4u, 2), dim3(256), 0, s, static_cast<const float*>(workspace), a.q.blocks,
                           a.k.blocks, a.D, dq_weight, dk_weight, d->weight_dtype);
        return launch_status();
    }
    return MI_OK;
}
