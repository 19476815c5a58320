// Low-rank adapters of many requests added to a shared projection (mi_lora_add), and the gradients
// (mi_lora_add_backward).  Token t with adapter a, A[a] [r,K], B[a] [N,r], factor s[a]:
//   u_t = A x_t                        out_t = y_t + s B u_t
//   d_t = s B^T g_t   (g = dy)         dx_t  = A^T d_t
//   dA  = sum_t d_t x_t^T              dB    = sum_t s g_t u_t^T
// With r small against K and N all of it is bound by reading x, y (g) and writing out (dx); the matrix
// cores have time to spare, and the kernels spend some of it on accuracy: u and d stay in 32 bits
// through being split into two 16-bit pieces, v = hi + lo, which both go through the matrix core
// (16 significand bits for bf16, 22 for fp16; a single piece would add an error of the size of the
// output's rounding).  fp16 pieces are taken after a scaling by a power of two, so that neither large
// nor very small values (gradients) leave the type's range.
//
// Tokens come grouped by adapter (adapter_plan.hpp), in tiles of up to 64 of one adapter.
//   contract_rows   P[split][position][r] = sum over a part of the long axis of row . M[a]:  u, and d / s
//   expand_rows     out = y + s (sum of P) M'[a]^T:  the forward output, and dx
//   transpose       B^T and A^T of the adapters in use, which give the backward pass the layouts of the
//                   forward one
//   weight_pieces   d and s u, transposed and split, for the contraction over tokens
//   weight_rows     dA and dB of up to 512 tokens;  weight_sum adds these up
// All sums are in a fixed order.
#include <type_traits>

#include "adapter_plan.hpp"

namespace mi {
namespace adapters {
namespace {

constexpr uint32_t kThreads = 256;

// A matrix-core step on 16-byte fragments: lane l holds row (or column) l % 16 and the VEC values of the
// contracted axis that start at VEC * (l / 16).  Any assignment of the contracted axis to (lane group,
// element) is right as long as both operands share it.
template <class E> struct Mx;
template <> struct Mx<__bf16> {
    static constexpr uint32_t VEC = 8, STEP = 32, PIECES = 2;
    static constexpr bool SCALED = false;
    using V = bf16x8;
    static __device__ __forceinline__ f32x4 mma(V a, V b, f32x4 c) { return BF16::mfma32(a, b, c); }
};
template <> struct Mx<_Float16> {
    static constexpr uint32_t VEC = 8, STEP = 32, PIECES = 2;
    static constexpr bool SCALED = true;
    using V = f16x8;
    static __device__ __forceinline__ f32x4 mma(V a, V b, f32x4 c) { return F16::mfma32(a, b, c); }
};
template <> struct Mx<float> {
    static constexpr uint32_t VEC = 4, STEP = 16, PIECES = 1;
    static constexpr bool SCALED = false;
    using V = f32x4;
    static __device__ __forceinline__ f32x4 mma(V a, V b, f32x4 c)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// hi + lo = v but for the last bits; lo = 0 where hi is not finite, so that an infinity stays one.
template <class E>
__device__ __forceinline__ void split(float v, E& hi, E& lo)
{
    hi = (E)v;
    const float rest = v - (float)hi;
    lo = (E)(__builtin_fabsf((float)hi) < __builtin_inff() ? rest : 0.0f);
}

// A magnitude for half_scale: what is not finite takes no part.
__device__ __forceinline__ float finite_magnitude(float v)
{
    const float m = __builtin_fabsf(v);
    return m < __builtin_inff() ? m : 0.0f;
}

// Power of two that brings a largest magnitude m to [2^14, 2^15), and its inverse.  Magnitudes below
// 2^-106 (and zero) take the factor of that border; both factors are normal numbers.
__device__ __forceinline__ void half_scale(float m, float& up, float& down)
{
    uint32_t e = __builtin_bit_cast(uint32_t, m) >> 23 & 255u;
    e = e < 21u ? 21u : e;
    up = __builtin_bit_cast(float, (268u - e) << 23);
    down = __builtin_bit_cast(float, (e - 14u) << 23);
}

// The wavefront's number in a scalar register.  Matrix-core instructions ignore the lane mask, so what decides
// about them has to be a branch that the whole wavefront takes or does not take.
__device__ __forceinline__ uint32_t this_wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

template <class V>
__device__ __forceinline__ V load16(const void* p)
{
    return *static_cast<const V*>(p);
}

struct Rows {            // token rows
    const void* p;
    uint64_t stride;     // elements
};

// ------------------------------------------------------------------------------------------------
struct ContractArgs {
    const int32_t* plan;
    Rows x;
    const void* M;       // [n][rank][K]
    float* P;            // [splits][tokens][16 RT]
    uint64_t tokens;
    uint32_t n, rank, K, splits, part;  // part: extent of K per workgroup, a multiple of 8 * STEP
};

// P^T tile = M (rows: r) . x^T (columns: tokens).  The four wavefronts take turns along the part of K, two
// steps (a 128-byte line of every row) at a time with the next two requested, and add their sums through
// LDS.  Columns behind the tile's tokens repeat its first one and rows behind the rank the first rank: the
// loads need no masks, and what they give is not stored.
template <class E, int RT, int SUB>
__device__ __forceinline__ void contract_tile(const ContractArgs& a, const Tile& tile, uint32_t split, f32x4* red)
{
    using X = Mx<E>;
    using V = typename X::V;
    constexpr uint32_t kBlock = 2u * X::STEP;
    const uint32_t lane = threadIdx.x & 63u, wave = this_wave(), lo = lane & 15u, g = lane >> 4;
    const PlanLayout L(a.tokens, a.n);
    const uint32_t k0 = split * a.part;
    const uint32_t k1 = a.K - k0 < a.part ? a.K : k0 + a.part;

    const E* xr[SUB];
#pragma unroll
    for (int i = 0; i < SUB; ++i) {
        const uint32_t at = 16u * i + lo;
        const int32_t t = a.plan[L.order + (uint32_t)tile.first + (at < (uint32_t)tile.count ? at : 0u)];
        xr[i] = static_cast<const E*>(a.x.p) + (uint64_t)t * a.x.stride + X::VEC * g;
    }
    const E* mr[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const uint32_t r = 16u * i + lo;
        mr[i] = static_cast<const E*>(a.M) + ((uint64_t)tile.adapter * a.rank + (r < a.rank ? r : 0u)) * a.K + X::VEC * g;
    }
    struct Block { V x[2][SUB], m[2][RT]; };
    f32x4 acc[SUB][RT] = {};
    const uint32_t full = (k1 - k0) / kBlock, mine = full > wave ? (full - wave + 3u) / 4u : 0u;
    auto load = [&](Block& b, uint32_t i) __attribute__((always_inline)) {
        const uint32_t k = k0 + (wave + 4u * i) * kBlock;
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < SUB; ++j) b.x[h][j] = load16<V>(xr[j] + k + h * X::STEP);
#pragma unroll
            for (int j = 0; j < RT; ++j) b.m[h][j] = load16<V>(mr[j] + k + h * X::STEP);
        }
    };
    auto multiply = [&](const Block& b) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
                for (int i = 0; i < SUB; ++i) acc[i][j] = X::mma(b.m[h][j], b.x[h][i], acc[i][j]);
    };
    if (mine) {
        Block p, q;
        uint32_t i = 0;
        load(p, 0);
        for (; i + 2u < mine; i += 2u) {
            load(q, i + 1u);
            multiply(p);
            load(p, i + 2u);
            multiply(q);
        }
        if (i + 1u < mine) load(q, i + 1u);
        multiply(p);
        if (i + 1u < mine) multiply(q);
    }
    if ((full & 3u) == wave) {  // the rest of K: less than a block, values behind the end are zeros on both sides
        for (uint32_t k = k0 + full * kBlock; k < k1; k += X::STEP) {
            V xf[SUB] = {}, mf[RT] = {};
            if (k + X::VEC * g < k1) {
#pragma unroll
                for (int i = 0; i < SUB; ++i) xf[i] = load16<V>(xr[i] + k);
#pragma unroll
                for (int i = 0; i < RT; ++i) mf[i] = load16<V>(mr[i] + k);
            }
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
                for (int i = 0; i < SUB; ++i) acc[i][j] = X::mma(mf[j], xf[i], acc[i][j]);
        }
    }
    // wavefronts 2, 3 to 0, 1, then 1 to 0
#pragma unroll
    for (uint32_t half = 2; half; half >>= 1) {
        if (wave >= half && wave < 2u * half) {
#pragma unroll
            for (int i = 0; i < SUB; ++i)
#pragma unroll
                for (int j = 0; j < RT; ++j) red[(((wave - half) * SUB + i) * RT + j) * 64u + lane] = acc[i][j];
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int i = 0; i < SUB; ++i)
#pragma unroll
                for (int j = 0; j < RT; ++j) acc[i][j] += red[((wave * SUB + i) * RT + j) * 64u + lane];
        }
        __syncthreads();
    }
    if (wave) return;
    float* P = a.P + ((uint64_t)split * a.tokens + (uint32_t)tile.first) * (16u * RT);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < SUB; ++i)
        if (16u * i + lo < (uint32_t)tile.count)
#pragma unroll
            for (int j = 0; j < RT; ++j)
                *reinterpret_cast<f32x4*>(P + (16u * i + lo) * (16u * RT) + 16u * j + 4u * g) =
                    16u * j + 4u * g < a.rank ? acc[i][j] : zero;
}

// The work of a workgroup: a tile, or with FEW 16 of its tokens, and one of `parts` parts of an axis.  Consecutive
// workgroups take the parts of one tile: they run on different XCDs, so an XCD's L2 holds its part of the
// adapters for all tiles.  False where the plan has no such tile.
template <bool FEW>
__device__ __forceinline__ bool take_tile(const int32_t* plan, const PlanLayout& L, uint32_t parts, Tile& tile, uint32_t& part)
{
    uint32_t t = blockIdx.x / parts, sub = 0;
    part = blockIdx.x - t * parts;
    if (FEW) {
        sub = 16u * (t & 3u);
        t >>= 2;
    }
    tile = reinterpret_cast<const Tile*>(plan)[t];
    if (t >= (uint32_t)plan[L.counts]) return false;
    if (FEW) {
        tile.first += (int32_t)sub;
        tile.count -= (int32_t)sub;
        if (tile.count > 16) tile.count = 16;
    }
    return tile.count > 0;
}

template <class E, int RT, bool FEW>
__global__ void __launch_bounds__(256, FEW || RT == 8 ? 1 : 2) contract_rows_kernel(ContractArgs a)
{
    __shared__ f32x4 red[2 * (FEW ? 1 : 4) * RT * 64];
    const PlanLayout L(a.tokens, a.n);
    Tile tile;
    uint32_t split;
    if (!take_tile<FEW>(a.plan, L, a.splits, tile, split) || (uint32_t)tile.adapter >= a.n) return;
    if constexpr (FEW) contract_tile<E, RT, 1>(a, tile, split, red);
    else if (tile.count <= 32) contract_tile<E, RT, 2>(a, tile, split, red);
    else contract_tile<E, RT, 4>(a, tile, split, red);
}

// ------------------------------------------------------------------------------------------------
struct ExpandArgs {
    const int32_t* plan;
    Rows y;              // added to
    void* out;
    uint64_t out_stride;
    const void* M;       // [n][N][rank]
    const float* scales; // [n] or NULL
    const float* P;      // [splits][tokens][16 RT]
    float* shrunk;       // [tokens][rank] or NULL: the sums of P in the tokens' own order
    uint64_t tokens;
    uint32_t n, rank, N, splits, part, parts;  // part: extent of N per workgroup
};

// The rank-space vectors of a tile as matrix-core operands in LDS: fragment (sub, f, p) of the 16 tokens of
// sub, the STEP ranks of f (PAIR: all 16 ranks, hi in lane groups 0, 1 and lo in 2, 3) and piece p.
template <class E, int RT>
struct Operand {
    using X = Mx<E>;
    static constexpr bool PAIR = X::PIECES == 2 && RT == 1;
    static constexpr int NF = X::PIECES == 2 ? (RT + 1) / 2 : RT;
    static constexpr int NP = PAIR ? 1 : (int)X::PIECES;
    static constexpr uint32_t BYTES = 4u * NF * NP * 1024u;
    // byte offset of piece p of rank r of token t (0 ... 63)
    static __device__ __forceinline__ uint32_t at(uint32_t t, uint32_t r, uint32_t p)
    {
        const uint32_t f = PAIR ? 0u : r / X::STEP, g = PAIR ? r / 8u + 2u * p : r % X::STEP / X::VEC;
        return (((t >> 4) * NF + f) * NP + (PAIR ? 0u : p)) * 1024u + (16u * g + (t & 15u)) * 16u + r % X::VEC * (uint32_t)sizeof(E);
    }
};

// Sums of P, times the factor, split: four threads per token, 4 RT ranks each.  Tokens behind the tile's
// repeat its first one.
template <class E, int RT, bool FEW>
__device__ __forceinline__ void make_operand(const ExpandArgs& a, const Tile& tile, unsigned char* lds, float* down, bool first_part)
{
    using X = Mx<E>;
    using O = Operand<E, RT>;
    typedef E E4 __attribute__((ext_vector_type(4)));
    const PlanLayout L(a.tokens, a.n);
    const uint32_t t = threadIdx.x >> 2, r0 = (threadIdx.x & 3u) * 4u * RT;
    if (FEW && t >= 16u) return;
    const bool live = t < (uint32_t)tile.count;
    const float s = a.scales ? a.scales[tile.adapter] : 1.0f;
    const float* P = a.P + ((uint64_t)(uint32_t)tile.first + (live ? t : 0u)) * (16u * RT) + r0;
    f32x4 sum[RT] = {};
#pragma unroll 4
    for (uint32_t sp = 0; sp < a.splits; ++sp)
#pragma unroll
        for (int i = 0; i < RT; ++i) sum[i] += load16<f32x4>(P + (uint64_t)sp * a.tokens * (16u * RT) + 4 * i);
    if (a.shrunk && first_part && live) {
        float* u = a.shrunk + (uint64_t)(uint32_t)a.plan[L.order + (uint32_t)tile.first + t] * a.rank;
#pragma unroll
        for (int i = 0; i < RT; ++i)
            if (r0 + 4u * i < a.rank)
#pragma unroll
                for (int c = 0; c < 4; ++c) u[r0 + 4u * i + c] = sum[i][c];
    }
    float up = 1.0f;
#pragma unroll
    for (int i = 0; i < RT; ++i) sum[i] = sum[i] * s;
    if constexpr (X::SCALED) {
        float m = 0.0f, d;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) m = fmaxf(m, finite_magnitude(sum[i][c]));
        m = fmaxf(m, __shfl_xor(m, 1));
        m = fmaxf(m, __shfl_xor(m, 2));
        half_scale(m, up, d);
        if ((threadIdx.x & 3u) == 0) down[t] = d;
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        if constexpr (X::PIECES == 1) {
            *reinterpret_cast<f32x4*>(lds + O::at(t, r0 + 4u * i, 0)) = sum[i];
        } else {
            E4 hi, low;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                E h, l;
                split<E>(sum[i][c] * up, h, l);
                hi[c] = h;
                low[c] = l;
            }
            *reinterpret_cast<E4*>(lds + O::at(t, r0 + 4u * i, 0)) = hi;
            *reinterpret_cast<E4*>(lds + O::at(t, r0 + 4u * i, 1)) = low;
        }
    }
}

// out^T tile = M (rows: n) . v^T (columns: tokens).  Row m = 4 g + q of the 16-row operand t stands for
// n = base + VEC g + 4 t + q, so that a lane's results are VEC consecutive values of its token: 16-byte loads
// of y and stores of out.  A wavefront takes two such bases (a 128-byte line of every token) at a time
// with the next two requested.  Tokens behind the tile's are its first token again and columns behind N
// the last VEC ones: these lanes compute and store what the owner does, from a y that was loaded before
// the owner stores (out may be y), so that no load or store stands behind a branch.
template <class E, int RT, int SUB, bool HAS_Y>
__device__ __forceinline__ void expand_tile(const ExpandArgs& a, const Tile& tile, uint32_t part, const unsigned char* lds, const float* down)
{
    using X = Mx<E>;
    using V = typename X::V;
    using O = Operand<E, RT>;
    constexpr uint32_t VEC = X::VEC, NT = VEC / 4u, ROWS = 16u * NT;
    constexpr uint32_t U = X::PIECES == 1 && RT == 8 ? 1 : 2, BLOCK = U * ROWS;  // fp32 of rank 128: one base, as the registers allow
    constexpr int NF = O::NF, NP = O::NP;
    const uint32_t lane = threadIdx.x & 63u, wave = this_wave(), lo = lane & 15u, g = lane >> 4;
    const PlanLayout L(a.tokens, a.n);
    const uint32_t n0 = part * a.part;
    const uint32_t n1 = a.N - n0 < a.part ? a.N : n0 + a.part;
    const uint32_t blocks = (n1 - n0 + BLOCK - 1u) / BLOCK, mine = blocks > wave ? (blocks - wave + 3u) / 4u : 0u;
    const bool ragged = a.rank != 16u * RT;

    const E* yr[SUB];
    E* outr[SUB];
#pragma unroll
    for (int i = 0; i < SUB; ++i) {
        const uint32_t at = 16u * i + lo;
        const uint64_t t = (uint64_t)(uint32_t)a.plan[L.order + (uint32_t)tile.first + (at < (uint32_t)tile.count ? at : 0u)];
        yr[i] = static_cast<const E*>(a.y.p) + t * a.y.stride;
        outr[i] = static_cast<E*>(a.out) + t * a.out_stride;
    }
    const E* M = static_cast<const E*>(a.M) + (uint64_t)tile.adapter * a.N * a.rank;
    uint32_t r0[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        r0[f] = O::PAIR ? 8u * (g & 1u) : X::STEP * f + VEC * g;
        if (r0[f] >= a.rank) r0[f] = a.rank;  // zeros
    }
    struct Block { V m[U][NT][NF], y[U][SUB]; };
    auto column = [&](uint32_t i, uint32_t u, uint32_t group) {
        const uint32_t n = n0 + (wave + 4u * i) * BLOCK + u * ROWS + VEC * group;
        return n < a.N ? n : a.N - VEC;
    };
    auto load = [&](Block& b, uint32_t i) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t row = column(i, u, lo >> 2) + (lo & 3u);
#pragma unroll
            for (uint32_t t = 0; t < NT; ++t)
#pragma unroll
                for (int f = 0; f < NF; ++f)
                    b.m[u][t][f] = load16<V>(M + (uint64_t)(row + 4u * t) * a.rank + (r0[f] < a.rank ? r0[f] : 0u));
            if (HAS_Y)
#pragma unroll
                for (int j = 0; j < SUB; ++j) b.y[u][j] = load16<V>(yr[j] + column(i, u, g));
        }
    };
    auto finish = [&](Block& b, uint32_t i) __attribute__((always_inline)) {
        if (ragged)
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
#pragma unroll
                for (uint32_t t = 0; t < NT; ++t)
#pragma unroll
                    for (int f = 0; f < NF; ++f) b.m[u][t][f] = r0[f] < a.rank ? b.m[u][t][f] : V{};
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            f32x4 acc[U][NT] = {};
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    const V v = *reinterpret_cast<const V*>(lds + ((j * NF + f) * NP + p) * 1024u + lane * 16u);
#pragma unroll
                    for (uint32_t u = 0; u < U; ++u)
#pragma unroll
                        for (uint32_t t = 0; t < NT; ++t) acc[u][t] = X::mma(b.m[u][t][f], v, acc[u][t]);
                }
            const float d = X::SCALED ? down[16u * j + lo] : 1.0f;
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                V o;
#pragma unroll
                for (uint32_t e = 0; e < VEC; ++e) {
                    float v = acc[u][e / 4u][e % 4u];
                    if (HAS_Y) v = X::SCALED ? __builtin_fmaf(v, d, (float)b.y[u][j][e]) : v + (float)b.y[u][j][e];
                    else if (X::SCALED) v *= d;
                    o[e] = (E)v;
                }
                __builtin_nontemporal_store(o, reinterpret_cast<V*>(outr[j] + column(i, u, g)));
            }
        }
    };
    if (!mine) return;
    Block p, q;
    uint32_t i = 0;
    load(p, 0);
    for (; i + 2u < mine; i += 2u) {
        load(q, i + 1u);
        finish(p, i);
        load(p, i + 2u);
        finish(q, i + 1u);
    }
    if (i + 1u < mine) {
        load(q, i + 1u);
        finish(p, i);
        finish(q, i + 1u);
    } else {
        finish(p, i);
    }
}

template <class E, int RT, bool HAS_Y, bool FEW>
__global__ void __launch_bounds__(256, FEW || RT == 8 ? 1 : 2) expand_rows_kernel(ExpandArgs a)
{
    using V = typename Mx<E>::V;
    constexpr uint32_t VEC = Mx<E>::VEC;
    __shared__ __attribute__((aligned(16))) unsigned char lds[Operand<E, RT>::BYTES];
    __shared__ float down[64];
    const PlanLayout L(a.tokens, a.n);
    Tile tile;
    uint32_t part;
    if (!take_tile<FEW>(a.plan, L, a.parts, tile, part)) return;
    if ((uint32_t)tile.adapter < a.n) {
        make_operand<E, RT, FEW>(a, tile, lds, down, part == 0u);
        if (a.N == 0u) return;
        __syncthreads();
        if constexpr (FEW) expand_tile<E, RT, 1, HAS_Y>(a, tile, part, lds, down);
        else if (tile.count <= 32) expand_tile<E, RT, 2, HAS_Y>(a, tile, part, lds, down);
        else expand_tile<E, RT, 4, HAS_Y>(a, tile, part, lds, down);
        return;
    }
    // tokens without an adapter: y as it is, or zeros
    const uint32_t n0 = part * a.part;
    const uint32_t n1 = a.N - n0 < a.part ? a.N : n0 + a.part;
    if (a.N && (!HAS_Y || a.y.p != a.out))
        for (uint32_t i = threadIdx.x >> 6; i < (uint32_t)tile.count; i += 4u) {
            const uint64_t t = (uint64_t)(uint32_t)a.plan[L.order + (uint32_t)tile.first + i];
            for (uint32_t c = n0 + VEC * (threadIdx.x & 63u); c < n1; c += VEC * 64u) {
                V v = {};
                if (HAS_Y) v = load16<V>(static_cast<const E*>(a.y.p) + t * a.y.stride + c);
                *reinterpret_cast<V*>(static_cast<E*>(a.out) + t * a.out_stride + c) = v;
            }
        }
    if (a.shrunk && part == 0u)
        for (uint32_t i = threadIdx.x; i < (uint32_t)tile.count * a.rank; i += kThreads) {
            const uint32_t at = i / a.rank;
            a.shrunk[(uint64_t)(uint32_t)a.plan[L.order + (uint32_t)tile.first + at] * a.rank + (i - at * a.rank)] = 0.0f;
        }
}

// ------------------------------------------------------------------------------------------------
struct TransposeArgs {
    const int32_t* plan;
    const void* src[2];  // A [n][rank][K], B [n][N][rank]
    void* dst[2];        // [n][K][rank], [n][rank][N]
    uint64_t tokens;
    uint32_t n, rows[2], cols[2];
    uint32_t blocks0;    // workgroups of the first matrix
};

// 64 x 64 pieces of the adapters in use.
template <class E>
__global__ void __launch_bounds__(256) transpose_kernel(TransposeArgs a)
{
    __shared__ E tile[64][66];
    const PlanLayout L(a.tokens, a.n);
    const uint32_t ad = blockIdx.y;
    if (a.plan[L.starts + ad] == a.plan[L.starts + ad + 1u]) return;
    const uint32_t which = blockIdx.x >= a.blocks0;
    const uint32_t b = blockIdx.x - which * a.blocks0, rows = a.rows[which], cols = a.cols[which];
    const uint32_t across = (cols + 63u) / 64u, r0 = b / across * 64u, c0 = b % across * 64u;
    const E* src = static_cast<const E*>(a.src[which]) + (uint64_t)ad * rows * cols;
    E* dst = static_cast<E*>(a.dst[which]) + (uint64_t)ad * rows * cols;
    const uint32_t x = threadIdx.x & 63u, y0 = threadIdx.x >> 6;
    for (uint32_t y = y0; y < 64u; y += 4u)
        if (r0 + y < rows && c0 + x < cols) tile[y][x] = src[(uint64_t)(r0 + y) * cols + c0 + x];
    __syncthreads();
    for (uint32_t y = y0; y < 64u; y += 4u)
        if (c0 + y < cols && r0 + x < rows) dst[(uint64_t)(c0 + y) * rows + r0 + x] = tile[x][y];
}

// ------------------------------------------------------------------------------------------------
struct PiecesArgs {
    const int32_t* plan;
    const float* P;       // d / s: [splits][tokens][16 RT]
    const float* shrunk;  // u: [tokens][rank]
    const float* scales;
    void* pieces[2];      // d, s u: [tiles][16 RT][PIECES][64]
    float* down;          // fp16: [2][tiles], the inverse of the tile's scaling
    uint64_t tokens, max_tiles;
    uint32_t n, rank, rp, splits;
};

// Transposes a tile's d (or s u) and splits it.  Tokens behind the tile's count and ranks behind the
// adapter's are zeros.
template <class E>
__global__ void __launch_bounds__(256) weight_pieces_kernel(PiecesArgs a)
{
    using X = Mx<E>;
    __shared__ float top[4];
    const PlanLayout L(a.tokens, a.n);
    if (blockIdx.x >= (uint32_t)a.plan[L.counts]) return;
    const Tile tile = reinterpret_cast<const Tile*>(a.plan)[blockIdx.x];
    if ((uint32_t)tile.adapter >= a.n) return;
    const uint32_t which = blockIdx.y, lane = threadIdx.x & 63u, wave = this_wave();
    const float s = a.scales ? a.scales[tile.adapter] : 1.0f;
    const bool live = lane < (uint32_t)tile.count;
    const uint64_t pos = (uint64_t)(uint32_t)tile.first + lane;
    const int64_t token = live ? a.plan[L.order + pos] : 0;
    auto value = [&](uint32_t r) {
        if (!live || r >= a.rank) return 0.0f;
        if (which) return a.shrunk[token * a.rank + r] * s;
        float sum = 0.0f;
        for (uint32_t sp = 0; sp < a.splits; ++sp) sum += a.P[((uint64_t)sp * a.tokens + pos) * a.rp + r];
        return sum * s;
    };
    float up = 1.0f;
    if constexpr (X::SCALED) {
        float m = 0.0f, down;
        for (uint32_t r = wave; r < a.rp; r += 4u) m = fmaxf(m, finite_magnitude(value(r)));
        for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
        if (lane == 0) top[wave] = m;
        __syncthreads();
        m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        half_scale(m, up, down);
        if (threadIdx.x == 0) a.down[which * a.max_tiles + blockIdx.x] = down;
    }
    E* out = static_cast<E*>(a.pieces[which]) + (uint64_t)blockIdx.x * a.rp * X::PIECES * 64u;
    for (uint32_t r = wave; r < a.rp; r += 4u) {
        const float v = value(r) * up;
        if constexpr (X::PIECES == 1) {
            out[r * 64u + lane] = v;
        } else {
            E hi, low;
            split<E>(v, hi, low);
            out[(2u * r) * 64u + lane] = hi;
            out[(2u * r + 1u) * 64u + lane] = low;
        }
    }
}

// ------------------------------------------------------------------------------------------------
struct WeightArgs {
    const int32_t* plan;
    Rows rows[2];         // x, dy
    const void* pieces[2];
    const float* down;
    float* partials;      // [slots][rank * (K + N)]
    void* grad[2];        // dA [n][rank][K], dB [n][N][rank]
    uint64_t tokens, max_tiles;
    uint32_t n, rank, rp, len[2];
    uint32_t blocks0;     // workgroups along K
};

// Four 16-byte rows' registers to fragments along the tokens: in[i] holds VEC consecutive columns of
// token i, out[c] the VEC tokens of column c.
__device__ __forceinline__ void turn_over(const u32x4 (&in)[8], u32x4 (&out)[8])
{
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
        for (int p = 0; p < 4; ++p)
            out[c][p] = __builtin_amdgcn_perm(in[2 * p + 1][c / 2], in[2 * p][c / 2], c & 1 ? 0x07060302u : 0x05040100u);
}
__device__ __forceinline__ void turn_over(const u32x4 (&in)[4], u32x4 (&out)[4])
{
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int p = 0; p < 4; ++p) out[c][p] = in[p][c];
}

// Workgroup: a chunk of up to 512 tokens of one adapter, 16 VEC columns, up to RT * 16 ranks.  A wavefront
// takes every fourth step of STEP tokens; a lane reads 16 bytes of VEC consecutive tokens (the 16 lanes of a
// group read 256 contiguous bytes of a row) and turns them over in registers, one byte permute for two
// values, so the contraction over tokens needs no LDS.  The wavefronts' sums meet in LDS at the end.
template <class E, int RT>
__global__ void __launch_bounds__(256) weight_rows_kernel(WeightArgs a)
{
    using X = Mx<E>;
    using V = typename X::V;
    constexpr uint32_t VEC = X::VEC, STEP = X::STEP;
    __shared__ f32x4 red[2 * RT * VEC * 64];
    __shared__ int32_t order[kChunk];
    const PlanLayout L(a.tokens, a.n);
    if (blockIdx.y >= (uint32_t)a.plan[L.counts + 1u]) return;
    const Chunk chunk = reinterpret_cast<const Chunk*>(a.plan + L.chunks)[blockIdx.y];
    const uint32_t lane = threadIdx.x & 63u, wave = this_wave(), lo = lane & 15u, g = lane >> 4;
    for (uint32_t i = threadIdx.x; i < (uint32_t)chunk.count; i += kThreads)
        order[i] = a.plan[L.order + (uint32_t)chunk.first + i];
    __syncthreads();
    const uint32_t which = blockIdx.x >= a.blocks0;
    const uint32_t len = a.len[which], col = (blockIdx.x - which * a.blocks0) * 16u * VEC + VEC * lo;
    const uint32_t rank0 = blockIdx.z * 16u * RT;
    const bool inside = col < len;
    const E* rows = static_cast<const E*>(a.rows[which].p) + (inside ? col : 0u);
    const uint64_t stride = a.rows[which].stride;
    const E* pieces = static_cast<const E*>(a.pieces[which]);

    f32x4 acc[RT][VEC] = {};
    for (uint32_t t0 = wave * STEP; t0 < (uint32_t)chunk.count; t0 += 4u * STEP) {
        u32x4 in[VEC], turned[VEC];
#pragma unroll
        for (uint32_t i = 0; i < VEC; ++i) {
            const uint32_t t = t0 + VEC * g + i;
            in[i] = u32x4{0u, 0u, 0u, 0u};  // tokens behind the chunk: zeros on both sides
            if (t < (uint32_t)chunk.count) in[i] = load16<u32x4>(rows + (uint64_t)order[t] * stride);
        }
        const uint32_t tile = (uint32_t)chunk.tile + t0 / kTile;
        V wf[RT][X::PIECES];
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
            for (uint32_t p = 0; p < X::PIECES; ++p)
                wf[j][p] = load16<V>(pieces + (((uint64_t)tile * a.rp + rank0 + 16u * j + lo) * X::PIECES + p) * 64u + t0 % kTile + VEC * g);
        turn_over(in, turned);
        if constexpr (X::SCALED) {
            const float down = a.down[which * a.max_tiles + tile];
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
                for (uint32_t c = 0; c < VEC; ++c) {
                    f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (uint32_t p = 0; p < X::PIECES; ++p) d = X::mma(wf[j][p], __builtin_bit_cast(V, turned[c]), d);
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc[j][c][q] = __builtin_fmaf(d[q], down, acc[j][c][q]);
                }
        } else {
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
                for (uint32_t p = 0; p < X::PIECES; ++p)
#pragma unroll
                    for (uint32_t c = 0; c < VEC; ++c) acc[j][c] = X::mma(wf[j][p], __builtin_bit_cast(V, turned[c]), acc[j][c]);
        }
    }
#pragma unroll
    for (uint32_t half = 2; half; half >>= 1) {
        if (wave >= half && wave < 2u * half) {
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
                for (uint32_t c = 0; c < VEC; ++c) red[(((wave - half) * RT + j) * VEC + c) * 64u + lane] = acc[j][c];
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
                for (uint32_t c = 0; c < VEC; ++c) acc[j][c] += red[((wave * RT + j) * VEC + c) * 64u + lane];
        }
        __syncthreads();
    }
    if (wave || !inside) return;
    // lane: columns col ... col + VEC - 1, ranks rank0 + 16 j + 4 g + q
    const uint64_t per = (uint64_t)a.rank * (a.len[0] + a.len[1]);
    float* part = chunk.slot >= 0 ? a.partials + (uint64_t)chunk.slot * per + (which ? (uint64_t)a.rank * a.len[0] : 0u) : nullptr;
    E* grad = static_cast<E*>(a.grad[which]) + (uint64_t)chunk.adapter * a.rank * len;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
        const uint32_t r = rank0 + 16u * j + 4u * g;
        if (r >= a.rank) continue;
        if (which) {  // [n][rank]
#pragma unroll
            for (uint32_t c = 0; c < VEC; ++c) {
                const uint64_t at = (uint64_t)(col + c) * a.rank + r;
                if (part) {
                    *reinterpret_cast<f32x4*>(part + at) = acc[j][c];
                } else {
                    typedef E E4 __attribute__((ext_vector_type(4)));
                    E4 o;
#pragma unroll
                    for (int q = 0; q < 4; ++q) o[q] = (E)acc[j][c][q];
                    *reinterpret_cast<E4*>(grad + at) = o;
                }
            }
        } else {  // [rank][k]
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint64_t at = (uint64_t)(r + q) * len + col;
                if (part) {
#pragma unroll
                    for (uint32_t c = 0; c < VEC; c += 4)
                        *reinterpret_cast<f32x4*>(part + at + c) = f32x4{acc[j][c][q], acc[j][c + 1][q], acc[j][c + 2][q], acc[j][c + 3][q]};
                } else {
                    V o;
#pragma unroll
                    for (uint32_t c = 0; c < VEC; ++c) o[c] = (E)acc[j][c][q];
                    *reinterpret_cast<V*>(grad + at) = o;
                }
            }
        }
    }
}

struct WeightSumArgs {
    const int32_t* plan;
    const float* partials;
    void* grad[2];
    uint64_t tokens;
    uint32_t n, rank, len[2];
};

// Gradients of adapters with several chunks, and the zeros of those with none.
template <class E>
__global__ void __launch_bounds__(256) weight_sum_kernel(WeightSumArgs a)
{
    typedef E E4 __attribute__((ext_vector_type(4)));
    const PlanLayout L(a.tokens, a.n);
    const uint32_t ad = blockIdx.y;
    const uint32_t count = (uint32_t)(a.plan[L.starts + ad + 1u] - a.plan[L.starts + ad]);
    if (count > 0u && count <= kChunk) return;  // complete already
    const uint32_t chunks = (count + kChunk - 1u) / kChunk;
    const uint64_t first = (uint64_t)a.rank * a.len[0], per = first + (uint64_t)a.rank * a.len[1];
    const float* part = a.partials + (uint64_t)(uint32_t)a.plan[L.slot_start + ad] * per;
    for (uint64_t i = 4u * ((uint64_t)blockIdx.x * kThreads + threadIdx.x); i < per; i += 4u * (uint64_t)gridDim.x * kThreads) {
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t c = 0; c < chunks; ++c) sum += load16<f32x4>(part + c * per + i);
        E4 o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = (E)sum[q];
        E* out = i < first ? static_cast<E*>(a.grad[0]) + ad * first + i : static_cast<E*>(a.grad[1]) + ad * (per - first) + (i - first);
        *reinterpret_cast<E4*>(out) = o;
    }
}

// ------------------------------------------------------------------------------------------------
uint32_t padded_rank(uint32_t rank) { return rank <= 16u ? 16u : rank <= 32u ? 32u : rank <= 64u ? 64u : 128u; }

// How an axis is cut: `most` workgroups or a little fewer, but no part smaller than a unit; where there are eight
// parts or more, a multiple of eight, one XCD's share each.
void cut(uint64_t tiles, uint32_t length, uint32_t unit, uint32_t most, uint32_t& part, uint32_t& parts)
{
    const uint32_t units = (length + unit - 1u) / unit;
    uint64_t want = tiles && units ? most / tiles : 1u;
    if (want < 1u) want = 1u;
    if (want > units) want = units ? units : 1u;
    if (want > 8u) want = want / 8u * 8u;
    part = (units + (uint32_t)want - 1u) / (uint32_t)want * unit;
    if (!part) part = unit;
    parts = length ? (length + part - 1u) / part : 1u;
}

#ifndef MC
#define MC 512u
#endif
#ifndef ME
#define ME 1024u
#endif
template <class F>
void for_rank(uint32_t rp, F f)
{
    switch (rp) {
        case 16: f(std::integral_constant<int, 1>{}); break;
        case 32: f(std::integral_constant<int, 2>{}); break;
        case 64: f(std::integral_constant<int, 4>{}); break;
        default: f(std::integral_constant<int, 8>{}); break;
    }
}

uint32_t elements_of(int dtype) { return dtype == MI_F32 ? 4u : 8u; }
uint64_t up256(uint64_t bytes) { return (bytes + 255u) / 256u * 256u; }

int check(const mi_lora* d)
{
    if (!d) return MI_ERR_NULL;
    if (d->dtype != MI_F32 && d->dtype != MI_BF16 && d->dtype != MI_F16) return MI_ERR_DTYPE;
    if (d->tokens > kMaxTokens || d->n_adapters < 1u || d->n_adapters > kMaxAdapters) return MI_ERR_SHAPE;
    if (d->rank < 8u || d->rank > 128u || d->rank % 8u) return MI_ERR_SIZE;
    if (d->K < 8u || d->K % 8u || d->N < 8u || d->N % 8u || d->K > kMaxWidth || d->N > kMaxWidth) return MI_ERR_SHAPE;
    const uint64_t unit = elements_of(d->dtype);
    if (d->x_stride % unit || d->y_stride % unit || d->out_stride % unit) return MI_ERR_ALIGN;
    return MI_OK;
}

// How a batch is cut, and the forward pass's workspace: the partial sums P.  With few tokens for each adapter
// (16 on the average, or 256 in all) workgroups take 16 tokens instead of 64: a fourth of the registers, so
// that four times as many wavefronts hide the latencies that such a batch consists of.
struct ForwardPlan {
    bool few;
    uint32_t rp, part, splits, npart, nparts;
    uint64_t tiles, bytes;  // tiles: that the grids provide for, absent ones among them
    ForwardPlan(const mi_lora* d, uint32_t K, uint32_t N)
    {
        const PlanLayout L(d->tokens, d->n_adapters);
        few = d->tokens <= 256u || d->tokens <= 16u * d->n_adapters;
        tiles = L.max_tiles;
        rp = padded_rank(d->rank);
        const uint32_t step = 4u * elements_of(d->dtype);
        cut(tiles, K, 8u * step, few ? 1024u : MC, part, splits);  // each wavefront two blocks of two steps at least
        cut(tiles, N, 8u * step, few ? 1024u : ME, npart, nparts);  // each wavefront a 128-byte line at least
        if (few) tiles *= 4u;
        bytes = up256((uint64_t)splits * d->tokens * rp * 4u);
    }
};

struct BackwardPlan {
    ForwardPlan f;  // contraction over N, expansion to K
    ForwardPlan u;  // contraction over K alone, when the forward pass's sums are not given
    uint64_t at, bt, shrunk, pieces[2], down, partials, bytes;
    explicit BackwardPlan(const mi_lora* d) : f(d, d->N, d->K), u(d, d->K, 0u)
    {
        const PlanLayout L(d->tokens, d->n_adapters);
        const uint64_t e = d->dtype == MI_F32 ? 4u : 2u, pieces_n = d->dtype == MI_F32 ? 1u : 2u;
        uint64_t at_ = f.bytes > u.bytes ? f.bytes : u.bytes;  // P first, in turn
        auto take = [&](uint64_t n) { const uint64_t here = at_; at_ += up256(n); return here; };
        at = take((uint64_t)d->n_adapters * d->rank * d->K * e);
        bt = take((uint64_t)d->n_adapters * d->rank * d->N * e);
        shrunk = take(d->tokens * d->rank * 4u);
        for (int i = 0; i < 2; ++i) pieces[i] = take(L.max_tiles * f.rp * pieces_n * 64u * e);
        down = take(2u * L.max_tiles * 4u);
        partials = take(L.max_slots * d->rank * ((uint64_t)d->K + d->N) * 4u);
        bytes = at_;
    }
};

template <class E>
int contract(const mi_lora* d, const int32_t* plan, Rows x, const void* M, uint32_t K, const ForwardPlan& f, float* P, hipStream_t s)
{
    ContractArgs a{plan, x, M, P, d->tokens, d->n_adapters, d->rank, K, f.splits, f.part};
    for_rank(f.rp, [&](auto rt) {
        constexpr int RT = decltype(rt)::value;
        const dim3 grid((uint32_t)f.tiles * f.splits);
        if (f.few) hipLaunchKernelGGL((contract_rows_kernel<E, RT, true>), grid, dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((contract_rows_kernel<E, RT, false>), grid, dim3(kThreads), 0, s, a);
    });
    return launch_status();
}

template <class E>
int expand(const mi_lora* d, const int32_t* plan, Rows y, void* out, uint64_t out_stride, const void* M, uint32_t N, const float* scales,
           const ForwardPlan& f, const float* P, float* shrunk, hipStream_t s)
{
    ExpandArgs a{plan, y, out, out_stride, M, scales, P, shrunk, d->tokens, d->n_adapters, d->rank, N, f.splits, f.npart, f.nparts};
    const dim3 grid((uint32_t)f.tiles * f.nparts);
    for_rank(f.rp, [&](auto rt) {
        constexpr int RT = decltype(rt)::value;
        if (y.p && f.few) hipLaunchKernelGGL((expand_rows_kernel<E, RT, true, true>), grid, dim3(kThreads), 0, s, a);
        else if (y.p) hipLaunchKernelGGL((expand_rows_kernel<E, RT, true, false>), grid, dim3(kThreads), 0, s, a);
        else if (f.few) hipLaunchKernelGGL((expand_rows_kernel<E, RT, false, true>), grid, dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((expand_rows_kernel<E, RT, false, false>), grid, dim3(kThreads), 0, s, a);
    });
    return launch_status();
}

template <class E>
int backward(const mi_lora* d, const void* dy, const void* x, const void* A, const void* B, const float* scales, const int32_t* plan,
             const float* shrunk, const void* dx_in, void* dx, void* dA, void* dB, unsigned char* ws, hipStream_t s)
{
    const BackwardPlan b(d);
    float* P = reinterpret_cast<float*>(ws);
    const Rows rx{x, d->x_stride}, rdy{dy, d->y_stride};
    int st;
    if (d->tokens == 0) {
        WeightSumArgs w{plan, P, {dA, dB}, 0, d->n_adapters, d->rank, {d->K, d->N}};
        hipLaunchKernelGGL((weight_sum_kernel<E>), dim3(64, d->n_adapters), dim3(kThreads), 0, s, w);
        return launch_status();
    }
    if (!shrunk) {  // u again
        if ((st = contract<E>(d, plan, rx, A, d->K, b.u, P, s)) != MI_OK) return st;
        float* u = reinterpret_cast<float*>(ws + b.shrunk);
        // the sums into the tokens' order: an expansion to no columns
        if ((st = expand<E>(d, plan, {nullptr, 0}, nullptr, 0, A, 0, nullptr, b.u, P, u, s)) != MI_OK) return st;
        shrunk = u;
    }
    const uint32_t across = (d->rank + 63u) / 64u;
    TransposeArgs t{plan, {A, B}, {ws + b.at, ws + b.bt}, d->tokens, d->n_adapters, {d->rank, d->N}, {d->K, d->rank}, across * ((d->K + 63u) / 64u)};
    hipLaunchKernelGGL((transpose_kernel<E>), dim3(t.blocks0 + across * ((d->N + 63u) / 64u), d->n_adapters), dim3(kThreads), 0, s, t);
    if ((st = launch_status()) != MI_OK) return st;
    if ((st = contract<E>(d, plan, rdy, ws + b.bt, d->N, b.f, P, s)) != MI_OK) return st;
    if ((st = expand<E>(d, plan, {dx_in, d->out_stride}, dx, d->out_stride, ws + b.at, d->K, scales, b.f, P, nullptr, s)) != MI_OK) return st;
    const PlanLayout L(d->tokens, d->n_adapters);
    PiecesArgs p{plan, P, shrunk, scales, {ws + b.pieces[0], ws + b.pieces[1]}, reinterpret_cast<float*>(ws + b.down),
                 d->tokens, L.max_tiles, d->n_adapters, d->rank, b.f.rp, b.f.splits};
    hipLaunchKernelGGL((weight_pieces_kernel<E>), dim3((uint32_t)L.max_tiles, 2), dim3(kThreads), 0, s, p);
    if ((st = launch_status()) != MI_OK) return st;
    const uint32_t cols = 16u * Mx<E>::VEC, blocks0 = (d->K + cols - 1u) / cols, blocks1 = (d->N + cols - 1u) / cols;
    WeightArgs w{plan, {rx, rdy}, {p.pieces[0], p.pieces[1]}, p.down, reinterpret_cast<float*>(ws + b.partials), {dA, dB},
                 d->tokens, L.max_tiles, d->n_adapters, d->rank, b.f.rp, {d->K, d->N}, blocks0};
    const uint32_t rt = b.f.rp <= 64u ? b.f.rp : 64u;
    const dim3 grid(blocks0 + blocks1, (uint32_t)L.max_chunks, b.f.rp / rt);
    if (rt == 16u) hipLaunchKernelGGL((weight_rows_kernel<E, 1>), grid, dim3(kThreads), 0, s, w);
    else if (rt == 32u) hipLaunchKernelGGL((weight_rows_kernel<E, 2>), grid, dim3(kThreads), 0, s, w);
    else hipLaunchKernelGGL((weight_rows_kernel<E, 4>), grid, dim3(kThreads), 0, s, w);
    if ((st = launch_status()) != MI_OK) return st;
    WeightSumArgs sum{plan, w.partials, {dA, dB}, d->tokens, d->n_adapters, d->rank, {d->K, d->N}};
    hipLaunchKernelGGL((weight_sum_kernel<E>), dim3(64, d->n_adapters), dim3(kThreads), 0, s, sum);
    return launch_status();
}

}  // namespace
}  // namespace adapters
}  // namespace mi

extern "C" uint64_t mi_lora_workspace(const mi_lora* d, int backward)
{
    using namespace mi::adapters;
    if (check(d) != MI_OK) return 0;
    return backward ? BackwardPlan(d).bytes : ForwardPlan(d, d->K, d->N).bytes;
}

extern "C" int mi_lora_add(const void* y, const void* x, const void* A, const void* B, const float* scales, const int32_t* plan, void* out,
                           float* shrunk, void* workspace, const mi_lora* d, void* stream)
{
    using namespace mi;
    using namespace mi::adapters;
    int st = check(d);
    if (st != MI_OK || d->tokens == 0) return st;
    if (!y || !x || !A || !B || !plan || !out || !workspace) return MI_ERR_NULL;
    if (!aligned16(y) || !aligned16(x) || !aligned16(A) || !aligned16(B) || !aligned16(plan) || !aligned16(out) || !aligned16(workspace) ||
        reinterpret_cast<uintptr_t>(scales) & 3u || reinterpret_cast<uintptr_t>(shrunk) & 3u)
        return MI_ERR_ALIGN;
    if (y == out && d->y_stride != d->out_stride && d->tokens > 1u) return MI_ERR_ALIAS;
    const ForwardPlan f(d, d->K, d->N);
    hipStream_t s = static_cast<hipStream_t>(stream);
    float* P = static_cast<float*>(workspace);
    auto both = [&](auto e) {
        using E = decltype(e);
        const int first = contract<E>(d, plan, {x, d->x_stride}, A, d->K, f, P, s);
        return first != MI_OK ? first
                              : expand<E>(d, plan, {y, d->y_stride}, out, d->out_stride, B, d->N, scales, f, P, shrunk, s);
    };
    return d->dtype == MI_F32 ? both(float{}) : d->dtype == MI_BF16 ? both(__bf16{}) : both(_Float16{});
}

extern "C" int mi_lora_add_backward(const void* dy, const void* x, const void* A, const void* B, const float* scales, const int32_t* plan,
                                    const float* shrunk, const void* dx_in, void* dx, void* dA, void* dB, void* workspace,
                                    const mi_lora* d, void* stream)
{
    using namespace mi;
    using namespace mi::adapters;
    const int st = check(d);
    if (st != MI_OK) return st;
    if (!A || !B || !plan || !dA || !dB || !workspace || (d->tokens && (!dy || !x || !dx))) return MI_ERR_NULL;
    if (!aligned16(dy) || !aligned16(x) || !aligned16(A) || !aligned16(B) || !aligned16(plan) || !aligned16(dx_in) || !aligned16(dx) ||
        !aligned16(dA) || !aligned16(dB) || !aligned16(workspace) || reinterpret_cast<uintptr_t>(scales) & 3u ||
        reinterpret_cast<uintptr_t>(shrunk) & 3u)
        return MI_ERR_ALIGN;
    hipStream_t s = static_cast<hipStream_t>(stream);
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    if (d->dtype == MI_F32) return backward<float>(d, dy, x, A, B, scales, plan, shrunk, dx_in, dx, dA, dB, ws, s);
    if (d->dtype == MI_BF16) return backward<__bf16>(d, dy, x, A, B, scales, plan, shrunk, dx_in, dx, dA, dB, ws, s);
    return backward<_Float16>(d, dy, x, A, B, scales, plan, shrunk, dx_in, dx, dA, dB, ws, s);
}
