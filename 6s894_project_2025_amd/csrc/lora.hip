// Low-rank adapters of many requests added to a shared projection (mi_lora_add), and the gradients
// (mi_lora_add_backward).  Token t with adapter a, A[a] [r,K], B[a] [N,r], factor s[a]:
//   u_t = A x_t                        out_t = y_t + s B u_t
//   d_t = s B^T g_t   (g = dy)         dx_t  = A^T d_t
//   dA  = sum_t d_t x_t^T              dB    = sum_t s g_t u_t^T
// With r small against K and N all of it is bound by reading x, y (g) and writing out (dx); the matrix
// cores have time to spare, and the kernels spend some of it on accuracy: u and d stay in 32 bits
// through being split into 16-bit pieces that all go through the matrix core.  Three bf16 pieces are the
// fp32 value itself (8 significand bits each).  Two fp16 pieces are within 2^-24 of it (11 bits, 11 of the rest
// and the rest's sign), what one fp32 rounding adds and less than the sums behind u and d have; they are taken
// after a scaling by a power of two, so that neither large nor very small values (gradients) leave the
// type's range.  (Two bf16 pieces, within 2^-18, moved one output in 1500 to a neighbouring bf16 value.)
//
// Tokens come grouped by adapter (adapter_plan.hpp), in tiles of up to 64 of one adapter.
//   contract_rows   P[split][position][r] = sum over a part of the long axis of row . M[a]:  u, and d / s
//   expand_rows     out = y + s (sum of P) M'[a]^T:  the forward output, and dx
//   gradient_rows   dB of a chunk of tokens and P of d, from one pass over g
//   tile_vectors    the sums of P times s, split, as operands of expand_rows and, transposed, of weight_rows;
//                   and A^T of the adapters in use, for dx by expand_rows
//   weight_rows     dA of a chunk of tokens;  weight_sum adds the weights' parts up
// All sums are in a fixed order.
//
// Bound: HBM.  A rank r is 2r operations a value of x and 4r or 6r (two or three pieces) a value of y, and the matrix cores do
// hundreds in the time of reading one from memory, so each kernel is one pass over a long matrix, and only
// rank-space vectors (4r bytes a token and part of the axis) go between them.  8192 tokens, 4096 -> 14336, bf16:
//   forward, 8 adapters, rank 64: contract_rows 23 us (67 MB in, 15 out), tile_vectors 6, expand_rows 104
//     (470 MB, 4.8 TB/s with what it reads again; a plain copy of 4 GB reaches 4.7, of 512 MB 5.4)
//   backward, 4 adapters, rank 16: gradient_rows 50 (206 MB in, 26 out, 4.6 TB/s), weight_rows 14 (67 MB),
//     expand_rows 15 (67 MB out), weight_sum 5, tile_vectors 5 twice
//   the same of rank 64: gradient_rows 149 (235 MB in, 107 out), weight_rows 35, expand_rows 20, weight_sum 14,
//     tile_vectors 5 and 12: no longer the bytes, but what a step waits for with one wavefront per SIMD
// Few tokens are bound by their launches (one token: 3 and 4 us).
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
    static constexpr int DTYPE = MI_BF16;
    static constexpr uint32_t VEC = 8, STEP = 32, PIECES = 3;
    static constexpr bool SCALED = false;
    using V = bf16x8;
    static __device__ __forceinline__ f32x4 mma(V a, V b, f32x4 c) { return BF16::mfma32(a, b, c); }
};
template <> struct Mx<_Float16> {
    static constexpr int DTYPE = MI_F16;
    static constexpr uint32_t VEC = 8, STEP = 32, PIECES = 2;
    static constexpr bool SCALED = true;
    using V = f16x8;
    static __device__ __forceinline__ f32x4 mma(V a, V b, f32x4 c) { return F16::mfma32(a, b, c); }
};
template <> struct Mx<float> {
    static constexpr int DTYPE = MI_F32;
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

// The sum of the pieces is v (but for the last bits of two); behind a first one that is not finite they are zero, so
// that an infinity stays one.
template <class E, uint32_t N>
__device__ __forceinline__ void split(float v, E (&piece)[N])
{
    piece[0] = (E)v;
    float rest = __builtin_fabsf((float)piece[0]) < __builtin_inff() ? v - (float)piece[0] : 0.0f;
#pragma unroll
    for (uint32_t p = 1; p < N; ++p) {
        piece[p] = (E)rest;
        rest -= (float)piece[p];  // exact
    }
}

// Bytes of a tile's 64 vectors of padded rank rp: as pieces, and as the expansion's operand, where three pieces
// of 16 ranks take the place of four (Operand::PAIR).
constexpr uint64_t pieces_bytes(int dtype, uint32_t rp) { return (uint64_t)rp * 64u * (dtype == MI_BF16 ? 6u : 4u); }
constexpr uint64_t vectors_bytes(int dtype, uint32_t rp) { return dtype == MI_BF16 && rp == 16u ? 8192u : pieces_bytes(dtype, rp); }

// Pieces meet an infinite operand one by one, and the later ones, zero or of the other sign, would make NaN of its
// infinity.  The first piece alone gives the sign and the class of the whole product, so results that are not
// finite are replaced by those of the first pieces (computed again: no cost but a sum where all is finite, as
// a finite result of all pieces has met finite operands only).  An fp16 value below 2^-40 of the largest that it is
// scaled with has a first piece of zero: that one makes NaN of an infinity.
template <int N>
__device__ __forceinline__ bool any_not_finite(const f32x4 (&v)[N])  // the same answer in all lanes
{
    f32x4 sum = v[0];  // what is not finite stays so; sums of finite values that overflow only cost time
#pragma unroll
    for (int i = 1; i < N; ++i) sum += v[i];
    return __ballot(!(__builtin_fabsf((sum[0] + sum[1]) + (sum[2] + sum[3])) < __builtin_inff())) != 0;
}
__device__ __forceinline__ void take_if_not_finite(f32x4& v, f32x4 first)
{
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = __builtin_fabsf(v[q]) < __builtin_inff() ? v[q] : first[q];
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
    uint32_t n, rank, K, splits;  // workgroup `split` takes every splits-th block of K
};

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

// P^T tile = M (rows: r) . x^T (columns: tokens), in blocks of 256 bytes of every row, which is how x and M are
// read (16 lanes a row) on their way into LDS; there the 16-byte pieces of row i are permuted by i, so that 16
// rows' pieces of one column come from 16 different groups of banks.  The workgroup's wavefronts take 16 tokens
// each and share the block of M, which has two buffers; with FEW they take every fourth block for the same 16
// tokens, each with its own M, and add up at the end.  The next block is requested before the present one is
// computed.  Columns behind the tile's tokens repeat the first of the 16 and rows behind the rank the first
// rank: the loads need no masks, and what they give is not stored.  LIVE: the wavefront has tokens.
template <class E, int RT, bool FEW>
struct Contraction {
    static constexpr uint32_t COLS = 256u / sizeof(E);            // k of a block
    static constexpr uint32_t ROWS_X = 16u * 256u;                // bytes of a wavefront's x
    static constexpr uint32_t ROWS_M = 16u * RT * 256u;           // bytes of M of a block
    static constexpr uint32_t LDS = 4u * ROWS_X + (FEW ? 4u : 2u) * ROWS_M;
    static __device__ __forceinline__ uint32_t at(uint32_t row, uint32_t piece) { return row * 256u + ((piece ^ row) & 15u) * 16u; }
};

template <class E, int RT, bool FEW, bool LIVE>
__device__ __forceinline__ void contract_blocks(const ContractArgs& a, const Tile& tile, uint32_t split, unsigned char* lds)
{
    using X = Mx<E>;
    using V = typename X::V;
    using C = Contraction<E, RT, FEW>;
    constexpr uint32_t VEC = X::VEC, MROWS = FEW ? 4u : 16u, MLOADS = 16u * RT / MROWS;  // rows of M per round of loads, rounds
    const uint32_t lane = threadIdx.x & 63u, wave = this_wave(), lo = lane & 15u, g = lane >> 4;
    const PlanLayout L(a.tokens, a.n);
    // every step-th block of K from the first
    const uint32_t all = (a.K + C::COLS - 1u) / C::COLS, first = FEW ? split + a.splits * wave : split, step = FEW ? 4u * a.splits : a.splits;
    const uint32_t blocks = all > first ? (all - first + step - 1u) / step : 0u;
    const uint32_t sub = FEW ? 0u : 16u * wave;
    unsigned char* const xl = lds + wave * C::ROWS_X;
    unsigned char* const ml = lds + 4u * C::ROWS_X + (FEW ? wave * C::ROWS_M : 0u);

    const E* xr[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t at = sub + 4u * j + g;
        const int32_t t = LIVE ? a.plan[L.order + (uint32_t)tile.first + (at < (uint32_t)tile.count ? at : sub)] : 0;
        xr[j] = static_cast<const E*>(a.x.p) + (uint64_t)(uint32_t)t * a.x.stride;
    }
    const uint32_t mrow = FEW ? g : threadIdx.x >> 4;
    const E* M = static_cast<const E*>(a.M) + (uint64_t)tile.adapter * a.rank * a.K;

    u32x4 xs[4], ms[MLOADS];
    auto column = [&](uint32_t i) { return (first + step * i) * C::COLS + VEC * lo; };
    auto request = [&](uint32_t i) __attribute__((always_inline)) {
        const uint32_t k = column(i) < a.K ? column(i) : 0u;
        if (LIVE)
#pragma unroll
            for (int j = 0; j < 4; ++j) xs[j] = load16<u32x4>(xr[j] + k);
#pragma unroll
        for (uint32_t j = 0; j < MLOADS; ++j) {
            const uint32_t r = mrow + MROWS * j;
            ms[j] = load16<u32x4>(M + (uint64_t)(r < a.rank ? r : 0u) * a.K + k);
        }
    };
    auto stage = [&](uint32_t i, unsigned char* to) __attribute__((always_inline)) {
        const u32x4 zero = {0u, 0u, 0u, 0u};
        const bool in = column(i) < a.K;
        if (LIVE)
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<u32x4*>(xl + C::at(4u * j + g, lo)) = in ? xs[j] : zero;
#pragma unroll
        for (uint32_t j = 0; j < MLOADS; ++j) *reinterpret_cast<u32x4*>(to + C::at(mrow + MROWS * j, lo)) = in ? ms[j] : zero;
    };
    f32x4 acc[RT] = {};
    auto compute = [&](const unsigned char* from) __attribute__((always_inline)) {
        if (!LIVE) return;
#pragma unroll
        for (uint32_t h = 0; h < 4; ++h) {
            const V x = *reinterpret_cast<const V*>(xl + C::at(lo, 4u * h + g));
#pragma unroll
            for (uint32_t j = 0; j < RT; ++j) acc[j] = X::mma(*reinterpret_cast<const V*>(from + C::at(16u * j + lo, 4u * h + g)), x, acc[j]);
        }
    };
    auto meet = [&]() __attribute__((always_inline)) {
        if (FEW) __builtin_amdgcn_wave_barrier();
        else __syncthreads();
    };
    if (blocks) {
        request(0);
        stage(0, ml);
        meet();
        uint32_t at = 0;
        for (uint32_t i = 0; i + 1u < blocks; ++i) {
            request(i + 1u);
            compute(ml + at);
            if (!FEW) at ^= C::ROWS_M;
            __builtin_amdgcn_wave_barrier();  // x is the wavefront's own
            stage(i + 1u, ml + at);
            meet();
        }
        compute(ml + at);
    }
    if constexpr (FEW) {  // wavefronts 2, 3 to 0, 1, then 1 to 0
        f32x4* const red = reinterpret_cast<f32x4*>(lds);
        __syncthreads();
#pragma unroll
        for (uint32_t half = 2; half; half >>= 1) {
            if (wave >= half && wave < 2u * half) {
#pragma unroll
                for (int j = 0; j < RT; ++j) red[((wave - half) * RT + j) * 64u + lane] = acc[j];
            }
            __syncthreads();
            if (wave < half) {
#pragma unroll
                for (int j = 0; j < RT; ++j) acc[j] += red[(wave * RT + j) * 64u + lane];
            }
            __syncthreads();
        }
        if (wave) return;
    }
    if (!LIVE) return;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    if (sub + lo >= (uint32_t)tile.count) return;
    float* P = a.P + ((uint64_t)split * a.tokens + (uint32_t)tile.first + sub + lo) * (16u * RT);
#pragma unroll
    for (int j = 0; j < RT; ++j) *reinterpret_cast<f32x4*>(P + 16u * j + 4u * g) = 16u * j + 4u * g < a.rank ? acc[j] : zero;
}

template <class E, int RT, bool FEW>
__global__ void __launch_bounds__(256, RT == 8 ? 1 : 2) contract_rows_kernel(ContractArgs a)
{
    __shared__ __attribute__((aligned(16))) unsigned char lds[Contraction<E, RT, FEW>::LDS];
    const PlanLayout L(a.tokens, a.n);
    Tile tile;
    uint32_t split;
    if (!take_tile<FEW>(a.plan, L, a.splits, tile, split) || (uint32_t)tile.adapter >= a.n) return;
    // every wavefront meets the same barriers on either way
    if (FEW || 16u * this_wave() < (uint32_t)tile.count) contract_blocks<E, RT, FEW, true>(a, tile, split, lds);
    else contract_blocks<E, RT, FEW, false>(a, tile, split, lds);
}

// ------------------------------------------------------------------------------------------------
// The expansion's matrix-core operands.  out tile = v (rows: 16 tokens) . M^T (columns: n), and column c of the
// operand t stands for n = base + VEC c + t: a lane's results over t are then VEC consecutive values of a
// token, and 16 lanes have 256 contiguous bytes of it, which is how y is read and out written.  (With 64
// contiguous bytes of 16 tokens, the other way round, the address units bound the kernel.)
template <class E, int RT>
struct Operand {
    using X = Mx<E>;
    static constexpr bool PAIR = X::PIECES > 1 && RT == 1;  // two pieces a step, one in lane groups 0, 1, one in 2, 3
    static constexpr int NF = X::PIECES > 1 ? (RT + 1) / 2 : RT;
    static constexpr int NP = PAIR ? (X::PIECES + 1) / 2 : X::PIECES;
    static constexpr uint32_t COLS = 16u * X::VEC;           // n of a block
    static constexpr uint32_t VECTORS = 4u * NF * NP * 1024u;  // bytes: v of 64 tokens
    static constexpr uint32_t BLOCK = 16u * RT * 256u;         // bytes: M of a block
    // byte offset of piece p of rank r of token t (0 ... 63)
    static __device__ __forceinline__ uint32_t vector_at(uint32_t t, uint32_t r, uint32_t p)
    {
        const uint32_t f = PAIR ? 0u : r / X::STEP, g = PAIR ? r / 8u + 2u * (p & 1u) : r % X::STEP / X::VEC;
        return (((t >> 4) * NF + f) * NP + (PAIR ? p / 2u : p)) * 1024u + (16u * g + (t & 15u)) * 16u + r % X::VEC * (uint32_t)sizeof(E);
    }
    // byte offset of the 16 bytes that lane (c, g) reads for operand t and fragment f.  Rows n and n + 1 of M
    // come in together and go to operands t and t + 1; the exclusive or spreads them over the banks.
    static __device__ __forceinline__ uint32_t row_at(uint32_t t, uint32_t f, uint32_t c, uint32_t g)
    {
        return (t * NF + f) * (PAIR ? 512u : 1024u) + (16u * g + (c ^ (t | (f & 1u) << 3))) * 16u;
    }
};

// The sums of P of four threads per token, 4 RT ranks each (token threadIdx.x / 4).
template <int RT>
__device__ __forceinline__ void sum_parts(const float* P, uint64_t tokens, uint32_t splits, uint64_t position, f32x4 (&sum)[RT])
{
    P += position * (16u * RT) + (threadIdx.x & 3u) * 4u * RT;
#pragma unroll
    for (int i = 0; i < RT; ++i) sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t sp = 0; sp < splits; ++sp)
#pragma unroll
        for (int i = 0; i < RT; ++i) sum[i] += load16<f32x4>(P + (uint64_t)sp * tokens * (16u * RT) + 4 * i);
}

template <int RT>
__device__ __forceinline__ void store_shrunk(float* u, uint32_t rank, const f32x4 (&sum)[RT])
{
    const uint32_t r0 = (threadIdx.x & 3u) * 4u * RT;
#pragma unroll
    for (int i = 0; i < RT; ++i)
        if (r0 + 4u * i < rank)
#pragma unroll
            for (int c = 0; c < 4; ++c) u[r0 + 4u * i + c] = sum[i][c];
}

// A token's vector as the expansion's operand; returns the inverse of its scaling.
template <class E, int RT>
__device__ __forceinline__ float store_vector(const f32x4 (&v)[RT], uint32_t t, unsigned char* to)
{
    using X = Mx<E>;
    using O = Operand<E, RT>;
    typedef E E4 __attribute__((ext_vector_type(4)));
    const uint32_t r0 = (threadIdx.x & 3u) * 4u * RT;
    float up = 1.0f, down = 1.0f;
    if constexpr (X::SCALED) {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) m = fmaxf(m, finite_magnitude(v[i][c]));
        m = fmaxf(m, __shfl_xor(m, 1));
        m = fmaxf(m, __shfl_xor(m, 2));
        half_scale(m, up, down);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        if constexpr (X::PIECES == 1) {
            *reinterpret_cast<f32x4*>(to + O::vector_at(t, r0 + 4u * i, 0)) = v[i];
        } else {
            E4 four[X::PIECES + 1] = {};  // and zeros in an odd pair's other half
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                E piece[X::PIECES];
                split(v[i][c] * up, piece);
#pragma unroll
                for (uint32_t p = 0; p < X::PIECES; ++p) four[p][c] = piece[p];
            }
#pragma unroll
            for (uint32_t p = 0; p < (O::PAIR ? 2u * O::NP : X::PIECES); ++p)
                *reinterpret_cast<E4*>(to + O::vector_at(t, r0 + 4u * i, p)) = four[p];
        }
    }
    return down;
}

// The source of a tile's token t: tokens behind the tile's repeat the first of their 16, if there is one.
__device__ __forceinline__ uint32_t source_token(uint32_t t, uint32_t count)
{
    return t < count ? t : (t & ~15u) < count ? t & ~15u : 0u;
}

// ------------------------------------------------------------------------------------------------
// A^T of the adapters in use, for dx: a thread has eight ranks of one k, so that reads are whole lines along k and
// the stores 16 or 32 bytes of neighbouring rows.
template <class E>
__device__ __forceinline__ void transpose_adapters(const int32_t* plan, const PlanLayout& L, const E* A, E* At, uint32_t rank, uint32_t K,
                                                   uint32_t block)
{
    typedef E E4 __attribute__((ext_vector_type(4)));
    const uint32_t blocks_k = (K + kThreads - 1u) / kThreads, rest = block / blocks_k;
    const uint32_t k = (block - rest * blocks_k) * kThreads + threadIdx.x, r0 = rest % (rank / 8u) * 8u, ad = rest / (rank / 8u);
    if (k >= K || plan[L.starts + ad] == plan[L.starts + ad + 1u]) return;
    const E* src = A + ((uint64_t)ad * rank + r0) * K + k;
    E4 v[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = src[(uint64_t)i * K];
    E4* dst = reinterpret_cast<E4*>(At + ((uint64_t)ad * K + k) * rank + r0);
    dst[0] = v[0];
    dst[1] = v[1];
}

struct VectorArgs {
    const int32_t* plan;
    const float* P;        // [splits][tokens][16 RT]
    const float* scales;   // [n] or NULL
    float* shrunk;         // NULL, or [tokens][rank]: receives the sums of P; with `given`, holds them
    unsigned char* vectors;  // NULL, or [tiles][Operand::VECTORS]
    float* down;             // [tiles][64]
    void* pieces;            // NULL, or [tiles][16 RT][PIECES][64]: transposed, for the contraction over tokens
    float* tile_down;        // [tiles]
    uint64_t tokens;
    uint32_t n, rank, splits;
    bool given;
    const void* A;         // NULL, or [n][rank][K]: workgroups behind the tiles' transpose it
    void* At;              // [n][K][rank]
    uint32_t K, tiles;     // workgroups of the tiles
};

// Where a tile is used by many workgroups: its vectors once, from the sums of P (or from the given ones) times
// the factor.
template <class E, int RT>
__global__ void __launch_bounds__(256) tile_vectors_kernel(VectorArgs a)
{
    using X = Mx<E>;
    using O = Operand<E, RT>;
    constexpr uint32_t RP = 16u * RT;
    __shared__ float top[4];
    __shared__ E turned[RP * X::PIECES * 64u];
    const PlanLayout L(a.tokens, a.n);
    if (blockIdx.x >= a.tiles)
        return transpose_adapters<E>(a.plan, L, static_cast<const E*>(a.A), static_cast<E*>(a.At), a.rank, a.K, blockIdx.x - a.tiles);
    const Tile tile = reinterpret_cast<const Tile*>(a.plan)[blockIdx.x];
    if (blockIdx.x >= (uint32_t)a.plan[L.counts]) return;
    const uint32_t t = threadIdx.x >> 2, r0 = (threadIdx.x & 3u) * 4u * RT, count = (uint32_t)tile.count;
    const bool live = t < count;
    const uint64_t position = (uint64_t)(uint32_t)tile.first + source_token(t, count);
    const uint64_t token = (uint64_t)(uint32_t)a.plan[L.order + position];
    if ((uint32_t)tile.adapter >= a.n) {
        if (a.shrunk && !a.given && live) {
            f32x4 zero[RT] = {};
            store_shrunk<RT>(a.shrunk + token * a.rank, a.rank, zero);
        }
        return;
    }
    const float s = a.scales ? a.scales[tile.adapter] : 1.0f;
    f32x4 sum[RT] = {};
    if (a.given) {
#pragma unroll
        for (int i = 0; i < RT; ++i)
            if (r0 + 4u * i < a.rank)
#pragma unroll
                for (int c = 0; c < 4; ++c) sum[i][c] = a.shrunk[token * a.rank + r0 + 4u * i + c];
    } else {
        sum_parts<RT>(a.P, a.tokens, a.splits, position, sum);
        if (a.shrunk && live) store_shrunk<RT>(a.shrunk + token * a.rank, a.rank, sum);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) sum[i] = sum[i] * s;
    if (a.vectors) {
        const float d = store_vector<E, RT>(sum, t, a.vectors + (uint64_t)blockIdx.x * O::VECTORS);
        if (X::SCALED && (threadIdx.x & 3u) == 0) a.down[(uint64_t)blockIdx.x * 64u + t] = d;
    }
    if (!a.pieces) return;
    float up = 1.0f;
    if constexpr (X::SCALED) {
        float m = 0.0f, d;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) m = fmaxf(m, finite_magnitude(sum[i][c]));
        for (int w = 1; w < 64; w <<= 1) m = fmaxf(m, __shfl_xor(m, w));
        if ((threadIdx.x & 63u) == 0) top[threadIdx.x >> 6] = m;
        __syncthreads();
        m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        half_scale(m, up, d);
        if (threadIdx.x == 0) a.tile_down[blockIdx.x] = d;
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float v = live ? sum[i][c] * up : 0.0f;  // zeros behind the tile's tokens
            E* to = turned + (r0 + 4u * i + c) * X::PIECES * 64u + t;
            if constexpr (X::PIECES == 1) {
                to[0] = v;
            } else {
                E piece[X::PIECES];
                split(v, piece);
#pragma unroll
                for (uint32_t p = 0; p < X::PIECES; ++p) to[64u * p] = piece[p];
            }
        }
    __syncthreads();
    constexpr uint32_t BYTES = RP * X::PIECES * 64u * sizeof(E);
    static_assert(BYTES == pieces_bytes(X::DTYPE, RP) && O::VECTORS == vectors_bytes(X::DTYPE, RP), "what the workspace has");
    for (uint32_t i = 16u * threadIdx.x; i < BYTES; i += 16u * kThreads)
        *reinterpret_cast<u32x4*>(static_cast<unsigned char*>(a.pieces) + (uint64_t)blockIdx.x * BYTES + i) =
            *reinterpret_cast<const u32x4*>(reinterpret_cast<const unsigned char*>(turned) + i);
}

// ------------------------------------------------------------------------------------------------
struct ExpandArgs {
    const int32_t* plan;
    Rows y;              // added to
    void* out;
    uint64_t out_stride;
    const void* M;       // [n][N][rank]
    // either: the tiles' vectors, and what undoes their scaling
    const unsigned char* vectors;  // [tiles][Operand::VECTORS], NULL with OWN
    const float* down;             // [tiles][64]
    // or, with OWN: what they are made from, and u as an output
    const float* scales;           // [n] or NULL
    const float* P;                // [splits][tokens][16 RT]
    float* shrunk;                 // [tokens][rank] or NULL
    uint64_t tokens;
    uint32_t n, rank, N, splits, parts;  // workgroup `part` takes every parts-th block of N
};

// A wavefront's blocks of the part, COLS columns each.  The workgroup's wavefronts take 16 tokens each and share
// the block of M, which goes through one of two LDS buffers; with FEW each has its own blocks for the same 16
// tokens, and a buffer of its own.  The next block of M and y is requested before the present one is
// computed.  LIVE: the wavefront has tokens.  Tokens behind the tile's are the first of the 16 again and
// columns behind N the last VEC: these lanes compute and store what the owner does, from a y that was loaded
// before the owner stores (out may be y), so that no load or store stands behind a branch.
template <class E, int RT, bool HAS_Y, bool FEW, bool OWN, bool LIVE>
__device__ __forceinline__ void expand_blocks(const ExpandArgs& a, const Tile& tile, uint32_t part, unsigned char* lds,
                                              const unsigned char* vectors, const float* down)
{
    using X = Mx<E>;
    using V = typename X::V;
    using O = Operand<E, RT>;
    constexpr uint32_t VEC = X::VEC, COLS = O::COLS;
    constexpr int NF = O::NF, NP = O::NP;
    constexpr uint32_t STAGERS = FEW ? 64u : 256u, CHUNKS = 16u * RT * 16u / STAGERS;  // 16-byte pieces of M per thread
    constexpr uint32_t PER_ROW = 16u * RT / VEC;
    const uint32_t lane = threadIdx.x & 63u, wave = this_wave(), c = lane & 15u, g = lane >> 4;
    const PlanLayout L(a.tokens, a.n);
    // every step-th block of N from the first
    const uint32_t all = (a.N + COLS - 1u) / COLS, first = FEW ? part + a.parts * wave : part, step = FEW ? 4u * a.parts : a.parts;
    const uint32_t blocks = all > first ? (all - first + step - 1u) / step : 0u;

    // v of the wavefront's tokens, and where their rows are
    V vf[NF][NP];
    const E* yr[4];
    E* outr[4];
    float d[4];
    if (LIVE) {
        const uint32_t sub = FEW ? 0u : wave;
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int p = 0; p < NP; ++p) vf[f][p] = *reinterpret_cast<const V*>(vectors + ((sub * NF + f) * NP + p) * 1024u + lane * 16u);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t at = 16u * sub + 4u * g + q;
            if (at >= (uint32_t)tile.count) at = 16u * sub;
            const uint64_t t = (uint64_t)(uint32_t)a.plan[L.order + (uint32_t)tile.first + at];
            yr[q] = static_cast<const E*>(a.y.p) + t * a.y.stride;
            outr[q] = static_cast<E*>(a.out) + t * a.out_stride;
            d[q] = X::SCALED ? down[at] : 1.0f;
        }
    }
    if (OWN) __syncthreads();  // the buffers of M take the place of the vectors
    if (FEW && !blocks) return;
    unsigned char* const buffer = FEW ? lds + wave * O::BLOCK : lds;

    const E* M = static_cast<const E*>(a.M) + (uint64_t)tile.adapter * a.N * a.rank;
    auto first_column = [&](uint32_t i) { return (first + step * i) * COLS; };
    u32x4 staged[CHUNKS];
    auto request_rows = [&](uint32_t i) __attribute__((always_inline)) {
        const uint32_t base = first_column(i);
#pragma unroll
        for (uint32_t k = 0; k < CHUNKS; ++k) {
            const uint32_t id = (FEW ? lane : threadIdx.x) + k * STAGERS, row = id / PER_ROW, r = id % PER_ROW * VEC;
            const uint32_t n = base + row < a.N ? base + row : a.N - 1u;  // rows behind N are not read back
            staged[k] = load16<u32x4>(M + (uint64_t)n * a.rank + (r < a.rank ? r : 0u));
        }
    };
    auto stage_rows = [&](unsigned char* to) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t k = 0; k < CHUNKS; ++k) {
            const uint32_t id = (FEW ? lane : threadIdx.x) + k * STAGERS, row = id / PER_ROW, r = id % PER_ROW * VEC;
            const u32x4 zero = {0u, 0u, 0u, 0u};
            const uint32_t chunk = r / VEC;
            *reinterpret_cast<u32x4*>(to + O::row_at(row % VEC, chunk / 4u, row / VEC, chunk % 4u)) = r < a.rank ? staged[k] : zero;
        }
    };
    V y[2][4];
    auto column = [&](uint32_t i) {
        const uint32_t n = first_column(i) + VEC * c;
        return n < a.N ? n : a.N - VEC;
    };
    auto request_y = [&](V (&to)[4], uint32_t i) __attribute__((always_inline)) {
        if (LIVE && HAS_Y)
#pragma unroll
            for (int q = 0; q < 4; ++q) to[q] = load16<V>(yr[q] + column(i));
    };
    auto compute = [&](const unsigned char* from, const V (&y)[4], uint32_t i) __attribute__((always_inline)) {
        if (!LIVE) return;
        const uint32_t base = first_column(i), col = column(i), cc = (col - base) / VEC;
        f32x4 acc[VEC] = {};
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (uint32_t t = 0; t < VEC; ++t) {
                const V m = *reinterpret_cast<const V*>(from + O::row_at(t, f, cc, O::PAIR ? g & 1u : g));
#pragma unroll
                for (int p = 0; p < NP; ++p) acc[t] = X::mma(vf[f][p], m, acc[t]);
            }
        if constexpr (X::PIECES > 1) {
            if (any_not_finite(acc)) {
                uint32_t again = cc, group = g;
                asm volatile("" : "+v"(again), "+v"(group));  // nothing of this is kept in registers on the usual way
#pragma unroll
                for (uint32_t t = 0; t < VEC; ++t) {
                    f32x4 first = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int f = 0; f < NF; ++f) {
                        V m = *reinterpret_cast<const V*>(from + O::row_at(t, f, again, O::PAIR ? group & 1u : group));
                        if (O::PAIR && group >= 2u) m = V{};  // what meets the second piece of a pair
                        first = X::mma(vf[f][0], m, first);
                    }
                    take_if_not_finite(acc[t], first);
                }
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            V o;
#pragma unroll
            for (uint32_t t = 0; t < VEC; ++t) {
                float v = acc[t][q];
                if (HAS_Y) v = X::SCALED ? __builtin_fmaf(v, d[q], (float)y[q][t]) : v + (float)y[q][t];
                else if (X::SCALED) v *= d[q];
                o[t] = (E)v;
            }
            __builtin_nontemporal_store(o, reinterpret_cast<V*>(outr[q] + col));
        }
    };
    auto meet = [&]() __attribute__((always_inline)) {
        if (FEW) __builtin_amdgcn_wave_barrier();
        else __syncthreads();
    };
    // block i from its buffer while block i + 1 comes in
    auto advance = [&](const V (&now)[4], V (&next)[4], uint32_t i) __attribute__((always_inline)) {
        request_rows(i + 1u);
        request_y(next, i + 1u);
        compute(buffer + (FEW ? 0u : (i & 1u) * O::BLOCK), now, i);
        if (FEW) meet();
        stage_rows(buffer + (FEW ? 0u : (i + 1u & 1u) * O::BLOCK));
        meet();
    };
    request_rows(0);
    request_y(y[0], 0);
    stage_rows(buffer);
    meet();
    uint32_t i = 0;
    for (; i + 2u < blocks; i += 2u) {
        advance(y[0], y[1], i);
        advance(y[1], y[0], i + 1u);
    }
    if (i + 1u < blocks) {
        advance(y[0], y[1], i);
        compute(buffer + (FEW ? 0u : O::BLOCK), y[1], i + 1u);
    } else {
        compute(buffer, y[0], i);
    }
}

// OWN: the workgroup makes its tile's vectors from the sums of P itself; otherwise tile_vectors_kernel has.
template <class E, int RT, bool HAS_Y, bool FEW, bool OWN>
__global__ void __launch_bounds__(256, RT == 8 || FEW ? 1 : 2) expand_rows_kernel(ExpandArgs a)
{
    using V = typename Mx<E>::V;
    using O = Operand<E, RT>;
    constexpr uint32_t VEC = Mx<E>::VEC;
    constexpr uint32_t buffers = (FEW ? 4u : 2u) * O::BLOCK;
    __shared__ __attribute__((aligned(16))) unsigned char lds[OWN && buffers < O::VECTORS ? O::VECTORS : buffers];
    __shared__ float own_down[64];
    const PlanLayout L(a.tokens, a.n);
    Tile tile;
    uint32_t part;
    if (!take_tile<FEW>(a.plan, L, a.parts, tile, part)) return;
    if ((uint32_t)tile.adapter < a.n) {
        const unsigned char* vectors = lds;
        const float* down = own_down;
        if constexpr (OWN) {
            const uint32_t t = threadIdx.x >> 2, count = (uint32_t)tile.count;
            if (!FEW || t < 16u) {
                const uint64_t position = (uint64_t)(uint32_t)tile.first + source_token(t, count);
                f32x4 v[RT];
                sum_parts<RT>(a.P, a.tokens, a.splits, position, v);
                if (a.shrunk && part == 0u && t < count)
                    store_shrunk<RT>(a.shrunk + (uint64_t)(uint32_t)a.plan[L.order + position] * a.rank, a.rank, v);
                const float s = a.scales ? a.scales[tile.adapter] : 1.0f;
#pragma unroll
                for (int i = 0; i < RT; ++i) v[i] = v[i] * s;
                const float d = store_vector<E, RT>(v, t, lds);
                if (Mx<E>::SCALED && (threadIdx.x & 3u) == 0) own_down[t] = d;
            }
            __syncthreads();
        } else {
            const uint64_t id = blockIdx.x / a.parts;
            vectors = a.vectors + id * O::VECTORS;
            down = a.down + id * 64u;
        }
        // every wavefront meets the same barriers on either way
        if (FEW || 16u * this_wave() < (uint32_t)tile.count) expand_blocks<E, RT, HAS_Y, FEW, OWN, true>(a, tile, part, lds, vectors, down);
        else expand_blocks<E, RT, HAS_Y, FEW, OWN, false>(a, tile, part, lds, vectors, down);
        return;
    }
    // tokens without an adapter: y as it is, or zeros
    if (!HAS_Y || a.y.p != a.out)
        for (uint32_t i = threadIdx.x >> 6; i < (uint32_t)tile.count; i += 4u) {
            const uint64_t t = (uint64_t)(uint32_t)a.plan[L.order + (uint32_t)tile.first + i];
            for (uint32_t c = VEC * (64u * part + (threadIdx.x & 63u)); c < a.N; c += VEC * 64u * a.parts) {
                V v = {};
                if (HAS_Y) v = load16<V>(static_cast<const E*>(a.y.p) + t * a.y.stride + c);
                __builtin_nontemporal_store(v, reinterpret_cast<V*>(static_cast<E*>(a.out) + t * a.out_stride + c));
            }
        }
    if (OWN && a.shrunk && part == 0u)
        for (uint32_t i = threadIdx.x; i < (uint32_t)tile.count * a.rank; i += kThreads) {
            const uint32_t at = i / a.rank;
            a.shrunk[(uint64_t)(uint32_t)a.plan[L.order + (uint32_t)tile.first + at] * a.rank + (i - at * a.rank)] = 0.0f;
        }
}

// ------------------------------------------------------------------------------------------------
struct WeightArgs {
    const int32_t* plan;
    Rows rows;            // x, dy
    const void* pieces;
    const float* down;    // fp16: [tiles], the inverse of the pieces' scaling
    float* partials;      // [slots][rank * (K + N)]
    void* grad;           // dA [n][rank][K], dB [n][N][rank]
    const void* B;        // [n][N][rank], with dy
    float* P;             // [slices][tokens][rp], with dy: d / s by slices of N
    uint64_t tokens;
    uint32_t n, rank, rp, K, N;
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

// The pieces of a step's tokens, 16 ranks (rows) each.
template <class E, int RT>
struct Pieces {
    typename Mx<E>::V of[RT][Mx<E>::PIECES];
    float down;
};

template <class E, int RT>
__device__ __forceinline__ void load_pieces(const WeightArgs& a, uint32_t tile, uint32_t t0, uint32_t rank0, Pieces<E, RT>& w)
{
    using X = Mx<E>;
    const uint32_t lane = threadIdx.x & 63u, lo = lane & 15u, g = lane >> 4;
    const E* pieces = static_cast<const E*>(a.pieces) + ((uint64_t)tile * a.rp + rank0 + lo) * X::PIECES * 64u + t0 % kTile + X::VEC * g;
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
        for (uint32_t p = 0; p < X::PIECES; ++p) w.of[j][p] = load16<typename X::V>(pieces + (16u * j * X::PIECES + p) * 64u);
    w.down = X::SCALED ? a.down[tile] : 1.0f;
}

// One step of the contraction over tokens: acc[j][c] += pieces . column VEC lo + c.
template <class E, int RT>
__device__ __forceinline__ void weight_step(const Pieces<E, RT>& w, const u32x4 (&in)[Mx<E>::VEC], f32x4 (&acc)[RT][Mx<E>::VEC])
{
    using X = Mx<E>;
    using V = typename X::V;
    constexpr uint32_t VEC = X::VEC;
    u32x4 turned[VEC];
    turn_over(in, turned);
    if constexpr (X::SCALED) {
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
            for (uint32_t c = 0; c < VEC; ++c) {
                f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (uint32_t p = 0; p < X::PIECES; ++p) d = X::mma(w.of[j][p], __builtin_bit_cast(V, turned[c]), d);
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[j][c][q] = __builtin_fmaf(d[q], w.down, acc[j][c][q]);
            }
    } else {
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
            for (uint32_t p = 0; p < X::PIECES; ++p)
#pragma unroll
                for (uint32_t c = 0; c < VEC; ++c) acc[j][c] = X::mma(w.of[j][p], __builtin_bit_cast(V, turned[c]), acc[j][c]);
    }
}

// What infinite rows need (any_not_finite): acc again from the first pieces, for steps t0, t0 + step, ... of the chunk.
template <class E, int RT>
__device__ __forceinline__ void mend_infinities(const WeightArgs& a, const E* rows, const int32_t* order, const Chunk& chunk, uint32_t t0, uint32_t step,
                                                uint32_t rank0, f32x4 (&acc)[RT][Mx<E>::VEC])
{
    using X = Mx<E>;
    using V = typename X::V;
    constexpr uint32_t VEC = X::VEC;
    if constexpr (X::PIECES > 1) {
        const uint32_t count = (uint32_t)chunk.count, lo = threadIdx.x & 15u, g = (threadIdx.x & 63u) >> 4;
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            if (!any_not_finite(acc[j])) continue;
            f32x4 first[VEC] = {};
            for (uint32_t t = t0; t < count; t += step) {
                const uint32_t tile = (uint32_t)chunk.tile + t / kTile;
                const V w = load16<V>(static_cast<const E*>(a.pieces) +
                                      ((uint64_t)tile * a.rp + rank0 + 16u * j + lo) * X::PIECES * 64u + t % kTile + VEC * g);
                const float down = X::SCALED ? a.down[tile] : 1.0f;
                u32x4 in[VEC], turned[VEC];
#pragma unroll
                for (uint32_t i = 0; i < VEC; ++i) {
                    const uint32_t at = t + VEC * g + i;
                    in[i] = load16<u32x4>(rows + (uint64_t)(uint32_t)order[at < count ? at : count - 1u] * a.rows.stride);
                    if (at >= count) in[i] = u32x4{0u, 0u, 0u, 0u};
                }
                turn_over(in, turned);
#pragma unroll
                for (uint32_t c = 0; c < VEC; ++c) {
                    const f32x4 d = X::mma(w, __builtin_bit_cast(V, turned[c]), X::SCALED ? f32x4{0.f, 0.f, 0.f, 0.f} : first[c]);
#pragma unroll
                    for (int q = 0; q < 4; ++q) first[c][q] = X::SCALED ? __builtin_fmaf(d[q], down, first[c][q]) : d[q];
                }
            }
#pragma unroll
            for (uint32_t c = 0; c < VEC; ++c) take_if_not_finite(acc[j][c], first[c]);
        }
    }
}

// A wavefront's sums: columns col ... col + VEC - 1, ranks rank0 + 16 j + 4 g + q.  To the chunk's partial sums, or
// rounded to the gradient where the adapter has no other chunk.
template <class E, int RT, bool DB>
__device__ __forceinline__ void store_weights(const WeightArgs& a, const Chunk& chunk, uint32_t rank0, uint32_t col, const f32x4 (&acc)[RT][Mx<E>::VEC])
{
    using V = typename Mx<E>::V;
    typedef E E4 __attribute__((ext_vector_type(4)));
    constexpr uint32_t VEC = Mx<E>::VEC;
    const uint32_t g = (threadIdx.x & 63u) >> 4, len = DB ? a.N : a.K;
    if (col >= len) return;
    const uint64_t per = (uint64_t)a.rank * (a.K + (uint64_t)a.N);
    float* part = chunk.slot >= 0 ? a.partials + (uint64_t)chunk.slot * per + (DB ? (uint64_t)a.rank * a.K : 0u) : nullptr;
    E* grad = static_cast<E*>(a.grad) + (uint64_t)chunk.adapter * a.rank * len;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
        const uint32_t r = rank0 + 16u * j + 4u * g;
        if (r >= a.rank) continue;
        if (DB) {  // [n][rank]
#pragma unroll
            for (uint32_t c = 0; c < VEC; ++c) {
                const uint64_t at = (uint64_t)(col + c) * a.rank + r;
                if (part) {
                    *reinterpret_cast<f32x4*>(part + at) = acc[j][c];
                } else {
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

// The slice of columns and the ranks of workgroup blockIdx.x, of the grid's `slices` rounded up to eights with
// several `halves` of the ranks: these read the same rows, and eight apart they run on one XCD soon after each
// other, where the second finds them in L2.
struct Share {
    uint32_t slice, half;
};

__device__ __forceinline__ Share share(uint32_t halves)
{
    const uint32_t group = blockIdx.x / (8u * halves), in = blockIdx.x - group * 8u * halves;
    return halves == 1u ? Share{blockIdx.x, 0u} : Share{group * 8u + (in & 7u), in >> 3};
}

uint32_t shares(uint32_t slices, uint32_t halves) { return halves == 1u ? slices : (slices + 7u) / 8u * 8u * halves; }

// dA.  Workgroup: a chunk of tokens of one adapter, 16 VEC columns of x, RT * 16 ranks (32 at most: with 64 the
// registers leave one wavefront per SIMD: a backward pass of 8192 tokens, 4096 -> 4096, rank 64, two pieces, took
// 130 us against 109, though rows are then read once less).  A wavefront takes
// every fourth step of STEP tokens; a lane reads 16 bytes of VEC consecutive tokens (the 16 lanes of a group
// read 256 contiguous bytes of a row) and turns them over in registers, one byte permute for two values,
// so the contraction over tokens needs no LDS.  The wavefronts' sums meet in LDS at the end.  (With three pieces and
// 32 ranks the compiler takes 192 registers, which leave room for two workgroups on a compute unit; it needs 162.)
template <class E, int RT>
__global__ void __launch_bounds__(256, Mx<E>::PIECES == 3 ? 3 : 1) weight_rows_kernel(WeightArgs a)
{
    using X = Mx<E>;
    constexpr uint32_t VEC = X::VEC, STEP = X::STEP;
    __shared__ f32x4 red[2 * RT * VEC * 64];
    __shared__ int32_t order[kMaxChunk];
    const PlanLayout L(a.tokens, a.n);
    const Chunk chunk = reinterpret_cast<const Chunk*>(a.plan + L.chunks)[blockIdx.y];
    if (blockIdx.y >= (uint32_t)a.plan[L.counts + 1u]) return;
    const uint32_t lane = threadIdx.x & 63u, wave = this_wave(), lo = lane & 15u, g = lane >> 4, count = (uint32_t)chunk.count;
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) order[i] = a.plan[L.order + (uint32_t)chunk.first + i];
    __syncthreads();
    const Share mine = share(a.rp / (16u * RT));
    const uint32_t col = mine.slice * 16u * VEC + VEC * lo, rank0 = mine.half * 16u * RT;
    if (mine.slice * 16u * VEC >= a.K) return;
    const E* rows = static_cast<const E*>(a.rows.p) + (col < a.K ? col : 0u);

    f32x4 acc[RT][VEC] = {};
    for (uint32_t t0 = wave * STEP; t0 < count; t0 += 4u * STEP) {
        u32x4 in[VEC];
        Pieces<E, RT> w;
        load_pieces(a, (uint32_t)chunk.tile + t0 / kTile, t0, rank0, w);
#pragma unroll
        for (uint32_t i = 0; i < VEC; ++i) {
            const uint32_t t = t0 + VEC * g + i;
            in[i] = u32x4{0u, 0u, 0u, 0u};  // tokens behind the chunk: zeros on both sides
            if (t < count) in[i] = load16<u32x4>(rows + (uint64_t)(uint32_t)order[t] * a.rows.stride);
        }
        weight_step<E, RT>(w, in, acc);
    }
    mend_infinities<E, RT>(a, rows, order, chunk, wave * STEP, 4u * STEP, rank0, acc);
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
    if (wave == 0) store_weights<E, RT, false>(a, chunk, rank0, col, acc);
}

// dB and the parts of d, from one pass over dy, which is most of what the backward pass has to read.
// Workgroup: a chunk of tokens of one adapter, a slice of 64 VEC columns of dy, up to RT * 16 ranks; a wavefront has
// 16 VEC of the columns and all tokens, STEP at a time with the next requested.  For dB the lanes' registers
// are turned over as above; for d the same registers go through LDS to become operands along the columns, B
// stays in registers, and the four wavefronts' sums of a step meet in LDS (two buffers, one barrier a step).
// A step's pieces are requested before the next step's rows: loads come back in order, and a wait for the
// pieces must not be one for those rows (8192 tokens, 4096 -> 14336, rank 64, two pieces: 200 us a call against 220).
// STREAM: dy is read past the caches (kStreamed).
template <class E, int RT, bool STREAM>
__global__ void __launch_bounds__(256, RT == 2 ? 1 : 2) gradient_rows_kernel(WeightArgs a)
{
    using X = Mx<E>;
    using V = typename X::V;
    using C = Contraction<E, RT, false>;
    constexpr uint32_t VEC = X::VEC, STEP = X::STEP, SUBS = STEP / 16u, UNITS = SUBS * RT * 64u;
    __shared__ __attribute__((aligned(16))) unsigned char own[4][STEP * 256u];
    __shared__ f32x4 red[2][4][UNITS];
    __shared__ int32_t order[kMaxChunk];
    const PlanLayout L(a.tokens, a.n);
    const Chunk chunk = reinterpret_cast<const Chunk*>(a.plan + L.chunks)[blockIdx.y];
    if (blockIdx.y >= (uint32_t)a.plan[L.counts + 1u]) return;
    const uint32_t lane = threadIdx.x & 63u, wave = this_wave(), lo = lane & 15u, g = lane >> 4, count = (uint32_t)chunk.count;
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) order[i] = a.plan[L.order + (uint32_t)chunk.first + i];
    __syncthreads();
    const Share part = share(a.rp / (16u * RT));
    const uint32_t slice = part.slice, rank0 = part.half * 16u * RT;
    if (slice * 64u * VEC >= a.N) return;
    const uint32_t base = (slice * 4u + wave) * 16u * VEC, col = base + VEC * lo;
    const bool inside = col < a.N;
    const E* rows = static_cast<const E*>(a.rows.p) + (inside ? col : 0u);

    // B of the wavefront's columns: operand j, step h, rank 16 j + lo, columns base + STEP h + VEC g ...
    V bf[4][RT];
#pragma unroll
    for (uint32_t h = 0; h < 4; ++h)
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
            for (uint32_t e = 0; e < VEC; ++e) {
                const uint32_t n = base + STEP * h + VEC * g + e, r = rank0 + 16u * j + lo;
                const bool in = n < a.N && r < a.rank;
                const E v = static_cast<const E*>(a.B)[((uint64_t)chunk.adapter * a.N + (in ? n : 0u)) * a.rank + (in ? r : 0u)];
                bf[h][j][e] = in ? v : (E)0.0f;
            }
    f32x4 acc[RT][VEC] = {};
    Pieces<E, RT> w;
    auto request = [&](u32x4 (&in)[VEC], uint32_t t0) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t i = 0; i < VEC; ++i) {
            const uint32_t t = t0 + VEC * g + i;
            const E* p = rows + (uint64_t)(uint32_t)order[t < count ? t : count - 1u] * a.rows.stride;
            in[i] = STREAM ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)) : load16<u32x4>(p);
        }
    };
    auto pieces = [&](uint32_t t0) __attribute__((always_inline)) { load_pieces(a, (uint32_t)chunk.tile + t0 / kTile, t0, rank0, w); };
    auto work = [&](u32x4 (&in)[VEC], uint32_t t0, uint32_t buffer) __attribute__((always_inline)) {
        const u32x4 zero = {0u, 0u, 0u, 0u};
        unsigned char* const mine = own[wave];
#pragma unroll
        for (uint32_t i = 0; i < VEC; ++i) {
            const uint32_t row = VEC * g + i;
            in[i] = inside && t0 + row < count ? in[i] : zero;  // zeros on both sides of the sums
            *reinterpret_cast<u32x4*>(mine + C::at(row, lo)) = in[i];
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (uint32_t s = 0; s < SUBS; ++s) {
            f32x4 d[RT] = {};
#pragma unroll
            for (uint32_t h = 0; h < 4; ++h) {
                const V x = *reinterpret_cast<const V*>(mine + C::at(16u * s + lo, 4u * h + g));
#pragma unroll
                for (int j = 0; j < RT; ++j) d[j] = X::mma(bf[h][j], x, d[j]);
            }
#pragma unroll
            for (int j = 0; j < RT; ++j) red[buffer][wave][(s * RT + j) * 64u + lane] = d[j];
        }
        weight_step<E, RT>(w, in, acc);
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < (UNITS + kThreads - 1u) / kThreads; ++k) {
            const uint32_t u = threadIdx.x + k * kThreads, l = u & 63u, j = u / 64u % RT, s = u / (64u * RT);
            const uint32_t t = t0 + 16u * s + (l & 15u), r = 16u * j + 4u * (l >> 4);
            if (u < UNITS && t < count) {
                const f32x4 sum = (red[buffer][0][u] + red[buffer][1][u]) + (red[buffer][2][u] + red[buffer][3][u]);
                float* P = a.P + ((uint64_t)slice * a.tokens + (uint32_t)chunk.first + t) * a.rp + rank0 + r;
                *reinterpret_cast<f32x4*>(P) = rank0 + r < a.rank ? sum : f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
    };
    u32x4 p[VEC], q[VEC];
    request(p, 0);
    uint32_t t0 = 0;
    for (; t0 + 2u * STEP < count; t0 += 2u * STEP) {
        pieces(t0);
        request(q, t0 + STEP);
        work(p, t0, 0);
        pieces(t0 + STEP);
        request(p, t0 + 2u * STEP);
        work(q, t0 + STEP, 1);
    }
    pieces(t0);
    if (t0 + STEP < count) {
        request(q, t0 + STEP);
        work(p, t0, 0);
        pieces(t0 + STEP);
        work(q, t0 + STEP, 1);
    } else {
        work(p, t0, 0);
    }
    mend_infinities<E, RT>(a, rows, order, chunk, 0, STEP, rank0, acc);
    store_weights<E, RT, true>(a, chunk, rank0, col, acc);
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
    if (count > 0u && count <= L.chunk) return;  // complete already
    const uint32_t chunks = (count + L.chunk - 1u) / L.chunk;
    const uint64_t first = (uint64_t)a.rank * a.len[0], per = first + (uint64_t)a.rank * a.len[1];
    const float* part = a.partials + (uint64_t)(uint32_t)a.plan[L.slot_start + ad] * per;
    for (uint64_t i = 4u * ((uint64_t)blockIdx.x * kThreads + threadIdx.x); i < per; i += 4u * (uint64_t)gridDim.x * kThreads) {
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
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

// How many workgroups share the blocks of an axis: so many that there are `most` in all, each with at least
// `least` blocks; eight, one for each XCD, or a multiple of eight where the blocks allow it.
uint32_t cut(uint64_t tiles, uint32_t blocks, uint32_t least, uint32_t most)
{
    uint32_t parts = (uint32_t)(tiles && most / tiles > 8u ? most / tiles : 8u);
    const uint32_t limit = blocks / least ? blocks / least : 1u;
    if (parts > limit) parts = limit;
    return parts > 8u ? parts / 8u * 8u : parts;
}

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

// How a batch is cut.  With at most 16 tiles workgroups take 16 tokens instead of 64, their wavefronts take
// different parts of the adapter, which is then most of what there is to read, and the expansion adds up the
// parts of P itself, a launch less (rank 16, 4096 -> 4096, in a graph: one token 7.1 us against 8.5, 64 tokens of
// four adapters 7.1 against 9.5).  With more tiles the four times as many workgroups cost more than that (64
// tokens of 48 adapters, 4096 -> 14336: 19.8 us against 16.4).
struct Cut {
    bool few;
    uint32_t rp, splits, parts;
    uint64_t max_tiles, grid_tiles;  // of the plan; that the grids provide for
    Cut(const mi_lora* d, uint32_t K, uint32_t N)
    {
        max_tiles = PlanLayout(d->tokens, d->n_adapters).max_tiles;
        few = max_tiles <= 16u;
        grid_tiles = few ? 4u * max_tiles : max_tiles;
        rp = padded_rank(d->rank);
        const uint32_t block = 16u * elements_of(d->dtype);  // columns of a block, of x and of y
        // x: the workgroups that run at once.  y: ten times that, as one round and a little of long ones leaves
        // compute units idle (8192 tokens, N = 14336: 128 us with 1100 workgroups, 100 with 7700), but two
        // blocks each, so that one is requested while the other is computed (one each: 116 us).
        splits = cut(max_tiles, (K + block - 1u) / block, few ? 4u : 2u, 1024u);
        parts = cut(max_tiles, (N + block - 1u) / block, few ? 4u : 2u, few ? 1024u : 8192u);
    }
    uint64_t sums() const { return (uint64_t)splits * rp * 4u; }  // bytes of P per token
};

// From so many bytes of dy on it is read past the caches, a quarter of the last of which it would fill.  Rank 16:
// 235 MB 92.6 us a call against 100.1, 67 MB 69 against 74; but 59 MB 48.4 against 45.9, 29 MB 38.5 against 35.
// Several halves of the ranks, which read the same rows soon after each other, gain less but lose nothing by it:
// 235 MB at rank 64 221 against 224, in fp16 207 against 210, at rank 128 416 against 419.
constexpr uint64_t kStreamed = 64u << 20;

struct Take {  // places in a workspace
    uint64_t end = 0;
    uint64_t operator()(uint64_t bytes)
    {
        const uint64_t here = end;
        end += (bytes + 255u) / 256u * 256u;
        return here;
    }
};

struct ForwardPlan {
    Cut c;
    bool own;
    uint64_t P, vectors, down, bytes;
    explicit ForwardPlan(const mi_lora* d) : c(d, d->K, d->N)
    {
        // A launch less where adding up P again in every workgroup moves no more than 16 MB of sums, and where the
        // workgroups, which read 64 tokens' whatever their tile has, read no more than 192 MB from the caches.  4096 ->
        // 14336, us a call (in a graph): 64 tokens of 48 adapters, rank 16 (176 MB read) 18.5 (16.4) against 21.2
        // (15.7), rank 32 (350) 22.8 (23.4) against 21.2 (19.1), rank 64 (700) 50 (50) against 32 (32); 256 tokens
        // of 64, rank 16 (120) 20.7 (20.9) against 21.2 (19.9).  4096 -> 4096, rank 64 (200) 23.8 (24.5) against 21.5
        // (21.6).  512 tokens of 64 adapters, 4096 -> 14336, rank 64 (58 MB moved): 62 against 51.
        own = c.few || (c.sums() * c.parts * d->tokens <= 16u << 20 && c.sums() * c.parts * c.max_tiles * 64u <= 192u << 20);
        Take take;
        P = take(c.sums() * d->tokens);
        vectors = take(own ? 0u : c.max_tiles * vectors_bytes(d->dtype, c.rp));
        down = take(own ? 0u : c.max_tiles * 64u * 4u);
        bytes = take.end;
    }
};

struct BackwardPlan {
    Cut c;           // expansion to K; the contraction over N is by slices
    Cut u;           // contraction over K as the forward pass does it, when its sums are not given
    uint32_t slices; // of N
    uint64_t P, at, vectors, down, pieces[2], tile_down[2], partials, bytes;
    explicit BackwardPlan(const mi_lora* d) : c(d, d->N, d->K), u(d, d->K, d->N)
    {
        const PlanLayout L(d->tokens, d->n_adapters);
        const uint64_t e = d->dtype == MI_F32 ? 4u : 2u;
        c.few = false;
        c.grid_tiles = c.max_tiles;
        const uint32_t slice = 64u * elements_of(d->dtype);
        c.splits = slices = (d->N + slice - 1u) / slice;
        Take take;
        P = take((c.sums() > u.sums() ? c.sums() : u.sums()) * d->tokens);  // in turn
        at = take((uint64_t)d->n_adapters * d->rank * d->K * e);
        vectors = take(c.max_tiles * vectors_bytes(d->dtype, c.rp));
        down = take(c.max_tiles * 64u * 4u);
        for (int i = 0; i < 2; ++i) {
            pieces[i] = take(c.max_tiles * pieces_bytes(d->dtype, c.rp));
            tile_down[i] = take(c.max_tiles * 4u);
        }
        partials = take(L.max_slots * d->rank * ((uint64_t)d->K + d->N) * 4u);
        bytes = take.end;
    }
};

template <class E>
int contract(const mi_lora* d, const int32_t* plan, Rows x, const void* M, uint32_t K, const Cut& c, float* P, hipStream_t s)
{
    ContractArgs a{plan, x, M, P, d->tokens, d->n_adapters, d->rank, K, c.splits};
    const dim3 grid((uint32_t)c.grid_tiles * c.splits);
    for_rank(c.rp, [&](auto rt) {
        constexpr int RT = decltype(rt)::value;
        if (c.few) hipLaunchKernelGGL((contract_rows_kernel<E, RT, true>), grid, dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((contract_rows_kernel<E, RT, false>), grid, dim3(kThreads), 0, s, a);
    });
    return launch_status();
}

template <class E>
int tile_vectors(const Cut& c, VectorArgs a, hipStream_t s)
{
    a.tiles = (uint32_t)c.max_tiles;
    const uint32_t more = a.A ? (a.K + kThreads - 1u) / kThreads * (a.rank / 8u) * a.n : 0u;
    for_rank(c.rp, [&](auto rt) {
        hipLaunchKernelGGL((tile_vectors_kernel<E, decltype(rt)::value>), dim3(a.tiles + more), dim3(kThreads), 0, s, a);
    });
    return launch_status();
}

template <class E>
int expand(const Cut& c, ExpandArgs a, hipStream_t s)
{
    a.parts = c.parts;
    a.splits = c.splits;
    const dim3 grid((uint32_t)c.grid_tiles * c.parts);
    for_rank(c.rp, [&](auto rt) {
        constexpr int RT = decltype(rt)::value;
        if (!a.y.p) hipLaunchKernelGGL((expand_rows_kernel<E, RT, false, false, false>), grid, dim3(kThreads), 0, s, a);
        else if (a.vectors) hipLaunchKernelGGL((expand_rows_kernel<E, RT, true, false, false>), grid, dim3(kThreads), 0, s, a);
        else if (c.few) hipLaunchKernelGGL((expand_rows_kernel<E, RT, true, true, true>), grid, dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((expand_rows_kernel<E, RT, true, false, true>), grid, dim3(kThreads), 0, s, a);
    });
    return launch_status();
}

template <class E>
int forward(const mi_lora* d, const void* y, const void* x, const void* A, const void* B, const float* scales, const int32_t* plan, void* out,
            float* shrunk, unsigned char* ws, hipStream_t s)
{
    const ForwardPlan f(d);
    float* P = reinterpret_cast<float*>(ws + f.P);
    float* down = reinterpret_cast<float*>(ws + f.down);
    int st;
    if ((st = contract<E>(d, plan, {x, d->x_stride}, A, d->K, f.c, P, s)) != MI_OK) return st;
    if (!f.own) {
        const VectorArgs v{plan, P, scales, shrunk, ws + f.vectors, down, nullptr, nullptr, d->tokens, d->n_adapters, d->rank, f.c.splits, false, nullptr, nullptr, 0, 0};
        if ((st = tile_vectors<E>(f.c, v, s)) != MI_OK) return st;
    }
    return expand<E>(f.c, {plan, {y, d->y_stride}, out, d->out_stride, B, f.own ? nullptr : ws + f.vectors, down, scales, P, shrunk, d->tokens, d->n_adapters,
                           d->rank, d->N, 0, 0}, s);
}

template <class E>
int backward(const mi_lora* d, const void* dy, const void* x, const void* A, const void* B, const float* scales, const int32_t* plan,
             const float* shrunk, const void* dx_in, void* dx, void* dA, void* dB, unsigned char* ws, hipStream_t s)
{
    const BackwardPlan b(d);
    float* P = reinterpret_cast<float*>(ws + b.P);
    float* down = reinterpret_cast<float*>(ws + b.down);
    float* tile_down[2] = {reinterpret_cast<float*>(ws + b.tile_down[0]), reinterpret_cast<float*>(ws + b.tile_down[1])};
    const Rows rx{x, d->x_stride}, rdy{dy, d->y_stride};
    int st;
    if (d->tokens) {
        // s u, transposed, and A^T
        VectorArgs v{plan, P, scales, const_cast<float*>(shrunk), nullptr, nullptr, ws + b.pieces[1], tile_down[1],
                     d->tokens, d->n_adapters, d->rank, b.u.splits, shrunk != nullptr, A, ws + b.at, d->K, 0};
        if (!shrunk && (st = contract<E>(d, plan, rx, A, d->K, b.u, P, s)) != MI_OK) return st;
        if ((st = tile_vectors<E>(b.c, v, s)) != MI_OK) return st;
        const PlanLayout L(d->tokens, d->n_adapters);
        const uint32_t rt = b.c.rp <= 32u ? b.c.rp : 32u, cols = 16u * Mx<E>::VEC;
        auto for_weights = [&](auto f) {
            if (rt == 16u) f(std::integral_constant<int, 1>{});
            else f(std::integral_constant<int, 2>{});
            return launch_status();
        };
        // dB and d
        float* partials = reinterpret_cast<float*>(ws + b.partials);
        WeightArgs w{plan, rdy, ws + b.pieces[1], tile_down[1], partials, dB, B, P, d->tokens, d->n_adapters, d->rank, b.c.rp, d->K, d->N};
        const uint32_t halves = b.c.rp / rt;
        dim3 grid(shares(b.slices, halves), (uint32_t)L.max_chunks);
        st = for_weights([&](auto r) {
            constexpr int RT = decltype(r)::value;
            if (d->tokens * d->N * sizeof(E) >= kStreamed) hipLaunchKernelGGL((gradient_rows_kernel<E, RT, true>), grid, dim3(kThreads), 0, s, w);
            else hipLaunchKernelGGL((gradient_rows_kernel<E, RT, false>), grid, dim3(kThreads), 0, s, w);
        });
        if (st != MI_OK) return st;
        v.A = nullptr;
        v.shrunk = nullptr;
        v.given = false;
        v.splits = b.slices;
        v.vectors = ws + b.vectors;
        v.down = down;
        v.pieces = ws + b.pieces[0];
        v.tile_down = tile_down[0];
        if ((st = tile_vectors<E>(b.c, v, s)) != MI_OK) return st;
        // dA
        w.rows = rx;
        w.pieces = ws + b.pieces[0];
        w.down = tile_down[0];
        w.grad = dA;
        grid.x = shares((d->K + cols - 1u) / cols, halves);
        st = for_weights([&](auto r) {
            hipLaunchKernelGGL((weight_rows_kernel<E, decltype(r)::value>), grid, dim3(kThreads), 0, s, w);
        });
        if (st != MI_OK) return st;
        // dx, after dA: it may lie in x
        if ((st = expand<E>(b.c, {plan, {dx_in, d->out_stride}, dx, d->out_stride, ws + b.at, ws + b.vectors, down, nullptr, nullptr, nullptr,
                                  d->tokens, d->n_adapters, d->rank, d->K, 0, 0}, s)) != MI_OK)
            return st;
    }
    WeightSumArgs sum{plan, reinterpret_cast<float*>(ws + b.partials), {dA, dB}, d->tokens, d->n_adapters, d->rank, {d->K, d->N}};
    hipLaunchKernelGGL((weight_sum_kernel<E>), dim3(512, d->n_adapters), dim3(kThreads), 0, s, sum);
    return launch_status();
}

}  // namespace
}  // namespace adapters
}  // namespace mi

extern "C" uint64_t mi_lora_workspace(const mi_lora* d, int backward)
{
    using namespace mi::adapters;
    if (check(d) != MI_OK) return 0;
    return backward ? BackwardPlan(d).bytes : ForwardPlan(d).bytes;
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
    if (d->tokens > 1u && d->out_stride < d->N) return MI_ERR_SHAPE;  // rows that overlap
    if (y == out && d->y_stride != d->out_stride && d->tokens > 1u) return MI_ERR_ALIAS;
    hipStream_t s = static_cast<hipStream_t>(stream);
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    if (d->dtype == MI_F32) return forward<float>(d, y, x, A, B, scales, plan, out, shrunk, ws, s);
    if (d->dtype == MI_BF16) return forward<__bf16>(d, y, x, A, B, scales, plan, out, shrunk, ws, s);
    return forward<_Float16>(d, y, x, A, B, scales, plan, out, shrunk, ws, s);
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
    if (d->tokens > 1u && d->out_stride < d->K) return MI_ERR_SHAPE;
    // A^T is made by a workgroup for every 2048 values, in one grid with the tiles: below 2^32 threads
    if ((uint64_t)d->n_adapters * d->rank * ((d->K + 255u) / 256u * 256u) >= 1ull << 35) return MI_ERR_SHAPE;
    hipStream_t s = static_cast<hipStream_t>(stream);
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    if (d->dtype == MI_F32) return backward<float>(d, dy, x, A, B, scales, plan, shrunk, dx_in, dx, dA, dB, ws, s);
    if (d->dtype == MI_BF16) return backward<__bf16>(d, dy, x, A, B, scales, plan, shrunk, dx_in, dx, dA, dB, ws, s);
    return backward<_Float16>(d, dy, x, A, B, scales, plan, shrunk, dx_in, dx, dA, dB, ws, s);
}
