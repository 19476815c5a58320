/*
 * mi_hadamard.h -- C ABI of the MI355X (gfx950) fast Hadamard transform library.
 *
 * Plain pointers and sizes only; no torch or HIP types appear in the signatures (`stream` is a
 * hipStream_t passed as void*, NULL = the null stream).  Every entry point
 *   - enqueues its kernels on `stream` and returns without synchronising,
 *   - allocates no device memory and keeps no mutable global state (safe from any host thread),
 *   - returns MI_OK (0) or a negative mi_status; mi_status_string() turns it into text.
 * All matrices are dense row-major with no padding between rows.
 */
#ifndef MI_HADAMARD_H
#define MI_HADAMARD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum mi_dtype {
    MI_F32 = 0,
    MI_BF16 = 1,
    MI_F16 = 2,
} mi_dtype;

typedef enum mi_status {
    MI_OK = 0,
    MI_ERR_DTYPE = -1,     /* dtype code not supported by this entry point            */
    MI_ERR_SIZE = -2,      /* transform length not a power of two in the valid range  */
    MI_ERR_ALIGN = -3,     /* a pointer is not 16-byte aligned                        */
    MI_ERR_NULL = -4,      /* a required pointer is NULL                              */
    MI_ERR_SHAPE = -5,     /* a dimension violates the entry point's tiling contract  */
    MI_ERR_LAUNCH = -6,    /* hipGetLastError() reported a launch failure             */
    MI_ERR_ALIAS = -7,     /* input/output overlap that the entry point cannot honour */
} mi_status;

/* Library version (major*10000 + minor*100 + patch). */
int mi_version(void);

/* Text for a status code; never NULL. */
const char* mi_status_string(int status);

/*
 * Walsh-Hadamard transform over the last dimension:  out[r, :] = scale * H_n * in[r, :]
 * for r in [0, rows), H_n the Sylvester matrix H[i][j] = (-1)^popcount(i & j).
 *
 * Replaces the reference's internal seam
 *     template<DType> void run_fht(void* a, void* out, uint32_t numel, uint32_t had_size,
 *                                  cudaStream_t)                 csrc/main.cuh:5-6,
 *                                                                HadaCore/hadamard_transform.cpp:8-9
 * which its pybind op hadamard_transform(x, inplace) calls (csrc/hadamard_transform.cpp:49-59).
 * Differences: `rows` is 64-bit (the reference's numel is u32); any row count is accepted (the
 * reference pads numel to a multiple of 256 first, csrc/hadamard_transform.cpp:31-39); fp32 is
 * accepted; `scale` is explicit (the reference hard-wires n^-1/2 in its kernel constants,
 * HadaCore/hadamard_transform_cuda.cu:139-142).
 *
 *   in, out : device pointers, 16-byte aligned, rows*n elements; in == out is allowed
 *             (in place); partial overlap is not.
 *   n       : power of two, 1 <= n <= 32768.
 *   dtype   : mi_dtype.  bf16/fp16 accumulate in fp32 on the matrix cores and round to the
 *             storage type between MFMA stages and at the store; fp32 stays fp32 throughout.
 */
int mi_fwht(const void* in, void* out, uint64_t rows, uint32_t n, int dtype, float scale,
            void* stream);

/*
 * Fused Hadamard + GEMV-batch:  Y[M,B] = W[M,N] * (scale * H_N * X[N,B]),
 * the transform running down each column of X (dimension 0).
 *
 * Replaces  fused_hadamard_gemv_kernel(const float* W, const float* X, float* Y, int M, int N,
 * int B)  and its _vec variant, fused_ht/fwht_gemv_fusion.cu:98-105,176-183, launched from
 * benchmark_fused (:371-420).  Layouts are the ones that file indexes: X[i*B + b] (:50-51),
 * W[row*N + k] (:146), Y[row*B + b] (:156).  scale = 1 reproduces the reference (raw +-1
 * butterfly, :118-133).
 *
 *   dtype : MI_F32 only.   N : power of two, 2 <= N <= 2048 (the 16-column tile of the
 *   transformed operand must fit in LDS).   M, B >= 1.
 *   Y must not overlap W or X.
 */
int mi_fused_ht_gemv(const void* W, const void* X, void* Y, uint32_t M, uint32_t N, uint32_t B,
                     int dtype, float scale, void* stream);

/*
 * Fused Hadamard -> GEMM:  C[M,N] = W[M,K] * (scale * H_K * X[K,N]),  X given as Xt[N,K]
 * (each logical column of X contiguous).  The transformed operand never goes to HBM.
 *
 * Replaces  fused_ht_gemm_pipelined(const float* X, const float* W, float* C)  with compile-time
 * KDIM/NDIM/MDIM, fused_ht/fusion_pipelined.cu:306-310, launched at :662-683.  Layouts:
 * X[col*KDIM + k] (:164,612), W[row*KDIM + k] (:211,498), C[row*NDIM + col] (:220,558).
 * scale = 1 reproduces the reference.
 *
 *   in_dtype  : MI_F32 (fp32 MFMA) or MI_BF16 / MI_F16 (16-bit MFMA, fp32 accumulate).
 *   out_dtype : MI_F32, or the same 16-bit type as in_dtype.
 *   K : power of two, 32 <= K <= 4096.   M, N >= 1 (edge tiles are masked).
 *   The register-resident kernels (16-bit inputs with K >= 512, MI_F32 with K >= 256) address W
 *   with 32-bit byte offsets: W larger than 4 GiB, or N >= 2^24, is MI_ERR_SHAPE.
 * K = 4096 enqueues two kernels on `stream` for every dtype (the second adds to what the first
 * stored in C, so nothing else may touch C between them); every other case is one kernel.
 * Precision at K = 4096: each kernel accumulates its half of the K range in fp32.  With MI_F32
 * output the halves meet in fp32 (one more fp32 rounding than a single pass).  With 16-bit output
 * the first kernel stores its half-K sum P0 rounded to the 16-bit type and the second adds its own
 * half P1, rounded to 16 bits, in 16-bit arithmetic (a packed add performed by the L2; masked edge
 * blocks add in fp32 and round once), so the result carries up to three 16-bit roundings instead of
 * the single one of K <= 2048:
 *     |C - exact| <= ulp16(P0) + ulp16(P1) + ulp16(C),   ulp16(v) = the 16-bit type's spacing at |v|,
 * which is a larger *relative* error than usual when P0 and P1 nearly cancel, and for MI_F16 a half-K
 * sum beyond 65504 becomes infinite even if the total is representable.  Callers that need the
 * single rounding ask for MI_F32 output.
 */
int mi_fused_ht_gemm(const void* W, const void* Xt, void* C, uint32_t M, uint32_t N, uint32_t K,
                     int in_dtype, int out_dtype, float scale, void* stream);

/*
 * Randomized Hadamard + FP8 quantize:  y[t,:] = scale * H_n * (sign .* x[t,:]) rounded to bf16,
 * then per row   amax = max|y|,  a = max(amax, 1e-30f),  row_scale[t] = a / 448,
 * q[t,j] = e4m3fn_rne(clamp(y[t,j] * (448 / a), -448, 448))   (OCP E4M3FN; IEEE fp32 ops; for
 * finite y the clamp never changes a value because |y| <= amax).
 *
 * No counterpart in the reference (it has no FP8 path); part of the build contract's hot path.
 *
 *   x         : bf16 [T,n];  n power of two, 16 <= n <= 4096.
 *   sign      : int8 [n], entries +1 / -1.
 *   q         : uint8 [T,n] E4M3FN codes.      row_scale : fp32 [T] (dequantisation factors).
 *   y_out     : optional bf16 [T,n] dump of the pre-quant values (NULL to skip).
 */
int mi_rht_quant_fp8(const void* x, const int8_t* sign, void* q, float* row_scale, void* y_out,
                     uint64_t T, uint32_t n, float scale, void* stream);

/*
 * FP8 GEMM with per-row scales:  out[T,N] = bf16( (qa[T,K] . qb[N,K]^T) * sa[t] * sb[n] ),
 * E4M3FN operands, fp32 accumulate.  No counterpart in the reference.
 *   K multiple of 128;  T, N >= 1.
 */
int mi_fp8_gemm_rowscale(const void* qa, const float* sa, const void* qb, const float* sb,
                         void* out, uint32_t T, uint32_t N, uint32_t K, void* stream);

/*
 * Groups the tokens of a batch by the low-rank adapter they use: ids[t] in [0, n_adapters), anything
 * else for a token without an adapter.  `plan` is an int32 buffer of layout[0] entries, 16-byte aligned,
 * layout from mi_adapter_plan_layout for the same sizes; it stays valid for every call with this batch.
 *   plan[layout[1] + i], i < tokens      : the tokens in grouped order (adapter by adapter, the tokens of
 *                                          one in their own order, those without an adapter last)
 *   plan[layout[2] + a], a <= n_adapters : first position of adapter a; [n_adapters] of the tokens without
 * The rest is the kernels' own.  tokens <= 2^24, 1 <= n_adapters <= 1024, id_bits 32 or 64.
 * One kernel up to 4096 tokens, two beyond; the result depends on the ids alone.  No counterpart in the reference.
 */
int mi_adapter_plan(const void* ids, int id_bits, uint64_t tokens, uint32_t n_adapters, int32_t* plan,
                    void* stream);
int mi_adapter_plan_layout(uint64_t tokens, uint32_t n_adapters, uint64_t layout[3]);

/* Sizes of a batch with low-rank adapters.  Strides are row strides in elements, multiples of 16 bytes. */
typedef struct mi_lora {
    uint64_t tokens;      /* at most 2^24                                                   */
    uint64_t x_stride;    /* of x                                                           */
    uint64_t y_stride;    /* of y (forward), dy (backward)                                  */
    uint64_t out_stride;  /* of out (forward), dx_in and dx (backward)                      */
    uint32_t n_adapters;  /* 1 ... 1024, as in the plan                                     */
    uint32_t rank;        /* a multiple of 8, 8 ... 128                                     */
    uint32_t K, N;        /* input and output width: multiples of 8, 8 ... 2^22             */
    int32_t dtype;        /* mi_dtype of every matrix                                       */
} mi_lora;

/*
 * Low-rank adapters beside a shared projection, each token with its own:
 *     u[t] = A[a] . x[t]      out[t] = y[t] + scales[a] * B[a] . u[t]      a = ids[t] of the plan
 * and out[t] = y[t] for tokens without an adapter.  A [n_adapters][rank][K] and B [n_adapters][N][rank]
 * are dense.  fp32 sums; u is kept to 23 significand bits (fp16; else 24) between the products; out is rounded
 * once.  An adapter of a smaller rank is padded with zeros.  No counterpart in the reference.
 *   scales    : fp32 [n_adapters], or NULL for 1.
 *   out       : may be y with the same stride (in place; other tokens' rows are then not touched); no
 *               other overlap with any operand.
 *   shrunk    : NULL, or fp32 [tokens][rank]: receives u (zeros for tokens without an adapter).
 *   workspace : mi_lora_workspace(sizes, 0) bytes.
 * All pointers 16-byte aligned (scales, shrunk: 4).  Two kernels, or three where that is faster.
 */
int mi_lora_add(const void* y, const void* x, const void* A, const void* B, const float* scales,
                const int32_t* plan, void* out, float* shrunk, void* workspace, const mi_lora* sizes,
                void* stream);

/*
 * Gradients of mi_lora_add (that of y is dy itself):
 *     d[t] = scales[a] * B[a]^T . dy[t]        dx[t] = dx_in[t] + A[a]^T . d[t]
 *     dA[a] = sum over its tokens of d[t] x[t]^T,   dB[a] = sum of scales[a] * dy[t] u[t]^T
 * in a fixed order; dA, dB are shaped like A, B, zeros for adapters without tokens.
 *   shrunk    : u from the forward pass, or NULL (it is computed again from x).
 *   dx_in     : NULL for zeros, or added; may be dx (in place).
 *   workspace : mi_lora_workspace(sizes, 1) bytes.  Outputs overlap no input, but dx may lie on dx_in (at
 *               the same address) and on x, which is read before dx is written.
 * A holds fewer than 2^35 values (K rounded up to a multiple of 256), or MI_ERR_SHAPE.
 */
int mi_lora_add_backward(const void* dy, const void* x, const void* A, const void* B, const float* scales,
                         const int32_t* plan, const float* shrunk, const void* dx_in, void* dx, void* dA,
                         void* dB, void* workspace, const mi_lora* sizes, void* stream);
/*
 * Bytes of workspace, 16-byte aligned; 0 for sizes that the calls refuse.  With R the rank padded to 16, 32, 64 or
 * 128: the forward pass takes 4 R tokens for each part of K, eight of them (more with few tokens), and 6 R tokens
 * for vectors.  The backward pass grows with the batch in three ways: 4 R tokens N / 512 (fp32: N / 256) for parts of d, 18 R tokens
 * for vectors, and, from 8192 tokens on, 4 rank (K + N) bytes for each 512 tokens and for each adapter with more
 * than 512 (smaller batches: 256 and 128); and it holds a transposed copy of all of A.  65536 tokens of 8
 * adapters of rank 64, 4096 -> 14336, bf16: 1.2 GB.
 */
uint64_t mi_lora_workspace(const mi_lora* sizes, int backward);

/*
 * Query and key heads of a batch of tokens, for mi_qk_norm_rope and its backward pass.  Strides are in
 * elements; base pointers are 16-byte aligned and strides multiples of 16 bytes; the values of a head
 * are contiguous.  The stride arrays are indexed like the call's tensors: forward {q, k, q_out, k_out},
 * backward {q, k, q_grad, k_grad, dq, dk}.
 */
typedef struct mi_heads {
    uint64_t tokens;
    uint64_t token_stride[6], head_stride[6];
    uint32_t q_heads, k_heads;
    uint32_t head_dim;        /* D: a multiple of 16, 16 ... 512                                     */
    uint32_t rotary_dim;      /* R: a multiple of 16, 0 ... D; the first R values of a head turn     */
    uint32_t axes;            /* position axes, 1 ... 4                                              */
    uint32_t section_end[4];  /* frequencies [section_end[i-1], section_end[i]) take axis i; the last
                                 of the `axes` entries is R / 2                                      */
    int32_t dtype;            /* of q, k, the outputs and gradients                                  */
    int32_t weight_dtype;     /* dtype, or MI_F32                                                    */
    uint32_t position_bits;   /* 32 or 64: signed integers                                           */
    uint32_t freq_bits;       /* 32 or 64: floats                                                    */
    uint32_t flags;           /* MI_HEADS_...                                                        */
    float eps;                /* >= 0                                                                */
} mi_heads;
#define MI_HEADS_NEIGHBOURS 1u /* the pairs are (2i, 2i+1); without it (i, i + R/2)                  */
#define MI_HEADS_HADAMARD 2u   /* the heads leave rotated by H_D / sqrt(D); D a power of two         */

/*
 * Norm of each query and key head, position rotation and optional Hadamard rotation, in one pass:
 *     n_i = x_i * (mean_j x_j^2 + eps)^-1/2 * weight_i
 *     pair f of n turns by  positions[axis(f)][token] * inv_freq[f]  radians:
 *     (a, b) -> (a cos - b sin, b cos + a sin);   values R ... D-1 stay
 *     out = H_D n / sqrt(D)   with MI_HEADS_HADAMARD
 * fp32 between the load and one rounding at the store; angles are formed and reduced in fp64.  The
 * Hadamard rotation of queries and keys alike leaves their products as they are and spreads outlier
 * channels before the keys are quantized.  No counterpart in the reference.
 *   q_weight, k_weight : [D] or NULL (all ones).
 *   positions          : [axes][tokens].      inv_freq : [R / 2].   (Not read when R = 0.)
 *   q_out, k_out       : may be q, k (in place, same strides); no other overlap.
 */
int mi_qk_norm_rope(const void* q, const void* k, const void* q_weight, const void* k_weight,
                    const void* positions, const void* inv_freq, void* q_out, void* k_out,
                    const mi_heads* heads, void* stream);

/*
 * Gradients of mi_qk_norm_rope.  q, k are the forward pass's inputs, q_grad, k_grad the gradients of its
 * outputs; dq, dk receive the gradients of q, k and overlap none of them.  dq_weight, dk_weight: [D] in
 * weight_dtype, or NULL; they are sums over all tokens and heads, in a fixed order.
 *   workspace : mi_qk_norm_rope_workspace(tokens, D) bytes, 16-byte aligned; not needed (NULL) when
 *               both weight gradients are NULL.  Two kernels with weight gradients, else one.
 */
int mi_qk_norm_rope_backward(const void* q, const void* k, const void* q_grad, const void* k_grad,
                             const void* q_weight, const void* k_weight, const void* positions,
                             const void* inv_freq, void* dq, void* dk, void* dq_weight, void* dk_weight,
                             void* workspace, const mi_heads* heads, void* stream);
uint64_t mi_qk_norm_rope_workspace(uint64_t tokens, uint32_t head_dim);

/*
 * One-wavefront MFMA layout check:  D[16,16] = A[16,Kk] * B[Kk,16]  with exactly one matrix-core
 * instruction, operands gathered under the register layout the kernels assume.
 * Mirrors the reference's test hook  test_mma_m16_n8_k16(x, y)  (csrc/test_frag.cu:8-62,
 * exported at csrc/hadamard_transform.cpp:83-89).
 *   kind 0: v_mfma_f32_16x16x32_bf16 (Kk = 32)    kind 1: v_mfma_f32_16x16x16_bf16 (Kk = 16)
 *   kind 2: v_mfma_f32_16x16x32_f16  (Kk = 32)    kind 3: v_mfma_f32_16x16x16_f16  (Kk = 16)
 *   kind 4: v_mfma_f32_16x16x4_f32   (Kk = 4, A and B fp32)
 *   A, B: row-major, element type per kind;  D: fp32 row-major.
 */
int mi_debug_mfma_16x16(int kind, const void* A, const void* B, float* D, void* stream);

/*
 * Element-wise narrowing conversions as the kernels perform them (hardware RNE), for unit tests
 * (the reference's  test_bit_convert, csrc/test_bit.cu:8-42).
 *   kind 0: fp32 -> bf16 bits (uint16)    kind 1: fp32 -> fp16 bits (uint16)
 *   kind 2: fp32 -> E4M3FN code (uint8), input clamped to +-448 first
 */
int mi_debug_convert(int kind, const float* in, void* out, uint64_t count, void* stream);

/*
 * Same contract as mi_fwht, but computed by a minimal kernel written against the device-side
 * embedding API (csrc/hadamard_device.hpp: HadamardTransformDevice<IO, LOG_N>), one call of
 * hadamard_transform_device per workgroup.  Exists so the embedding API -- the counterpart of the
 * reference's  HadamardTransform<dtype,N>::hadamard_transform_device  (csrc/hada_handler.cuh:
 * 227-264, thin caller csrc/main.cu:42-53) -- is tested for every length and element type.
 *   rows must be a multiple of the API's N_ROWS (512 / n for n <= 512, else 1): MI_ERR_SHAPE.
 */
int mi_debug_device_fwht(const void* in, void* out, uint64_t rows, uint32_t n, int dtype,
                         float scale, void* stream);

/*
 * Host-only: how mi_fused_ht_gemm cuts a 16-bit problem with K = 512 ... 4096 into workgroups (no
 * GPU call; MI_ERR_SIZE for any other K).
 * The (column group, M slice) grid, the XCD rectangles and the map from workgroup id to tile are
 * what decides L2 reuse and the number of launch rounds; this hook lets a test check on the CPU
 * that every tile is handled by exactly one workgroup.  No counterpart in the reference.
 *   header[8] : ngroups (groups of 131072 / K columns, 64 at K = 4096), msplit (M slices), m_per_block (rows per slice),
 *               mpx, cgx (rectangle extents in M slices and column groups), nrect, grid
 *               (workgroups launched), 0
 *   tiles     : NULL, or 2 * capacity uint32: for workgroup id i, tiles[2i] = column group and
 *               tiles[2i+1] = M slice, or 0xffffffff twice for an id without work
 * Returns MI_ERR_SIZE when capacity < grid (header is filled in either way).
 */
int mi_debug_fused_gemm_tiling(uint32_t M, uint32_t N, uint32_t K, uint32_t* header, uint32_t* tiles,
                               uint32_t capacity);

#ifdef __cplusplus
}
#endif
#endif /* MI_HADAMARD_H */
