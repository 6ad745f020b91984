/*
 * sbx.h -- C ABI of the MI355X (gfx950) GEMM hot path of SushiBLAS.
 *
 * This is the drop-in boundary.  In the reference, Level3::gemm
 * (src/ops/blas/level3/gemm.cpp:82-198) records a task whose body,
 * gemm_dispatch<T> (gemm.cpp:44-79), calls oneMKL on a sycl::queue.  Each
 * entry point below replaces one of those oneMKL calls one-for-one: the same
 * argument set as gemm_dispatch (gemm.cpp:45-51), with the sycl::queue
 * replaced by a hipStream_t and the dependency-event vector replaced by
 * stream order.
 *
 * Conventions
 *   - Plain pointers and sizes only; every buffer is caller-owned device
 *     memory (or pinned host memory mapped into the device address space).
 *     The library never frees or retains a caller pointer.
 *   - Launches are asynchronous on `stream` (NULL = the null stream of the
 *     current device; hipStreamPerThread is accepted).  The only allocation
 *     is the workspace for split-K GEMM/SYRK partials and chunked GEMV
 *     partials: cached per (device, stream), grown with hipMalloc (at least
 *     doubling) the first time a larger one is needed and reused after that;
 *     an outgrown buffer is kept, not freed, until the process ends.  Uses of
 *     a workspace are ordered by its stream.  Calls on hipStreamPerThread get
 *     no workspace and run unsplit.  If the allocation fails the call runs
 *     without splitting instead of failing.
 *   - Return value is a status code (sbx_status); nothing throws across the
 *     ABI.  The C++ layer turns codes into std::runtime_error, as the
 *     reference's SB_THROW_IF does (include/SushiBLAS/core/logger.hpp:316-323).
 *   - BLAS semantics: m == 0 || n == 0 is a no-op; alpha == 0 || k == 0 gives
 *     C = beta*C; beta == 0 means C is never read (NaN/Inf in C do not
 *     propagate).
 *   - layout 0 = row-major, 1 = column-major (Core::Layout,
 *     include/SushiBLAS/core/common.hpp:41-45).  transA/transB: 0 or 1.
 *   - fp32 GEMM and SYRK on the tiles of 128x128, 256x64, 64x256 and more
 *     multiply on the bf16 matrix cores, each operand value as the exact sum of
 *     three bf16 values: results are nearer to the exact sums than fp32 products
 *     added in order (3.0e-7 against 1.6e-6 at K = 8192).  Where the sum is not
 *     exact (bits below 2^-133, which only values below 2^-110 have) and that
 *     could move a result by 2^-24 of its terms' magnitudes, and where
 *     infinities, NaN or values next to fp32's largest meet, the tile is
 *     computed again with fp32 products: it then gives what fp32 arithmetic gives.
 *   - Re-entrant: the only global state is the per-device CU count and the
 *     workspace cache, both behind mutexes; safe to call from any host thread
 *     (the reference runs the GEMM closure on a scheduler worker thread).
 *     Calls on one stream share its workspace and run in stream order; the
 *     two kernels of a split call are enqueued under that stream's lock, so
 *     concurrent host threads on one stream cannot interleave with them.
 */
#ifndef SBX_H
#define SBX_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum sbx_status {
    SBX_OK = 0,
    SBX_INVALID_ARGUMENT = 1, /* bad layout/trans flag, negative size, ld too small, null ptr */
    SBX_UNSUPPORTED = 2,      /* dtype or shape this build cannot run                       */
    SBX_HIP_ERROR = 3         /* a HIP runtime call or kernel launch failed                */
} sbx_status;

/* SBX_BF16 and SBX_F16: the dropout, norm, MXFP4 and MXFP8 entry points only (the
 * others return SBX_UNSUPPORTED). */
typedef enum sbx_dtype { SBX_F32 = 0, SBX_F64 = 1, SBX_BF16 = 2, SBX_F16 = 3 } sbx_dtype;

/* Replaces oneapi::mkl::blas::row_major::gemm<float> (gemm.cpp:63) and
 * column_major::gemm<float> (gemm.cpp:76), reached from the FLOAT32 case of
 * Level3::gemm (gemm.cpp:146-157). */
int sbx_sgemm(void* stream, int layout, int transA, int transB, int64_t m, int64_t n, int64_t k,
              float alpha, const float* A, int64_t lda, const float* B, int64_t ldb, float beta,
              float* C, int64_t ldc);

/* Replaces row_major::gemm<double> (gemm.cpp:63) / column_major::gemm<double>
 * (gemm.cpp:76), reached from the FLOAT64 case (gemm.cpp:158-169), where the
 * float alpha/beta are widened to double (gemm.cpp:161). */
int sbx_dgemm(void* stream, int layout, int transA, int transB, int64_t m, int64_t n, int64_t k,
              double alpha, const double* A, int64_t lda, const double* B, int64_t ldb,
              double beta, double* C, int64_t ldc);

/* Replaces row_major::gemm_batch<float> (gemm.cpp:58) and
 * column_major::gemm_batch<float> (gemm.cpp:71): `batch` problems, problem b
 * using A + b*str_a, B + b*str_b, C + b*str_c (strides in elements, as
 * derived at gemm.cpp:103-105). */
int sbx_sgemm_strided_batched(void* stream, int layout, int transA, int transB, int64_t m,
                              int64_t n, int64_t k, float alpha, const float* A, int64_t lda,
                              int64_t str_a, const float* B, int64_t ldb, int64_t str_b,
                              float beta, float* C, int64_t ldc, int64_t str_c, int64_t batch);

/* Replaces row_major::gemm_batch<double> (gemm.cpp:58) / column_major::gemm_batch<double>
 * (gemm.cpp:71). */
int sbx_dgemm_strided_batched(void* stream, int layout, int transA, int transB, int64_t m,
                              int64_t n, int64_t k, double alpha, const double* A, int64_t lda,
                              int64_t str_a, const double* B, int64_t ldb, int64_t str_b,
                              double beta, double* C, int64_t ldc, int64_t str_c,
                              int64_t batch);

/* Algorithm override for tests and tuning (no counterpart in the reference,
 * where oneMKL chooses internally): SBX_ALGO_AUTO is what the four entry
 * points above use.  SBX_ALGO_MFMA: any MFMA kernel (model's choice);
 * SBX_ALGO_MFMA_TILE: the LDS-tiled MFMA kernels only; SBX_ALGO_MFMA_SMALL:
 * the one-launch small-problem kernel.  A forced choice the
 * problem cannot use returns SBX_UNSUPPORTED. */
typedef enum sbx_algo {
    SBX_ALGO_AUTO = 0,
    SBX_ALGO_GENERIC = 1,
    SBX_ALGO_MFMA = 2,
    SBX_ALGO_MFMA_TILE = 3,
    SBX_ALGO_MFMA_SMALL = 4
} sbx_algo;

/* dtype-generic form of the four entry points above; alpha/beta point to a
 * float (SBX_F32) or double (SBX_F64). */
int sbx_gemm_ex(void* stream, int dtype, int layout, int transA, int transB, int64_t m,
                int64_t n, int64_t k, const void* alpha, const void* A, int64_t lda,
                int64_t str_a, const void* B, int64_t ldb, int64_t str_b, const void* beta,
                void* C, int64_t ldc, int64_t str_c, int64_t batch, int algo);

/* Bytes of the fixed per-device scratch that sbx_gemm_ex_noalloc uses. */
#define SBX_NOALLOC_SCRATCH_BYTES ((size_t)32 << 20)

/* sbx_gemm_ex without any allocation.  No counterpart in the reference: it
 * is for callers that cannot allocate device memory -- code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc.  Same
 * arguments and results as sbx_gemm_ex, except that split-K partials go to a
 * fixed array of SBX_NOALLOC_SCRATCH_BYTES in device memory (one per GPU,
 * held from the library's first use on that GPU until the process ends)
 * instead of the stream's workspace, and the tiling heuristics only consider
 * splits whose partials fit in it (a problem whose preferred split would not
 * fit runs with fewer k-parts or unsplit, so results may differ from
 * sbx_gemm_ex by rounding only; none is refused for its size).  It calls no
 * hipMalloc/hipFree.  Every call on one GPU shares that GPU's array.  A call
 * that splits holds a per-GPU host lock while it enqueues its two kernels
 * (the partial pass and the reduction), so concurrent host threads are
 * serialised at enqueue: on one stream, one call's kernels never interleave
 * with another's, whatever thread issued them.  Calls on different streams
 * of one GPU are not ordered by that lock: when their kernels run at the
 * same time they race on the array, and the caller must order them (one
 * stream, or events).  Every partial is written before it is read, so
 * nothing in the array needs clearing. */
int sbx_gemm_ex_noalloc(void* stream, int dtype, int layout, int transA, int transB, int64_t m,
                        int64_t n, int64_t k, const void* alpha, const void* A, int64_t lda,
                        int64_t str_a, const void* B, int64_t ldb, int64_t str_b,
                        const void* beta, void* C, int64_t ldc, int64_t str_c, int64_t batch,
                        int algo);

/* Epilogues that can be fused into the GEMM (no counterpart on the
 * reference's GEMM path, where they are separate tasks). */
typedef enum sbx_epilogue { SBX_EPILOGUE_NONE = 0, SBX_EPILOGUE_RELU = 1 } sbx_epilogue;

/* C = epilogue(alpha*op(A)*op(B) + beta*C), same arguments as sbx_gemm_ex.
 * SBX_EPILOGUE_RELU fuses the caller pattern of the reference's integration
 * tests -- Level3::gemm followed by NonLinearOps::relu on C
 * (tests/runtime/test_framework_sim.cpp:51-57,109-110; ReLU is
 * src/ops/math/nonlinear/relu.cpp:38-41: x > 0 ? x : 0) -- into one kernel,
 * saving the extra read and write of C. */
int sbx_gemm_fused(void* stream, int dtype, int layout, int transA, int transB, int64_t m,
                   int64_t n, int64_t k, const void* alpha, const void* A, int64_t lda,
                   int64_t str_a, const void* B, int64_t ldb, int64_t str_b, const void* beta,
                   void* C, int64_t ldc, int64_t str_c, int64_t batch, int epilogue);

/* Grouped GEMM: `count` problems C_i = epilogue(alpha*op(A_i)*op(B_i) +
 * beta*C_i) with one shape, one set of leading dimensions and scalars, and
 * operands anywhere in device memory: `table` is a DEVICE array of 3*count
 * pointers (A_0, B_0, C_0, A_1, B_1, C_1, ...), read by the kernel in stream
 * order.  aligned16 != 0 promises every C pointer is 16-byte aligned (enables
 * 16-byte C stores; operand loads are 16 bytes at any alignment).  One launch for all of them.  No single counterpart in the
 * reference: it is how the task graph issues a run of independent,
 * same-shaped Level3::gemm tasks (each one gemm.cpp:63 / :76 call in the
 * reference, run on worker threads) without one launch per task. */
int sbx_gemm_grouped(void* stream, int dtype, int layout, int transA, int transB, int64_t m,
                     int64_t n, int64_t k, const void* alpha, int64_t lda, int64_t ldb,
                     const void* beta, int64_t ldc, const void* const* table, int64_t count,
                     int aligned16, int epilogue);

/* x[i] = x[i] > 0 ? x[i] : 0 for n contiguous elements of dtype: the
 * stand-alone ReLU (replaces the body of NonLinearOps::relu,
 * src/ops/math/nonlinear/relu.cpp:38-41, for FLOAT32/FLOAT64). */
int sbx_relu(void* stream, int dtype, void* x, int64_t n);

/* GEMV, y = alpha*op(A)*x + beta*y with op(A) = A (m x n) or A^T: replaces
 * oneapi::mkl::blas::row_major::gemv (src/ops/blas/level2/gemv.cpp:55) and
 * column_major::gemv (gemv.cpp:60), reached from Level2::gemv (gemv.cpp:65-148)
 * for FLOAT32 / FLOAT64 (float alpha/beta widened, gemv.cpp:125).  x has
 * (transA ? m : n) elements x[i*incx], y has (transA ? n : m) elements
 * y[i*incy]; increments must be positive (the reference passes 1 or a rank-1
 * tensor's stride, utils.hpp:47-60).  Netlib quick returns: m == 0 or n == 0
 * leaves y untouched; alpha == 0 gives y = beta*y; beta == 0 never reads y. */
int sbx_sgemv(void* stream, int layout, int transA, int64_t m, int64_t n, float alpha,
              const float* A, int64_t lda, const float* x, int64_t incx, float beta, float* y,
              int64_t incy);
int sbx_dgemv(void* stream, int layout, int transA, int64_t m, int64_t n, double alpha,
              const double* A, int64_t lda, const double* x, int64_t incx, double beta,
              double* y, int64_t incy);

/* SYRK on one triangle of the n x n C: C = alpha*op(A)*op(A)^T + beta*C with
 * op(A) = A (n x k) when trans == 0 and A^T (A is k x n) when trans == 1;
 * upper != 0 updates the upper triangle, else the lower; the other triangle
 * is neither read nor written.  Replaces row_major::syrk / syrk_batch
 * (src/ops/blas/level3/syrk.cpp:65,60) and column_major::syrk / syrk_batch
 * (syrk.cpp:78,73), reached from Level3::syrk (syrk.cpp:84-194); batch b uses
 * A + b*str_a and C + b*str_c.  Quick returns as for GEMM: n == 0 is a
 * no-op, alpha == 0 or k == 0 gives C = beta*C on the triangle. */
int sbx_ssyrk(void* stream, int layout, int upper, int trans, int64_t n, int64_t k, float alpha,
              const float* A, int64_t lda, float beta, float* C, int64_t ldc);
int sbx_dsyrk(void* stream, int layout, int upper, int trans, int64_t n, int64_t k,
              double alpha, const double* A, int64_t lda, double beta, double* C, int64_t ldc);
int sbx_ssyrk_strided_batched(void* stream, int layout, int upper, int trans, int64_t n,
                              int64_t k, float alpha, const float* A, int64_t lda, int64_t str_a,
                              float beta, float* C, int64_t ldc, int64_t str_c, int64_t batch);
int sbx_dsyrk_strided_batched(void* stream, int layout, int upper, int trans, int64_t n,
                              int64_t k, double alpha, const double* A, int64_t lda,
                              int64_t str_a, double beta, double* C, int64_t ldc, int64_t str_c,
                              int64_t batch);

/* ---- Dropout and MXFP4: a dense layer's training and serving in 4 bits ----
 *
 * None of these has a counterpart in the reference.  They make a feed-forward
 * block whose products run on the 4-bit matrix cores: quantise activations,
 * weights and gradients along the axis that a product sums over, multiply, and
 * drop activations out on their way.  All matrices are row-major; nothing is
 * allocated and no workspace used.  Sides are 2^30 at most (m, n too; and what
 * would take 2^31 tiles of 128 x 128 to quantise, or 2^23 of 256 x 256 to
 * multiply, is refused too): SBX_UNSUPPORTED. */

/* Dropout, Y = keep ? X / (1 - p) : 0 (rows x cols, F32, F64, BF16 or F16).
 * keep is a function of (seed, stream_id, row, column) alone, by the
 * counter-based Philox4x32-10: 16 bits h per element -- word c % 8 / 2, half
 * c % 2, of the counter (c / 8, row, stream_id, 0x44524F50) under the key seed --
 * and an element stays if h >= t, t = floor(65536 p + 0.5).  The factor is
 * 65536 / (65536 - t), rounded to the arithmetic's type (fp64 for F64, else fp32):
 * that of the rate that p is rounded to, so the mean is kept.  From p = 1 - 2^-17
 * on (t = 65536) everything is dropped.  The mask is never stored: the backward pass is the same
 * call on dY with the same p, seed and stream_id.
 * gate (may be NULL): values that pass only where gate > 0, else 0.  Backward:
 * the output of the ReLU that the dropout followed, so the call is the gradient
 * through both; forward: gate == X is the ReLU itself.
 * Dropped and gated values are 0 whatever X holds there, NaN included.  Y may
 * be X or the gate itself (same leading dimension).  0 <= p <= 1. */
int sbx_dropout(void* stream, int dtype, int64_t rows, int64_t cols, const void* X, int64_t ldx,
                const void* gate, int64_t ldg, void* Y, int64_t ldy, double p, uint64_t seed,
                uint32_t stream_id);

/* Quantisation to MXFP4, the OCP microscaling format with 4-bit e2m1 elements
 * (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), of V: the rows x cols matrix X
 * (F32, BF16 or F16) after sbx_dropout's p, seed, stream_id and gate (p = 0 and
 * gate = NULL: X itself; V is held in 32 bits, not rounded to dtype).
 *   P, S (NULL: not wanted): V in blocks of 32 along its rows.  Element
 * (r, c) is half c % 2 (0: low) of byte P[r*ldp + c/2]; a row's last block is
 * filled with zeros.  Block b of row r has its scale 2^(code - 127) at
 * S[(b/8)*lds + 8*r + b%8]: 8 blocks of a row lie together (codes past a row's
 * last block are 0), groups of 8 blocks lds bytes apart.
 *   PT, ST: the same of V^T (cols x rows), blocks of 32 along V's columns.
 * code = max(floor(log2 max|v|) - 2, -127) + 127 over the block; elements are
 * v / 2^(code - 127) rounded to nearest even, saturated at 6.  A block with an
 * infinity or NaN has code 255: all of it is NaN.
 * P, PT 16-byte aligned, ldp >= 16*ceil(cols/32) and a multiple of 16; S, ST
 * 8-byte aligned, lds >= 8*rows and a multiple of 8 (ldpt, ldst: of rows and
 * cols).  As everywhere here this is asked of a leading dimension also where one
 * row, or one group of codes, leaves it without a use (the Python binding, which
 * is given torch's strides, puts the packed one there). */
int sbx_mx4_quantize(void* stream, int dtype, int64_t rows, int64_t cols, const void* X,
                     int64_t ldx, const void* gate, int64_t ldg, double p, uint64_t seed,
                     uint32_t stream_id, void* P, int64_t ldp, void* S, int64_t lds, void* PT,
                     int64_t ldpt, void* ST, int64_t ldst);

/* The values an MXFP4 matrix (P, S as above) stands for, rounded to dtype
 * (F32: exact). */
int sbx_mx4_dequantize(void* stream, int dtype, int64_t rows, int64_t cols, const void* P,
                       int64_t ldp, const void* S, int64_t lds, void* Y, int64_t ldy);

/* C = epilogue(alpha * A * B^T + beta * C): A (m x k) and B (n x k) MXFP4
 * matrices (A, SA with lda, ldsa; B, SB with ldb, ldsb, as written by
 * sbx_mx4_quantize), C (m x n) of dtype F32, BF16 or F16 in `layout`.  Products
 * are exact (down to 2^-149), sums are held in 32 bits and rounded to dtype once.  What lies
 * past the k-th term's block is not used, nor are the codes there.  BLAS
 * semantics as for GEMM (beta == 0: C is not read; alpha == 0 or k == 0: A and
 * B are not).  A layer's three products are this one on the right quantisations:
 *   forward Y = X W^T    : X along rows, W (n x k) along rows
 *   dX = dY W            : dY along rows, W's PT
 *   dW = dY^T X          : dY's PT, X's PT
 * k <= 2^23 and lda, ldb < 2^23 - 15 (else SBX_UNSUPPORTED). */
int sbx_mx4_gemm(void* stream, int dtype, int layout, int64_t m, int64_t n, int64_t k, float alpha,
                 const void* A, int64_t lda, const void* SA, int64_t ldsa, const void* B,
                 int64_t ldb, const void* SB, int64_t ldsb, float beta, void* C, int64_t ldc,
                 int epilogue);

/* ---- Norm, and MXFP4 weights for a few tokens -------------------------------
 *
 * None of these has a counterpart in the reference.  They are what stands around a
 * dense layer: the norm before it, with the residual's addition, in training and
 * serving, and products for a few tokens whose weights are MXFP4 matrices
 * (sbx_mx4_quantize along rows) and whose activations keep their type, or 8 bits.
 * dtype is F32, BF16 or F16, all dense matrices are row-major and of it.  Nothing is
 * allocated: what needs memory of its own takes it from the caller, as many bytes
 * as its _workspace function says (0: sizes that are refused), 16-byte aligned; its
 * contents are nobody's business before or after, and calls that may run at the
 * same time need one each. */

/* H = X + R in dtype's precision (rounded to dtype; R NULL: H = X), and row by row
 *   V = H * W / sqrt(mean(H^2) + eps)
 * with W one value per column.  Sums and statistics are held in 64 bits, V in 32.
 *   H, Y (NULL: not wanted): rows x cols, Y is V rounded to dtype.
 *   P, S (NULL: not wanted): V as an MXFP8 matrix, blocks of 32 along its rows:
 * element (r, c) is the e4m3 byte P[r*ldp + c], a row's last block filled with
 * zeros; codes as MXFP4's (sbx_mx4_quantize).  code = max(floor(log2 max|v|) - 8,
 * -127) + 127; elements are v / 2^(code - 127) rounded to nearest even and saturated
 * at 448.  A block with an infinity or NaN has code 255: all of it is NaN.  P 16-byte
 * aligned, ldp >= 32*ceil(cols/32) and a multiple of 16; S, lds as MXFP4's.
 * One of H, Y, P at least.  H may be X or R; Y may be X or R too where H is neither
 * (same leading dimension).  eps >= 0 and finite; with eps = 0 a row of zeros is NaN. */
int sbx_rms_norm(void* stream, int dtype, int64_t rows, int64_t cols, const void* X, int64_t ldx,
                 const void* R, int64_t ldr, const void* W, double eps, void* H, int64_t ldh, void* Y,
                 int64_t ldy, void* P, int64_t ldp, void* S, int64_t lds);

/* The gradient of Y = H * W / sqrt(mean(H^2) + eps): with s = 1 / sqrt(mean(H^2) + eps)
 *   DX = s * DY * W - H * s^3 * mean(DY * W * H)  (+ DR, if there is one: a gradient that
 *        reaches H along the residual), which is X's and R's of sbx_rms_norm alike
 *   DW = the sum over rows of s * DY * H, in 32 bits (NULL: not wanted, and no workspace)
 * s is computed again from H, so the forward call stores none.  DX may be DY or DR
 * (same leading dimension).  The order of DW's sums depends on rows, cols and
 * dtype alone.  Without rows DW is zero. */
int sbx_rms_norm_grad(void* stream, int dtype, int64_t rows, int64_t cols, const void* H, int64_t ldh,
                      const void* W, double eps, const void* DY, int64_t lddy, const void* DR,
                      int64_t lddr, void* DX, int64_t lddx, float* DW, void* workspace,
                      size_t workspace_bytes);
size_t sbx_rms_norm_grad_workspace(int64_t rows, int64_t cols);

/* The values an MXFP8 matrix (P, S as above) stands for, rounded to dtype
 * (F32: exact, below 2^128). */
int sbx_mx8_dequantize(void* stream, int dtype, int64_t rows, int64_t cols, const void* P,
                       int64_t ldp, const void* S, int64_t lds, void* Y, int64_t ldy);

/* Y = epilogue(alpha * X * B^T + beta * Y) for a few rows: X (m x k) keeps its type
 * (SX NULL) or is an MXFP8 matrix (X, SX), B (n x k) is an MXFP4 matrix, Y (m x n) of
 * dtype.  X is not rounded (but for bits of fp32 and MXFP8 values below 2^-133, which do not
 * count); sums are held in 32 bits and rounded to dtype once.  A value of 2^128 or more, which 32
 * bits do not hold either (MXFP4's of 4 and 6 under code 253 and of 2 and more under 254, MXFP8's under
 * codes from 247 on; no quantiser here writes one), is an infinity: results that it is a term of are
 * infinite or NaN, and those of a row of B that has it past the k-th term, in the same block, may be
 * NaN.  What else lies past the k-th term is not used; Y lies apart from X and B.  BLAS semantics as for GEMM (beta == 0: Y is
 * not read; alpha == 0 or k == 0: X and B are not).  Rows are computed apart: those of
 * one call have the bits that they have alone.  m <= 1024, n <= 2^30, k <= 2^23, ldb <
 * 2^23 - 15, a row of X (ldx) at most 2^26 bytes (else SBX_UNSUPPORTED). */
int sbx_mx4_linear(void* stream, int dtype, int64_t m, int64_t n, int64_t k, float alpha,
                   const void* X, int64_t ldx, const void* SX, int64_t ldsx, const void* B,
                   int64_t ldb, const void* SB, int64_t ldsb, float beta, void* Y, int64_t ldy,
                   int epilogue);

/* A mixture-of-experts layer for a few tokens.  For each token x (a row of X, tokens x
 * width): logits WR x (WR: experts x width, dense) in 64 bits; the topk experts with
 * the highest ones, in that order, equal ones by index (NaN counts as the highest);
 * p = softmax over the chosen ones' logits (normalize != 0) or over all (0); and
 *   y = sum_j p_j * W2_e (silu(G_e x) * (U_e x)),  silu(z) = z / (1 + exp(-z)),  e the j-th expert
 * W1, S1: an MXFP4 matrix of experts * 2 * hidden rows over width, expert e's G at rows
 * e * 2 * hidden, its U hidden rows later.  W2, S2: of experts * width rows over hidden.
 * For W1 and W2 sbx_mx4_linear's words about values past 32 bits hold.
 * Activations are not rounded before W1's product (but for bits of fp32 values below 2^-133);
 * before W2's they are held as the sum of three bf16 values, 24 bits.  Sums are held in 32 bits and
 * rounded to dtype once.
 * A token's result has the same bits in calls of the same sizes, wherever it stands and whatever the
 * others are; in a call of another number of tokens its sums may be in another order.
 * chosen (int32), weights (p): tokens x topk, packed; NULL: not wanted.  Y may be X
 * (same leading dimension).
 * tokens <= 256, topk <= 16, experts <= 512, width and hidden <= 2^18, ld1, ld2 < 2^23 -
 * 15, of several tokens a row of X (ldx) less than 2^23 - 15 bytes (else SBX_UNSUPPORTED). */
int sbx_mx4_moe(void* stream, int dtype, int64_t tokens, int64_t width, int64_t hidden,
                int64_t experts, int64_t topk, const void* X, int64_t ldx, const void* WR,
                int64_t ldwr, int normalize, const void* W1, int64_t ld1, const void* S1,
                int64_t lds1, const void* W2, int64_t ld2, const void* S2, int64_t lds2, void* Y,
                int64_t ldy, int32_t* chosen, float* weights, void* workspace,
                size_t workspace_bytes);
size_t sbx_mx4_moe_workspace(int64_t tokens, int64_t width, int64_t hidden, int64_t experts,
                             int64_t topk);

/* Name of the plan (kernel tile and k-split) the dispatcher would launch for
 * this problem (tiling heuristics introspection for benchmarks).  A name is a
 * plan's handle, not a description of the kernel's inside: an unsplit
 * 256x128 plan may run its tiles in neighbouring pairs.  Pointers are assumed 16-byte
 * aligned.  Writes a NUL-terminated string of at most cap bytes. */
int sbx_gemm_select(int dtype, int layout, int transA, int transB, int64_t m, int64_t n,
                    int64_t k, int64_t lda, int64_t ldb, int64_t ldc, char* name, size_t cap);

/* The same for a strided batch of `batch` packed entries (stride = the stored
 * extent of each operand): a batch whose grid fills less than one round of
 * the device cuts K too, so its pick can differ from a single problem's.
 * No counterpart in the reference (introspection, as above). */
int sbx_gemm_select_batched(int dtype, int layout, int transA, int transB, int64_t m, int64_t n,
                            int64_t k, int64_t lda, int64_t ldb, int64_t ldc, int64_t batch,
                            char* name, size_t cap);

/* The plans the tiling heuristics weigh for this (packed, as above) problem:
 * one line "<plan name> <predicted microseconds>\n" per candidate kernel and
 * k-split, in the names sbx_gemm_select reports (NUL-terminated, at most cap
 * bytes; SBX_INVALID_ARGUMENT if they do not fit).  No counterpart in the
 * reference: it serves measurements of the heuristics against every
 * candidate (regret), with sbx_gemm_ex_plan. */
int sbx_gemm_plans(int dtype, int layout, int transA, int transB, int64_t m, int64_t n,
                   int64_t k, int64_t lda, int64_t ldb, int64_t ldc, int64_t batch, char* out,
                   size_t cap);

/* sbx_gemm_ex (algo = AUTO) with the named plan -- a name from sbx_gemm_plans
 * or sbx_gemm_select -- instead of the heuristics' pick.  Same results as any
 * plan within the tolerance.  SBX_INVALID_ARGUMENT for a name that is no
 * plan, SBX_UNSUPPORTED for a plan the problem cannot use (another element
 * type, offsets beyond the kernel's range, more k-ranges than its tail
 * allows).  No counterpart in the reference (measurement hook, as above). */
int sbx_gemm_ex_plan(void* stream, int dtype, int layout, int transA, int transB, int64_t m,
                     int64_t n, int64_t k, const void* alpha, const void* A, int64_t lda,
                     int64_t str_a, const void* B, int64_t ldb, int64_t str_b, const void* beta,
                     void* C, int64_t ldc, int64_t str_c, int64_t batch, const char* plan);

/* The same for sbx_{s,d}syrk[_strided_batched] (single problem): the kernel
 * and split that would compute the triangle. */
int sbx_syrk_select(int dtype, int layout, int upper, int trans, int64_t n, int64_t k,
                    int64_t lda, int64_t ldc, char* name, size_t cap);

/* sbx_gemm_plans for a single SYRK problem: the plans (square tile configs
 * over the triangle, unsplit and split) the heuristics weigh.  No counterpart
 * in the reference (measurement hook, as above). */
int sbx_syrk_plans(int dtype, int layout, int upper, int trans, int64_t n, int64_t k,
                   int64_t lda, int64_t ldc, char* out, size_t cap);

/* sbx_{s,d}syrk_strided_batched with the named plan (a name from
 * sbx_syrk_plans or sbx_syrk_select) instead of the heuristics' pick; status
 * as sbx_gemm_ex_plan (a config that is not a triangle's is
 * SBX_UNSUPPORTED).  alpha and beta point to the element type's scalar.  No
 * counterpart in the reference (measurement hook, as above). */
int sbx_syrk_ex_plan(void* stream, int dtype, int layout, int upper, int trans, int64_t n,
                     int64_t k, const void* alpha, const void* A, int64_t lda, int64_t str_a,
                     const void* beta, void* C, int64_t ldc, int64_t str_c, int64_t batch,
                     const char* plan);

/* Human-readable text for a status code (static storage). */
const char* sbx_status_string(int status);

/* Synthetic-input generators (Philox4x32-10, counter-based), writing n
 * elements of dtype into device memory on `stream`.  They stand in for the
 * reference's RandomOps::uniform / normal (src/ops/math/random/uniform.cpp:40-62)
 * only as a source of benchmark inputs; the stream layout is this library's
 * own: key = seed, counter = (element block, stream_id, 0).
 * uniform: [-1, 1).  normal: N(0, 1) * scale. */
int sbx_fill_uniform(void* stream, int dtype, void* out, int64_t n, uint64_t seed,
                     uint32_t stream_id);
int sbx_fill_normal(void* stream, int dtype, void* out, int64_t n, uint64_t seed,
                    uint32_t stream_id, double scale);

/* Library version string. */
const char* sbx_version(void);

#ifdef __cplusplus
}
#endif

#endif /* SBX_H */
