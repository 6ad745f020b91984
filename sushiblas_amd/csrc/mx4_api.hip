// mx4_api.hip -- C entry points of the dropout and the MXFP4 operators
// (include/sbx.h): argument checks, the column-major mapping, quick returns.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/sbx.h"
#include "mx4.hpp"

namespace sbx {
namespace {

constexpr int64_t kMaxSide = (int64_t)1 << 30;  // rows, columns
// terms of a product and bytes of its operands' rows: 256 rows stay within the
// kernel's 32-bit offsets
constexpr int64_t kMaxTerms = (int64_t)1 << 23;
constexpr int64_t kMaxRowBytes = ((int64_t)1 << 23) - 16;

int64_t blocks(int64_t k) { return (k + 31) / 32; }

size_t elem_size(int dtype) { return dtype == SBX_F64 ? 8 : dtype == SBX_F32 ? 4 : 2; }

bool is_dtype(int dtype, bool f64)
{
    return dtype == SBX_F32 || dtype == SBX_BF16 || dtype == SBX_F16 || (f64 && dtype == SBX_F64);
}

// A row-major rows x cols matrix of `elem`-byte values.
bool bad_dense(const void* X, int64_t cols, int64_t ld, size_t elem)
{
    return !X || (uintptr_t)X % elem || ld < cols;
}

// The packed elements and codes of a rows x cols MXFP4 matrix.
bool bad_mx4(const void* P, int64_t ldp, const void* S, int64_t lds, int64_t rows, int64_t cols)
{
    return !P || !S || (uintptr_t)P % 16 || (uintptr_t)S % 8 || ldp % 16 || lds % 8 ||
           ldp < 16 * blocks(cols) || lds < 8 * rows;
}

int dropout_args(DropoutArgs* a, const void* X, int64_t ldx, const void* gate, int64_t ldg,
                 int64_t rows, int64_t cols, double p, uint64_t seed, uint32_t stream_id,
                 size_t elem)
{
    if (!(p >= 0.0 && p <= 1.0)) return SBX_INVALID_ARGUMENT;
    if (bad_dense(X, cols, ldx, elem)) return SBX_INVALID_ARGUMENT;
    if (gate && bad_dense(gate, cols, ldg, elem)) return SBX_INVALID_ARGUMENT;
    a->X = X; a->ldx = ldx;
    a->gate = gate; a->ldg = ldg;
    a->rows = rows; a->cols = cols;
    a->seed = seed; a->stream_id = stream_id;
    a->threshold = (uint32_t)floor(65536.0 * p + 0.5);
    a->scale = a->threshold < 65536 ? 65536.0 / (65536 - a->threshold) : 0.0;
    return SBX_OK;
}

int status_of(hipError_t e)
{
    return e == hipSuccess ? SBX_OK : e == hipErrorNotSupported ? SBX_UNSUPPORTED : SBX_HIP_ERROR;
}

}  // namespace
}  // namespace sbx

extern "C" {

int sbx_dropout(void* stream, int dtype, int64_t rows, int64_t cols, const void* X, int64_t ldx,
                const void* gate, int64_t ldg, void* Y, int64_t ldy, double p, uint64_t seed,
                uint32_t stream_id)
{
    if (stream == (void*)-1) return SBX_INVALID_ARGUMENT;
    if (!sbx::is_dtype(dtype, true)) return SBX_UNSUPPORTED;
    if (rows < 0 || cols < 0) return SBX_INVALID_ARGUMENT;
    if (rows > sbx::kMaxSide || cols > sbx::kMaxSide) return SBX_UNSUPPORTED;
    if (rows == 0 || cols == 0) return SBX_OK;
    const size_t elem = sbx::elem_size(dtype);
    sbx::DropoutArgs a;
    const int st = sbx::dropout_args(&a, X, ldx, gate, ldg, rows, cols, p, seed, stream_id, elem);
    if (st != SBX_OK) return st;
    if (sbx::bad_dense(Y, cols, ldy, elem)) return SBX_INVALID_ARGUMENT;
    return sbx::status_of(sbx::launch_dropout(dtype, a, Y, ldy, (hipStream_t)stream));
}

int sbx_mx4_quantize(void* stream, int dtype, int64_t rows, int64_t cols, const void* X,
                     int64_t ldx, const void* gate, int64_t ldg, double p, uint64_t seed,
                     uint32_t stream_id, void* P, int64_t ldp, void* S, int64_t lds, void* PT,
                     int64_t ldpt, void* ST, int64_t ldst)
{
    if (stream == (void*)-1) return SBX_INVALID_ARGUMENT;
    if (!sbx::is_dtype(dtype, false)) return SBX_UNSUPPORTED;
    if (rows < 0 || cols < 0) return SBX_INVALID_ARGUMENT;
    if (rows > sbx::kMaxSide || cols > sbx::kMaxSide) return SBX_UNSUPPORTED;
    if (rows == 0 || cols == 0) return SBX_OK;
    sbx::DropoutArgs a;
    const int st = sbx::dropout_args(&a, X, ldx, gate, ldg, rows, cols, p, seed, stream_id,
                                     sbx::elem_size(dtype));
    if (st != SBX_OK) return st;
    const bool row = P || S, col = PT || ST;
    if (!row && !col) return SBX_INVALID_ARGUMENT;
    if (row && sbx::bad_mx4(P, ldp, S, lds, rows, cols)) return SBX_INVALID_ARGUMENT;
    if (col && sbx::bad_mx4(PT, ldpt, ST, ldst, cols, rows)) return SBX_INVALID_ARGUMENT;
    const sbx::Mx4Out ro{(uint8_t*)P, ldp, (uint8_t*)S, lds}, co{(uint8_t*)PT, ldpt, (uint8_t*)ST, ldst};
    return sbx::status_of(sbx::launch_mx4_quantize(dtype, a, ro, co, (hipStream_t)stream));
}

int sbx_mx4_dequantize(void* stream, int dtype, int64_t rows, int64_t cols, const void* P,
                       int64_t ldp, const void* S, int64_t lds, void* Y, int64_t ldy)
{
    if (stream == (void*)-1) return SBX_INVALID_ARGUMENT;
    if (!sbx::is_dtype(dtype, false)) return SBX_UNSUPPORTED;
    if (rows < 0 || cols < 0) return SBX_INVALID_ARGUMENT;
    if (rows > sbx::kMaxSide || cols > sbx::kMaxSide) return SBX_UNSUPPORTED;
    if (rows == 0 || cols == 0) return SBX_OK;
    if (sbx::bad_mx4(P, ldp, S, lds, rows, cols)) return SBX_INVALID_ARGUMENT;
    if (sbx::bad_dense(Y, cols, ldy, sbx::elem_size(dtype))) return SBX_INVALID_ARGUMENT;
    return sbx::status_of(sbx::launch_mx4_dequantize(dtype, rows, cols, (const uint8_t*)P, ldp,
                                                     (const uint8_t*)S, lds, Y, ldy,
                                                     (hipStream_t)stream));
}

int sbx_mx4_gemm(void* stream, int dtype, int layout, int64_t m, int64_t n, int64_t k, float alpha,
                 const void* A, int64_t lda, const void* SA, int64_t ldsa, const void* B,
                 int64_t ldb, const void* SB, int64_t ldsb, float beta, void* C, int64_t ldc,
                 int epilogue)
{
    if (stream == (void*)-1) return SBX_INVALID_ARGUMENT;
    if (!sbx::is_dtype(dtype, false)) return SBX_UNSUPPORTED;
    if (epilogue != SBX_EPILOGUE_NONE && epilogue != SBX_EPILOGUE_RELU) return SBX_INVALID_ARGUMENT;
    if (layout != 0 && layout != 1) return SBX_INVALID_ARGUMENT;
    if (m < 0 || n < 0 || k < 0) return SBX_INVALID_ARGUMENT;
    if (m > sbx::kMaxSide || n > sbx::kMaxSide || k > sbx::kMaxTerms) return SBX_UNSUPPORTED;
    if (m == 0 || n == 0) return SBX_OK;
    if (sbx::bad_dense(C, layout == 0 ? n : m, ldc, sbx::elem_size(dtype))) return SBX_INVALID_ARGUMENT;
    if (alpha == 0.0f) k = 0;  // A and B are not read
    if (k > 0) {
        if (sbx::bad_mx4(A, lda, SA, ldsa, m, k) || sbx::bad_mx4(B, ldb, SB, ldsb, n, k))
            return SBX_INVALID_ARGUMENT;
        if (lda > sbx::kMaxRowBytes || ldb > sbx::kMaxRowBytes) return SBX_UNSUPPORTED;
    }
    sbx::Mx4GemmArgs a;
    a.A = (const uint8_t*)A; a.lda = lda; a.SA = (const uint8_t*)SA; a.ldsa = ldsa;
    a.B = (const uint8_t*)B; a.ldb = ldb; a.SB = (const uint8_t*)SB; a.ldsb = ldsb;
    a.C = C; a.ldc = ldc;
    a.m = (int)m; a.n = (int)n; a.k = (int)k;
    a.alpha = alpha; a.beta = beta;
    a.relu = epilogue == SBX_EPILOGUE_RELU;
    a.past = ((uintptr_t)C | (uint64_t)ldc * sbx::elem_size(dtype)) % 64 == 0;
    a.down = dtype == SBX_F32 && ((uintptr_t)C | (uint64_t)ldc * 4) % 16 != 0 &&
             ldc <= (32 << 20) / (layout == 0 ? m : n);
    if (layout == 1) {  // column-major C (m x n) is row-major C^T = B * A^T
        const uint8_t *t = a.A, *ts = a.SA;
        a.A = a.B; a.SA = a.SB; a.B = t; a.SB = ts;
        const int64_t l = a.lda, ls = a.ldsa;
        a.lda = a.ldb; a.ldsa = a.ldsb; a.ldb = l; a.ldsb = ls;
        a.m = (int)n; a.n = (int)m;
    }
    return sbx::status_of(sbx::launch_mx4_gemm(dtype, a, (hipStream_t)stream));
}

}  // extern "C"
