// Arguments of the 8-bit linear layer's kernels (linear_i8.hip), filled by the C entries in api_ops.hip after their checks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cmdi {

constexpr int kI8KAlign = 128;   // columns of a quantised row: padded with zeros to this
constexpr int kI8MaxK = 130048;  // 127 * 127 * K (and 128 * 128 * K) stays below 2^31

struct QuantRowsArgs {
    const void* x;
    int64_t rows, ld;            // ld: elements between rows
    int32_t cols, dtype;
    int8_t* q;                   // [rows][kp]
    int32_t kp;
    float* scale;                // [rows]
};
hipError_t launch_quant_rows_i8(const QuantRowsArgs& a, hipStream_t stream);

struct GemmI8Args {
    const int8_t *a, *w;         // [m][lda], [n][ldw], k columns each
    const float *a_scale, *w_scale, *bias;
    const void* resid;           // [m][ldr] of the output's type, or null
    void* c;                     // [m][ldc]
    int32_t m, n, k;
    int64_t lda, ldw, ldc, ldr;
    int32_t dtype, epi;          // epi: 0 bias, 1 bias + GELU, 3 bias + residual
};
hipError_t launch_gemm_i8(const GemmI8Args& a, hipStream_t stream);

// Few rows: quantising and product in one launch (p.a and p.a_scale are not read).
constexpr int kI8FusedBytes = 65536;   // bytes of the activations, their rows rounded up to a power of two
bool linear_i8_fused(int m, int n, int kp, int dtype);
hipError_t launch_linear_i8_fused(const QuantRowsArgs& x, const GemmI8Args& p, hipStream_t stream);

}  // namespace cmdi
