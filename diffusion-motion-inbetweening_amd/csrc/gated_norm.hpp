// Arguments of the gated-norm kernels (gated_norm.hip), filled by the C entries in api_ops.hip after their checks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cmdi {

struct Rows {               // [batch, seq] rows of `dim` contiguous elements
    const void* p = nullptr;
    int64_t bs = 0, ss = 0; // elements between samples / between rows
};
struct NormParam {          // one row for all samples (bs == 0) or one for each
    const void* p = nullptr;
    int64_t bs = 0;
};

struct GatedNormArgs {
    int32_t batch, seq, dim;
    int32_t dtype, param_dtype, post, pre;
    float alpha, eps;
    Rows x, y, gr, gh;                       // gr, gh: gradients of r and h (vjp)
    NormParam gate, scale, shift;
    const void *w, *b, *wp, *bp;             // N_pre's weight and bias, N_post's
    void *r, *h;                             // forward: contiguous outputs
    void *gx, *gy;                           // vjp: contiguous outputs, either may be null
    void *g_gate, *g_scale, *g_shift, *g_w, *g_b, *g_wp, *g_bp;
    float* work;                             // vjp: partial column sums
    // split of the rows (gated_norm_plan)
    int64_t groups, rows_per_group, chunks, rows_per_chunk;
    uint32_t first = 0;                      // block or (joins) group that the launch's first block takes
    int32_t span;                            // vjp: teams take whole samples (many short ones); rows_per_chunk = samples a team
    int32_t slots;                           // column sums kept: bit 0 sum dh, 1 sum dh n, 2 sum dr ny, 3 sum dr (span: times 1 + s, g)
};

constexpr int kGatedNormMaxDim = 16384;

void gated_norm_plan(GatedNormArgs& a, bool vjp);         // (at least one row)
int64_t gated_norm_work_floats(const GatedNormArgs& a);   // after gated_norm_plan(a, true)
hipError_t launch_gated_norm_fwd(const GatedNormArgs& a, hipStream_t stream);
hipError_t launch_gated_norm_vjp(const GatedNormArgs& a, hipStream_t stream);

}  // namespace cmdi
