// C-ABI of libcondmdi_hip.so, block operators: argument checks of the gated norms, the 8-bit linear layer and shared-prefix
// attention, then one call of the kernels' launchers.  Nothing here allocates, synchronises or throws.
#include <cmath>

#include "common.hpp"
#include "engine.hpp"
#include "gated_norm.hpp"
#include "linear_i8.hpp"
#include "prefix_attention.hpp"

using namespace cmdi;
using namespace cmdi::host;

namespace {

int dt_bytes(int dt) { return dt == CMDI_DT_F32 ? 4 : 2; }
bool dt_known(int dt) { return dt == CMDI_DT_F32 || dt == CMDI_DT_BF16 || dt == CMDI_DT_F16; }
bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool at_elem(const void* p, int dt) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(dt_bytes(dt) - 1)) == 0; }

// Blocks of a launch of the 8-bit and attention kernels, 256 or 512 threads each (threads of a launch stay below 2^32); the norms'
// kernels go out in as many launches as their blocks need (launches.hpp).
constexpr int64_t kMaxBlocks = (int64_t)1 << 22;

int norm_args(const cmdi_gated_norm_desc* d, const cmdi_gated_norm_grads* g, GatedNormArgs& a) {
    if (!d) return fail(CMDI_E_INVALID, "null descriptor");
    if (d->batch < 0 || d->seq < 0 || (int64_t)d->batch * d->seq >= ((int64_t)1 << 31)) return fail(CMDI_E_INVALID, "batch * seq must lie in [0, 2^31)");
    if (d->dim < 1 || d->dim > kGatedNormMaxDim) return fail(CMDI_E_INVALID, "dim must lie in [1, 16384]");
    if (!dt_known(d->dtype)) return fail(CMDI_E_INVALID, "dtype must be CMDI_DT_F32, CMDI_DT_BF16 or CMDI_DT_F16");
    if (d->param_dtype != CMDI_DT_F32 && d->param_dtype != d->dtype) return fail(CMDI_E_INVALID, "param_dtype must be CMDI_DT_F32 or dtype");
    if (d->post < CMDI_NORM_NONE || d->post > CMDI_NORM_LAYER) return fail(CMDI_E_INVALID, "post must be CMDI_NORM_NONE, CMDI_NORM_RMS or CMDI_NORM_LAYER");
    if (d->pre != CMDI_NORM_RMS && d->pre != CMDI_NORM_LAYER) return fail(CMDI_E_INVALID, "pre must be CMDI_NORM_RMS or CMDI_NORM_LAYER");
    if (!(d->eps > 0.f) || !std::isfinite(d->eps)) return fail(CMDI_E_INVALID, "eps must be positive and finite");
    if (!std::isfinite(d->residual_scale)) return fail(CMDI_E_INVALID, "residual_scale must be finite");
    const bool some = d->batch > 0 && d->seq > 0;
    if (some && !d->d_x) return fail(CMDI_E_INVALID, "null x");
    if (!d->d_y && (d->post != CMDI_NORM_NONE || d->d_gate)) return fail(CMDI_E_INVALID, "post and gate need y");
    if (d->post == CMDI_NORM_NONE && (d->d_post_weight || d->d_post_bias)) return fail(CMDI_E_INVALID, "post_weight and post_bias need post");
    const int64_t strides[] = {d->x_stride[0], d->x_stride[1], d->y_stride[0], d->y_stride[1], d->gate_stride, d->scale_stride, d->shift_stride};
    for (int64_t s : strides)
        if (s < 0) return fail(CMDI_E_INVALID, "negative stride");
    const void* rows[] = {d->d_x, d->d_y, g ? g->d_gr : nullptr, g ? g->d_gh : nullptr, g ? g->d_gx : nullptr, g ? g->d_gy : nullptr};
    const void* params[] = {d->d_gate, d->d_scale, d->d_shift, d->d_weight, d->d_bias, d->d_post_weight, d->d_post_bias};
    for (const void* p : rows)
        if (!at_elem(p, d->dtype)) return fail(CMDI_E_INVALID, "a tensor is not aligned to its element");
    for (const void* p : params)
        if (!at_elem(p, d->param_dtype)) return fail(CMDI_E_INVALID, "a parameter is not aligned to its element");
    a.batch = d->batch; a.seq = d->seq; a.dim = d->dim;
    a.dtype = d->dtype; a.param_dtype = d->param_dtype; a.post = d->post; a.pre = d->pre;
    a.alpha = d->residual_scale; a.eps = d->eps;
    a.x = Rows{d->d_x, d->x_stride[0], d->x_stride[1]};
    a.y = Rows{d->d_y, d->y_stride[0], d->y_stride[1]};
    a.gate = NormParam{d->d_gate, d->gate_stride};
    a.scale = NormParam{d->d_scale, d->scale_stride};
    a.shift = NormParam{d->d_shift, d->shift_stride};
    a.w = d->d_weight; a.b = d->d_bias; a.wp = d->d_post_weight; a.bp = d->d_post_bias;
    if (g) {
        for (int64_t s : {g->gr_stride[0], g->gr_stride[1], g->gh_stride[0], g->gh_stride[1]})
            if (s < 0) return fail(CMDI_E_INVALID, "negative stride");
        a.gr = Rows{g->d_gr, g->gr_stride[0], g->gr_stride[1]};
        a.gh = Rows{g->d_gh, g->gh_stride[0], g->gh_stride[1]};
        a.gx = g->d_gx; a.gy = g->d_gy;
        a.g_gate = g->d_ggate; a.g_scale = g->d_gscale; a.g_shift = g->d_gshift;
        a.g_w = g->d_gweight; a.g_b = g->d_gbias; a.g_wp = g->d_gpost_weight; a.g_bp = g->d_gpost_bias;
        if ((a.gy || a.g_gate || a.g_wp || a.g_bp) && !d->d_y) return fail(CMDI_E_INVALID, "gradients of y, gate and the post norm need y");
        if ((a.g_gate && !d->d_gate) || (a.g_scale && !d->d_scale) || (a.g_shift && !d->d_shift) || (a.g_w && !d->d_weight) ||
            (a.g_b && !d->d_bias) || (a.g_wp && !d->d_post_weight) || (a.g_bp && !d->d_post_bias))
            return fail(CMDI_E_INVALID, "gradient wanted of a parameter that is not there");
    }
    return CMDI_OK;
}

int prefix_args(const cmdi_prefix_attention_desc* d, PrefixAttnArgs& a) {
    if (!d) return fail(CMDI_E_INVALID, "null descriptor");
    if (d->batch < 0 || d->queries < 0 || d->prefix < 0 || d->own_max < 0) return fail(CMDI_E_INVALID, "negative size");
    if (d->heads < 1 || d->kv_heads < 1 || d->heads % d->kv_heads != 0) return fail(CMDI_E_INVALID, "heads must be a positive multiple of kv_heads");
    if (d->dim != 64 && d->dim != 128) return fail(CMDI_E_INVALID, "dim must be 64 or 128");
    if (d->dtype != CMDI_DT_BF16 && d->dtype != CMDI_DT_F16) return fail(CMDI_E_INVALID, "dtype must be CMDI_DT_BF16 or CMDI_DT_F16");
    if (!(d->scale > 0.f) || !std::isfinite(d->scale)) return fail(CMDI_E_INVALID, "scale must be positive and finite");
    const int64_t lim = (int64_t)1 << 31;
    if (d->batch > 0 && d->queries > 0 && (int64_t)d->batch * d->queries >= lim / d->heads) return fail(CMDI_E_INVALID, "batch * queries * heads must stay below 2^31");
    if ((int64_t)d->prefix + d->own_max >= lim - 4096) return fail(CMDI_E_INVALID, "prefix + own_max must stay below 2^31 - 4096");
    const bool some = d->batch > 0 && d->queries > 0;
    if (some && !d->d_q) return fail(CMDI_E_INVALID, "null q");
    if (some && d->prefix > 0 && (!d->d_prefix_k || !d->d_prefix_v)) return fail(CMDI_E_INVALID, "null prefix");
    if (some && d->own_max > 0 && (!d->d_own_k || !d->d_own_v)) return fail(CMDI_E_INVALID, "null own keys or values");
    const void* at[] = {d->d_q, d->d_prefix_k, d->d_prefix_v, d->d_own_k, d->d_own_v};
    for (const void* p : at)
        if (!at16(p)) return fail(CMDI_E_INVALID, "q, keys and values must be 16-byte aligned");
    const int64_t strides[] = {d->q_stride[0], d->q_stride[1], d->q_stride[2], d->prefix_k_stride[0], d->prefix_k_stride[1], d->prefix_v_stride[0],
                               d->prefix_v_stride[1], d->own_k_stride[0], d->own_k_stride[1], d->own_k_stride[2], d->own_v_stride[0],
                               d->own_v_stride[1], d->own_v_stride[2]};
    for (int64_t s : strides)
        if (s < 0 || s % 8 != 0) return fail(CMDI_E_INVALID, "strides must be non-negative multiples of 8 elements");
    const int64_t tokens[] = {d->prefix_k_stride[0], d->prefix_v_stride[0], d->own_k_stride[1], d->own_v_stride[1]};
    for (int64_t s : tokens)
        if (s > ((int64_t)1 << 23)) return fail(CMDI_E_INVALID, "token strides of keys and values must be at most 2^23 elements");
    a.q = d->d_q; a.pk = d->d_prefix_k; a.pv = d->d_prefix_v; a.ok = d->d_own_k; a.ov = d->d_own_v;
    a.q_bs = d->q_stride[0]; a.q_ss = d->q_stride[1]; a.q_hs = d->q_stride[2];
    a.pk_ss = d->prefix_k_stride[0]; a.pk_hs = d->prefix_k_stride[1];
    a.pv_ss = d->prefix_v_stride[0]; a.pv_hs = d->prefix_v_stride[1];
    a.ok_bs = d->own_k_stride[0]; a.ok_ss = d->own_k_stride[1]; a.ok_hs = d->own_k_stride[2];
    a.ov_bs = d->own_v_stride[0]; a.ov_ss = d->own_v_stride[1]; a.ov_hs = d->own_v_stride[2];
    a.own_len = d->d_own_len;
    a.batch = d->batch; a.queries = d->queries; a.heads = d->heads; a.kv_heads = d->kv_heads; a.dim = d->dim;
    a.prefix = d->prefix; a.own_max = d->own_max; a.causal = d->causal != 0; a.dtype = d->dtype; a.scale = d->scale;
    return CMDI_OK;
}

int64_t prefix_blocks(const PrefixAttnArgs& a, const PrefixAttnPlan& p) {
    int64_t most = 0;
    for (int i = 0; i < p.n; ++i) {
        const int64_t n = (int64_t)(p.l[i].packed ? 1 : a.batch) * a.kv_heads * p.l[i].tiles * p.l[i].chunks;
        most = n > most ? n : most;
    }
    return most;
}

// argument checks of the product, then (go) its launch
int gemm_i8_checked(const void* d_a, const float* d_a_scale, const void* d_w, const float* d_w_scale, const float* d_bias, const void* d_resid,
                 void* d_c, int32_t m, int32_t n, int32_t k, int64_t lda, int64_t ldw, int64_t ldc, int64_t ldr, int32_t dtype, int32_t epi,
                 cmdi_stream stream, bool go) {
    if (!dt_known(dtype)) return fail(CMDI_E_INVALID, "dtype must be CMDI_DT_F32, CMDI_DT_BF16 or CMDI_DT_F16");
    if (epi != 0 && epi != 1 && epi != 3) return fail(CMDI_E_INVALID, "epi must be 0 (bias), 1 (bias+gelu) or 3 (bias+residual)");
    if (m < 0 || n < 1 || k < kI8KAlign || k % kI8KAlign != 0 || k > kI8MaxK) return fail(CMDI_E_INVALID, "m >= 0, n >= 1, k a multiple of 128 up to 130048");
    if (lda < k || ldw < k || lda % 16 != 0 || ldw % 16 != 0 || lda > (1 << 22) || ldw > (1 << 22))
        return fail(CMDI_E_INVALID, "lda and ldw must be multiples of 16 from k to 2^22");
    if (ldc < n || (epi == 3 && ldr < n)) return fail(CMDI_E_INVALID, "ldc and ldr must be at least n");
    if (m == 0) return CMDI_OK;
    if (!d_a || !d_a_scale || !d_w || !d_w_scale || !d_c) return fail(CMDI_E_INVALID, "null tensor");
    if (epi == 3 && !d_resid) return fail(CMDI_E_INVALID, "residual epilogue needs d_resid");
    if (!at16(d_a) || !at16(d_w)) return fail(CMDI_E_INVALID, "a and w must be 16-byte aligned");
    if (!at_elem(d_c, dtype) || !at_elem(d_resid, dtype) || !at_elem(d_a_scale, CMDI_DT_F32) || !at_elem(d_w_scale, CMDI_DT_F32) || !at_elem(d_bias, CMDI_DT_F32))
        return fail(CMDI_E_INVALID, "a tensor is not aligned to its element");
    // (up to 16 rows have four blocks where others have a tile)
    if (((int64_t)m + 63) / 64 * (((int64_t)n + 63) / 64) >= kMaxBlocks) return fail(CMDI_E_INVALID, "m * n: 2^22 tiles of 64 x 64 or more");
    GemmI8Args p{static_cast<const int8_t*>(d_a), static_cast<const int8_t*>(d_w), d_a_scale, d_w_scale, d_bias, epi == 3 ? d_resid : nullptr, d_c,
                 m, n, k, lda, ldw, ldc, ldr, dtype, epi};
    if (!go) return CMDI_OK;
    HIPCHK(launch_gemm_i8(p, static_cast<hipStream_t>(stream)));
    return CMDI_OK;
}

int quant_checked(const void* d_x, int32_t dtype, int64_t rows, int32_t cols, int64_t ld, void* d_q, int32_t kp, float* d_scale, cmdi_stream stream,
                  bool go) {
    if (!dt_known(dtype)) return fail(CMDI_E_INVALID, "dtype must be CMDI_DT_F32, CMDI_DT_BF16 or CMDI_DT_F16");
    if (rows < 0 || rows > kMaxBlocks || cols < 1 || ld < 0) return fail(CMDI_E_INVALID, "rows must lie in [0, 2^22], cols be positive, ld not negative");
    if (kp < cols || kp % kI8KAlign != 0 || kp > kI8MaxK) return fail(CMDI_E_INVALID, "kp must be a multiple of 128 from cols to 130048");
    if (rows == 0) return CMDI_OK;
    if (!d_x || !d_q || !d_scale) return fail(CMDI_E_INVALID, "null tensor");
    if (!at16(d_q) || !at_elem(d_x, dtype) || !at_elem(d_scale, CMDI_DT_F32)) return fail(CMDI_E_INVALID, "q must be 16-byte aligned, x and scale to their elements");
    if (!go) return CMDI_OK;
    QuantRowsArgs a{d_x, rows, ld, cols, dtype, static_cast<int8_t*>(d_q), kp, d_scale};
    HIPCHK(launch_quant_rows_i8(a, static_cast<hipStream_t>(stream)));
    return CMDI_OK;
}

}  // namespace

extern "C" {

int cmdi_gated_norm_fwd(const cmdi_gated_norm_desc* d, void* d_r, void* d_h, cmdi_stream stream) {
    GatedNormArgs a{};
    if (int rc = norm_args(d, nullptr, a)) return rc;
    if (a.batch == 0 || a.seq == 0) return CMDI_OK;
    if (!d_h) return fail(CMDI_E_INVALID, "null h");
    if (!at_elem(d_r, a.dtype) || !at_elem(d_h, a.dtype)) return fail(CMDI_E_INVALID, "an output is not aligned to its element");
    a.r = d_r; a.h = d_h;
    gated_norm_plan(a, false);
    HIPCHK(launch_gated_norm_fwd(a, static_cast<hipStream_t>(stream)));
    return CMDI_OK;
}

int64_t cmdi_gated_norm_vjp_workspace(const cmdi_gated_norm_desc* d, const cmdi_gated_norm_grads* g) {
    GatedNormArgs a{};
    if (!g) return fail(CMDI_E_INVALID, "null gradients");
    if (int rc = norm_args(d, g, a)) return rc;
    if (a.batch == 0 || a.seq == 0) return 0;
    gated_norm_plan(a, true);
    return gated_norm_work_floats(a) * (int64_t)sizeof(float);
}

int cmdi_gated_norm_vjp(const cmdi_gated_norm_desc* d, const cmdi_gated_norm_grads* g, cmdi_stream stream) {
    GatedNormArgs a{};
    if (!g) return fail(CMDI_E_INVALID, "null gradients");
    if (int rc = norm_args(d, g, a)) return rc;
    if (a.batch == 0 || a.seq == 0)
        return a.g_gate || a.g_scale || a.g_shift || a.g_w || a.g_b || a.g_wp || a.g_bp ? fail(CMDI_E_INVALID, "no rows: parameter gradients are the caller's zeros")
                                                                                         : CMDI_OK;
    gated_norm_plan(a, true);
    const int64_t need = gated_norm_work_floats(a) * (int64_t)sizeof(float);
    if (need > 0 && (!g->d_work || g->work_bytes < need)) return fail(CMDI_E_INVALID, "workspace too small (cmdi_gated_norm_vjp_workspace)");
    if (!at_elem(g->d_work, CMDI_DT_F32)) return fail(CMDI_E_INVALID, "workspace is not aligned");
    a.work = static_cast<float*>(g->d_work);
    HIPCHK(launch_gated_norm_vjp(a, static_cast<hipStream_t>(stream)));
    return CMDI_OK;
}

int cmdi_quant_rows_i8(const void* d_x, int32_t dtype, int64_t rows, int32_t cols, int64_t ld, void* d_q, int32_t kp, float* d_scale,
                       cmdi_stream stream) {
    return quant_checked(d_x, dtype, rows, cols, ld, d_q, kp, d_scale, stream, true);
}

int cmdi_gemm_i8(const void* d_a, const float* d_a_scale, const void* d_w, const float* d_w_scale, const float* d_bias, const void* d_resid,
                 void* d_c, int32_t m, int32_t n, int32_t k, int64_t lda, int64_t ldw, int64_t ldc, int64_t ldr, int32_t dtype, int32_t epi,
                 cmdi_stream stream) {
    return gemm_i8_checked(d_a, d_a_scale, d_w, d_w_scale, d_bias, d_resid, d_c, m, n, k, lda, ldw, ldc, ldr, dtype, epi, stream, true);
}

int cmdi_linear_i8(const void* d_x, int32_t dtype, int32_t m, int32_t cols, int64_t ldx, const void* d_w, const float* d_w_scale,
                   const float* d_bias, const void* d_resid, void* d_c, int32_t n, int32_t kp, int64_t ldw, int64_t ldc, int64_t ldr,
                   int32_t epi, void* d_work, int64_t work_bytes, cmdi_stream stream) {
    if (m < 0 || cols < 1 || kp != (int64_t)(cols + (int64_t)kI8KAlign - 1) / kI8KAlign * kI8KAlign)
        return fail(CMDI_E_INVALID, "m >= 0, cols >= 1, kp = cols rounded up to 128");
    if (m > 0 && (!d_work || !at16(d_work) || work_bytes < (int64_t)m * (kp + 4)))
        return fail(CMDI_E_INVALID, "workspace must be 16-byte aligned and hold m * (kp + 4) bytes");
    int8_t* q = static_cast<int8_t*>(d_work);
    float* scale = reinterpret_cast<float*>(q + (int64_t)m * kp);
    // the checks of both halves first (m = 0: they need no tensors), so that a refused call has launched nothing
    if (int rc = gemm_i8_checked(q, scale, d_w, d_w_scale, d_bias, d_resid, d_c, m, n, kp, kp, ldw, ldc, ldr, dtype, epi, nullptr, false)) return rc;
    if (int rc = quant_checked(d_x, dtype, m, cols, ldx, q, kp, scale, nullptr, false)) return rc;
    if (m == 0) return CMDI_OK;
    if (linear_i8_fused(m, n, kp, dtype)) {
        const QuantRowsArgs x{d_x, m, ldx, cols, dtype, nullptr, kp, nullptr};
        const GemmI8Args p{nullptr, static_cast<const int8_t*>(d_w), nullptr, d_w_scale, d_bias, epi == 3 ? d_resid : nullptr, d_c,
                           m, n, kp, kp, ldw, ldc, ldr, dtype, epi};
        HIPCHK(launch_linear_i8_fused(x, p, static_cast<hipStream_t>(stream)));
        return CMDI_OK;
    }
    if (int rc = quant_checked(d_x, dtype, m, cols, ldx, q, kp, scale, stream, true)) return rc;
    return gemm_i8_checked(q, scale, d_w, d_w_scale, d_bias, d_resid, d_c, m, n, kp, kp, ldw, ldc, ldr, dtype, epi, stream, true);
}

int64_t cmdi_prefix_attention_workspace(const cmdi_prefix_attention_desc* d) {
    PrefixAttnArgs a{};
    if (int rc = prefix_args(d, a)) return rc;
    if (a.batch == 0 || a.queries == 0) return 0;
    return prefix_attention_work_floats(a, prefix_attention_plan(a, device_cu_count())) * (int64_t)sizeof(float);
}

int cmdi_prefix_attention(const cmdi_prefix_attention_desc* d, void* d_out, float* d_lse, void* d_work, int64_t work_bytes, cmdi_stream stream) {
    PrefixAttnArgs a{};
    if (int rc = prefix_args(d, a)) return rc;
    if (a.batch == 0 || a.queries == 0) return CMDI_OK;
    if (!d_out || !at16(d_out)) return fail(CMDI_E_INVALID, "out must be there and 16-byte aligned");
    if (!at_elem(d_lse, CMDI_DT_F32)) return fail(CMDI_E_INVALID, "lse is not aligned");
    const PrefixAttnPlan plan = prefix_attention_plan(a, device_cu_count());
    // (the join takes four rows a block)
    if (prefix_blocks(a, plan) > kMaxBlocks || (plan.slots > 1 && (int64_t)a.batch * a.queries * a.heads > 4 * kMaxBlocks)) return fail(CMDI_E_INVALID, "batch * heads * queries too large");
    const int64_t need = prefix_attention_work_floats(a, plan) * (int64_t)sizeof(float);
    if (need > 0 && (!d_work || work_bytes < need)) return fail(CMDI_E_INVALID, "workspace too small (cmdi_prefix_attention_workspace)");
    if (!at16(d_work)) return fail(CMDI_E_INVALID, "workspace must be 16-byte aligned");
    a.out = d_out; a.lse = d_lse; a.work = static_cast<float*>(d_work);
    HIPCHK(launch_prefix_attention(a, plan, static_cast<hipStream_t>(stream)));
    return CMDI_OK;
}

}  // extern "C"
