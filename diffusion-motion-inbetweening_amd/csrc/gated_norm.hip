// The norms around a block with its gate and residual scale, and their gradients.
//
//   m = N_post(y) wp + bp          N: v -> v / sqrt(mean v^2 + eps)  (rms), the same of v - mean v  (layer), or v  (none)
//   r = alpha x + g m              the residual stream behind the block
//   n = N_pre(r),  u = n w + b
//   h = u (1 + s) + t              the next block's input
//
// Backward, with dh, dr' the gradients of h and r, k = 1 / sqrt(.. + eps) of a norm and <.> the mean over a row:
//   dn = dh (1 + s) w              dr = dr' + k_pre (dn - n <dn n> - [layer] <dn>)        dx = alpha dr
//   dm = dr g                      dy = k_post (dm wp - ny <dm wp ny> - [layer] <dm wp>)
// and every gradient of a parameter follows from FOUR column sums over the rows of a sample
//   A = sum dh,  N = sum dh n,  P = sum dr ny,  Q = sum dr:
//   ds = w N + b A,  dt = A,  dg = wp P + bp Q,  dw = sum_b (1 + s) N,  db = sum_b (1 + s) A,  dwp = sum_b g P,  dbp = sum_b g Q,
// because s, t, g are constant along a sample.  So the pass over the rows adds four numbers a column in registers, writes them
// once per block, and two small kernels join them in a fixed order: no atomics, the same bits every run.
//
// Bound by memory: forward reads x, y and writes r, h; backward reads x, y, dr', dh and writes dx, dy (r is computed again from
// x and y, unrounded, which costs no more reads than r itself would).  A row stays in the registers of its team of lanes, so the
// variance is taken of the centred values at no extra reads.
#include "gated_norm.hpp"

#include <type_traits>

#include "../../include/condmdi.h"
#include "ops_common.hpp"

namespace cmdi {
namespace {

// A team of TEAM lanes holds one row: element (c * TEAM + lane) * W + i, c < NV.  TEAM = 64: the row's sums never leave the wave;
// wider teams are whole blocks and join their waves through LDS, one barrier a sum (two slots in turn).
template <int TEAM>
struct TeamSum {
    float* lds;      // [2][2][TEAM / 64]
    int slot = 0;
    __device__ __forceinline__ explicit TeamSum(float* l) : lds(l) {}
    __device__ __forceinline__ void two(float& a, float& b) {
        a = wave_total(a);
        b = wave_total(b);
        if constexpr (TEAM > 64) {
            constexpr int NW = TEAM / 64;
            float* at = lds + slot * 2 * NW;
            slot ^= 1;
            if ((threadIdx.x & 63) == 0) {
                at[threadIdx.x >> 6] = a;
                at[NW + (threadIdx.x >> 6)] = b;
            }
            __syncthreads();
            a = 0.f;
            b = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) { a += at[i]; b += at[NW + i]; }
        }
    }
    __device__ __forceinline__ float one(float a) {
        a = wave_total(a);
        if constexpr (TEAM > 64) {
            constexpr int NW = TEAM / 64;
            float* at = lds + slot * 2 * NW;
            slot ^= 1;
            if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = a;
            __syncthreads();
            a = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) a += at[i];
        }
        return a;
    }
};

template <int W, int NV>
struct Row { float v[NV][W]; };

template <class T, int W, int TEAM, int NV>
__device__ __forceinline__ void load_row(Row<W, NV>& r, const T* p, int lane, int dim) {
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int e = (c * TEAM + lane) * W;
        if (e < dim) {
            load_vec<T, W>(p + e, r.v[c]);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) r.v[c][i] = 0.f;
        }
    }
}
template <class T, int W, int TEAM, int NV>
__device__ __forceinline__ void store_row(T* p, const Row<W, NV>& r, int lane, int dim) {
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int e = (c * TEAM + lane) * W;
        if (e < dim) store_vec<T, W>(p + e, r.v[c]);
    }
}
// a parameter row, or `fill` where there is none (columns behind `dim` hold 0)
template <class P, int W, int TEAM, int NV>
__device__ __forceinline__ void load_param_as(Row<W, NV>& r, const P* p, int lane, int dim, bool vec) {
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int e = (c * TEAM + lane) * W;
        if (vec && e < dim) {
            load_vec<P, W>(p + e, r.v[c]);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) r.v[c][i] = e + i < dim ? Elem<P>::up(p[e + i]) : 0.f;
        }
    }
}
template <class T, int W, int TEAM, int NV>
__device__ __forceinline__ void load_param(Row<W, NV>& r, const void* p, int64_t off, float fill, const GatedNormArgs& a, int lane) {
    if (!p) {
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
            for (int i = 0; i < W; ++i) r.v[c][i] = (c * TEAM + lane) * W + i < a.dim ? fill : 0.f;
    } else if (a.param_dtype == CMDI_DT_F32) {
        load_param_as<float, W, TEAM, NV>(r, static_cast<const float*>(p) + off, lane, a.dim, a.pvec);
    } else {   // the entries allow 32 bits or the rows' own type
        load_param_as<T, W, TEAM, NV>(r, static_cast<const T*>(p) + off, lane, a.dim, a.pvec);
    }
}

// v <- N(v), returns k = 1 / sqrt(mean + eps).  Columns behind `dim` stay 0.
template <int W, int TEAM, int NV>
__device__ __forceinline__ float normalise(Row<W, NV>& r, int kind, const GatedNormArgs& a, float inv_dim, int lane, TeamSum<TEAM>& sum) {
    if (kind == CMDI_NORM_NONE) return 1.f;
    if (kind == CMDI_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
            for (int i = 0; i < W; ++i) s += r.v[c][i];
        const float mean = sum.one(s) * inv_dim;
#pragma unroll
        for (int c = 0; c < NV; ++c)
            if ((c * TEAM + lane) * W < a.dim) {
#pragma unroll
                for (int i = 0; i < W; ++i) r.v[c][i] -= mean;
            }
    }
    float q = 0.f;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int i = 0; i < W; ++i) q += r.v[c][i] * r.v[c][i];
    const float k = 1.f / sqrtf(sum.one(q) * inv_dim + a.eps);
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int i = 0; i < W; ++i) r.v[c][i] *= k;
    return k;
}

// row numbers stay below 2^31 (checked at the entry): one 32-bit division a row, offsets in 64 bits
__device__ __forceinline__ int64_t row_at(const Rows& t, unsigned row, unsigned seq) {
    const unsigned b = row / seq, s = row - b * seq;
    return (int64_t)b * t.bs + (int64_t)s * t.ss;
}

#define FOR_ROW(c, i) _Pragma("unroll") for (int c = 0; c < NV; ++c) _Pragma("unroll") for (int i = 0; i < W; ++i)

template <class T, int W, int TEAM, int NV>
__global__ __launch_bounds__(TEAM < 256 ? 256 : TEAM) void gated_norm_fwd_kernel(const GatedNormArgs a) {
    constexpr int BLOCK = TEAM < 256 ? 256 : TEAM, TPB = BLOCK / TEAM;
    __shared__ float lds[4 * (TEAM / 64)];
    TeamSum<TEAM> sum(lds);
    const int lane = threadIdx.x % TEAM, team = TPB == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / TEAM);
    const int64_t group = blockIdx.x / (unsigned)a.chunks, chunk = blockIdx.x % (unsigned)a.chunks;
    const int64_t total = (int64_t)a.batch * a.seq;
    const int64_t first = group * a.rows_per_group + chunk * a.rows_per_chunk;
    int64_t end = group * a.rows_per_group + (chunk + 1) * a.rows_per_chunk;
    if (end > (group + 1) * a.rows_per_group) end = (group + 1) * a.rows_per_group;
    if (end > total) end = total;
    const float inv_dim = 1.f / (float)a.dim;

    Row<W, NV> g, wp, bp, w, t;
    // h = n w (1 + s) + (b (1 + s) + t); r = alpha x + ny (wp g) + bp g
    load_param<T, W, TEAM, NV>(g, a.gate.p, group * a.gate.bs, 1.f, a, lane);
    load_param<T, W, TEAM, NV>(wp, a.wp, 0, 1.f, a, lane);
    load_param<T, W, TEAM, NV>(bp, a.bp, 0, 0.f, a, lane);
    load_param<T, W, TEAM, NV>(w, a.w, 0, 1.f, a, lane);
    load_param<T, W, TEAM, NV>(t, a.b, 0, 0.f, a, lane);
    FOR_ROW(c, i) { wp.v[c][i] *= g.v[c][i]; bp.v[c][i] *= g.v[c][i]; }
    load_param<T, W, TEAM, NV>(g, a.scale.p, group * a.scale.bs, 0.f, a, lane);
    FOR_ROW(c, i) { w.v[c][i] *= 1.f + g.v[c][i]; t.v[c][i] *= 1.f + g.v[c][i]; }
    load_param<T, W, TEAM, NV>(g, a.shift.p, group * a.shift.bs, 0.f, a, lane);
    FOR_ROW(c, i) t.v[c][i] += g.v[c][i];

    for (int64_t row0 = first; row0 < end; row0 += TPB) {
        const int64_t row = row0 + team;
        if (row >= end) break;                     // a whole wave (TEAM = 64) or never (TPB = 1)
        Row<W, NV> x, y;
        load_row<T, W, TEAM, NV>(x, static_cast<const T*>(a.x.p) + row_at(a.x, (unsigned)row, a.seq), lane, a.dim);
        if (a.y.p) {
            load_row<T, W, TEAM, NV>(y, static_cast<const T*>(a.y.p) + row_at(a.y, (unsigned)row, a.seq), lane, a.dim);
            normalise<W, TEAM, NV>(y, a.post, a, inv_dim, lane, sum);
            FOR_ROW(c, i) x.v[c][i] = a.alpha * x.v[c][i] + (y.v[c][i] * wp.v[c][i] + bp.v[c][i]);
        } else {
            FOR_ROW(c, i) x.v[c][i] *= a.alpha;
        }
        if (a.r) store_row<T, W, TEAM, NV>(static_cast<T*>(a.r) + row * a.dim, x, lane, a.dim);
        normalise<W, TEAM, NV>(x, a.pre, a, inv_dim, lane, sum);
        FOR_ROW(c, i) x.v[c][i] = x.v[c][i] * w.v[c][i] + t.v[c][i];
        store_row<T, W, TEAM, NV>(static_cast<T*>(a.h) + row * a.dim, x, lane, a.dim);
    }
}

template <class T, int W, int TEAM, int NV>
__global__ __launch_bounds__(TEAM < 256 ? 256 : TEAM) void gated_norm_vjp_kernel(const GatedNormArgs a) {
    constexpr int BLOCK = TEAM < 256 ? 256 : TEAM, TPB = BLOCK / TEAM;
    __shared__ float lds[4 * (TEAM / 64)];
    __shared__ float joined[TPB > 1 ? TEAM * NV * W : 1];
    TeamSum<TEAM> sum(lds);
    const int lane = threadIdx.x % TEAM, team = TPB == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / TEAM);
    const int64_t group = blockIdx.x / (unsigned)a.chunks, chunk = blockIdx.x % (unsigned)a.chunks;
    const int64_t total = (int64_t)a.batch * a.seq;
    const int64_t first = group * a.rows_per_group + chunk * a.rows_per_chunk;
    int64_t end = group * a.rows_per_group + (chunk + 1) * a.rows_per_chunk;
    if (end > (group + 1) * a.rows_per_group) end = (group + 1) * a.rows_per_group;
    if (end > total) end = total;
    const float inv_dim = 1.f / (float)a.dim;

    Row<W, NV> g, wp, bp, w;     // gate, N_post's weight and bias, w (1 + s)
    load_param<T, W, TEAM, NV>(w, a.w, 0, 1.f, a, lane);
    load_param<T, W, TEAM, NV>(g, a.scale.p, group * a.scale.bs, 0.f, a, lane);
    FOR_ROW(c, i) w.v[c][i] *= 1.f + g.v[c][i];
    load_param<T, W, TEAM, NV>(g, a.gate.p, group * a.gate.bs, 1.f, a, lane);
    load_param<T, W, TEAM, NV>(wp, a.wp, 0, 1.f, a, lane);
    load_param<T, W, TEAM, NV>(bp, a.bp, 0, 0.f, a, lane);

    Row<W, NV> sA, sN, sP, sQ;
    FOR_ROW(c, i) { sA.v[c][i] = 0.f; sN.v[c][i] = 0.f; sP.v[c][i] = 0.f; sQ.v[c][i] = 0.f; }

    for (int64_t row0 = first; row0 < end; row0 += TPB) {
        const int64_t row = row0 + team;
        if (row >= end) break;
        Row<W, NV> x, y, d;
        float ky = 1.f;
        load_row<T, W, TEAM, NV>(x, static_cast<const T*>(a.x.p) + row_at(a.x, (unsigned)row, a.seq), lane, a.dim);
        if (a.gh.p) {
            load_row<T, W, TEAM, NV>(d, static_cast<const T*>(a.gh.p) + row_at(a.gh, (unsigned)row, a.seq), lane, a.dim);
        } else {
            FOR_ROW(c, i) d.v[c][i] = 0.f;
        }
        if (a.y.p) {
            load_row<T, W, TEAM, NV>(y, static_cast<const T*>(a.y.p) + row_at(a.y, (unsigned)row, a.seq), lane, a.dim);
            ky = normalise<W, TEAM, NV>(y, a.post, a, inv_dim, lane, sum);
            FOR_ROW(c, i) x.v[c][i] = a.alpha * x.v[c][i] + (y.v[c][i] * wp.v[c][i] + bp.v[c][i]) * g.v[c][i];
        } else {
            FOR_ROW(c, i) { y.v[c][i] = 0.f; x.v[c][i] *= a.alpha; }
        }
        const float kr = normalise<W, TEAM, NV>(x, a.pre, a, inv_dim, lane, sum);     // x = n
        float m1 = 0.f, m2 = 0.f;
        FOR_ROW(c, i) {
            sA.v[c][i] += d.v[c][i];
            sN.v[c][i] += d.v[c][i] * x.v[c][i];
            d.v[c][i] *= w.v[c][i];                                                   // dn
            m1 += d.v[c][i];
            m2 += d.v[c][i] * x.v[c][i];
        }
        sum.two(m1, m2);
        m1 = a.pre == CMDI_NORM_LAYER ? m1 * inv_dim : 0.f;
        m2 *= inv_dim;
        FOR_ROW(c, i) d.v[c][i] = kr * (d.v[c][i] - x.v[c][i] * m2 - m1);
        if (a.gr.p) {
            load_row<T, W, TEAM, NV>(x, static_cast<const T*>(a.gr.p) + row_at(a.gr, (unsigned)row, a.seq), lane, a.dim);
            FOR_ROW(c, i) d.v[c][i] += x.v[c][i];                                     // dr
        }
        if (a.gx) {
            FOR_ROW(c, i) x.v[c][i] = a.alpha * d.v[c][i];
            store_row<T, W, TEAM, NV>(static_cast<T*>(a.gx) + row * a.dim, x, lane, a.dim);
        }
        if (a.y.p) {
            m1 = 0.f;
            m2 = 0.f;
            FOR_ROW(c, i) {
                // columns behind `dim` (only the last chunk has them) hold -kr m1 in d; their weights are 0
                sP.v[c][i] += d.v[c][i] * y.v[c][i];
                sQ.v[c][i] += d.v[c][i];
                d.v[c][i] *= g.v[c][i] * wp.v[c][i];
                m1 += d.v[c][i];
                m2 += d.v[c][i] * y.v[c][i];
            }
            if (a.gy) {
                if (a.post != CMDI_NORM_NONE) {
                    sum.two(m1, m2);
                    m1 = a.post == CMDI_NORM_LAYER ? m1 * inv_dim : 0.f;
                    m2 *= inv_dim;
                    FOR_ROW(c, i) d.v[c][i] = ky * (d.v[c][i] - y.v[c][i] * m2 - m1);
                }
                store_row<T, W, TEAM, NV>(static_cast<T*>(a.gy) + row * a.dim, d, lane, a.dim);
            }
        }
    }
    // the block's column sums: teams add in order, one sum after another, then one write
    float* out = a.work + (group * a.chunks + chunk) * (int64_t)__builtin_popcount(a.slots) * a.dim;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (!(a.slots >> k & 1)) continue;
        Row<W, NV>& s = k == 0 ? sA : k == 1 ? sN : k == 2 ? sP : sQ;
        if constexpr (TPB > 1) {
            for (int tm = 0; tm < TPB; ++tm) {
                __syncthreads();
                if (team == tm) {
                    FOR_ROW(c, i) {
                        float& at = joined[(c * W + i) * TEAM + lane];
                        s.v[c][i] += tm ? at : 0.f;
                        at = s.v[c][i];
                    }
                }
            }
            if (team == TPB - 1) {
#pragma unroll
                for (int c = 0; c < NV; ++c) {
                    const int e = (c * TEAM + lane) * W;
#pragma unroll
                    for (int i = 0; i < W; ++i)
                        if (e + i < a.dim) out[e + i] = s.v[c][i];
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < NV; ++c) {
                const int e = (c * TEAM + lane) * W;
#pragma unroll
                for (int i = 0; i < W; ++i)
                    if (e + i < a.dim) out[e + i] = s.v[c][i];
            }
        }
        out += a.dim;
    }
}

__device__ __forceinline__ float param_at(const void* p, int64_t i, float none, int param_dtype) {
    if (!p) return none;
    if (param_dtype == CMDI_DT_F32) return static_cast<const float*>(p)[i];
    if (param_dtype == CMDI_DT_BF16) return Elem<Bf16>::up(static_cast<const Bf16*>(p)[i]);
    return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void param_put(void* p, int64_t i, float v, int param_dtype) {
    if (param_dtype == CMDI_DT_F32) static_cast<float*>(p)[i] = v;
    else if (param_dtype == CMDI_DT_BF16) static_cast<Bf16*>(p)[i] = Elem<Bf16>::down(v);
    else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

constexpr int JOIN_COLS = 64, JOIN_SLICES = 16;

// The chunks of one group, 64 columns a block, 16 slices of chunks each joined in order.  Writes the gradients
// that belong to the group's own sample; where more is needed, leaves the group's sums in its first chunk's place.
__global__ __launch_bounds__(JOIN_COLS * JOIN_SLICES) void gated_norm_join_kernel(const GatedNormArgs a, int per_sample, int keep) {
    __shared__ float part[JOIN_SLICES][JOIN_COLS];
    const unsigned cols = (unsigned)(a.dim + JOIN_COLS - 1) / JOIN_COLS;
    const int64_t group = blockIdx.x / cols;
    const int col = (int)(blockIdx.x % cols) * JOIN_COLS + threadIdx.x % JOIN_COLS, slice = threadIdx.x / JOIN_COLS;
    const int nslot = __builtin_popcount(a.slots);
    const int64_t pitch = (int64_t)nslot * a.dim;
    float* base = a.work + group * a.chunks * pitch;
    float tot[4] = {0.f, 0.f, 0.f, 0.f};
    int at = 0;
    for (int k = 0; k < 4; ++k) {
        if (!(a.slots >> k & 1)) continue;
        float s = 0.f;
        if (col < a.dim)
            for (int64_t c = slice; c < a.chunks; c += JOIN_SLICES) s += base[c * pitch + (int64_t)at * a.dim + col];
        __syncthreads();
        part[slice][threadIdx.x % JOIN_COLS] = s;
        __syncthreads();
        if (slice == 0) {
#pragma unroll
            for (int i = 1; i < JOIN_SLICES; ++i) s += part[i][threadIdx.x % JOIN_COLS];
            tot[k] = s;
        }
        ++at;
    }
    if (slice != 0 || col >= a.dim) return;
    const int pd = a.param_dtype;
    if (per_sample) {
        const int64_t o = group * a.dim + col;
        if (a.g_scale && a.scale.bs) param_put(a.g_scale, o, param_at(a.w, col, 1.f, pd) * tot[1] + param_at(a.b, col, 0.f, pd) * tot[0], pd);
        if (a.g_shift && a.shift.bs) param_put(a.g_shift, o, tot[0], pd);
        if (a.g_gate && a.gate.bs) param_put(a.g_gate, o, param_at(a.wp, col, 1.f, pd) * tot[2] + param_at(a.bp, col, 0.f, pd) * tot[3], pd);
    }
    if (keep) {
        at = 0;
        for (int k = 0; k < 4; ++k)
            if (a.slots >> k & 1) base[(int64_t)(at++) * a.dim + col] = tot[k];
    }
}

// All groups' sums -> the gradients that belong to every sample.
__global__ __launch_bounds__(JOIN_COLS * JOIN_SLICES) void gated_norm_join_all_kernel(const GatedNormArgs a) {
    __shared__ float part[JOIN_SLICES][JOIN_COLS];
    const int lane = threadIdx.x % JOIN_COLS, col = blockIdx.x * JOIN_COLS + lane, slice = threadIdx.x / JOIN_COLS;
    const int nslot = __builtin_popcount(a.slots), pd = a.param_dtype;
    const int64_t pitch = (int64_t)nslot * a.dim * a.chunks;
    // sums over the samples: 0 A, 1 N, 2 P, 3 Q plain; 4 (1 + s) A, 5 (1 + s) N, 6 g P, 7 g Q
    float tot[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) tot[k] = 0.f;
    if (col < a.dim)
        for (int64_t gi = slice; gi < a.groups; gi += JOIN_SLICES) {
            const float* p = a.work + gi * pitch + col;
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[k] = 0.f;
                if (a.slots >> k & 1) { v[k] = *p; p += a.dim; }
            }
            const float s1 = 1.f + param_at(a.scale.p, gi * a.scale.bs + col, 0.f, pd);
            const float gg = param_at(a.gate.p, gi * a.gate.bs + col, 1.f, pd);
#pragma unroll
            for (int k = 0; k < 4; ++k) { tot[k] += v[k]; tot[4 + k] += (k < 2 ? s1 : gg) * v[k]; }
        }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        __syncthreads();
        part[slice][lane] = tot[k];
        __syncthreads();
        if (slice == 0) {
#pragma unroll
            for (int i = 1; i < JOIN_SLICES; ++i) tot[k] += part[i][lane];
        }
    }
    if (slice != 0 || col >= a.dim) return;
    if (a.g_scale && !a.scale.bs) param_put(a.g_scale, col, param_at(a.w, col, 1.f, pd) * tot[1] + param_at(a.b, col, 0.f, pd) * tot[0], pd);
    if (a.g_shift && !a.shift.bs) param_put(a.g_shift, col, tot[0], pd);
    if (a.g_gate && !a.gate.bs) param_put(a.g_gate, col, param_at(a.wp, col, 1.f, pd) * tot[2] + param_at(a.bp, col, 0.f, pd) * tot[3], pd);
    if (a.g_w) param_put(a.g_w, col, tot[5], pd);
    if (a.g_b) param_put(a.g_b, col, tot[4], pd);
    if (a.g_wp) param_put(a.g_wp, col, tot[6], pd);
    if (a.g_bp) param_put(a.g_bp, col, tot[7], pd);
}

bool per_sample(const GatedNormArgs& a) {
    return (a.gate.p && a.gate.bs) || (a.scale.p && a.scale.bs) || (a.shift.p && a.shift.bs);
}
int teams_per_block(int dim) { return dim <= 1024 ? 4 : 1; }

// Width of the team by the row's length: 8 or 16 elements a lane (a lane's registers hold the row, the parameters and, backward,
// four column sums of each of its columns).
template <class T, int W, class F>
hipError_t by_width(int dim, F&& f) {
    if (dim <= 512) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 8 / W>());
    if (dim <= 1024) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 16 / W>());
    if (dim <= 2048) return f(std::integral_constant<int, 256>(), std::integral_constant<int, 8 / W>());
    if (dim <= 4096) return f(std::integral_constant<int, 256>(), std::integral_constant<int, 16 / W>());
    if (dim <= 8192) return f(std::integral_constant<int, 512>(), std::integral_constant<int, 16 / W>());
    return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 16 / W>());
}
template <class F>
hipError_t by_type(const GatedNormArgs& a, F&& f) {
    switch (a.dtype) {
        case CMDI_DT_F32: return a.vec ? f(float(), std::integral_constant<int, 4>()) : f(float(), std::integral_constant<int, 1>());
        case CMDI_DT_BF16: return a.vec ? f(Bf16(), std::integral_constant<int, 8>()) : f(Bf16(), std::integral_constant<int, 1>());
        default: return a.vec ? f(_Float16(), std::integral_constant<int, 8>()) : f(_Float16(), std::integral_constant<int, 1>());
    }
}

}  // namespace

void gated_norm_plan(GatedNormArgs& a, bool vjp) {
    const int64_t total = (int64_t)a.batch * a.seq;
    const int tpb = teams_per_block(a.dim);
    // blocks that keep the chip busy; a block's rows share its parameter registers and, backward, its column sums
    const int64_t want = 2048;
    if (per_sample(a)) {
        a.groups = a.batch;
        a.rows_per_group = a.seq;
    } else {
        // no sample of its own anywhere: cut the rows into pieces so that the joins run beside each other
        a.groups = vjp ? (total + 31) / 32 : 1;
        if (a.groups > 32) a.groups = 32;
        if (a.groups < 1) a.groups = 1;
        a.rows_per_group = (total + a.groups - 1) / a.groups;
        if (a.rows_per_group < 1) a.rows_per_group = 1;
        a.groups = (total + a.rows_per_group - 1) / a.rows_per_group;
        if (a.groups < 1) a.groups = 1;
    }
    int64_t chunks = (want + a.groups - 1) / a.groups;
    const int64_t most = (a.rows_per_group + tpb - 1) / tpb;
    if (chunks > most) chunks = most;
    if (chunks < 1) chunks = 1;
    int64_t rows = (a.rows_per_group + chunks - 1) / chunks;
    rows = (rows + tpb - 1) / tpb * tpb;
    a.rows_per_chunk = rows;
    a.chunks = (a.rows_per_group + rows - 1) / rows;
    if (a.chunks < 1) a.chunks = 1;
    a.slots = 0;
    if (a.g_shift || a.g_b || (a.g_scale && a.b)) a.slots |= 1;
    if (a.g_scale || a.g_w) a.slots |= 2;
    if (a.g_gate || a.g_wp) a.slots |= 4;
    if (a.g_bp || (a.g_gate && a.bp)) a.slots |= 8;
}

int64_t gated_norm_work_floats(const GatedNormArgs& a) {
    return a.groups * a.chunks * (int64_t)__builtin_popcount(a.slots) * a.dim;
}

hipError_t launch_gated_norm_fwd(const GatedNormArgs& a, hipStream_t stream) {
    return by_type(a, [&](auto t, auto w) {
        using T = decltype(t);
        constexpr int W = decltype(w)::value;
        return by_width<T, W>(a.dim, [&](auto team, auto nv) {
            constexpr int TEAM = decltype(team)::value, NV = decltype(nv)::value;
            gated_norm_fwd_kernel<T, W, TEAM, NV><<<dim3((unsigned)(a.groups * a.chunks)), dim3(TEAM < 256 ? 256 : TEAM), 0, stream>>>(a);
            return hipGetLastError();
        });
    });
}

hipError_t launch_gated_norm_vjp(const GatedNormArgs& a, hipStream_t stream) {
    hipError_t err = by_type(a, [&](auto t, auto w) {
        using T = decltype(t);
        constexpr int W = decltype(w)::value;
        return by_width<T, W>(a.dim, [&](auto team, auto nv) {
            constexpr int TEAM = decltype(team)::value, NV = decltype(nv)::value;
            gated_norm_vjp_kernel<T, W, TEAM, NV><<<dim3((unsigned)(a.groups * a.chunks)), dim3(TEAM < 256 ? 256 : TEAM), 0, stream>>>(a);
            return hipGetLastError();
        });
    });
    if (err != hipSuccess || !a.slots) return err;
    const bool own = (a.g_scale && a.scale.bs) || (a.g_shift && a.shift.bs) || (a.g_gate && a.gate.bs);
    const bool all = a.g_w || a.g_b || a.g_wp || a.g_bp || (a.g_scale && !a.scale.bs) || (a.g_shift && !a.shift.bs) || (a.g_gate && !a.gate.bs);
    const unsigned cols = (unsigned)((a.dim + JOIN_COLS - 1) / JOIN_COLS);
    gated_norm_join_kernel<<<dim3(cols * (unsigned)a.groups), dim3(JOIN_COLS * JOIN_SLICES), 0, stream>>>(a, own, all);
    err = hipGetLastError();
    if (err != hipSuccess || !all) return err;
    gated_norm_join_all_kernel<<<dim3(cols), dim3(JOIN_COLS * JOIN_SLICES), 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace cmdi
