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
// once per block, and two small kernels join them in a fixed order: no atomics, the same bits every run.  Where samples are many and
// short, a team of lanes takes whole samples instead: it writes their gradients itself and carries only the sums over all samples.
//
// Bound by memory: forward reads x, y and writes r, h; backward reads x, y, dr', dh and writes dx, dy (r is computed again from
// x and y, unrounded, which costs no more reads than r itself would).  A row stays in the registers of its team of lanes, so the
// variance is taken of the centred values at no extra reads.  16 x 2048 rows of 2048 bf16: forward 95 - 100 us (5.4 - 5.7 TB/s, part of it
// from the last-level cache), backward 193 - 208 us (3.9 - 4.2 TB/s; 60 registers a lane for a row's values and its four sums), its joins
// 14 - 15 us; 64 x 197 rows of 512 fp32: 18 us.
#include "gated_norm.hpp"

#include <type_traits>

#include "../../include/condmdi.h"
#include "launches.hpp"
#include "ops_common.hpp"

namespace cmdi {
namespace {

// A team of TEAM lanes holds a row: element (c * TEAM + lane) * W + i, c < NV.  TEAM = 64: the row's sums never leave the wave;
// wider teams are whole blocks and join their waves through LDS, one barrier for all sums of a step (two slots in turn).
template <int TEAM>
struct TeamSum {
    static constexpr int NW = TEAM / 64, MOST = 4;
    float* lds;      // [2][MOST][NW]
    int slot = 0;
    __device__ __forceinline__ explicit TeamSum(float* l) : lds(l) {}
    template <int N>
    __device__ __forceinline__ void all(float (&v)[N]) {
        static_assert(N <= MOST, "");
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = wave_total(v[k]);
        if constexpr (TEAM > 64) {
            float* at = lds + slot * MOST * NW;
            slot ^= 1;
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int k = 0; k < N; ++k) at[k * NW + (threadIdx.x >> 6)] = v[k];
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < N; ++k) {
                v[k] = 0.f;
#pragma unroll
                for (int i = 0; i < NW; ++i) v[k] += at[k * NW + i];
            }
        }
    }
};

template <int W, int NV>
struct Row { float v[NV][W]; };

// How a team's lanes lie on a row.  WHOLE: W divides the row, a lane's access is all in or all out (a row's odd end costs every
// access a branch: 130 us against 112 us for 16 x 2048 rows of 2048 forward).
template <int W_, int TEAM_, int NV_, bool WHOLE_>
struct Shape {
    static constexpr int W = W_, TEAM = TEAM_, NV = NV_;
    static constexpr bool WHOLE = WHOLE_;
    static constexpr int BLOCK = TEAM == 64 ? 256 : TEAM, TPB = BLOCK / TEAM;
    using R = Row<W, NV>;
};
#define SHAPE                                                      \
    constexpr int W = S::W, TEAM = S::TEAM, NV = S::NV;            \
    using R = typename S::R;                                       \
    (void)W, (void)TEAM, (void)NV

#define FOR_ROW(c, i) _Pragma("unroll") for (int c = 0; c < NV; ++c) _Pragma("unroll") for (int i = 0; i < W; ++i)

// columns behind `dim` read as 0
// `over`: the W - 1 elements behind the row may be read (they are the tensor's own): one access then also at an odd end, whose
// separate elements would cost the row a second trip to memory
template <class S, class T>
__device__ __forceinline__ void load_row(typename S::R& r, const T* p, int lane, int dim, bool over = false) {
    SHAPE;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int e = (c * TEAM + lane) * W;
        if constexpr (S::WHOLE) {
            if (e < dim) {
                load_vec<T, W>(p + e, r.v[c]);
            } else {
#pragma unroll
                for (int i = 0; i < W; ++i) r.v[c][i] = 0.f;
            }
        } else if (over) {
            load_part<T, W>(p + e, r.v[c], e < dim ? W : 0);
            if (e + W > dim) {
#pragma unroll
                for (int i = 0; i < W; ++i) r.v[c][i] = e + i < dim ? r.v[c][i] : 0.f;
            }
        } else {
            load_part<T, W>(p + e, r.v[c], dim - e);
        }
    }
}
template <class S, class T>
__device__ __forceinline__ void store_row(T* p, const typename S::R& r, int lane, int dim) {
    SHAPE;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int e = (c * TEAM + lane) * W;
        if constexpr (S::WHOLE) {
            if (e < dim) store_vec<T, W>(p + e, r.v[c]);
        } else {
            store_part<T, W>(p + e, r.v[c], dim - e);
        }
    }
}
// a parameter row, or `fill` where there is none (columns behind `dim` hold 0); the entries allow 32 bits or the rows' own type
template <class S, class T>
__device__ __forceinline__ void load_param(typename S::R& r, const void* p, int64_t off, float fill, const GatedNormArgs& a, int lane) {
    SHAPE;
    if (!p) {
        FOR_ROW(c, i) r.v[c][i] = (c * TEAM + lane) * W + i < a.dim ? fill : 0.f;
    } else if (a.param_dtype == CMDI_DT_F32) {
        load_row<S, float>(r, static_cast<const float*>(p) + off, lane, a.dim);
    } else {
        load_row<S, T>(r, static_cast<const T*>(p) + off, lane, a.dim);
    }
}
template <class S, class T>
__device__ __forceinline__ void store_param(void* p, int64_t off, const typename S::R& r, const GatedNormArgs& a, int lane) {
    if (a.param_dtype == CMDI_DT_F32) store_row<S, float>(static_cast<float*>(p) + off, r, lane, a.dim);
    else store_row<S, T>(static_cast<T*>(p) + off, r, lane, a.dim);
}

// v <- N(v), returns k = 1 / sqrt(mean + eps).  Columns behind `dim` stay 0.
template <class S>
__device__ __forceinline__ float normalise(typename S::R& r, int kind, const GatedNormArgs& a, float inv_dim, int lane, TeamSum<S::TEAM>& sum) {
    SHAPE;
    if (kind == CMDI_NORM_NONE) return 1.f;
    float v[1];
    if (kind == CMDI_NORM_LAYER) {
        v[0] = 0.f;
        FOR_ROW(c, i) v[0] += r.v[c][i];
        sum.all(v);
        const float mean = v[0] * inv_dim;
        FOR_ROW(c, i) r.v[c][i] = (c * TEAM + lane) * W + i < a.dim ? r.v[c][i] - mean : 0.f;
    }
    v[0] = 0.f;
    FOR_ROW(c, i) v[0] += r.v[c][i] * r.v[c][i];
    sum.all(v);
    const float k = 1.f / sqrtf(v[0] * inv_dim + a.eps);
    FOR_ROW(c, i) r.v[c][i] *= k;
    return k;
}

// row numbers stay below 2^31 (checked at the entry): one 32-bit division a row, offsets in 64 bits
__device__ __forceinline__ int64_t row_at(const Rows& t, unsigned row, unsigned seq) {
    const unsigned b = row / seq, s = row - b * seq;
    return (int64_t)b * t.bs + (int64_t)s * t.ss;
}
template <class S, class T>
__device__ __forceinline__ void load_at(typename S::R& r, const Rows& t, int64_t row, const GatedNormArgs& a, int lane) {
    const int64_t at = row_at(t, (unsigned)row, a.seq), last = (int64_t)(a.batch - 1) * t.bs + (int64_t)(a.seq - 1) * t.ss;
    load_row<S, T>(r, static_cast<const T*>(t.p) + at, lane, a.dim, at + S::W - 1 <= last);
}

// this block's number over all launches of the pass
__device__ __forceinline__ unsigned block_at(const GatedNormArgs& a) { return a.first + blockIdx.x; }

// the rows of a block: a chunk of a group
__device__ __forceinline__ void chunk_rows(const GatedNormArgs& a, int64_t& group, int64_t& chunk, int64_t& first, int64_t& end) {
    group = block_at(a) / (unsigned)a.chunks;
    chunk = block_at(a) % (unsigned)a.chunks;
    first = group * a.rows_per_group + chunk * a.rows_per_chunk;
    end = first + a.rows_per_chunk;
    const int64_t total = (int64_t)a.batch * a.seq, stop = (group + 1) * a.rows_per_group;
    if (end > stop) end = stop;
    if (end > total) end = total;
}

template <class T, class S>
__global__ __launch_bounds__(S::BLOCK) void gated_norm_fwd_kernel(const GatedNormArgs a) {
    SHAPE;
    constexpr int TPB = S::TPB;
    __shared__ float lds[2 * TeamSum<TEAM>::MOST * (TEAM / 64)];
    TeamSum<TEAM> sum(lds);
    const int lane = threadIdx.x % TEAM, team = TPB == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / TEAM);
    int64_t group, chunk, first, end;
    chunk_rows(a, group, chunk, first, end);
    const float inv_dim = 1.f / (float)a.dim;

    R g, wp, bp, w, t;
    // h = n w (1 + s) + (b (1 + s) + t); r = alpha x + ny (wp g) + bp g
    load_param<S, T>(g, a.gate.p, group * a.gate.bs, 1.f, a, lane);
    load_param<S, T>(wp, a.wp, 0, 1.f, a, lane);
    load_param<S, T>(bp, a.bp, 0, 0.f, a, lane);
    load_param<S, T>(w, a.w, 0, 1.f, a, lane);
    load_param<S, T>(t, a.b, 0, 0.f, a, lane);
    FOR_ROW(c, i) { wp.v[c][i] *= g.v[c][i]; bp.v[c][i] *= g.v[c][i]; }
    load_param<S, T>(g, a.scale.p, group * a.scale.bs, 0.f, a, lane);
    FOR_ROW(c, i) { w.v[c][i] *= 1.f + g.v[c][i]; t.v[c][i] *= 1.f + g.v[c][i]; }
    load_param<S, T>(g, a.shift.p, group * a.shift.bs, 0.f, a, lane);
    FOR_ROW(c, i) t.v[c][i] += g.v[c][i];

    for (int64_t row = first + team; row < end; row += TPB) {     // (TPB > 1: a team is a wave, nothing in here waits for another)
        R x, y;
        load_at<S, T>(x, a.x, row, a, lane);
        if (a.y.p) {
            load_at<S, T>(y, a.y, row, a, lane);
            normalise<S>(y, a.post, a, inv_dim, lane, sum);
            FOR_ROW(c, i) x.v[c][i] = a.alpha * x.v[c][i] + (y.v[c][i] * wp.v[c][i] + bp.v[c][i]);
        } else {
            FOR_ROW(c, i) x.v[c][i] *= a.alpha;
        }
        if (a.r) store_row<S, T>(static_cast<T*>(a.r) + row * a.dim, x, lane, a.dim);
        normalise<S>(x, a.pre, a, inv_dim, lane, sum);
        FOR_ROW(c, i) x.v[c][i] = x.v[c][i] * w.v[c][i] + t.v[c][i];
        store_row<S, T>(static_cast<T*>(a.h) + row * a.dim, x, lane, a.dim);
    }
}

// Column sums of the rows seen so far.
template <int W, int NV>
struct Sums {
    Row<W, NV> A, N, P, Q;
    __device__ __forceinline__ void clear() {
        FOR_ROW(c, i) { A.v[c][i] = 0.f; N.v[c][i] = 0.f; P.v[c][i] = 0.f; Q.v[c][i] = 0.f; }
    }
};

// One row backward: gx, gy written, its column sums added.  wp, bp: N_post's weight and bias times the gate; w: weight (1 + s).
template <class S, class T>
__device__ __forceinline__ void vjp_row(const GatedNormArgs& a, int64_t row, const typename S::R& wp, const typename S::R& bp, const typename S::R& w, float inv_dim,
                                        int lane, TeamSum<S::TEAM>& sum, Sums<S::W, S::NV>& s) {
    SHAPE;
    R x, y, d;
    float ky = 1.f, m[2];
    load_at<S, T>(x, a.x, row, a, lane);
    if (a.gh.p) {
        load_at<S, T>(d, a.gh, row, a, lane);
    } else {
        FOR_ROW(c, i) d.v[c][i] = 0.f;
    }
    if (a.y.p) {
        load_at<S, T>(y, a.y, row, a, lane);
        ky = normalise<S>(y, a.post, a, inv_dim, lane, sum);
        FOR_ROW(c, i) x.v[c][i] = a.alpha * x.v[c][i] + (y.v[c][i] * wp.v[c][i] + bp.v[c][i]);
    } else {
        FOR_ROW(c, i) { y.v[c][i] = 0.f; x.v[c][i] *= a.alpha; }
    }
    const float kr = normalise<S>(x, a.pre, a, inv_dim, lane, sum);     // x = n
    m[0] = m[1] = 0.f;
    FOR_ROW(c, i) {
        s.A.v[c][i] += d.v[c][i];
        s.N.v[c][i] += d.v[c][i] * x.v[c][i];
        d.v[c][i] *= w.v[c][i];                                                   // dn
        m[0] += d.v[c][i];
        m[1] += d.v[c][i] * x.v[c][i];
    }
    sum.all(m);
    float m1 = a.pre == CMDI_NORM_LAYER ? m[0] * inv_dim : 0.f, m2 = m[1] * inv_dim;
    FOR_ROW(c, i) d.v[c][i] = kr * (d.v[c][i] - x.v[c][i] * m2 - m1);
    if (a.gr.p) {
        load_at<S, T>(x, a.gr, row, a, lane);
        FOR_ROW(c, i) d.v[c][i] += x.v[c][i];                                     // dr
    }
    if (a.gx) {
        FOR_ROW(c, i) x.v[c][i] = a.alpha * d.v[c][i];
        store_row<S, T>(static_cast<T*>(a.gx) + row * a.dim, x, lane, a.dim);
    }
    if (!a.y.p) return;
    m[0] = m[1] = 0.f;
    FOR_ROW(c, i) {
        // columns behind `dim` hold -kr m1 in d; their weights are 0 and their sums never written
        s.P.v[c][i] += d.v[c][i] * y.v[c][i];
        s.Q.v[c][i] += d.v[c][i];
        d.v[c][i] *= wp.v[c][i];
        m[0] += d.v[c][i];
        m[1] += d.v[c][i] * y.v[c][i];
    }
    if (!a.gy) return;
    if (a.post != CMDI_NORM_NONE) {
        sum.all(m);
        m1 = a.post == CMDI_NORM_LAYER ? m[0] * inv_dim : 0.f;
        m2 = m[1] * inv_dim;
        FOR_ROW(c, i) d.v[c][i] = ky * (d.v[c][i] - y.v[c][i] * m2 - m1);
    }
    store_row<S, T>(static_cast<T*>(a.gy) + row * a.dim, d, lane, a.dim);
}

// SPAN: a team takes a.rows_per_chunk whole samples one after the other; otherwise a block a chunk of one group's rows.
template <class T, class S, bool SPAN>
__global__ __launch_bounds__(S::BLOCK) void gated_norm_vjp_kernel(const GatedNormArgs a) {
    SHAPE;
    constexpr int TPB = S::TPB;
    __shared__ float lds[2 * TeamSum<TEAM>::MOST * (TEAM / 64)];
    __shared__ float joined[TPB > 1 ? TEAM * NV * W : 1];
    TeamSum<TEAM> sum(lds);
    const int lane = threadIdx.x % TEAM, team = TPB == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / TEAM);
    const float inv_dim = 1.f / (float)a.dim;
    R wp, bp, w;
    auto params = [&](int64_t sample) {
        R g;
        load_param<S, T>(w, a.w, 0, 1.f, a, lane);
        load_param<S, T>(g, a.scale.p, sample * a.scale.bs, 0.f, a, lane);
        FOR_ROW(c, i) w.v[c][i] *= 1.f + g.v[c][i];
        load_param<S, T>(g, a.gate.p, sample * a.gate.bs, 1.f, a, lane);
        load_param<S, T>(wp, a.wp, 0, 1.f, a, lane);
        load_param<S, T>(bp, a.bp, 0, 0.f, a, lane);
        FOR_ROW(c, i) { wp.v[c][i] *= g.v[c][i]; bp.v[c][i] *= g.v[c][i]; }
    };
    Sums<W, NV> s;
    s.clear();
    if constexpr (SPAN) {
        Sums<W, NV> own;
        const int64_t s0 = ((int64_t)block_at(a) * TPB + team) * a.rows_per_chunk;
        const int64_t s1 = s0 + a.rows_per_chunk < a.batch ? s0 + a.rows_per_chunk : a.batch;
        for (int64_t b = s0; b < s1; ++b) {
            params(b);
            own.clear();
            for (int i = 0; i < a.seq; ++i) vjp_row<S, T>(a, b * a.seq + i, wp, bp, w, inv_dim, lane, sum, own);
            // ds = w N + b A, dt = A, dg = wp P + bp Q; the other parameters' sums take (1 + s) or g along
            R u, v;
            load_param<S, T>(u, a.scale.p, b * a.scale.bs, 0.f, a, lane);
            FOR_ROW(c, i) { s.A.v[c][i] += (1.f + u.v[c][i]) * own.A.v[c][i]; s.N.v[c][i] += (1.f + u.v[c][i]) * own.N.v[c][i]; }
            load_param<S, T>(u, a.gate.p, b * a.gate.bs, 1.f, a, lane);
            FOR_ROW(c, i) { s.P.v[c][i] += u.v[c][i] * own.P.v[c][i]; s.Q.v[c][i] += u.v[c][i] * own.Q.v[c][i]; }
            if (a.g_shift) store_param<S, T>(a.g_shift, b * a.dim, own.A, a, lane);
            if (a.g_scale) {
                load_param<S, T>(u, a.w, 0, 1.f, a, lane);
                load_param<S, T>(v, a.b, 0, 0.f, a, lane);
                FOR_ROW(c, i) u.v[c][i] = u.v[c][i] * own.N.v[c][i] + v.v[c][i] * own.A.v[c][i];
                store_param<S, T>(a.g_scale, b * a.dim, u, a, lane);
            }
            if (a.g_gate) {
                load_param<S, T>(u, a.wp, 0, 1.f, a, lane);
                load_param<S, T>(v, a.bp, 0, 0.f, a, lane);
                FOR_ROW(c, i) u.v[c][i] = u.v[c][i] * own.P.v[c][i] + v.v[c][i] * own.Q.v[c][i];
                store_param<S, T>(a.g_gate, b * a.dim, u, a, lane);
            }
        }
    } else {
        int64_t group, chunk, first, end;
        chunk_rows(a, group, chunk, first, end);
        params(group);
        for (int64_t row = first + team; row < end; row += TPB) vjp_row<S, T>(a, row, wp, bp, w, inv_dim, lane, sum, s);
    }
    // the block's column sums: teams add in order, one sum after another, then one write
    float* out = a.work + (int64_t)block_at(a) * __builtin_popcount(a.slots) * a.dim;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (!(a.slots >> k & 1)) continue;
        typename S::R& r = k == 0 ? s.A : k == 1 ? s.N : k == 2 ? s.P : s.Q;
        if constexpr (TPB > 1) {
            for (int tm = 0; tm < TPB; ++tm) {
                __syncthreads();
                if (team == tm) {
                    FOR_ROW(c, i) {
                        float& at = joined[(c * W + i) * TEAM + lane];
                        r.v[c][i] += tm ? at : 0.f;
                        at = r.v[c][i];
                    }
                }
            }
        }
        if (team == TPB - 1) store_row<S, float>(out, r, lane, a.dim);
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
    const int64_t group = a.first + blockIdx.x / cols;
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
#pragma unroll 4
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
    const bool apart = !a.span && (a.scale.bs || a.gate.bs);          // (span: g and 1 + s are taken along already)
    float s1 = a.span || apart ? 1.f : 1.f + param_at(a.scale.p, col < a.dim ? col : 0, 0.f, pd);
    float gg = a.span || apart ? 1.f : param_at(a.gate.p, col < a.dim ? col : 0, 1.f, pd);
    constexpr int U = 4;                                              // groups whose sums are on their way together
    if (col < a.dim)
        for (int64_t g0 = slice; g0 < a.groups; g0 += U * JOIN_SLICES) {
            float v[U][4];
#pragma unroll
            for (int k = 0, at = 0; k < 4; ++k) {
                const bool there = a.slots >> k & 1;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t gi = g0 + u * JOIN_SLICES;
                    v[u][k] = there && gi < a.groups ? a.work[gi * pitch + (int64_t)at * a.dim + col] : 0.f;
                }
                at += there;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t gi = g0 + u * JOIN_SLICES;
                if (gi >= a.groups) break;
                if (apart) {
                    s1 = 1.f + param_at(a.scale.p, gi * a.scale.bs + col, 0.f, pd);
                    gg = param_at(a.gate.p, gi * a.gate.bs + col, 1.f, pd);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) { tot[k] += v[u][k]; tot[4 + k] += (k < 2 ? s1 : gg) * v[u][k]; }
            }
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
int teams_per_block(int dim) { return dim <= 512 ? 4 : 1; }
int block_threads(int dim) { return dim <= 512 ? 256 : dim <= 1024 ? 128 : dim <= 2048 ? 256 : dim <= 4096 ? 512 : 1024; }

// Width of the team by the row's length: 8 elements a lane as long as a block can be that wide (backward a lane's registers also
// hold four column sums of each of its columns).
template <class T, class F>
hipError_t by_shape(int dim, F&& f) {
    constexpr int W = Elem<T>::W;
    auto go = [&](auto team, auto nv) {
        constexpr int TEAM = decltype(team)::value, NV = decltype(nv)::value;
        return dim % W == 0 ? f(Shape<W, TEAM, NV, true>()) : f(Shape<W, TEAM, NV, false>());
    };
    using std::integral_constant;
    if (dim <= 512) return go(integral_constant<int, 64>(), integral_constant<int, 8 / W>());
    if (dim <= 1024) return go(integral_constant<int, 128>(), integral_constant<int, 8 / W>());
    if (dim <= 2048) return go(integral_constant<int, 256>(), integral_constant<int, 8 / W>());
    if (dim <= 4096) return go(integral_constant<int, 512>(), integral_constant<int, 8 / W>());
    if (dim <= 8192) return go(integral_constant<int, 1024>(), integral_constant<int, 8 / W>());
    return go(integral_constant<int, 1024>(), integral_constant<int, 16 / W>());
}
template <class F>
hipError_t by_type(const GatedNormArgs& a, F&& f) {
    switch (a.dtype) {
        case CMDI_DT_F32: return f(float());
        case CMDI_DT_BF16: return f(Bf16());
        default: return f(_Float16());
    }
}

}  // namespace

void gated_norm_plan(GatedNormArgs& a, bool vjp) {
    const int64_t total = (int64_t)a.batch * a.seq;
    const int tpb = teams_per_block(a.dim);
    // blocks that keep the chip busy; a block's rows share its parameter registers and, backward, its column sums (whose partial
    // results the joins read back: fewer, longer blocks there)
    const int64_t want = (vjp ? 262144 : 524288) / block_threads(a.dim);
    const bool own = per_sample(a);
    a.slots = 0;
    a.span = vjp && own && a.batch >= 256 && a.seq <= 32 && (!a.gate.p || a.gate.bs) && (!a.scale.p || a.scale.bs) && (!a.shift.p || a.shift.bs);
    if (a.span) {
        // many short samples: teams take whole ones (4096 of one row, width 2048: 86 us, with the joins below 959 us)
        const int64_t teams = want * tpb;
        a.rows_per_chunk = (a.batch + teams - 1) / teams;
        a.groups = ((a.batch + a.rows_per_chunk - 1) / a.rows_per_chunk + tpb - 1) / tpb;
        a.chunks = 1;
        a.rows_per_group = 0;
        a.slots = (a.g_b ? 1 : 0) | (a.g_w ? 2 : 0) | (a.g_wp ? 4 : 0) | (a.g_bp ? 8 : 0);
        return;
    }
    const int64_t span = own ? a.seq : total, spans = own ? a.batch : 1;
    int64_t chunks = (want + spans - 1) / spans;
    const int64_t most = (span + tpb - 1) / tpb;
    if (chunks > most) chunks = most;
    if (chunks < 1) chunks = 1;
    int64_t rows = (span + chunks - 1) / chunks;
    rows = (rows + tpb - 1) / tpb * tpb;
    chunks = (span + rows - 1) / rows;
    if (chunks < 1) chunks = 1;
    a.rows_per_chunk = rows < 1 ? 1 : rows;
    if (own) {
        a.groups = a.batch;
        a.chunks = chunks;
        a.rows_per_group = a.seq;
    } else if (vjp && chunks > 512) {
        // no sample of its own anywhere: 32 groups of chunks whose joins run beside each other, then one of the groups.  Against one join
        // of all chunks (us, whole backward pass): 1000 chunks of width 515: 23 / 34;  512 chunks of width 4096: 71 / 63;  385 of 1024: 18.8 / 19.4
        a.chunks = (chunks + 31) / 32;
        a.groups = (chunks + a.chunks - 1) / a.chunks;
        a.rows_per_group = a.chunks * a.rows_per_chunk;
    } else if (vjp) {
        a.chunks = 1;            // few chunks: the last join takes them all
        a.groups = chunks;
        a.rows_per_group = a.rows_per_chunk;
    } else {
        a.chunks = chunks;
        a.groups = 1;
        a.rows_per_group = total;
    }
    if (a.g_shift || a.g_b || (a.g_scale && a.b)) a.slots |= 1;
    if (a.g_scale || a.g_w) a.slots |= 2;
    if (a.g_gate || a.g_wp) a.slots |= 4;
    if (a.g_bp || (a.g_gate && a.bp)) a.slots |= 8;
}

int64_t gated_norm_work_floats(const GatedNormArgs& a) {
    return a.groups * a.chunks * (int64_t)__builtin_popcount(a.slots) * a.dim;
}

hipError_t launch_gated_norm_fwd(const GatedNormArgs& args, hipStream_t stream) {
    GatedNormArgs a = args;
    return by_type(a, [&](auto t) {
        using T = decltype(t);
        return by_shape<T>(a.dim, [&](auto shape) {
            using S = decltype(shape);
            return in_launches(a.groups * a.chunks, S::BLOCK, 1, [&](int64_t first, unsigned blocks) {
                a.first = (uint32_t)first;
                gated_norm_fwd_kernel<T, S><<<dim3(blocks), dim3(S::BLOCK), 0, stream>>>(a);
                return hipGetLastError();
            });
        });
    });
}

hipError_t launch_gated_norm_vjp(const GatedNormArgs& args, hipStream_t stream) {
    GatedNormArgs a = args;
    hipError_t err = by_type(a, [&](auto t) {
        using T = decltype(t);
        return by_shape<T>(a.dim, [&](auto shape) {
            using S = decltype(shape);
            return in_launches(a.groups * a.chunks, S::BLOCK, 1, [&](int64_t first, unsigned blocks) {
                a.first = (uint32_t)first;
                if (a.span) gated_norm_vjp_kernel<T, S, true><<<dim3(blocks), dim3(S::BLOCK), 0, stream>>>(a);
                else gated_norm_vjp_kernel<T, S, false><<<dim3(blocks), dim3(S::BLOCK), 0, stream>>>(a);
                return hipGetLastError();
            });
        });
    });
    if (err != hipSuccess || !a.slots) return err;
    const bool own = !a.span && ((a.g_scale && a.scale.bs) || (a.g_shift && a.shift.bs) || (a.g_gate && a.gate.bs));
    const bool all = a.g_w || a.g_b || a.g_wp || a.g_bp || (a.g_scale && !a.scale.bs) || (a.g_shift && !a.shift.bs) || (a.g_gate && !a.gate.bs);
    const unsigned cols = (unsigned)((a.dim + JOIN_COLS - 1) / JOIN_COLS);
    if (own || a.chunks > 1) {
        err = in_launches(cols * a.groups, JOIN_COLS * JOIN_SLICES, cols, [&](int64_t first, unsigned blocks) {
            a.first = (uint32_t)first;
            gated_norm_join_kernel<<<dim3(blocks), dim3(JOIN_COLS * JOIN_SLICES), 0, stream>>>(a, own, all);
            return hipGetLastError();
        });
        if (err != hipSuccess || !all) return err;
    }
    gated_norm_join_all_kernel<<<dim3(cols), dim3(JOIN_COLS * JOIN_SLICES), 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace cmdi
