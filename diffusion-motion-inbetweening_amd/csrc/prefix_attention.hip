// Attention of a batch whose sequences share one long prefix of keys and values and have some of their own:
//
//   out[b, i, h] = softmax_j (scale q . k_j) v_j   over the prefix's keys and the own keys j < visible(b, i)
//   visible = own_len[b], or with causal order own_len[b] - queries + i + 1 (the queries are the sequence's newest tokens)
//
// A pass over the keys keeps a running maximum and sum per row (fp32, base-2 exponentials):
//   m' = max(m, max s),  l' = l 2^(m - m') + sum 2^(s - m'),  o' = o 2^(m - m') + sum 2^(s - m') v
// and partial results over different keys join the same way, so the prefix can be read ONCE for all sequences: their rows
// (sequence, query, head of the key head's group) are packed into tiles that run over a chunk of the prefix; each sequence's own
// keys are a second set of items; a last kernel joins a row's partial results through their log-sums.  Few queries: bound by the
// keys' bytes, prefix read once instead of once a sequence.  Many queries: a tile of one sequence's rows runs over prefix and own
// keys in one loop, bound by the matrix units.
//
// Matrix instructions: v_mfma_f32_16x16x32 (bf16 / f16 operands, fp32 sums).  S^T = K Q^T puts a row of Q into a lane column,
// so maximum and sum stay in the lane but for two exchanges, and S^T's accumulators ARE the operand of O^T += V^T P^T: lane group
// g holds keys 4 g + r and 16 + 4 g + r of a 32-key block, and the transposed LDS reads (ds_read_b64_tr_b16) fetch V in that same
// order.  P is rounded to the operands' 16 bits (half a step relative, as the matrix unit asks), its sum l is taken before that.
#include "prefix_attention.hpp"

#include <algorithm>
#include <type_traits>

#include "../../include/condmdi.h"
#include "ops_common.hpp"

namespace cmdi {
namespace {

typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

template <class T> struct Mma;
template <> struct Mma<Bf16> {
    static __device__ __forceinline__ f32x4 mul(s8 a, s8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ unsigned pack(float x, float y) { return __builtin_bit_cast(unsigned, b2{(__bf16)x, (__bf16)y}); }
};
template <> struct Mma<_Float16> {
    static __device__ __forceinline__ f32x4 mul(s8 a, s8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ unsigned pack(float x, float y) { return __builtin_bit_cast(unsigned, h2{(_Float16)x, (_Float16)y}); }
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

// A key row of a stage is DIM elements in 16-byte slots; slot t of key k is stored at t ^ swz(k).  A ds_read_b128 serves lanes
// {0-3, 12-15, 20-27} and so on together: keys {0-3, 12-15} at one slot and {4-11} at its neighbour, so the swizzles of the first
// eight have to be four whole pairs; a transposed read takes 8 keys at two neighbouring slots, whose pairs have to differ.
template <int DIM>
__device__ __forceinline__ int swz(int k) {
    const int high = (k >> 3) & 1;
    return DIM == 128 ? (((k & 7) ^ (high << 2)) << 1) | high : ((((k >> 1) & 3) ^ (high << 1)) << 1) | high;
}

// 16 bytes a lane from `offset` behind the descriptor's base to LDS, lane after lane.  (The host's pass over this file knows no
// 16-byte form of the builtin.)
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, char* to, int offset) {
#ifdef __HIP_DEVICE_COMPILE__
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)to, 16, offset, 0, 0, 0);
#endif
}

// Maximum / sum over the four lane groups that share a row (lanes 16 apart).
__device__ __forceinline__ float over_groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float over_groups_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

template <int DIM, bool BYWAVE>
constexpr int lds_bytes() {
    // by rows: three stages of 64 keys, two of 64 values; by wave: each of the four has two stages of 32 values
    return BYWAVE ? 4 * 2 * 32 * DIM * 2 : 5 * 64 * DIM * 2;
}

// One item: a tile of rows over a chunk of keys.
//   By rows: wave w owns rows [16 RT w, +16 RT); K and V come in 64-key stages through LDS (LDS-DMA, three stages of K, two of V).
//   A stage is two units of 32 keys; the scores of the next unit are multiplied while the softmax of this one runs, so the matrix
//   units work under the exponentials.
//   BYWAVE: at most 16 rows (few queries): a wave takes every fourth 32-key tile, its K straight into registers, its V through its own
//   two LDS slots, no barrier until the four waves join at the end.
// A row's maximum is moved only when a score passes it by 2^8: until then its p stay below 256, which changes no relative
// rounding and saves the exchange between the lanes and the rescaling of o.
template <class T, int DIM, int RT, bool BYWAVE>
__device__ __forceinline__ void attend(const PrefixAttnArgs& a, const PrefixAttnLaunch& L, int slots, int block, int blocks, char* lds_all) {
    constexpr int KT = BYWAVE ? 32 : 64, ROWB = DIM * 2, TILE = KT * ROWB, KB = 2, DB = DIM / 16, DS = DIM / 32;
    constexpr int SLOTS = DIM / 8, RPP = 64 / SLOTS;              // 16-byte slots of a key row; key rows of a 1-KiB piece
    constexpr int PIECES = KT / RPP / (BYWAVE ? 1 : 4);           // pieces of a tile that a wave brings
    static_assert(!BYWAVE || RT == 1, "");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l15 = lane & 15, g = lane >> 4;
    // by rows: K slots at 0 .. 2, V slots at 3, 4 tiles; by wave: the wave's two V slots
    char* lds = lds_all + (BYWAVE ? wave * 2 * TILE : 0);

    // ---- which item ----
    const int grp = a.heads / a.kv_heads;
    const int id = xcd_remap(block, blocks);
    const int tile = id % L.tiles, rest = id / L.tiles;
    const int chunk = rest % L.chunks, bh = rest / L.chunks;
    const int hk = bh % a.kv_heads, b0 = bh / a.kv_heads;         // packed: b0 = 0, the sample comes from the row
    const int n_rows = (L.packed ? a.batch : 1) * a.queries * grp;
    constexpr int BM = BYWAVE ? 16 : 64 * RT;

    // ---- rows of this lane: column l15 of each of the wave's RT row tiles ----
    int row_b[RT], row_i[RT], row_h[RT], vis[RT];
    bool row_ok[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        int r = tile * BM + (BYWAVE ? 0 : wave * RT * 16) + t * 16 + l15;
        row_ok[t] = r < n_rows;
        if (!row_ok[t]) r = n_rows - 1;
        row_h[t] = hk * grp + r % grp;
        const int q = r / grp;
        row_i[t] = q % a.queries;
        row_b[t] = L.packed ? q / a.queries : b0;
        vis[t] = 0;
    }
    int vis_top = 0, vis_low = 0;                                 // own keys that the block's last and first row see
    if (L.k_end > a.prefix) {                                     // (never for packed rows)
        int len = a.own_len ? a.own_len[b0] : a.own_max;
        len = len < 0 ? 0 : len > a.own_max ? a.own_max : len;
        auto sees = [&](int i) {
            const int v = a.causal ? len - a.queries + i + 1 : len;
            return v < 0 ? 0 : v > len ? len : v;
        };
#pragma unroll
        for (int t = 0; t < RT; ++t) vis[t] = sees(row_i[t]);
        vis_top = sees(((tile + 1) * BM < n_rows ? (tile + 1) * BM - 1 : n_rows - 1) / grp);
        vis_low = sees(tile * BM / grp);
    }
    const int c0 = L.k_begin + chunk * L.chunk;
    const int c1 = c0 + L.chunk < L.k_end ? c0 + L.chunk : L.k_end;
    const int p0 = c0, p1 = c1 < a.prefix ? c1 : a.prefix;        // prefix keys [p0, p1)
    const int o0 = c0 > a.prefix ? c0 - a.prefix : 0;             // own keys [o0, o1)
    const int o1 = c1 - a.prefix < vis_top ? c1 - a.prefix : vis_top;
    const int np = p1 > p0 ? (p1 - p0 + KT - 1) / KT : 0;
    const int no = o1 > o0 ? (o1 - o0 + KT - 1) / KT : 0;
    const int stages = np + no;

    // ---- a stage's keys or values, through a descriptor that ends with the stage's last valid key: keys behind it read as zeros
    // whatever lies there ----
    const char* pk = static_cast<const char*>(a.pk) + (int64_t)hk * a.pk_hs * 2;
    const char* pv = static_cast<const char*>(a.pv) + (int64_t)hk * a.pv_hs * 2;
    const char* ok = static_cast<const char*>(a.ok) + ((int64_t)b0 * a.ok_bs + (int64_t)hk * a.ok_hs) * 2;
    const char* ov = static_cast<const char*>(a.ov) + ((int64_t)b0 * a.ov_bs + (int64_t)hk * a.ov_hs) * 2;
    auto rows_of = [&](int s, bool values, int64_t& stride) {
        const bool own = s >= np;
        const int k0 = own ? o0 + (s - np) * KT : p0 + s * KT;
        const int left = (own ? o1 : p1) - k0, valid = left < KT ? left : KT;
        stride = own ? (values ? a.ov_ss : a.ok_ss) : (values ? a.pv_ss : a.pk_ss);
        const char* base = (own ? (values ? ov : ok) : (values ? pv : pk)) + (int64_t)k0 * stride * 2;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, (int)((valid - 1) * stride * 2 + ROWB), 0x00020000);
    };
    const int w4 = BYWAVE ? 0 : wave;
    auto bring = [&](int s, bool values, char* to) {
        int64_t stride;
        const auto r = rows_of(s, values, stride);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int pc = i + w4 * PIECES, key = pc * RPP + lane / SLOTS, t = (lane % SLOTS) ^ swz<DIM>(key);
            dma16(r, to + pc * 1024, key * (int)stride * 2 + t * 16);
        }
    };
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    s8 kreg[2][BYWAVE ? KB : 1][DS];                              // by wave: the K operand, this tile's and the next one's
    auto load_k = [&](int s, int buf) {
        int64_t stride;
        const auto r = rows_of(s, false, stride);
#pragma unroll
        for (int kb = 0; kb < (BYWAVE ? KB : 0); ++kb)
#pragma unroll
            for (int d = 0; d < DS; ++d)
                kreg[buf][kb][d] = __builtin_bit_cast(s8, (u4)__builtin_amdgcn_raw_buffer_load_b128(r, (kb * 16 + l15) * (int)stride * 2 + (32 * d + 8 * g) * 2, 0, 0));
    };
    const int first = BYWAVE ? wave : 0, step = BYWAVE ? 4 : 1;
    if (first < stages) {
        if constexpr (BYWAVE) {
            load_k(first, 0);
            bring(first, true, lds);
        } else {
            bring(0, false, lds);
            bring(0, true, lds + 3 * TILE);
            if (stages > 1) bring(1, false, lds + TILE);
        }
    }

    // ---- Q as the B operand: lane (row l15, dims 32 s + 8 g ..) ----
    s8 q[RT][DS];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const short* p = static_cast<const short*>(a.q) + row_b[t] * a.q_bs + row_i[t] * a.q_ss + row_h[t] * a.q_hs + 8 * g;
#pragma unroll
        for (int s = 0; s < DS; ++s) q[t][s] = *reinterpret_cast<const s8*>(p + 32 * s);
    }

    f32x4 o[RT][DB];
    float m[RT], l[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float scale2 = a.scale * kLog2e;
    const int kswz = swz<DIM>(l15), krow = l15 * ROWB;            // K: key l15 of a 16-key block
    const int vkey = 4 * g + (l15 >> 2);                          // V: this lane's source key of a 16-key block
    const int vrow = vkey * ROWB + (l15 & 1) * 8, vsl = ((l15 & 3) >> 1) ^ swz<DIM>(vkey);

    auto scores = [&](const char* kt, int buf, f32x4 (&sc)[KB][RT]) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int t = 0; t < RT; ++t) sc[kb][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < DS; ++d) {
                s8 kf;
                if constexpr (BYWAVE) kf = kreg[buf][kb][d];
                else kf = *reinterpret_cast<const s8*>(kt + kb * 16 * ROWB + krow + (((4 * d + g) ^ kswz) << 4));
#pragma unroll
                for (int t = 0; t < RT; ++t) sc[kb][t] = Mma<T>::mul(kf, q[t][d], sc[kb][t]);
            }
        }
    };
    // masks of unit `u` of stage s, and the running maximum brought above the scores less 2^8
    auto settle = [&](int s, int u, f32x4 (&sc)[KB][RT]) {
        const bool own = s >= np;
        const int k0 = (own ? o0 + (s - np) * KT : p0 + s * KT) + 32 * u;
        const int end = own ? o1 : p1;
        if (k0 + 32 > end || (own && k0 + 32 > vis_low)) {        // keys behind the chunk's end, own keys a row does not see
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const int lim = own && vis[t] < end ? vis[t] : end;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (k0 + kb * 16 + 4 * g + r >= lim) sc[kb][t][r] = -INFINITY;
            }
        }
        float top[RT];
        bool move = false;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            top[t] = sc[0][t][0];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) top[t] = fmaxf(top[t], sc[kb][t][r]);
            top[t] *= scale2;
            move |= top[t] > m[t] + 8.f;
        }
        if (__any(move)) {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const float mn = fmaxf(m[t], over_groups_max(top[t]));
                const float k = mn == -INFINITY ? 0.f : exp2f(m[t] - mn);
                l[t] *= k;
#pragma unroll
                for (int d = 0; d < DB; ++d) o[t][d] *= k;
                m[t] = mn;
            }
        }
    };
    // P^T as the B operand of the unit's products, its sum into l
    auto weights = [&](const f32x4 (&sc)[KB][RT], s8 (&p)[RT]) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const float base = m[t] == -INFINITY ? 0.f : m[t];    // nothing seen yet: every p is 2^-inf = 0
            float e[8];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[0][t][r], scale2, -base));
                e[4 + r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[1][t][r], scale2, -base));
            }
            l[t] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
            struct { unsigned u[4]; } w;
#pragma unroll
            for (int r = 0; r < 4; ++r) w.u[r] = Mma<T>::pack(e[2 * r], e[2 * r + 1]);
            p[t] = __builtin_bit_cast(s8, w);
        }
    };
    // O^T += V^T P^T over 32 keys.  AHEAD fragments are on their way from LDS at any time, the first ones asked for before the softmax
    // ends (as the compiler orders it alone, each product waits for its own read)
    constexpr int AHEAD = 4;
    s8 vf[AHEAD];
    auto v_frag = [&](const char* vt, int d) {
        const char* at = vt + vrow + ((vsl ^ (2 * d)) << 4);
        const s4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)at);
        const s4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(at + 16 * ROWB));
        return __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto values_ahead = [&](const char* vt) {
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) vf[d] = v_frag(vt, d);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto values = [&](const char* vt, const s8 (&p)[RT]) {
#pragma unroll
        for (int d = 0; d < DB; ++d) {
#pragma unroll
            for (int t = 0; t < RT; ++t) o[t][d] = Mma<T>::mul(vf[d % AHEAD], p[t], o[t][d]);
            if (d + AHEAD < DB) vf[d % AHEAD] = v_frag(vt, d + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    s8 p[RT];
    if constexpr (BYWAVE) {
        auto one = [&](int s, int buf) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    // the other slot's reads are done
            const bool more = s + step < stages;
            if (more) {
                load_k(s + step, buf ^ 1);
                bring(s + step, true, lds + (buf ^ 1) * TILE);
            }
            f32x4 sc[KB][RT];
            scores(nullptr, buf, sc);
            settle(s, 0, sc);
            weights(sc, p);
            if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PIECES + KB * DS) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            values_ahead(lds + buf * TILE);
            values(lds + buf * TILE, p);
        };
        for (int s = first; s < stages; s += 2 * step) {
            one(s, 0);
            if (s + step < stages) one(s + step, 1);
        }
    } else if (stages > 0) {
        f32x4 sc[KB][RT], nx[KB][RT];
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        scores(lds, 0, sc);
        const char* kt = lds;                                     // K of stage s, s + 1; V of s
        char* kn = lds + TILE;
        char* k2 = lds + 2 * TILE;
        char* vt = lds + 3 * TILE;
        char* vn = lds + 4 * TILE;
        for (int s = 0; s < stages; ++s) {
            // K of s + 1 and V of s are in LDS, and every wave has left K and V of s - 1
            if (s > 0) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
            }
            if (s + 2 < stages) bring(s + 2, false, k2);
            if (s + 1 < stages) bring(s + 1, true, vn);
            settle(s, 0, sc);
            scores(kt + 32 * ROWB, 0, nx);
            weights(sc, p);
            values_ahead(vt);
            values(vt, p);
            settle(s, 1, nx);
            scores(kn, 0, sc);                                    // (the last stage: what lies there, not used)
            weights(nx, p);
            values_ahead(vt + 32 * ROWB);
            values(vt + 32 * ROWB, p);
            char* was = const_cast<char*>(kt);
            kt = kn;
            kn = k2;
            k2 = was;
            was = vt;
            vt = vn;
            vn = was;
        }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) l[t] = over_groups_sum(l[t]);

    if constexpr (BYWAVE) {                                       // the four waves' results join in order
        __syncthreads();                                          // the rings are free
        float* jo = reinterpret_cast<float*>(lds_all);            // [4][16 rows][DIM + 4]
        float* jm = jo + 4 * 16 * (DIM + 4);                      // [4][16], then the sums
#pragma unroll
        for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4*>(jo + (wave * 16 + l15) * (DIM + 4) + 16 * d + 4 * g) = o[0][d];
        if (g == 0) {
            jm[wave * 16 + l15] = m[0];
            jm[64 + wave * 16 + l15] = l[0];
        }
        __syncthreads();
        if (wave != 0) return;
        float mt = fmaxf(fmaxf(jm[l15], jm[16 + l15]), fmaxf(jm[32 + l15], jm[48 + l15]));
        const float base = mt == -INFINITY ? 0.f : mt;
        float lt = 0.f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[0][d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float k = exp2f(jm[w * 16 + l15] - base);
            lt += k * jm[64 + w * 16 + l15];
#pragma unroll
            for (int d = 0; d < DB; ++d) o[0][d] += k * *reinterpret_cast<const f32x4*>(jo + (w * 16 + l15) * (DIM + 4) + 16 * d + 4 * g);
        }
        m[0] = mt;
        l[0] = lt;
    }
    // ---- results: lane (row l15) holds dims 16 d + 4 g + r ----
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        if (!row_ok[t]) continue;
        const bool some = l[t] > 0.f || l[t] != l[t];             // a NaN sum is a result, an empty row is not
        const float inv = some ? 1.f / l[t] : 0.f;
        const float lse2 = some ? m[t] + log2f(l[t]) : -INFINITY;
        const int64_t row = ((int64_t)row_b[t] * a.queries + row_i[t]) * a.heads + row_h[t];
        if (slots == 1) {
            T* out = static_cast<T*>(a.out) + row * DIM + 4 * g;
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = some ? o[t][d][r] * inv : 0.f;
                store_vec<T, 4>(out + 16 * d, v);
            }
            if (a.lse && g == 0) a.lse[((int64_t)row_b[t] * a.heads + row_h[t]) * a.queries + row_i[t]] = lse2 * kLn2;
        } else {
            const int64_t rows = (int64_t)a.batch * a.queries * a.heads, at = (int64_t)(L.slot0 + chunk) * rows + row;
            float* out = a.work + at * DIM + 4 * g;
#pragma unroll
            for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4*>(out + 16 * d) = some ? o[t][d] * inv : f32x4{0.f, 0.f, 0.f, 0.f};
            if (g == 0) (a.work + (int64_t)slots * rows * DIM)[at] = lse2;
        }
    }
}

// The first `n0` blocks work on launch A, the others on B: the packed prefix and the own keys run beside each other.  KIND 0: by
// wave, 1, 2: by rows.
template <class T, int DIM, int KIND_A, int KIND_B>
__global__ __launch_bounds__(256, 2) void prefix_attention_kernel(const PrefixAttnArgs a, const PrefixAttnLaunch A, const PrefixAttnLaunch B, int n0,
                                                                  int slots) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int block = blockIdx.x;
    if constexpr (KIND_A == KIND_B) {
        const bool second = block >= n0;
        const PrefixAttnLaunch L = second ? B : A;
        attend<T, DIM, KIND_A == 0 ? 1 : KIND_A, KIND_A == 0>(a, L, slots, second ? block - n0 : block, second ? (int)gridDim.x - n0 : n0, lds);
    } else if (block < n0) {
        attend<T, DIM, KIND_A == 0 ? 1 : KIND_A, KIND_A == 0>(a, A, slots, block, n0, lds);
    } else {
        attend<T, DIM, KIND_B == 0 ? 1 : KIND_B, KIND_B == 0>(a, B, slots, block - n0, (int)gridDim.x - n0, lds);
    }
}

// Joins a row's partial results: out = sum_s 2^(lse_s - max) o_s / sum_s 2^(lse_s - max).  One wave a row, a lane a partial
// result's weight (at most 64), then a lane two columns or one.
template <class T, int DIM>
__global__ __launch_bounds__(256) void prefix_attention_join_kernel(const PrefixAttnArgs a, int slots, int rows) {
    constexpr int W = DIM / 64;
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= rows) return;
    const float mine = lane < slots ? a.work[(int64_t)slots * rows * DIM + (int64_t)lane * rows + row] : -INFINITY;
    const float top = wave_highest(mine), base = top == -INFINITY ? 0.f : top;
    const float k = exp2f(mine - base);                           // NaN stays NaN
    const float sum = wave_total(k);
    float acc[W];
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = 0.f;
    const float* o = a.work + (int64_t)row * DIM + lane * W;
#pragma unroll 8
    for (int s = 0; s < slots; ++s) {
        float v[W];
        load_vec<float, W>(o + (int64_t)s * rows * DIM, v);
        const float ks = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(k), s));
#pragma unroll
        for (int i = 0; i < W; ++i) acc[i] += ks * v[i];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] *= inv;
    store_vec<T, W>(static_cast<T*>(a.out) + (int64_t)row * DIM + lane * W, acc);
    if (a.lse && lane == 0) {
        const int h = row % a.heads, bq = row / a.heads, b = bq / a.queries, i = bq % a.queries;
        a.lse[((int64_t)b * a.heads + h) * a.queries + i] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
    }
}

template <class T, int DIM, int KIND_A, int KIND_B>
hipError_t launch_kinds(const PrefixAttnArgs& a, const PrefixAttnPlan& p, hipStream_t stream) {
    constexpr int LA = lds_bytes<DIM, KIND_A == 0>(), LB = lds_bytes<DIM, KIND_B == 0>(), LDS = LA > LB ? LA : LB;
    static_assert((KIND_A != 0 && KIND_B != 0) || LDS >= (4 * 16 * (DIM + 4) + 128) * 4, "the join fits the rings");
    static_assert(LDS <= 80 * 1024, "two blocks a CU");
    if (LDS > 64 * 1024) {
        static PerDevice<int> set;
        int& done = set.get();
        if (!done) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(prefix_attention_kernel<T, DIM, KIND_A, KIND_B>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
            if (e != hipSuccess) return e;
            done = 1;
        }
    }
    auto blocks = [&](const PrefixAttnLaunch& l) { return (int64_t)(l.packed ? 1 : a.batch) * a.kv_heads * l.tiles * l.chunks; };
    const int64_t n0 = blocks(p.l[0]), n1 = p.n > 1 ? blocks(p.l[1]) : 0;
    prefix_attention_kernel<T, DIM, KIND_A, KIND_B><<<dim3((unsigned)(n0 + n1)), 256, LDS, stream>>>(a, p.l[0], p.l[1], (int)n0, p.slots);
    return hipGetLastError();
}

template <class T, int DIM>
hipError_t launch_dim(const PrefixAttnArgs& a, const PrefixAttnPlan& p, hipStream_t stream) {
    const int ka = p.l[0].kind, kb = p.n > 1 ? p.l[1].kind : ka;   // the packed prefix has at least the own keys' rows: ka >= kb
    hipError_t e;
    if (ka == 0) e = launch_kinds<T, DIM, 0, 0>(a, p, stream);
    else if (ka == 1) e = kb == 0 ? launch_kinds<T, DIM, 1, 0>(a, p, stream) : launch_kinds<T, DIM, 1, 1>(a, p, stream);
    else e = kb == 0 ? launch_kinds<T, DIM, 2, 0>(a, p, stream) : kb == 1 ? launch_kinds<T, DIM, 2, 1>(a, p, stream) : launch_kinds<T, DIM, 2, 2>(a, p, stream);
    if (e != hipSuccess || p.slots == 1) return e;
    const int rows = a.batch * a.queries * a.heads;
    prefix_attention_join_kernel<T, DIM><<<dim3((unsigned)((rows + 3) / 4)), 256, 0, stream>>>(a, p.slots, rows);
    return hipGetLastError();
}

}  // namespace

PrefixAttnPlan prefix_attention_plan(const PrefixAttnArgs& a, int cus) {
    PrefixAttnPlan plan;
    const int grp = a.heads / a.kv_heads;
    const int64_t rows_own = (int64_t)a.queries * grp;
    auto add = [&](bool packed, int k_begin, int k_end) {
        PrefixAttnLaunch l{};
        l.packed = packed;
        l.k_begin = k_begin;
        l.k_end = k_end;
        const int64_t rows = rows_own * (packed ? a.batch : 1);
        l.kind = rows <= 16 ? 0 : rows <= 64 ? 1 : 2;
        const int bm = l.kind == 0 ? 16 : 64 * l.kind;
        l.tiles = (int)((rows + bm - 1) / bm);
        const int64_t items = (int64_t)(packed ? 1 : a.batch) * a.kv_heads * l.tiles;
        const int keys = k_end - k_begin, unit = 128;
        // fill the chip (two blocks a CU) with chunks of at least 256 keys (512 for the widest tiles, whose partial results are the
        // largest); at most 32 of them, so that a wave of the join holds all weights
        int64_t n = (2 * cus + items - 1) / items;
        n = std::min<int64_t>(n, std::max(1, keys / (l.kind == 2 ? 512 : 256)));
        n = std::min<int64_t>(n, 32);
        l.chunk = (int)std::max<int64_t>(unit, ((keys + n - 1) / n + unit - 1) / unit * unit);   // no keys at all: one empty chunk
        l.chunks = std::max(1, (keys + l.chunk - 1) / l.chunk);
        l.slot0 = plan.slots;
        plan.slots += l.chunks;
        plan.l[plan.n++] = l;
    };
    if (a.batch > 1 && a.prefix >= 256 && rows_own < 64) {
        add(true, 0, a.prefix);
        if (a.own_max > 0) add(false, a.prefix, a.prefix + a.own_max);
        else plan.l[1] = plan.l[0];
    } else {
        add(false, 0, a.prefix + a.own_max);
        plan.l[1] = plan.l[0];
    }
    return plan;
}

int64_t prefix_attention_work_floats(const PrefixAttnArgs& a, const PrefixAttnPlan& p) {
    return p.slots > 1 ? (int64_t)p.slots * a.batch * a.queries * a.heads * (a.dim + 1) : 0;
}

hipError_t launch_prefix_attention(const PrefixAttnArgs& a, const PrefixAttnPlan& p, hipStream_t stream) {
    if (a.dtype == CMDI_DT_BF16) return a.dim == 128 ? launch_dim<Bf16, 128>(a, p, stream) : launch_dim<Bf16, 64>(a, p, stream);
    return a.dim == 128 ? launch_dim<_Float16, 128>(a, p, stream) : launch_dim<_Float16, 64>(a, p, stream);
}

}  // namespace cmdi
