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
// Matrix instructions: v_mfma_f32_32x32x16 (bf16 / f16 operands, fp32 sums; an eighth more throughput here than 16x16x32).
// S^T = K Q^T puts a row of Q into a lane column, so maximum and sum stay in the lane but for one exchange, and S^T's accumulators
// ARE the operand of O^T += V^T P^T: lane half h holds keys 8 i + 4 h + r of a tile, and the transposed LDS reads
// (ds_read_b64_tr_b16) fetch V in that same order.  P is rounded to the operands' 16 bits (half a step relative, as the matrix unit
// asks), its sum l is taken before that.
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
    static __device__ __forceinline__ f32x16 mul(s8 a, s8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ unsigned pack(float x, float y) { return __builtin_bit_cast(unsigned, b2{(__bf16)x, (__bf16)y}); }
};
template <> struct Mma<_Float16> {
    static __device__ __forceinline__ f32x16 mul(s8 a, s8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ unsigned pack(float x, float y) { return __builtin_bit_cast(unsigned, h2{(_Float16)x, (_Float16)y}); }
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

// A key row in LDS is DIM elements in 16-byte slots; slot t of key k is stored at t ^ swz(k).  A ds_read_b128 serves lanes {0-3,
// 12-15, 20-27} and so on together: 16 keys at one slot have to lie in 16 different bank quads.  A transposed read takes 4 keys at
// two neighbouring slots, whose pairs have to differ.
template <int DIM>
__device__ __forceinline__ int swz(int k) {
    return DIM == 128 ? ((k & 3) << 2) | ((k >> 2) & 3) : (((k >> 1) & 3) << 1) | ((k >> 3) & 1);
}

// 16 bytes a lane from `offset` behind the descriptor's base to LDS at `to`, lane after lane.  In assembly because the compiler
// puts a wait for ALL requests in front of the next transposed LDS read when it knows of one: the waits below count them instead.
// (It has no result register; a wait that the compiler counts for its own loads only gets longer by requests it does not know of.)
typedef unsigned u4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void dma16(u4 descriptor, char* to, int offset) {
    const unsigned at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)to;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(at), "v"(offset), "s"(descriptor) : "memory", "m0");
}
// a raw buffer: `bytes` from `base`, accesses behind them return zeros
__device__ __forceinline__ u4 buffer(const char* base, int bytes) {
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    return u4{(unsigned)at, (unsigned)(at >> 32) & 0xffffu, (unsigned)bytes, 0x00020000u};
}

template <int DIM, bool BYWAVE>
constexpr int lds_bytes() {
    // by rows: three tiles of 64 keys, two of 64 values; by wave: each of the four waves has two tiles of 32 values
    return BYWAVE ? 4 * 2 * 32 * DIM * 2 : 5 * 64 * DIM * 2;
}

// The item's keys, tile by tile: its part of the prefix, then its part of the own keys.  A walker stands at one tile; a step costs
// a handful of scalar instructions but where it crosses into the own keys.
struct Segment { const char *k, *v; int ks, vs, n; };             // first key's addresses, bytes between keys, number of keys
template <int KT>
struct Walker {
    int tile, at;                                                 // tile number; first key of the tile within its segment
    bool own;
    __device__ __forceinline__ void go(int t, int prefix_tiles) {
        tile = t;
        own = t >= prefix_tiles;
        at = (own ? t - prefix_tiles : t) * KT;
    }
};

// One item: a tile of rows over a chunk of keys.
//   By rows: wave w owns 32 of 128 rows; K and V come in 64-key tiles through LDS (LDS-DMA, a ring of three tiles of K, of two of V).
//   A tile is two units of 32 keys; the scores of the next unit are multiplied while the softmax of this one runs, so the matrix
//   units work under the exponentials.
//   BYWAVE: at most 32 rows (few queries): a wave takes every fourth 32-key tile, its K straight into registers, its V through its own
//   two LDS tiles, no barrier until the four waves join at the end.
// A row's maximum is moved only when a score passes it by 2^8: until then its p stay below 256, which changes no relative
// rounding and saves the exchange between the lanes and the rescaling of o.
template <class T, int DIM, bool BYWAVE>
__device__ __forceinline__ void attend(const PrefixAttnArgs& a, const PrefixAttnLaunch& L, int slots, int block, int blocks, char* lds_all) {
    constexpr int KT = BYWAVE ? 32 : 64, ROWB = DIM * 2, TILE = KT * ROWB, DS = DIM / 16, DB = DIM / 32;
    constexpr int SLOTS = DIM / 8, RPP = 64 / SLOTS;              // 16-byte slots of a key row; key rows of a 1-KiB piece
    constexpr int PIECES = KT / RPP / (BYWAVE ? 1 : 4);           // pieces of a tile that a wave brings
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    char* lds = lds_all + (BYWAVE ? wave * 2 * TILE : 0);

    // ---- which item ----
    const int grp = a.heads / a.kv_heads;
    const int id = xcd_remap(block, blocks);
    const int tile = id % L.tiles, rest = id / L.tiles;
    const int chunk = rest % L.chunks, bh = rest / L.chunks;
    const int hk = bh % a.kv_heads, b0 = bh / a.kv_heads;         // packed: b0 = 0, the sample comes from the row
    const int n_rows = (L.packed ? a.batch : 1) * a.queries * grp;
    constexpr int BM = BYWAVE ? 32 : 128;
    const int row0 = tile * BM + (BYWAVE ? 0 : wave * 32);
    const bool busy = row0 < n_rows;                              // this wave has rows (it brings keys in any case)
    const bool row_ok = row0 + l31 < n_rows;
    const int r = row_ok ? row0 + l31 : n_rows - 1;               // this lane's row
    const int rq = r / grp, row_h = hk * grp + r - rq * grp, row_b = L.packed ? rq / a.queries : b0;
    const int row_i = L.packed ? rq - row_b * a.queries : rq;

    // ---- own keys that the lane's row, the block's last row and the wave's first one see ----
    int vis = 0, vis_top = 0, vis_low = 0;
    if (L.k_end > a.prefix) {                                     // (never for packed rows)
        int len = a.own_len ? a.own_len[b0] : a.own_max;
        len = len < 0 ? 0 : len > a.own_max ? a.own_max : len;
        auto sees = [&](int i) {
            const int v = a.causal ? len - a.queries + i + 1 : len;
            return v < 0 ? 0 : v > len ? len : v;
        };
        vis = sees(row_i);
        vis_top = sees(((tile + 1) * BM < n_rows ? (tile + 1) * BM - 1 : n_rows - 1) / grp);
        vis_low = sees(row0 / grp);
    }
    // ---- its keys: prefix [p0, p1), own [o0, o1) ----
    const int c0 = L.k_begin + chunk * L.chunk;
    const int c1 = c0 + L.chunk < L.k_end ? c0 + L.chunk : L.k_end;
    const int p1 = c1 < a.prefix ? c1 : a.prefix;
    const int o0 = c0 > a.prefix ? c0 - a.prefix : 0;
    const int o1 = c1 - a.prefix < vis_top ? c1 - a.prefix : vis_top;
    auto segment = [&](bool own) {
        Segment g;
        g.n = own ? (o1 > o0 ? o1 - o0 : 0) : (p1 > c0 ? p1 - c0 : 0);
        const int from = own ? o0 : c0;
        g.ks = (int)((own ? a.ok_ss : a.pk_ss) * 2);
        g.vs = (int)((own ? a.ov_ss : a.pv_ss) * 2);
        const char* k = static_cast<const char*>(own ? a.ok : a.pk);
        const char* v = static_cast<const char*>(own ? a.ov : a.pv);
        g.k = k + ((own ? b0 * a.ok_bs : 0) + hk * (own ? a.ok_hs : a.pk_hs)) * 2 + (int64_t)from * g.ks;
        g.v = v + ((own ? b0 * a.ov_bs : 0) + hk * (own ? a.ov_hs : a.pv_hs)) * 2 + (int64_t)from * g.vs;
        return g;
    };
    const int np = p1 > c0 ? (p1 - c0 + KT - 1) / KT : 0;
    const int no = o1 > o0 ? (o1 - o0 + KT - 1) / KT : 0;
    const int stages = np + no;
    const int first = BYWAVE ? wave : 0, step = BYWAVE ? 4 : 1;

    // A tile's keys or values through a descriptor that ends with the segment's last key: keys behind it read as zeros whatever lies
    // there.  The lane's offset within a tile changes with the segment's stride only.
    struct Cursor { Walker<KT> w; Segment g; };
    auto start = [&](Cursor& c, int t) {
        c.w.go(t, np);
        c.g = segment(c.w.own);
    };
    auto advance = [&](Cursor& c, int by) {
        const bool was = c.w.own;
        c.w.go(c.w.tile + by, np);
        if (c.w.own != was) c.g = segment(true);
    };
    auto tile_of = [&](const Cursor& c, bool values, const char*& base, int& bytes) {
        const int left = c.g.n - c.w.at, valid = left < KT ? left : KT, stride = values ? c.g.vs : c.g.ks;
        base = (values ? c.g.v : c.g.k) + (int64_t)c.w.at * stride;
        bytes = (valid - 1) * stride + ROWB;
    };
    const int w4 = BYWAVE ? 0 : wave;
    auto bring = [&](const Cursor& c, bool values, char* to) {
        const char* base;
        int bytes;
        tile_of(c, values, base, bytes);
        const u4 d = buffer(base, bytes);
        const int stride = values ? c.g.vs : c.g.ks;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int pc = i + w4 * PIECES, key = pc * RPP + lane / SLOTS, t = (lane % SLOTS) ^ swz<DIM>(key);
            dma16(d, to + pc * 1024, key * stride + t * 16);
        }
    };
    s8 kreg[2][BYWAVE ? DS : 1];                                  // by wave: the K operand, this tile's and the next one's
    auto load_k = [&](const Cursor& c, int buf) {
        const char* base;
        int bytes;
        tile_of(c, false, base, bytes);
        const auto d = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, bytes, 0x00020000);
#pragma unroll
        for (int s = 0; s < (BYWAVE ? DS : 0); ++s)
            kreg[buf][s] = __builtin_bit_cast(s8, (u4)__builtin_amdgcn_raw_buffer_load_b128(d, l31 * c.g.ks + 32 * s + 16 * hi, 0, 0));
    };
    Cursor ck, cv;                                                // the next tile of K and of V to ask for
    start(ck, first);
    cv = ck;
    if (first < stages) {
        if constexpr (BYWAVE) {
            load_k(ck, 0);
            bring(cv, true, lds);
        } else {
            bring(ck, false, lds);
            bring(cv, true, lds + 3 * TILE);
            advance(ck, 1);
            if (stages > 1) bring(ck, false, lds + TILE);
            advance(ck, 1);
        }
        advance(cv, step);
    }

    // ---- Q as the B operand: lane (row l31, dims 16 s + 8 hi ..) ----
    s8 q[DS];
    {
        const short* p = static_cast<const short*>(a.q) + row_b * a.q_bs + row_i * a.q_ss + row_h * a.q_hs + 8 * hi;
#pragma unroll
        for (int s = 0; s < DS; ++s) q[s] = *reinterpret_cast<const s8*>(p + 16 * s);
    }

    f32x16 o[DB];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    const float scale2 = a.scale * kLog2e;
    const int kswz = swz<DIM>(l31), krow = l31 * ROWB;            // K: key l31 of a 32-key unit
    // V, transposed reads: group G = lane / 16, lane L of it points at key 4 (G / 2) + L / 4, dims 16 (G % 2) + 4 (L % 4) .. + 3; the
    // group's lane i receives keys 4 (G / 2) .. + 3 of dim 16 (G % 2) + i
    const int vkey = 4 * hi + ((lane & 15) >> 2);
    const int vrow = vkey * ROWB + (lane & 1) * 8, vsl = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const int vs0 = vsl ^ swz<DIM>(vkey), vs1 = vsl ^ swz<DIM>(vkey + 8);

    // the K fragments of a unit are asked for before the softmax of the one before it begins
    s8 kf[BYWAVE ? 1 : DS];
    auto keys_ahead = [&](const char* kt) {
#pragma unroll
        for (int s = 0; s < (BYWAVE ? 0 : DS); ++s) kf[s] = *reinterpret_cast<const s8*>(kt + krow + (((2 * s + hi) ^ kswz) << 4));
        __builtin_amdgcn_sched_barrier(0);
    };
    auto scores = [&](int buf, f32x16& sc) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
        for (int s = 0; s < DS; ++s) {
            if constexpr (BYWAVE) sc = Mma<T>::mul(kreg[buf][s], q[s], sc);
            else sc = Mma<T>::mul(kf[s], q[s], sc);
        }
    };
    // masks of the unit whose first key is `k0` of the segment's, and the running maximum brought above the scores less 2^8
    auto settle = [&](const Walker<KT>& w, int unit, f32x16& sc) {
        const int k0 = w.at + 32 * unit, n = w.own ? o1 - o0 : p1 - c0;
        if (k0 + 32 > n || (w.own && o0 + k0 + 32 > vis_low)) {   // keys behind the chunk's end, own keys a row does not see
            const int lim = w.own && vis - o0 < n ? vis - o0 : n;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (k0 + mfma32_row(i, lane) >= lim) sc[i] = -INFINITY;
        }
        float top = sc[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, sc[i]);
        top *= scale2;
        if (__any(top > m + 8.f)) {
            const float mn = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
            const float k = mn == -INFINITY ? 0.f : exp2f(m - mn);
            l *= k;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= k;
            m = mn;
        }
    };
    // P^T as the B operand of the unit's two 16-key products, its sum into l
    s8 p[2];
    auto weights = [&](const f32x16& sc) {
        const float base = m == -INFINITY ? 0.f : m;              // nothing seen yet: every p is 2^-inf = 0
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * kb + i], scale2, -base));
            l += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
            struct { unsigned u[4]; } w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w.u[i] = Mma<T>::pack(e[2 * i], e[2 * i + 1]);
            p[kb] = __builtin_bit_cast(s8, w);
        }
    };
    // O^T += V^T P^T over 32 keys.  AHEAD fragments are on their way from LDS at any time, the first ones asked for before the softmax
    // ends (as the compiler orders it alone, each product waits for its own read)
    constexpr int FRAGS = 2 * DB, AHEAD = 4;
    s8 vf[AHEAD];
    auto v_frag = [&](const char* vt, int i) {
        const char* at = vt + (i / DB) * 16 * ROWB + vrow;
        const int db = i % DB;
        const s4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(at + ((vs0 ^ (4 * db)) << 4)));
        const s4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(at + 8 * ROWB + ((vs1 ^ (4 * db)) << 4)));
        return __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto values_ahead = [&](const char* vt) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) vf[i] = v_frag(vt, i);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto values = [&](const char* vt) {
#pragma unroll
        for (int i = 0; i < FRAGS; ++i) {
            o[i % DB] = Mma<T>::mul(vf[i % AHEAD], p[i / DB], o[i % DB]);
            if (i + AHEAD < FRAGS) vf[i % AHEAD] = v_frag(vt, i + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    Walker<KT> now;                                               // the tile that is worked on
    now.go(first, np);
    if constexpr (BYWAVE) {
        auto one = [&](int buf) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    // the other tile's reads are done
            const bool more = now.tile + step < stages;
            if (more) {
                load_k(cv, buf ^ 1);
                bring(cv, true, lds + (buf ^ 1) * TILE);
                advance(cv, step);
            }
            f32x16 sc;
            scores(buf, sc);
            settle(now, 0, sc);
            weights(sc);
            if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PIECES + DS) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            values_ahead(lds + buf * TILE);
            values(lds + buf * TILE);
            now.go(now.tile + step, np);
        };
        while (now.tile < stages) {
            one(0);
            if (now.tile < stages) one(1);
        }
    } else if (stages > 0) {
        f32x16 sc, nx;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        // Q is there too: said to the compiler, which would otherwise wait for it (and for every request) in each turn of the loop
#pragma unroll
        for (int i = 0; i < DS; ++i) asm volatile("" : "+v"(q[i]));
        __syncthreads();
        if (busy) {
            keys_ahead(lds);
            scores(0, sc);
        }
        char *kt = lds, *kn = lds + TILE, *k2 = lds + 2 * TILE;   // K of this tile and the next two, V of this one and the next
        char *vt = lds + 3 * TILE, *vn = lds + 4 * TILE;
        for (int s = 0; s < stages; ++s) {
            // K of s + 1 and V of s are in LDS, and every wave has left K and V of s - 1
            if (s > 0) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
            }
            if (s + 2 < stages) {
                bring(ck, false, k2);
                advance(ck, 1);
            }
            if (s + 1 < stages) {
                bring(cv, true, vn);
                advance(cv, 1);
            }
            if (busy) {
                keys_ahead(kt + 32 * ROWB);
                settle(now, 0, sc);
                scores(0, nx);
                weights(sc);
                values_ahead(vt);
                values(vt);
                keys_ahead(kn);
                settle(now, 1, nx);
                scores(0, sc);                                    // (the last tile: what lies there, not used)
                weights(nx);
                values_ahead(vt + 32 * ROWB);
                values(vt + 32 * ROWB);
            }
            now.go(s + 1, np);
            char* was = kt;
            kt = kn;
            kn = k2;
            k2 = was;
            was = vt;
            vt = vn;
            vn = was;
        }
    }
    l += __shfl_xor(l, 32, 64);

    if constexpr (BYWAVE) {                                       // the waves join in a fixed order: 2 into 0 and 3 into 1, then 1 into 0
        float* jo = reinterpret_cast<float*>(lds_all);            // [2][32 rows][DIM + 4], then [2][m | l][32]
        float* jm = jo + 2 * 32 * (DIM + 4);
#pragma unroll
        for (int half = 2; half > 0; half >>= 1) {
            __syncthreads();                                      // the LDS is free
            if (wave >= half && wave < 2 * half) {
                float* to = jo + ((wave - half) * 32 + l31) * (DIM + 4) + 4 * hi;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<f32x4*>(to + 32 * d + 8 * i) = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
                if (hi == 0) {
                    jm[(wave - half) * 64 + l31] = m;
                    jm[(wave - half) * 64 + 32 + l31] = l;
                }
            }
            __syncthreads();
            if (wave < half) {
                const float mo = jm[wave * 64 + l31], lo = jm[wave * 64 + 32 + l31], mt = fmaxf(m, mo), base = mt == -INFINITY ? 0.f : mt;
                const float ka = exp2f(m - base), kb = exp2f(mo - base);
                const float* from = jo + (wave * 32 + l31) * (DIM + 4) + 4 * hi;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x4 v = *reinterpret_cast<const f32x4*>(from + 32 * d + 8 * i);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[d][4 * i + e] = ka * o[d][4 * i + e] + kb * v[e];
                    }
                l = ka * l + kb * lo;
                m = mt;
            }
        }
        if (wave != 0) return;
    }
    // ---- results: lane (row l31) holds dims 32 d + 8 i + 4 hi + e ----
    if (!row_ok) return;
    const bool some = l > 0.f || l != l;                          // a NaN sum is a result, an empty row is not
    const float inv = some ? 1.f / l : 0.f;
    const float lse2 = some ? m + log2f(l) : -INFINITY;
    const int64_t row = ((int64_t)row_b * a.queries + row_i) * a.heads + row_h;
    if (slots == 1) {
        T* out = static_cast<T*>(a.out) + row * DIM + 4 * hi;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = some ? o[d][4 * i + e] * inv : 0.f;
                store_vec<T, 4>(out + 32 * d + 8 * i, v);
            }
        if (a.lse && hi == 0) a.lse[((int64_t)row_b * a.heads + row_h) * a.queries + row_i] = lse2 * kLn2;
    } else {
        const int64_t rows = (int64_t)a.batch * a.queries * a.heads, at = (int64_t)(L.slot0 + chunk) * rows + row;
        float* out = a.work + at * DIM + 4 * hi;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = some ? o[d][4 * i + e] * inv : 0.f;
                *reinterpret_cast<f32x4*>(out + 32 * d + 8 * i) = v;
            }
        if (hi == 0) (a.work + (int64_t)slots * rows * DIM)[at] = lse2;
    }
}

// The first `n0` blocks work on launch A, the others on B: the packed prefix and the own keys run beside each other.
template <class T, int DIM, bool WAVE_A, bool WAVE_B>
__global__ __launch_bounds__(256, 2) void prefix_attention_kernel(const PrefixAttnArgs a, const PrefixAttnLaunch A, const PrefixAttnLaunch B, int n0,
                                                                  int slots) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int block = blockIdx.x;
    if constexpr (WAVE_A == WAVE_B) {
        const bool second = block >= n0;
        const PrefixAttnLaunch L = second ? B : A;
        attend<T, DIM, WAVE_A>(a, L, slots, second ? block - n0 : block, second ? (int)gridDim.x - n0 : n0, lds);
    } else if (block < n0) {
        attend<T, DIM, WAVE_A>(a, A, slots, block, n0, lds);
    } else {
        attend<T, DIM, WAVE_B>(a, B, slots, block - n0, (int)gridDim.x - n0, lds);
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

template <class T, int DIM, bool WAVE_A, bool WAVE_B>
hipError_t launch_kinds(const PrefixAttnArgs& a, const PrefixAttnPlan& p, hipStream_t stream) {
    constexpr int LA = lds_bytes<DIM, WAVE_A>(), LB = lds_bytes<DIM, WAVE_B>(), LDS = LA > LB ? LA : LB;
    static_assert(lds_bytes<DIM, true>() >= (2 * 32 * (DIM + 4) + 128) * 4, "the join fits the rings");
    static_assert(LDS <= 80 * 1024, "two blocks a CU");
    if (LDS > 64 * 1024) {
        static PerDevice<int> set;
        int& done = set.get();
        if (!done) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(prefix_attention_kernel<T, DIM, WAVE_A, WAVE_B>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
            if (e != hipSuccess) return e;
            done = 1;
        }
    }
    auto blocks = [&](const PrefixAttnLaunch& l) { return (int64_t)(l.packed ? 1 : a.batch) * a.kv_heads * l.tiles * l.chunks; };
    const int64_t n0 = blocks(p.l[0]), n1 = p.n > 1 ? blocks(p.l[1]) : 0;
    prefix_attention_kernel<T, DIM, WAVE_A, WAVE_B><<<dim3((unsigned)(n0 + n1)), 256, LDS, stream>>>(a, p.l[0], p.l[1], (int)n0, p.slots);
    return hipGetLastError();
}

template <class T, int DIM>
hipError_t launch_dim(const PrefixAttnArgs& a, const PrefixAttnPlan& p, hipStream_t stream) {
    // the packed prefix has at least the own keys' rows: by wave there, by wave here
    const hipError_t e = p.l[0].by_wave ? launch_kinds<T, DIM, true, true>(a, p, stream)
                         : p.l[1].by_wave ? launch_kinds<T, DIM, false, true>(a, p, stream)
                                          : launch_kinds<T, DIM, false, false>(a, p, stream);
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
        l.by_wave = rows <= 32;
        const int bm = l.by_wave ? 32 : 128;
        l.tiles = (int)((rows + bm - 1) / bm);
        const int64_t items = (int64_t)(packed ? 1 : a.batch) * a.kv_heads * l.tiles;
        const int keys = k_end - k_begin, unit = 128;
        // fill the chip (two blocks a CU) with chunks of at least 256 keys (512 for 128 rows, whose partial results are the
        // largest); at most 32 of them, so that a wave of the join holds all weights
        int64_t n = (2 * cus + items - 1) / items;
        n = std::min<int64_t>(n, std::max(1, keys / (l.by_wave ? 256 : 512)));
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
