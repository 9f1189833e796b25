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
// (ds_read_b64_tr_b16) fetch V in that same order.  P is rounded to the operands' 16 bits, as the matrix unit asks: half a step
// relative, and in f16 a weight below 2^-14 of that by a fixed step, so that a long tail of small weights would be lost from o.  Their
// p are therefore 2^LIFT times as large (below 2^15 with what the maximum may lag behind): the step is 2^-32 of the row's largest
// weight.  l is summed in fp32 before the rounding.
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
    static constexpr unsigned short TOP = 0x7f80;     // exponent of an infinity or a NaN
    static constexpr float LIFT = 0.f;                // p are 2^LIFT times their formula
    static __device__ __forceinline__ float up(short v) { return __uint_as_float((unsigned)(unsigned short)v << 16); }
    static __device__ __forceinline__ f32x16 mul(s8 a, s8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ unsigned pack(float x, float y) { return __builtin_bit_cast(unsigned, b2{(__bf16)x, (__bf16)y}); }
};
template <> struct Mma<_Float16> {
    static constexpr unsigned short TOP = 0x7c00;
    static constexpr float LIFT = 7.f;
    static __device__ __forceinline__ float up(short v) { return (float)__builtin_bit_cast(_Float16, v); }
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

// 16 bytes a lane from `offset` behind the descriptor's base to LDS at `to` + PLUS, lane after lane.  In assembly because the compiler
// puts a wait for ALL requests in front of the next transposed LDS read when it knows of one: the waits below count them instead.
// (It has no result register; a wait that the compiler counts for its own loads only gets longer by requests it does not know of.)
typedef unsigned u4 __attribute__((ext_vector_type(4)));
template <int PLUS>
__device__ __forceinline__ void dma16(u4 descriptor, unsigned to, int offset) {
    asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(offset), "s"(descriptor), "n"(PLUS)
                 : "memory", "m0", "scc");
}
// a raw buffer: `bytes` from `base`, accesses behind them return zeros
__device__ __forceinline__ u4 buffer(const char* base, int bytes) {
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    return u4{(unsigned)at, (unsigned)(at >> 32) & 0xffffu, (unsigned)bytes, 0x00020000u};
}
__device__ __forceinline__ unsigned lds_at(const char* p) { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p; }

template <int DIM, bool BYWAVE>
constexpr int lds_bytes() {
    // by rows: three tiles of 64 keys, two of 64 values; by wave: each of the four waves has two tiles of 32 values
    return BYWAVE ? 4 * 2 * 32 * DIM * 2 : 5 * 64 * DIM * 2;
}

// A lane's row: sample, query, head.
struct Row {
    bool ok;                              // it exists (else it repeats the last one)
    int b, i, h;
};

// Which rows and which keys an item has; the same in all lanes of a wave.
template <int BM, int KT>
struct Item {
    int chunk, n_rows, row0, hk, b0;      // row0: the wave's first row;  b0: the sample (packed: 0, it comes from the row)
    int len;                              // own keys of the sample
    int vis_low, vis_first;               // own keys that the wave's first row sees, and the block's
    int c0, p1, o0, o1;                   // prefix keys [c0, p1), own keys [o0, o1)
    int np, tiles;                        // tiles of KT keys: prefix ones, all

    __device__ __forceinline__ Item(const PrefixAttnArgs& a, const PrefixAttnLaunch& L, int block, int blocks, int first_row) {
        const int grp = a.heads / a.kv_heads;
        const int id = xcd_remap(block, blocks);
        const int tile = id % L.tiles, rest = id / L.tiles;
        const int bh = rest / L.chunks;
        chunk = rest % L.chunks;
        hk = bh % a.kv_heads;
        b0 = bh / a.kv_heads;
        n_rows = (L.packed ? a.batch : 1) * a.queries * grp;
        row0 = tile * BM + first_row;
        len = vis_low = vis_first = 0;
        int vis_top = 0;                                          // own keys that the block's last row sees
        if (L.k_end > a.prefix) {                                 // (never for packed rows)
            len = a.own_len ? a.own_len[b0] : a.own_max;
            len = len < 0 ? 0 : len > a.own_max ? a.own_max : len;
            vis_top = sees(a, ((tile + 1) * BM < n_rows ? (tile + 1) * BM - 1 : n_rows - 1) / grp);
            vis_low = sees(a, row0 / grp);
            vis_first = sees(a, tile * BM / grp);
        }
        c0 = L.k_begin + chunk * L.chunk;
        const int c1 = c0 + L.chunk < L.k_end ? c0 + L.chunk : L.k_end;
        p1 = c1 < a.prefix ? c1 : a.prefix;
        o0 = c0 > a.prefix ? c0 - a.prefix : 0;
        o1 = c1 - a.prefix < vis_top ? c1 - a.prefix : vis_top;
        np = p1 > c0 ? (p1 - c0 + KT - 1) / KT : 0;
        tiles = np + (o1 > o0 ? (o1 - o0 + KT - 1) / KT : 0);
    }
    // own keys that query i sees
    __device__ __forceinline__ int sees(const PrefixAttnArgs& a, int i) const {
        const int v = a.causal ? len - a.queries + i + 1 : len;
        return v < 0 ? 0 : v > len ? len : v;
    }
    // worked out anew at each use: kept over the loop it would cost registers that the loop has not got
    __device__ __forceinline__ Row row(const PrefixAttnArgs& a, const PrefixAttnLaunch& L, int l31) const {
        asm volatile("" : "+v"(l31));
        const int grp = a.heads / a.kv_heads;
        Row to;
        to.ok = row0 + l31 < n_rows;
        const int r = to.ok ? row0 + l31 : n_rows - 1;
        const int rq = r / grp;
        to.h = hk * grp + r - rq * grp;
        to.b = L.packed ? rq / a.queries : b0;
        to.i = L.packed ? rq - to.b * a.queries : rq;
        return to;
    }
};

// A walk over an item's keys or values, tile by tile: its part of the prefix, then of the own keys.  `left` keys from `at` on are in
// the segment.  A tile is read through a descriptor that ends with the segment's last key: what lies behind it reads as zeros.
template <class I, int DIM, int KT>
struct Walk {
    const char* at;
    int left, stride;                     // stride: bytes between keys
    bool own;
    __device__ __forceinline__ void enter(const PrefixAttnArgs& a, const I& it, bool values, bool own_keys, int skip) {
        own = own_keys;
        const int64_t ss = own ? (values ? a.ov_ss : a.ok_ss) : (values ? a.pv_ss : a.pk_ss);
        const int64_t hs = own ? (values ? a.ov_hs : a.ok_hs) : (values ? a.pv_hs : a.pk_hs);
        const int64_t bs = own ? (values ? a.ov_bs : a.ok_bs) : 0;
        stride = (int)(ss * 2);
        left = (own ? it.o1 - it.o0 : it.p1 - it.c0) - skip;
        at = static_cast<const char*>(own ? (values ? a.ov : a.ok) : (values ? a.pv : a.pk)) +
             (it.b0 * bs + it.hk * hs + (int64_t)((own ? it.o0 : it.c0) + skip) * ss) * 2;
    }
    __device__ __forceinline__ void start(const PrefixAttnArgs& a, const I& it, bool values, int tile) {
        const bool o = tile >= it.np;
        enter(a, it, values, o, (o ? tile - it.np : tile) * KT);
    }
    __device__ __forceinline__ u4 tile() const { return buffer(at, ((left < KT ? left : KT) - 1) * stride + DIM * 2); }
    // `by` tiles on; true where that entered the own keys
    __device__ __forceinline__ bool step(const PrefixAttnArgs& a, const I& it, bool values, int by) {
        at += (int64_t)by * KT * stride;
        left -= by * KT;
        if (__builtin_expect(left <= 0 && !own, 0)) {
            const int np = (it.p1 - it.c0 + KT - 1) / KT * KT, over = (it.p1 - it.c0 - left) - np;   // keys walked behind the prefix's last tile
            enter(a, it, values, true, over);
            return true;
        }
        return false;
    }
};

// Does any of a tile's `N` KiB in LDS hold an infinity or a NaN (the same answer in all lanes), and zeros for those of the lane's parts
// (`from`, then every 1 KiB).
typedef unsigned short us8 __attribute__((ext_vector_type(8)));
template <class T, int N>
__device__ __forceinline__ bool any_odd(const char* at, int lane) {
    us8 top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
        top = __builtin_elementwise_max(top, (us8)(*reinterpret_cast<const us8*>(at + i * 1024 + lane * 16) & (unsigned short)0x7fff));
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) odd |= top[e] >= Mma<T>::TOP;
    return __any(odd);
}
template <class T>
__device__ __forceinline__ void clear_odd(char* from, int n) {
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        us8 v = *reinterpret_cast<us8*>(from + i * 1024);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if ((v[e] & 0x7fff) >= Mma<T>::TOP) v[e] = 0;
        *reinterpret_cast<us8*>(from + i * 1024) = v;
    }
}

// A wave's 32 rows against 32 keys at a time.  A row's maximum is moved only when a score passes it by 2^8: until then its p stay
// below 256, which changes no relative rounding and saves the exchange between the lanes and the rescaling of o.
//
// With s the raw score and c = scale log2 e, p = 2^(s c - m c) is one multiply-add and one exponential: m c, rounded to fp32, is the same
// addend for all of a row's keys, but its rounding is a factor of p, and beyond |m c| = 2^27 one that leaves the operands' range.  So a
// row is FAR once |m c| passes 2^16: its scores have m taken off before they are scaled (exact where p is not 0).  A far row's limit is
// -inf, which sends every unit through the seldom taken path that does so.
constexpr float kFar = 65536.f;
template <class T, int DIM>
struct Rows32 {
    static constexpr int ROWB = DIM * 2, DS = DIM / 16, DB = DIM / 32, FRAGS = 2 * DB, AHEAD = 4;
    s8 q[DS], p[2], vf[AHEAD];
    f32x16 o[DB];
    float m, l, limit, base;              // m: largest raw score;  limit: a raw score above it moves m;  base: LIFT - m c, LIFT for far rows and unseen ones
    float scale2;                         // c
    int krow[DS], vat[DB], vat8[DB];      // LDS offsets of the lane's fragments within a 32-key unit

    // `keys_at`: where the ring of K lies in LDS (in the offsets, so that every slot is within reach of an instruction's constant)
    __device__ __forceinline__ Rows32(float scale, int lane, int keys_at) {
        const int l31 = lane & 31, hi = lane >> 5;
        m = -INFINITY;
        l = 0.f;
        limit = -INFINITY;
        base = Mma<T>::LIFT;
        scale2 = scale * kLog2e;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
        // K: key l31, dims 16 s + 8 hi ..
#pragma unroll
        for (int s = 0; s < DS; ++s) krow[s] = keys_at + l31 * ROWB + (((2 * s + hi) ^ swz<DIM>(l31)) << 4);
        // V, transposed reads: group G = lane / 16, lane L of it points at key 4 (G / 2) + L / 4, dims 16 (G % 2) + 4 (L % 4) .. + 3; the
        // group's lane i receives keys 4 (G / 2) .. + 3 of dim 16 (G % 2) + i
        const int key = 4 * hi + ((lane & 15) >> 2), slot = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), byte = key * ROWB + (lane & 1) * 8;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            vat[d] = byte + (((slot + 4 * d) ^ swz<DIM>(key)) << 4);
            vat8[d] = byte + 8 * ROWB + (((slot + 4 * d) ^ swz<DIM>(key + 8)) << 4);
        }
    }
    __device__ __forceinline__ void load_q(const short* at) {
#pragma unroll
        for (int s = 0; s < DS; ++s) q[s] = *reinterpret_cast<const s8*>(at + 16 * s);
    }
    __device__ __forceinline__ void q_is_there() {
#pragma unroll
        for (int s = 0; s < DS; ++s) asm volatile("" : "+v"(q[s]));
    }
    // the fragments of a unit's keys, asked for before the softmax of the unit before it begins
    __device__ __forceinline__ void keys(const char* kt, s8 (&kf)[DS]) const {
#pragma unroll
        for (int s = 0; s < DS; ++s) kf[s] = *reinterpret_cast<const s8*>(kt + krow[s]);
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ void scores(const s8 (&kf)[DS], f32x16& sc) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
        for (int s = 0; s < DS; ++s) sc = Mma<T>::mul(kf[s], q[s], sc);
    }
    // keys from `lim` on (of the unit's 32) are hidden from the lane's row
    __device__ __forceinline__ void mask(f32x16& sc, int lim, int lane) const {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (mfma32_row(i, lane) >= lim) sc[i] = -INFINITY;
    }
    // p of a row whose largest score is m: 2^((s - off) c + base), 2^LIFT of the largest one's
    struct Frame { float off, base; };
    __device__ __forceinline__ Frame frame(float m) const {
#pragma clang fp contract(off)                        // (the product as it was rounded, wherever it is used)
        const float lift = Mma<T>::LIFT;
        if (m == -INFINITY) return {0.f, lift};
        return fabsf(m * scale2) >= kFar ? Frame{m, lift} : Frame{0.f, lift - m * scale2};
    }
    // the factor of what was summed while `from` was the largest score, now that `to`'s frame is t
    __device__ __forceinline__ float rescale(float from, const Frame& t) const {
#pragma clang fp contract(off)
        const Frame f = frame(from);
        return from == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(f.off - t.off, scale2, t.base - f.base));
    }
    // (not twice on the same scores: those of far rows are changed)
    __device__ __forceinline__ void settle(f32x16& sc) {
        float top = fmaxf(sc[0], sc[1]);
#pragma unroll
        for (int i = 2; i < 16; ++i) top = fmaxf(top, sc[i]);
        if (__builtin_expect(__any(top > limit), 0)) {
            const float mn = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
            const Frame f = frame(mn);
            const float k = rescale(m, f);
            l *= k;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= k;
            m = mn;
            base = f.base;
            const bool far = f.off != 0.f;
            limit = far || mn == -INFINITY ? -INFINITY : (Mma<T>::LIFT + 8.f - f.base) * __builtin_amdgcn_rcpf(scale2);
            if (__builtin_expect(__any(far), 0)) {
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[i] -= f.off;
            }
        }
    }
    // P^T as the B operand of the unit's two 16-key products, its sum into l
    __device__ __forceinline__ void weights(const f32x16& sc) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * kb + i], scale2, base));
            l += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
            struct { unsigned u[4]; } w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w.u[i] = Mma<T>::pack(e[2 * i], e[2 * i + 1]);
            p[kb] = __builtin_bit_cast(s8, w);
        }
    }
    // O^T += V^T P^T over 32 keys.  AHEAD fragments are on their way from LDS at any time, the first ones asked for before the softmax
    // ends (as the compiler orders it alone, each product waits for its own read)
    __device__ __forceinline__ s8 v_frag(const char* vt, int i) const {
        const char* at = vt + (i / DB) * 16 * ROWB;
        const s4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(at + vat[i % DB]));
        const s4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(at + vat8[i % DB]));
        return __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    __device__ __forceinline__ void values_ahead(const char* vt) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) vf[i] = v_frag(vt, i);
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ void values(const char* vt) {
#pragma unroll
        for (int i = 0; i < FRAGS; ++i) {
            o[i % DB] = Mma<T>::mul(vf[i % AHEAD], p[i / DB], o[i % DB]);
            if (i + AHEAD < FRAGS) vf[i % AHEAD] = v_frag(vt, i + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // Where rows see different keys, a value that is infinite or not a number must reach the rows that see its key and no others (0 times
    // it is not 0): it is added to their o as it is, which no weight above zero would change, and a zero takes its place in LDS.  The
    // tile's maximum is settled before: a row's first one multiplies its o by zero.  `lim`: keys of the tile that the lane's row sees.
    __device__ __forceinline__ void odd_values(const char* vt, int keys, int lim, int hi) {
#pragma unroll 1
        for (int key = 0; key < keys; ++key) {
            const char* row = vt + key * ROWB + 8 * hi;
            asm volatile("" : "+v"(row));                         // (no address of this path is kept in registers outside it)
#pragma unroll
            for (int i = 0; i < DIM / 8; ++i) {
                const s4 v = *reinterpret_cast<const s4*>(row + ((i ^ swz<DIM>(key)) << 4));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if ((v[e] & Mma<T>::TOP) == Mma<T>::TOP && key < lim) o[i / 4][4 * (i % 4) + e] += Mma<T>::up(v[e]);
            }
        }
    }
    // results: lane (row l31) holds dims 32 d + 8 i + 4 hi + e
    __device__ __forceinline__ void store(const PrefixAttnArgs& a, const PrefixAttnLaunch& L, int chunk, const Row& r, int slots, int hi) const {
        if (!r.ok) return;
        const bool some = l > 0.f || l != l;                      // a NaN sum is a result, an empty row is not
        const float inv = some ? 1.f / l : 0.f;
        const Frame f = frame(m);
        const float lse2 = some ? __builtin_fmaf(f.off, scale2, log2f(l) - f.base) : -INFINITY;
        const int64_t row = ((int64_t)r.b * a.queries + r.i) * a.heads + r.h;
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
            if (a.lse && hi == 0) a.lse[((int64_t)r.b * a.heads + r.h) * a.queries + r.i] = lse2 * kLn2;
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
};

// Many rows: wave w owns 32 of a block's 128; K and V come in 64-key tiles through LDS (LDS-DMA, a ring of three tiles of K and of two
// of V).  A tile is two units of 32 keys; the scores of the next unit are multiplied while the softmax of this one runs, so the
// matrix units work under the exponentials.  What bounds it is the waves' instruction issue (a wave issues one instruction in about
// eight cycles, two waves share a SIMD), so the loop is unrolled over the rings' six states: LDS addresses are constants.  4 x 1024
// queries, 32 heads over 8, 16384 + 1024 keys, bf16: 1.03 - 1.10 ms (1.03 - 1.10 PF/s; one block a CU reaches 0.8).
template <class T, int DIM>
__device__ __forceinline__ void attend_rows(const PrefixAttnArgs& a, const PrefixAttnLaunch& L, int slots, int block, int blocks, char* lds) {
    constexpr int KT = 64, ROWB = DIM * 2, TILE = KT * ROWB;
    constexpr int SLOTS = DIM / 8, RPP = 64 / SLOTS, PIECES = KT / RPP / 4;      // 16-byte slots of a key row; key rows of a 1-KiB piece; a wave's pieces
    using I = Item<128, KT>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    const I it(a, L, block, blocks, wave * 32);
    const bool busy = it.row0 < it.n_rows;                        // this wave has rows (it brings keys in any case)

    // the lane's offsets within a tile of K and of V; they change where the walk enters the own keys
    int ko[PIECES], vo[PIECES];
    auto offsets = [&](int (&to)[PIECES], int stride) {
        int at = lane;
        asm volatile("" : "+v"(at));                              // (nothing of it is kept in registers)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int key = (wave * PIECES + i) * RPP + at / SLOTS;
            to[i] = key * stride + ((at % SLOTS) ^ swz<DIM>(key)) * 16;
        }
    };
    Walk<I, DIM, KT> wk, wv;
    wk.start(a, it, false, 0);
    wv.start(a, it, true, 0);
    offsets(ko, wk.stride);
    offsets(vo, wv.stride);
    const unsigned mine = lds_at(lds) + wave * PIECES * 1024;     // the wave's first piece of tile slot 0
    auto bring_k = [&](auto at, unsigned mine) {
        const u4 d = wk.tile();
        dma16<(2 + decltype(at)::value) * TILE>(d, mine, ko[0]);
        dma16<(2 + decltype(at)::value) * TILE + 1024>(d, mine, ko[1]);
        if constexpr (PIECES == 4) {
            dma16<(2 + decltype(at)::value) * TILE + 2048>(d, mine, ko[2]);
            dma16<(2 + decltype(at)::value) * TILE + 3 * 1024>(d, mine, ko[3]);
        }
        if (wk.step(a, it, false, 1)) offsets(ko, wk.stride);
    };
    auto bring_v = [&](auto at, unsigned mine) {
        const u4 d = wv.tile();
        dma16<decltype(at)::value * TILE>(d, mine, vo[0]);
        dma16<decltype(at)::value * TILE + 1024>(d, mine, vo[1]);
        if constexpr (PIECES == 4) {
            dma16<decltype(at)::value * TILE + 2048>(d, mine, vo[2]);
            dma16<decltype(at)::value * TILE + 3 * 1024>(d, mine, vo[3]);
        }
        if (wv.step(a, it, true, 1)) offsets(vo, wv.stride);
    };
    static_assert(PIECES == 4 || PIECES == 2, "");
    constexpr std::integral_constant<int, 0> C0{};
    constexpr std::integral_constant<int, 1> C1{};
    constexpr std::integral_constant<int, 2> C2{};

    Rows32<T, DIM> w(a.scale, lane, 2 * TILE);
    const int tiles = it.tiles;
    if (tiles > 0) {
        bring_k(C0, mine);
        bring_v(C0, mine);
        if (tiles > 1) bring_k(C1, mine);
    }
    {
        const Row r = it.row(a, L, l31);
        w.load_q(static_cast<const short*>(a.q) + r.b * a.q_bs + r.i * a.q_ss + r.h * a.q_hs + 8 * hi);
    }
    if (tiles > 0) {
        // The tiles up to `plain` hide keys behind a segment's end only, the same for all rows; those behind it (the last ones of causal
        // own keys) hide keys from some of the block's rows.
        const int plain = it.vis_first >= it.o1 ? tiles : it.np + (it.vis_first > it.o0 ? (it.vis_first - it.o0) / KT : 0);
        bool own = it.np == 0;
        int left = own ? it.o1 - it.o0 : it.p1 - it.c0;           // keys from the tile's first one to the segment's end
        auto next_tile = [&]() {
            left -= KT;
            if (__builtin_expect(left <= 0 && !own, 0)) {
                own = true;
                left = it.o1 - it.o0;
            }
        };
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        w.q_is_there();       // said to the compiler, which would otherwise wait for Q (and for every request) in each turn of the loop
        __syncthreads();
        f32x16 sc, nx;
        s8 kf[DIM / 16];
        if (busy) {
            w.keys(lds, kf);
            w.scores(kf, sc);
        }
        int s = 0;
        auto meet = [&]() {   // K of s + 1 and V of s are in LDS, and every wave has left K and V of s - 1
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            meet_waves();
        };
        auto tile = [&](auto ks, auto vs) {
            constexpr int KS = decltype(ks)::value, VS = decltype(vs)::value;
            meet();
            if (__builtin_expect(s + 2 < tiles, 1)) bring_k(std::integral_constant<int, (KS + 2) % 3>{}, mine);
            if (__builtin_expect(s + 1 < tiles, 1)) bring_v(std::integral_constant<int, (VS + 1) % 2>{}, mine);
            if (__builtin_expect(busy, 1)) {
                const char *kt = lds + KS * TILE, *kn = lds + (KS + 1) % 3 * TILE, *vt = lds + VS * TILE;
                w.keys(kt + 32 * ROWB, kf);
                if (__builtin_expect(left < 32, 0)) w.mask(sc, left, lane);
                w.settle(sc);
                w.scores(kf, nx);
                w.weights(sc);
                w.values_ahead(vt);
                w.values(vt);
                w.keys(kn, kf);
                if (__builtin_expect(left < 64, 0)) w.mask(nx, left - 32, lane);
                w.settle(nx);
                w.scores(kf, sc);                                 // (behind the last tile: what lies there, not used)
                w.weights(nx);
                w.values_ahead(vt + 32 * ROWB);
                w.values(vt + 32 * ROWB);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    // this wave's reads are done when it meets the others
            next_tile();
            return ++s < plain;
        };
        while (s < plain) {
            if (!tile(C0, C0)) break;
            if (!tile(C1, C1)) break;
            if (!tile(C2, C0)) break;
            if (!tile(C0, C1)) break;
            if (!tile(C1, C0)) break;
            if (!tile(C2, C1)) break;
        }
        // the rest, tile by tile
        const int seen = it.sees(a, it.row(a, L, l31).i);
        for (; s < tiles; ++s) {
            const int ks = s % 3, vs = s & 1;
            meet();
            if (s + 2 < tiles) bring_k(C0, mine + (ks == 0 ? 2 : ks - 1) * TILE);
            if (s + 1 < tiles) bring_v(C0, mine + (vs ^ 1) * TILE);
            const int at = it.o0 + (s - it.np) * KT, lim = (seen < it.o1 ? seen : it.o1) - at;     // (only own keys are hidden from some rows)
            char* vt = lds + vs * TILE;
            if (__builtin_expect(any_odd<T, TILE / 1024>(vt, lane), 0)) {         // all waves say the same
                if (busy) {                                       // the maxima over both units: none moves in the loop below
                    w.mask(sc, lim, lane);
                    w.settle(sc);
                    w.keys(lds + ks * TILE + 32 * ROWB, kf);
                    w.scores(kf, nx);
                    w.mask(nx, lim - 32, lane);
                    w.settle(nx);
                    w.keys(lds + ks * TILE, kf);
                    w.scores(kf, sc);
                }
                w.odd_values(vt, KT, lim, hi);
                __syncthreads();
                clear_odd<T>(vt + wave * PIECES * 1024 + lane * 16, PIECES);
                __syncthreads();
            }
            if (busy) {
                for (int unit = 0; unit < 2; ++unit) {
                    w.mask(sc, lim - 32 * unit, lane);
                    w.settle(sc);
                    w.weights(sc);
                    w.values_ahead(vt + unit * 32 * ROWB);
                    w.values(vt + unit * 32 * ROWB);
                    w.keys(unit == 0 ? lds + ks * TILE + 32 * ROWB : lds + (ks == 2 ? 0 : ks + 1) * TILE, kf);
                    w.scores(kf, sc);
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
    w.l += __shfl_xor(w.l, 32, 64);
    w.store(a, L, it.chunk, it.row(a, L, l31), slots, hi);
}

// Few rows (at most 32): a wave takes every fourth 32-key tile, its K straight into registers, its V through its own two LDS tiles; no
// barrier until the four waves join at the end.  Bound by the keys' bytes: 16 x 1 query over 4096 + 4096 keys of 8 heads takes 44 us (4.5
// TB/s), one query over 32768 + 1024 keys 31 us with its join.
template <class T, int DIM>
__device__ __forceinline__ void attend_wave(const PrefixAttnArgs& a, const PrefixAttnLaunch& L, int slots, int block, int blocks, char* lds_all) {
    constexpr int KT = 32, ROWB = DIM * 2, TILE = KT * ROWB, DS = DIM / 16, DB = DIM / 32;
    constexpr int SLOTS = DIM / 8, RPP = 64 / SLOTS, PIECES = KT / RPP;
    using I = Item<32, KT>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    const I it(a, L, block, blocks, 0);
    char* lds = lds_all + wave * 2 * TILE;
    const unsigned mine = lds_at(lds);

    Walk<I, DIM, KT> wk, wv;                                      // the next tile to ask for
    auto bring_v = [&](auto buf, unsigned mine) {
        const u4 d = wv.tile();
        auto piece = [&](auto i) {
            constexpr int P = decltype(i)::value;
            if constexpr (P < PIECES) {
                const int key = P * RPP + lane / SLOTS;
                dma16<decltype(buf)::value * TILE + P * 1024>(d, mine, key * wv.stride + (((lane % SLOTS) ^ swz<DIM>(key)) << 4));
            }
        };
        piece(std::integral_constant<int, 0>{});
        piece(std::integral_constant<int, 1>{});
        piece(std::integral_constant<int, 2>{});
        piece(std::integral_constant<int, 3>{});
        piece(std::integral_constant<int, 4>{});
        piece(std::integral_constant<int, 5>{});
        piece(std::integral_constant<int, 6>{});
        piece(std::integral_constant<int, 7>{});
        wv.step(a, it, true, 4);
    };
    static_assert(PIECES <= 8, "");
    s8 kreg[2][DS];
    auto load_k = [&](int buf) {
        const auto d = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(wk.at), 0, ((wk.left < KT ? wk.left : KT) - 1) * wk.stride + ROWB, 0x00020000);
#pragma unroll
        for (int s = 0; s < DS; ++s)
            kreg[buf][s] = __builtin_bit_cast(s8, (u4)__builtin_amdgcn_raw_buffer_load_b128(d, l31 * wk.stride + 32 * s + 16 * hi, 0, 0));
        wk.step(a, it, false, 4);
    };
    constexpr std::integral_constant<int, 0> C0{};
    constexpr std::integral_constant<int, 1> C1{};
    Rows32<T, DIM> w(a.scale, lane, 0);
    int s = wave;
    if (s < it.tiles) {
        wk.start(a, it, false, s);
        wv.start(a, it, true, s);
        load_k(0);
        bring_v(C0, mine);
    }
    {
        const Row r = it.row(a, L, l31);
        w.load_q(static_cast<const short*>(a.q) + r.b * a.q_bs + r.i * a.q_ss + r.h * a.q_hs + 8 * hi);
    }
    // the tiles up to `plain` hide keys behind a segment's end only; those behind it (own keys in causal order) hide keys from some rows
    const int plain = it.vis_low >= it.o1 ? it.tiles : it.np + (it.vis_low > it.o0 ? (it.vis_low - it.o0) / KT : 0);
    f32x16 sc;
    auto landed = [&](bool more) {                                // this tile's values: all but the next one's pieces of V and fragments of K
        if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PIECES + DS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    auto one = [&](auto buf, auto other) {
        constexpr int B = decltype(buf)::value;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // the other tile's reads are done
        const bool more = s + 4 < it.tiles;
        if (more) {
            load_k(B ^ 1);
            bring_v(other, mine);
        }
        w.scores(kreg[B], sc);
        const int n = s >= it.np ? it.o1 - it.o0 - (s - it.np) * KT : it.p1 - it.c0 - s * KT;
        if (n < KT) w.mask(sc, n, lane);
        w.settle(sc);
        w.weights(sc);
        landed(more);
        w.values_ahead(lds + B * TILE);
        w.values(lds + B * TILE);
        s += 4;
    };
    int cur = 0;
    while (s < plain) {
        one(C0, C1);
        cur = 1;
        if (s >= plain) break;
        one(C1, C0);
        cur = 0;
    }
    if (s < it.tiles) {
        const int seen = it.sees(a, it.row(a, L, l31).i);
        if (cur)
#pragma unroll
            for (int i = 0; i < DS; ++i) kreg[0][i] = kreg[1][i];
#pragma unroll 1
        for (; s < it.tiles; s += 4, cur ^= 1) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            const bool more = s + 4 < it.tiles;
            w.scores(kreg[0], sc);
            if (more) {
                load_k(0);
                bring_v(C0, mine + (cur ^ 1) * TILE);
            }
            const int lim = (seen < it.o1 ? seen : it.o1) - it.o0 - (s - it.np) * KT;
            char* vt = lds + cur * TILE;
            w.mask(sc, lim, lane);
            w.settle(sc);
            w.weights(sc);
            landed(more);
            if (__builtin_expect(any_odd<T, TILE / 1024>(vt, lane), 0)) {
                w.odd_values(vt, KT, lim, hi);
                clear_odd<T>(vt + lane * 16, TILE / 1024);
            }
            w.values_ahead(vt);
            w.values(vt);
        }
    }
    w.l += __shfl_xor(w.l, 32, 64);

    // the waves join in a fixed order: 2 into 0 and 3 into 1, then 1 into 0
    float* jo = reinterpret_cast<float*>(lds_all);                // [2][32 rows][DIM + 4], then [2][m | l][32]
    float* jm = jo + 2 * 32 * (DIM + 4);
#pragma unroll
    for (int half = 2; half > 0; half >>= 1) {
        __syncthreads();                                          // the LDS is free
        if (wave >= half && wave < 2 * half) {
            float* to = jo + ((wave - half) * 32 + l31) * (DIM + 4) + 4 * hi;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4*>(to + 32 * d + 8 * i) = f32x4{w.o[d][4 * i], w.o[d][4 * i + 1], w.o[d][4 * i + 2], w.o[d][4 * i + 3]};
            if (hi == 0) {
                jm[(wave - half) * 64 + l31] = w.m;
                jm[(wave - half) * 64 + 32 + l31] = w.l;
            }
        }
        __syncthreads();
        if (wave < half) {
            const float mo = jm[wave * 64 + l31], lo = jm[wave * 64 + 32 + l31], mt = fmaxf(w.m, mo);
            const auto f = w.frame(mt);
            const float ka = w.rescale(w.m, f), kb = w.rescale(mo, f);
            const float* from = jo + (wave * 32 + l31) * (DIM + 4) + 4 * hi;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 v = *reinterpret_cast<const f32x4*>(from + 32 * d + 8 * i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) w.o[d][4 * i + e] = ka * w.o[d][4 * i + e] + kb * v[e];
                }
            w.l = ka * w.l + kb * lo;
            w.m = mt;
        }
    }
    if (wave == 0) w.store(a, L, it.chunk, it.row(a, L, l31), slots, hi);
}

// The first `n0` blocks work on launch A, the others on B: the packed prefix and the own keys run beside each other.
template <class T, int DIM, bool WAVE_A, bool WAVE_B>
__global__ __launch_bounds__(256, 2) void prefix_attention_kernel(const PrefixAttnArgs a, const PrefixAttnLaunch A, const PrefixAttnLaunch B, int n0,
                                                                  int slots) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int block = blockIdx.x;
    if constexpr (WAVE_A && WAVE_B) {
        const bool second = block >= n0;
        const PrefixAttnLaunch L = second ? B : A;
        attend_wave<T, DIM>(a, L, slots, second ? block - n0 : block, second ? (int)gridDim.x - n0 : n0, lds);
    } else if constexpr (!WAVE_A && !WAVE_B) {
        const bool second = block >= n0;
        const PrefixAttnLaunch L = second ? B : A;
        attend_rows<T, DIM>(a, L, slots, second ? block - n0 : block, second ? (int)gridDim.x - n0 : n0, lds);
    } else if (block < n0) {
        attend_rows<T, DIM>(a, A, slots, block, n0, lds);
    } else {
        attend_wave<T, DIM>(a, B, slots, block - n0, (int)gridDim.x - n0, lds);
    }
}

// Joins a row's partial results: out = sum_s 2^(lse_s - max) o_s / sum_s 2^(lse_s - max).  One wave a row, a lane a partial
// result's weight (at most 64), then a lane two columns or one, eight partial results in flight: bound by latency (64 x 32 rows of 12
// parts: 4.1 us).
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
    for (int s0 = 0; s0 < slots; s0 += 8) {
        float v[8][W];
#pragma unroll
        for (int u = 0; u < 8; ++u) load_vec<float, W>(o + (int64_t)(s0 + u < slots ? s0 + u : slots - 1) * rows * DIM, v[u]);
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (s0 + u < slots) {
                const float ks = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(k), s0 + u));
#pragma unroll
                for (int i = 0; i < W; ++i) acc[i] += ks * v[u][i];
            }
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
        // Chunks: every one more is a partial result of each row to write and join.  Measured (us, bf16, 32 heads over 8, dim 128):
        //   64 x 1 token behind 8192 + 512 keys, prefix in 16 / 8 chunks: 43.5 / 37.3;   256 x 1: 8 / 4 chunks: 122 / 109
        //   8 x 64 tokens behind 8192, 2 / 4 chunks (a block / two a CU): 93 / 85;   32 x 197 tokens, 4 heads, 1000 keys, 1 / 2: 28 / 37
        //   1 x 100 tokens behind 8192, 8 / 16 chunks: 29.5 / 23.7;   16 x 1 token, own 4096 by wave, 16 / 8 chunks: 46.3 / 42.4
        // so one block a CU with chunks of 512 keys or more (1024 where the own keys' items run beside them), two where they still have
        // 2048; by wave, whose blocks hold little, two a CU.  At most 32, so that a wave of the join holds all weights.
        auto fill = [&](int64_t per_cu, int least) { return std::min<int64_t>((per_cu * cus + items - 1) / items, std::max(1, keys / least)); };
        int64_t n = l.by_wave ? fill(2, 512) : std::max(fill(1, packed ? 1024 : 512), fill(2, 2048));
        n = std::min<int64_t>(n, 32);
        l.chunk = (int)std::max<int64_t>(unit, ((keys + n - 1) / n + unit - 1) / unit * unit);   // no keys at all: one empty chunk
        l.chunks = std::max(1, (keys + l.chunk - 1) / l.chunk);
        l.slot0 = plan.slots;
        plan.slots += l.chunks;
        plan.l[plan.n++] = l;
    };
    // Packing pays where the prefix would be read often enough (us, 8 heads, 16 tokens behind 300 keys, 32 samples: packed 18.0, each
    // for itself 12.4; one token behind 600, 32 samples: 16.5 both) and a sample alone does not fill half a tile of rows
    if (a.batch > 1 && a.prefix >= 256 && (int64_t)a.batch * a.prefix >= 16384 && rows_own < 64) {
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
