// The linear layer in 8-bit integers: rows of activations and weights carry a scale each.
//
//   s[r] = max_k |x[r, k]| / 127,  q[r, k] = round(x[r, k] * (127 / max)), halves to even        (quantise)
//   C[m, n] = (sum_k q_x[m, k] q_w[n, k]) s_x[m] s_w[n] + bias[n],  then GELU or + residual        (product)
//
// The sum is exact: 8-bit products in 32-bit integers (K <= kI8MaxK keeps them below 2^31), whatever order the tiles and waves
// add in, so every schedule below gives the same bits; it is rounded to fp32 once, before the scales.
#include "linear_i8.hpp"

#include <algorithm>
#include <type_traits>

#include "../../include/condmdi.h"
#include "ops_common.hpp"

namespace cmdi {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// ---- quantise ------------------------------------------------------------------------------------------------------------
// A team of TEAM lanes takes a row; its first NV vectors of a lane stay in registers between the two passes, the rest of a
// longer row is read again (from the L2).  Bound by memory: 2 or 4 bytes read, 1 written (12608 x 512 fp32: 7.6 us, 4.2 TB/s; 8192 x
// 4096 bf16: 26 us, 3.9 TB/s).
template <class T, int TEAM>
__global__ __launch_bounds__(256) void quant_rows_i8_kernel(const QuantRowsArgs a) {
    constexpr int W = Elem<T>::W;
    constexpr int NV = 4, TPB = 256 / TEAM;
    __shared__ float lds[2][4];
    const int lane = threadIdx.x % TEAM;
    const int team = TPB == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / TEAM);
    const int64_t row = (int64_t)blockIdx.x * TPB + team;
    if (row >= a.rows) return;                 // whole waves; never where the team is the block
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    float v[NV][W];
    float top = 0.f, odd = 0.f;                // odd: NaN once a value is not finite (0 * inf, 0 * nan)
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int e = (c * TEAM + lane) * W;
        load_part<T, W>(x + e, v[c], a.cols - e);
    }
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int i = 0; i < W; ++i) { top = fmaxf(top, fabsf(v[c][i])); odd += 0.f * v[c][i]; }
    for (int e = (NV * TEAM + lane) * W; e < a.cols; e += TEAM * W) {
        float u[W];
        load_part<T, W>(x + e, u, a.cols - e);
#pragma unroll
        for (int i = 0; i < W; ++i) { top = fmaxf(top, fabsf(u[i])); odd += 0.f * u[i]; }
    }
    top = wave_highest(top);
    odd = wave_total(odd);
    if constexpr (TEAM > 64) {
        if ((threadIdx.x & 63) == 0) { lds[0][threadIdx.x >> 6] = top; lds[1][threadIdx.x >> 6] = odd; }
        __syncthreads();
        top = fmaxf(fmaxf(lds[0][0], lds[0][1]), fmaxf(lds[0][2], lds[0][3]));
        odd = (lds[1][0] + lds[1][1]) + (lds[1][2] + lds[1][3]);
    }
    // below 1e-35 the factor 127 / top would leave the range: such a row is all zeros.  A row with an infinity or a NaN has the
    // scale NaN, so that its products say so
    const bool fine = odd == 0.f, some = fine && top >= 1e-35f;
    const float inv = some ? 127.f / top : 0.f;
    if (lane == 0) a.scale[row] = fine ? (some ? top / 127.f : 0.f) : __builtin_nanf("");
    int8_t* q = a.q + row * a.kp;
    struct alignas(W) Out { int8_t e[W]; };
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int e = (c * TEAM + lane) * W;
        if (e < a.kp) {                        // columns behind `cols` hold 0: the padding
            Out o;
#pragma unroll
            for (int i = 0; i < W; ++i) o.e[i] = (int8_t)(fine ? (int)rintf(v[c][i] * inv) : 0);
            *reinterpret_cast<Out*>(q + e) = o;
        }
    }
    for (int e = (NV * TEAM + lane) * W; e < a.kp; e += TEAM * W) {
        float u[W];
        load_part<T, W>(x + e, u, a.cols - e);
        Out o;
#pragma unroll
        for (int i = 0; i < W; ++i) o.e[i] = (int8_t)(fine ? (int)rintf(u[i] * inv) : 0);
        *reinterpret_cast<Out*>(q + e) = o;
    }
}

// ---- product -------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float finish(int acc, float sa, float sw, float bias) { return (float)acc * sa * sw + bias; }

template <class T>
__device__ __forceinline__ void finish_at(const GemmI8Args& p, int row, int col, int acc, float sa, float sw, float bias) {
    float v = finish(acc, sa, sw, bias);
    if (p.epi == 1) v = gelu_erf(v);
    if (p.epi == 3) v += Elem<T>::up(static_cast<const T*>(p.resid)[(int64_t)row * p.ldr + col]);
    static_cast<T*>(p.c)[(int64_t)row * p.ldc + col] = Elem<T>::down(v);
}

// W sums of a row at `at` in LDS, finished and stored from column `col` on; `whole`: all W lie in the matrix
template <class T, int W>
__device__ __forceinline__ void store_row(const GemmI8Args& p, int row, int col, bool whole, const int* at, float sa, const float (&ws)[W], const float (&bias)[W]) {
    if (whole) {
        float v[W];
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = finish(at[e], sa, ws[e], bias[e]);
        if (p.epi == 1) {
#pragma unroll
            for (int e = 0; e < W; ++e) v[e] = gelu_erf(v[e]);
        }
        if (p.epi == 3) {
            float r[W];
            load_vec<T, W>(static_cast<const T*>(p.resid) + (int64_t)row * p.ldr + col, r);
#pragma unroll
            for (int e = 0; e < W; ++e) v[e] += r[e];
        }
        store_vec<T, W>(static_cast<T*>(p.c) + (int64_t)row * p.ldc + col, v);
    } else {
#pragma unroll
        for (int e = 0; e < W; ++e)
            if (col + e < p.n) finish_at<T>(p, row, col + e, at[e], sa, ws[e], bias[e]);
    }
}

// Tiles: WM x WN waves, a wave owns TM x TN fragments of 32 x 32 (v_mfma_i32_32x32x32_i8).  K runs in steps of 128 columns
// through NST LDS stages filled by LDS-DMA.  A row of a stage is 128 bytes = eight 16-byte slots; slot t of row r holds columns
// 16 (t ^ (r >> 1 & 7)), which spreads the rows of a read's lane group over all banks.  Rows behind the matrix repeat its last
// one and are not stored.  NST stages: two where the products of a step cover a request's way, four where a step is short.
//
// A step is four substeps of 32 columns; the fragments of the next substep are read while this one multiplies.  The step's one
// barrier sits before its LAST substep: by then every wave has that substep's fragments in registers, so stage s may be
// overwritten (requests of step s + 2 go out) and, with the wait in front of it, step s + 1 has landed and its first fragments are
// read under the last products: the matrix pipe waits for other waves once a step, never for LDS.  8192 x 8192 x 4096: 285 - 340 us by
// the card's clock (1.6 - 1.9 POP/s); what it leaves is the epilogue of each of the four rounds, under which no other block of the CU runs.
template <class T, int TM, int TN, int WM, int WN, int NST>
__global__ __launch_bounds__(64 * WM * WN, TM * TN == 16 ? 1 : 2) void gemm_i8_tile_kernel(const GemmI8Args p, int tiles_m, int tiles_n) {
    constexpr int NW = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN, STAGE = (BM + BN) * 128;
    constexpr int PIECES = (BM + BN) / 8 / NW;       // 1-KiB pieces (8 rows) a wave brings per step
    static_assert((BM / 8) % NW == 0 && (BN / 8) % NW == 0, "a piece lies in one operand for every wave");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN, l31 = lane & 31, hi = lane >> 5;
    // neighbouring tiles of an XCD share operand panels in its L2: 8 rows of tiles, then the next column
    const int id = xcd_remap(blockIdx.x, tiles_m * tiles_n);
    const int band = id / (8 * tiles_n), in = id % (8 * tiles_n);
    const int bh = tiles_m - band * 8 < 8 ? tiles_m - band * 8 : 8;
    const int m0 = (band * 8 + in % bh) * BM, n0 = (in / bh) * BN;

    // the epilogue's scales and bias, asked for first of all where the registers allow it: its lane's W columns and 32 / RPI rows of
    // each strip
    constexpr bool EARLY = TM * TN <= 4;
    constexpr int W = Elem<T>::W, COLS = 32 * TN, PITCH = COLS + 4, LPR = COLS / W, RPI = 64 / LPR;
    const int col = n0 + wn * COLS + (lane % LPR) * W;
    float ws[W], bias[W], sa[EARLY ? TM : 1][32 / RPI];
    auto scales = [&]() {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int c = col + i < p.n ? col + i : p.n - 1;
            ws[i] = p.w_scale[c];
            bias[i] = p.bias ? p.bias[c] : 0.f;
        }
    };
    auto row_scales = [&](int i, float (&out)[32 / RPI]) {
#pragma unroll
        for (int it = 0; it < 32 / RPI; ++it) {
            const int row = m0 + (wm * TM + i) * 32 + it * RPI + lane / LPR;
            out[it] = p.a_scale[row < p.m ? row : p.m - 1];
        }
    };
    if constexpr (EARLY) {
        scales();
#pragma unroll
        for (int i = 0; i < TM; ++i) row_scales(i, sa[i]);
    }

    unsigned off[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int pc = i * NW + wave;                // pieces 0 .. BM/8 - 1: A, then W
        const bool is_a = pc < BM / 8;
        const int r = (is_a ? pc : pc - BM / 8) * 8 + (lane >> 3);
        const int last = (is_a ? p.m - m0 : p.n - n0) - 1;
        const int rr = r < last ? r : last;
        off[i] = (unsigned)(rr * (is_a ? p.lda : p.ldw)) + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
    }
    const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(p.a + (int64_t)m0 * p.lda), 0, 0x7fffffff, 0x00020000);
    const auto rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(p.w + (int64_t)n0 * p.ldw), 0, 0x7fffffff, 0x00020000);
    auto bring_one = [&](int i, int step, int stage) {
        char* dst = lds + stage * STAGE + (i * NW + wave) * 1024;
        if (i * NW < BM / 8)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (__attribute__((address_space(3))) void*)dst, 16, (int)off[i], step * 128, 0, 0);
        else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (__attribute__((address_space(3))) void*)dst, 16, (int)off[i], step * 128, 0, 0);
    };
    auto bring = [&](int step, int stage) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) bring_one(i, step, stage);
    };

    i32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

    const int arow = (wm * TM * 32 + l31) * 128, brow = (BM + wn * TN * 32 + l31) * 128, sw = (l31 >> 1) & 7;
    i32x4 fa[2][TM], fb[2][TN];
    auto read = [&](const char* st, int ks, int buf) {
        const int slot = ((ks * 2 + hi) ^ sw) << 4;
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[buf][i] = *reinterpret_cast<const i32x4*>(st + arow + i * 32 * 128 + slot);
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[buf][j] = *reinterpret_cast<const i32x4*>(st + brow + j * 32 * 128 + slot);
    };
    // the products of one substep; where `go`, pieces [from, to) of `step`'s request go out between them, evenly
    auto multiply = [&](int buf, int from, int to, bool go, int step, int stage) {
        int piece = from;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[buf][i], fb[buf][j], acc[i][j], 0, 0, 0);
                const int done = from + (to - from) * (i * TN + j + 1) / (TM * TN);
                if (done > piece) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (go) {
#pragma unroll
                        for (int k = piece; k < done; ++k) bring_one(k, step, stage);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    piece = done;
                }
            }
    };

    const int steps = p.k / 128;
#pragma unroll
    for (int i = 0; i < NST; ++i)
        if (i < steps) bring(i, i);
    if (steps >= NST) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 1) * PIECES) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    meet_waves();
    read(lds, 0, 0);
    int at = 0;                                       // s % NST
    for (int s = 0; s < steps; ++s) {
        const char* st = lds + at * STAGE;
        const int next = at + 1 == NST ? 0 : at + 1;
        read(st, 1, 1);
        // two stages: the second half of the request of s + 1 goes out here (step 1's went out whole in front of the loop)
        if constexpr (NST == 2) multiply(0, PIECES / 2, PIECES, s > 0 && s + 1 < steps, s + 1, next);
        else multiply(0, 0, 0, false, 0, 0);
        read(st, 2, 0);
        multiply(1, 0, 0, false, 0, 0);
        read(st, 3, 1);
        multiply(0, 0, 0, false, 0, 0);
        if (s + 1 < steps) {
            // step s + 1 has landed once at most the NST - 2 requests behind it are out
            if (s + NST <= steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * PIECES) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            meet_waves();
            read(lds + next * STAGE, 0, 0);
        }
        multiply(1, 0, NST == 2 ? PIECES / 2 : PIECES, s + NST < steps, s + NST, at);      // into the stage just left
        at = next;
    }

    // ---- epilogue: 32 rows of the wave's columns at a time through its own slice of LDS, so that a lane stores 16 consecutive
    // bytes of a row; its columns, their scales and their bias stay the same for all rows ----
    static_assert(NW * 32 * PITCH * 4 <= NST * STAGE, "the strips fit the stages");
    __syncthreads();
    int* strip = reinterpret_cast<int*>(lds) + wave * 32 * PITCH;
    if constexpr (!EARLY) scales();
    const bool whole = col + W <= p.n;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) strip[mfma32_row(r, lane) * PITCH + j * 32 + l31] = acc[i][j][r];
        if constexpr (!EARLY) row_scales(i, sa[0]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    // one wave writes and reads: no barrier
#pragma unroll
        for (int it = 0; it < 32 / RPI; ++it) {
            const int lr = it * RPI + lane / LPR, row = m0 + (wm * TM + i) * 32 + lr;
            if (row >= p.m) continue;
            store_row<T>(p, row, col, whole, strip + lr * PITCH + (lane % LPR) * W, sa[EARLY ? i : 0][it], ws, bias);
        }
        asm volatile("" ::: "memory");
    }
}

// Short K (STEPS * 128 <= 512 columns) and many rows: a tile's products are too short to hide its way in and out.  A block of 8 waves
// keeps the weights of its 256 columns in registers and walks down the rows, 32 at a time, whose activations wait in a ring of three
// LDS tiles; a wave's stores of one tile run under the products of the next, two blocks share a CU.  12608 x 1536 x 512 with fp32
// results: 22.1 us, of which the 77 MB of C alone would take 13.
constexpr int kShortTiles = 32;                                       // the most row tiles of a block
constexpr int kShortWeights = 8 * 8192;
template <class T, int STEPS>
__global__ __launch_bounds__(512, 4) void gemm_i8_short_kernel(const GemmI8Args p, int tiles_m, int per, int groups_n) {
    constexpr int TILE = STEPS * 32 * 128;
    constexpr int W = Elem<T>::W, PITCH = 36, LPR = 32 / W, RPI = 64 / LPR, STORES = 32 / RPI;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    static_assert(2 * TILE + 8 * 16 * PITCH * 4 + kShortTiles * 32 * 4 <= kShortWeights, "");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    const int id = xcd_remap(blockIdx.x, gridDim.x);                  // neighbours share rows
    const int n0 = id % groups_n * 256, t0 = id / groups_n * per, t1 = t0 + per < tiles_m ? t0 + per : tiles_m;
    if (t0 >= t1) return;

    const int r = (wave & 3) * 8 + (lane >> 3), at_slot = ((lane & 7) ^ ((r >> 1) & 7)) << 4;
    // LDS: the weights on their way in (64 KiB), later slots 1 and 2 of the ring, the strips and the rows' scales; behind it slot 0
    auto ring = [&](int slot) { return lds + (slot == 0 ? kShortWeights : (slot - 1) * TILE); };
    auto bring = [&](int t, int slot) {                               // waves 0 - 3 bring the even steps, 4 - 7 the odd ones
        const int last = p.m - 1 - t * 32;
        const int off = (r < last ? r : last) * (int)p.lda + at_slot;
        const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(p.a + (int64_t)t * 32 * p.lda), 0, 0x7fffffff, 0x00020000);
#pragma unroll
        for (int i = 0; i < (STEPS + 1) / 2; ++i) {
            const int s = 2 * i + (wave >> 2);
            if (s < STEPS)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (__attribute__((address_space(3))) void*)(ring(slot) + s * 4096 + (wave & 3) * 1024), 16,
                                                         off, s * 128, 0, 0);
        }
    };
    // the weights come through the LDS, two steps at a time in 8 KiB of each wave's own: as fragments straight from memory (32 bytes of
    // a row at once) they took 8 us of 26
    bring(t0, 0);
    i32x4 fw[STEPS * 4];
    char* mine = lds + wave * 8192;
    const int wr0 = n0 + wave * 32, sw = (l31 >> 1) & 7;
    const int8_t* wbase = p.w + (int64_t)(wr0 < p.n ? wr0 : p.n - 1) * p.ldw;
    const auto rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(wbase), 0, 0x7fffffff, 0x00020000);
#pragma unroll
    for (int s0 = 0; s0 < STEPS; s0 += 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {                                 // 8 rows of a step
            if (s0 + i / 4 >= STEPS) break;
            const int row = i % 4 * 8 + (lane >> 3), last = p.n - 1 - wr0;
            const int off = (row < last ? row : last > 0 ? last : 0) * (int)p.ldw + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (__attribute__((address_space(3))) void*)(mine + i * 1024), 16, off, (s0 + i / 4) * 128, 0, 0);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int k = 4 * s0; k < 4 * s0 + 8 && k < 4 * STEPS; ++k)
            fw[k] = *reinterpret_cast<const i32x4*>(mine + (k / 4 - s0) * 4096 + l31 * 128 + (((k % 4 * 2 + hi) ^ sw) << 4));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    meet_waves();                                                     // the LDS is the ring's now
    if (t0 + 1 < t1) bring(t0 + 1, 1);
    const int col = n0 + wave * 32 + (lane % LPR) * W;
    float ws[W], bias[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const int c = col + i < p.n ? col + i : p.n - 1;
        ws[i] = p.w_scale[c];
        bias[i] = p.bias ? p.bias[c] : 0.f;
    }
    int* strip = reinterpret_cast<int*>(lds + 2 * TILE) + wave * 16 * PITCH;
    float* scales = reinterpret_cast<float*>(lds + 2 * TILE + 8 * 16 * PITCH * 4);
    for (int i = threadIdx.x; i < (t1 - t0) * 32; i += 512) scales[i] = p.a_scale[t0 * 32 + i < p.m ? t0 * 32 + i : p.m - 1];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                // (read behind the loop's first barrier)

    const bool whole = col + W <= p.n, all = n0 + 256 <= p.n;         // all: every lane of the block stores whole vectors
    int slot = 0;
    for (int t = t0; t < t1; ++t) {
        // tile t has landed: behind its request there are at least that of t + 1 (STEPS / 2 of it by any wave) and, in a block that
        // stores whole vectors, t - 1's stores
        if (t == t0 || t + 1 >= t1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else if (all) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(STEPS / 2 + STORES) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(STEPS / 2) : "memory");
        meet_waves();                                                 // and every wave has left tile t - 1
        const char* a = ring(slot) + l31 * 128;
        slot = slot == 2 ? 0 : slot + 1;                              // t + 1's
        if (t + 2 < t1) bring(t + 2, slot == 2 ? 0 : slot + 1);
        i32x16 acc;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = 0;
#pragma unroll
        for (int k = 0; k < STEPS * 4; ++k) {
            const i32x4 fa = *reinterpret_cast<const i32x4*>(a + k / 4 * 4096 + (((k % 4 * 2 + hi) ^ sw) << 4));
            acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa, fw[k], acc, 0, 0, 0);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {                        // 16 rows: one wave writes and reads, no barrier
#pragma unroll
            for (int i = 0; i < 8; ++i) strip[mfma32_row(i, lane) * PITCH + l31] = acc[8 * half + i];
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int it = 0; it < STORES / 2; ++it) {
                const int lr = it * RPI + lane / LPR, row = t * 32 + 16 * half + lr;
                if (row < p.m)
                    store_row<T>(p, row, col, whole, strip + lr * PITCH + (lane % LPR) * W, scales[(t - t0) * 32 + 16 * half + lr], ws, bias);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
}

// Few rows (M <= 16): the weights' bytes are the time.  A block takes 16 weight rows, its 4 waves split K and read their
// weights straight into the registers of v_mfma_i32_16x16x64_i8 (weights as its rows, activations as its columns), 16 steps of
// 64 columns in flight; the waves' sums join through LDS.  8 x 28672 x 4096: 29 us (4.1 TB/s).
template <class T>
__global__ __launch_bounds__(256) void gemm_i8_rows_kernel(const GemmI8Args p) {
    __shared__ i32x4 part[4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l15 = lane & 15, kg = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int wr = n0 + l15 < p.n ? n0 + l15 : p.n - 1, ar = l15 < p.m ? l15 : p.m - 1;
    const int8_t* w = p.w + (int64_t)wr * p.ldw + kg * 16;
    const int8_t* a = p.a + (int64_t)ar * p.lda + kg * 16;
    i32x4 acc{0, 0, 0, 0};
    const int steps = p.k / 64;
    constexpr int U = 16;
    for (int s0 = wave * U; s0 < steps; s0 += 4 * U) {
        const int n = steps - s0 < U ? steps - s0 : U;
        if (n == U) {
            i32x4 fw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) fw[u] = *reinterpret_cast<const i32x4*>(w + (int64_t)(s0 + u) * 64);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const i32x4 fa = *reinterpret_cast<const i32x4*>(a + (int64_t)(s0 + u) * 64);
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u], fa, acc, 0, 0, 0);
            }
        } else {
            for (int u = 0; u < n; ++u) {
                const i32x4 f = *reinterpret_cast<const i32x4*>(w + (int64_t)(s0 + u) * 64);
                const i32x4 fa = *reinterpret_cast<const i32x4*>(a + (int64_t)(s0 + u) * 64);
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(f, fa, acc, 0, 0, 0);
            }
        }
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave != 0 || l15 >= p.m) return;
    // this lane: activation row l15, weight rows 4 kg + r
    const i32x4 s = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
    const float sa = p.a_scale[l15];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int col = n0 + 4 * kg + r;
        if (col < p.n) finish_at<T>(p, l15, col, s[r], sa, p.w_scale[col], p.bias ? p.bias[col] : 0.f);
    }
}

// Few rows with their quantising: every block rounds all the activations for itself, into its LDS, while its weights are on their way;
// the bits are those of quant_rows_i8_kernel and gemm_i8_rows_kernel.  2^lanes lanes share an activation row; a lane's vectors stay
// packed between the two passes.  Bound by the weights' bytes behind a launch's first request: 8 x 8192 x 4096 takes 11.4 us (2.9
// TB/s), 4 x 8192 x 8192 15.8 us (4.3 TB/s).
__device__ __forceinline__ float plus_apart(float x, float y) {     // never one instruction with the product that x is
#pragma clang fp contract(off)
    return x + y;
}
template <class T> struct Packed;
template <> struct Packed<float> {
    typedef unsigned U;
    typedef U V __attribute__((ext_vector_type(4)));
    static constexpr unsigned ABS = 0x7fffffffu, INF = 0x7f800000u;
    static __device__ __forceinline__ float up(unsigned v) { return __uint_as_float(v); }
};
template <> struct Packed<Bf16> {
    typedef unsigned short U;
    typedef U V __attribute__((ext_vector_type(8)));
    static constexpr unsigned short ABS = 0x7fff, INF = 0x7f80;
    static __device__ __forceinline__ float up(unsigned short v) { return __uint_as_float((unsigned)v << 16); }
};
template <> struct Packed<_Float16> {
    typedef unsigned short U;
    typedef U V __attribute__((ext_vector_type(8)));
    static constexpr unsigned short ABS = 0x7fff, INF = 0x7c00;
    static __device__ __forceinline__ float up(unsigned short v) { return (float)__builtin_bit_cast(_Float16, v); }
};

template <class T>
__global__ __launch_bounds__(256, 2) void linear_i8_rows_kernel(const QuantRowsArgs x, const GemmI8Args p, int lanes) {
    typedef Packed<T> P;
    typedef typename P::V V;
    constexpr int W = Elem<T>::W, NV = kI8FusedBytes / 256 / 16, U = 16;
    extern __shared__ __attribute__((aligned(16))) char rows8[];       // [m][kp + 16]
    __shared__ i32x4 part[4][64];
    __shared__ unsigned high[4];
    __shared__ float sas[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l15 = lane & 15, kg = lane >> 4;
    const int kp = p.k, ldq = kp + 16, steps = kp / 64;

    // the activations first: a wait for them must not be one for the weights
    const int team = 1 << lanes, at = threadIdx.x & (team - 1), row = threadIdx.x >> lanes;
    const T* xr = static_cast<const T*>(x.x) + (int64_t)(row < p.m ? row : p.m - 1) * x.ld;
    struct __attribute__((packed, aligned(sizeof(T)))) Raw { V v; };
    V v[NV];
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int e = (c * team + at) * W;
        v[c] = V(0);
        if (e + W <= x.cols) v[c] = reinterpret_cast<const Raw*>(xr + e)->v;
    }
    const int whole = x.cols / W, rest = x.cols - whole * W;           // a part of a vector at the row's end
    V end = V(0);
#pragma unroll
    for (int i = 0; i < W; ++i)
        if (i < rest) end[i] = reinterpret_cast<const typename P::U*>(xr)[whole * W + i];
    const int n0 = blockIdx.x * 16;
    const int wr = n0 + l15 < p.n ? n0 + l15 : p.n - 1, ar = l15 < p.m ? l15 : p.m - 1;
    const int8_t* w = p.w + (int64_t)wr * p.ldw + kg * 16;
    i32x4 fw[U];
    auto weights = [&](int s0) {
#pragma unroll
        for (int u = 0; u < U; ++u) fw[u] = *reinterpret_cast<const i32x4*>(w + (int64_t)(s0 + u < steps ? s0 + u : steps - 1) * 64);
        __builtin_amdgcn_sched_barrier(0);
    };
    weights(wave * U);

    if (rest > 0 && (whole & (team - 1)) == at) {
#pragma unroll
        for (int c = 0; c < NV; ++c)
            if (c == whole >> lanes) v[c] = end;
    }
    // absolute values order as their bits do, infinities and NaN on top
    V tops = V(0);
#pragma unroll
    for (int c = 0; c < NV; ++c) tops = __builtin_elementwise_max(tops, (V)(v[c] & P::ABS));
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) top = top > tops[i] ? top : tops[i];
    for (int d = team < 64 ? team / 2 : 32; d > 0; d >>= 1) {
        const unsigned other = __shfl_xor(top, d, 64);
        top = top > other ? top : other;
    }
    if (team > 64) {
        if (lane == 0) high[wave] = top;
        __syncthreads();
        const int first = threadIdx.x >> lanes << (lanes - 6);
        for (int i = 0; i < team / 64; ++i) top = top > high[first + i] ? top : high[first + i];
    }
    const bool fine = top < P::INF;
    const float most = fine ? P::up(top) : 0.f;
    const bool some = most >= 1e-35f;
    const float inv = some ? 127.f / most : 0.f;
    if (at == 0 && row < p.m) sas[row] = fine ? (some ? most / 127.f : 0.f) : __builtin_nanf("");
    if (row < p.m) {
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int e = (c * team + at) * W;
            if (e < kp) {
                unsigned o[W / 4];
#pragma unroll
                for (int i = 0; i < W; i += 4) {
                    unsigned b[4];
                    // 1.5 * 2^23 more: rounded to a whole number, halves to even, its lowest byte in front
#pragma unroll
                    for (int k = 0; k < 4; ++k) b[k] = __float_as_uint(plus_apart(P::up(v[c][i + k]) * inv, 12582912.f));
                    o[i / 4] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
                }
                __builtin_memcpy(__builtin_assume_aligned(rows8 + row * ldq + e, W), o, W);
            }
        }
    }
    __syncthreads();
    i32x4 acc{0, 0, 0, 0};
    const char* a = rows8 + ar * ldq + kg * 16;
    for (int s0 = wave * U; s0 < steps;) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u < steps) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u], *reinterpret_cast<const i32x4*>(a + (s0 + u) * 64), acc, 0, 0, 0);
        s0 += 4 * U;
        if (s0 < steps) weights(s0);
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave != 0 || l15 >= p.m) return;
    const i32x4 s = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
    const float sa = sas[l15];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int col = n0 + 4 * kg + r;
        if (col < p.n) finish_at<T>(p, l15, col, s[r], sa, p.w_scale[col], p.bias ? p.bias[col] : 0.f);
    }
}

template <class T, int TM, int TN, int WM, int WN, int NST>
hipError_t launch_tile(const GemmI8Args& p, hipStream_t stream) {
    constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN, LDS = NST * (BM + BN) * 128;
    auto* kernel = gemm_i8_tile_kernel<T, TM, TN, WM, WN, NST>;
    if (LDS > 64 * 1024) {
        static PerDevice<int> set;
        int& done = set.get();
        if (!done) {
            hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
            if (e != hipSuccess) return e;
            done = 1;
        }
    }
    const int tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
    kernel<<<dim3((unsigned)tm * tn), dim3(64 * WM * WN), LDS, stream>>>(p, tm, tn);
    return hipGetLastError();
}

template <class T, int STEPS>
hipError_t launch_short(const GemmI8Args& p, hipStream_t stream) {
    constexpr int LDS = kShortWeights + STEPS * 32 * 128;
    auto* kernel = gemm_i8_short_kernel<T, STEPS>;
    if (LDS > 64 * 1024) {
        static PerDevice<int> set;
        int& done = set.get();
        if (!done) {
            hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
            if (e != hipSuccess) return e;
            done = 1;
        }
    }
    const int tiles_m = (p.m + 31) / 32, groups_n = (p.n + 255) / 256;
    const int want = std::max(1, 2 * device_cu_count() / groups_n), per = std::min(kShortTiles, (tiles_m + want - 1) / want), groups_m = (tiles_m + per - 1) / per;
    kernel<<<dim3((unsigned)(groups_m * groups_n)), 512, LDS, stream>>>(p, tiles_m, per, groups_n);
    return hipGetLastError();
}

template <class T>
hipError_t launch_typed(const GemmI8Args& p, hipStream_t stream) {
    // Measured on an MI355X (us, 8-bit operands, bf16 out unless said):
    //   rows kernel / 64 x 64 tile:          16 x 8192 x 4096: 9.1 / 12.7        32 x 8192 x 4096: 14.1 / 12.7
    //   short K / the tile that is right:    12608 x 1536 x 512 fp32 out: 22.1 / 28.0    12608 x 512 x 512 fp32 + residual: 15.8 / 24.7
    //                                        50000 x 1000 x 384: 33.2 / 51.3     8192 x 8192 x 512: 47.9 / 58.2    4096 x 4096 x 512: 18.8 / 18.1
    //                                        and with 2^22 sums or fewer:        2048 x 2048 x 512: 8.8 / 8.1      64 x 65536 x 512: 15.3 / 14.5
    //   64 x 64, four stages / two stages:   65 x 8192 x 4096: 11.8 / 17.4       512 x 4096 x 4096: 15.5 / 17.8
    //   128 x 128, three stages / 64 x 64:   1024 x 4096 x 4096: 23.6 / 30.1     512 x 4096 x 4096 (half a chip of tiles): 20.6 / 15.5
    //   128 x 128, two stages / three:       2048 x 4096 x 4096: 39.7 / 44.8
    //   256 x 256 / 128 x 128, two stages:   4096^3: 64 / 75    2048 x 4096 x 4096 (half a chip): 50 / 40
    const int cus = device_cu_count();
    auto tiles = [&](int side) { return (int64_t)((p.m + side - 1) / side) * ((p.n + side - 1) / side); };
    const int64_t t256 = tiles(256), t128 = tiles(128);
    if (p.m <= 16) {
        gemm_i8_rows_kernel<T><<<dim3((unsigned)((p.n + 15) / 16)), 256, 0, stream>>>(p);
        return hipGetLastError();
    }
    if (p.k <= 512 && (int64_t)p.m * p.n > (1 << 22)) {
        switch (p.k / 128) {
            case 1: return launch_short<T, 1>(p, stream);
            case 2: return launch_short<T, 2>(p, stream);
            case 3: return launch_short<T, 3>(p, stream);
            default: return launch_short<T, 4>(p, stream);
        }
    }
    // one block a CU: worth it where its rounds are at least three quarters full
    if (t256 >= cus && 4 * t256 >= 3 * ((t256 + cus - 1) / cus) * cus) return launch_tile<T, 4, 2, 2, 4, 2>(p, stream);
    if (t128 >= 2 * cus) return launch_tile<T, 2, 2, 2, 2, 2>(p, stream);
    if (t128 >= cus) return launch_tile<T, 2, 2, 2, 2, 3>(p, stream);
    return launch_tile<T, 1, 1, 2, 2, 4>(p, stream);
}

// bits of the row's number among the (up to 16) rows
int fused_row_bits(int m) { return m <= 1 ? 0 : m <= 2 ? 1 : m <= 4 ? 2 : m <= 8 ? 3 : 4; }

}  // namespace

hipError_t launch_quant_rows_i8(const QuantRowsArgs& a, hipStream_t stream) {
    auto go = [&](auto t) {
        using T = decltype(t);
        if (a.cols <= 2048) quant_rows_i8_kernel<T, 64><<<dim3((unsigned)((a.rows + 3) / 4)), 256, 0, stream>>>(a);
        else quant_rows_i8_kernel<T, 256><<<dim3((unsigned)a.rows), 256, 0, stream>>>(a);
        return hipGetLastError();
    };
    switch (a.dtype) {
        case CMDI_DT_F32: return go(float());
        case CMDI_DT_BF16: return go(Bf16());
        default: return go(_Float16());
    }
}

hipError_t launch_gemm_i8(const GemmI8Args& p, hipStream_t stream) {
    switch (p.dtype) {
        case CMDI_DT_F32: return launch_typed<float>(p, stream);
        case CMDI_DT_BF16: return launch_typed<Bf16>(p, stream);
        default: return launch_typed<_Float16>(p, stream);
    }
}

bool linear_i8_fused(int m, int n, int kp, int dtype) {
    // Measured on an MI355X (us, one launch / quantise, then product):
    //   8 x 8192 x 4096: 11.6 / 13.5    16 x 8192 x 2048: 10.3 / 10.5   1 x 1024 x 32768: 20.7 / 34.5   16 x 512 x 512 fp32: 5.8 / 6.8
    //   where the weights take more than one round of blocks:  1 x 28672 x 4096: 27.6 / 26.8    8 x 28672 x 4096: 33.7 / 33.2
    return m <= 16 && (n + 15) / 16 <= 2 * device_cu_count() && (1 << fused_row_bits(m)) * (int64_t)kp * (dtype == CMDI_DT_F32 ? 4 : 2) <= kI8FusedBytes;
}

hipError_t launch_linear_i8_fused(const QuantRowsArgs& x, const GemmI8Args& p, hipStream_t stream) {
    const int lanes = 8 - fused_row_bits(p.m), lds = p.m * (p.k + 16);
    const dim3 grid((unsigned)((p.n + 15) / 16));
    switch (p.dtype) {
        case CMDI_DT_F32: linear_i8_rows_kernel<float><<<grid, 256, lds, stream>>>(x, p, lanes); break;
        case CMDI_DT_BF16: linear_i8_rows_kernel<Bf16><<<grid, 256, lds, stream>>>(x, p, lanes); break;
        default: linear_i8_rows_kernel<_Float16><<<grid, 256, lds, stream>>>(x, p, lanes); break;
    }
    return hipGetLastError();
}

}  // namespace cmdi
