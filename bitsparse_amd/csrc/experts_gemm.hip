// Products of ragged groups of rows with their experts' weights
// (bitsparse_amd/experts.py).  Expert e has the rows offsets[e] up to
// offsets[e + 1]:
//   forward  y[r, n]     = sum over d of x[src r, d] W[e][n, d]
//   dx       dx[r, d]    = sum over n of dy[r, n] W[e][n, d]
//   dW       dW[e][n, d] = sum over the expert's r of dy[r, n] x[r, d]
// src r is r, or in forward the row's token: gathered rows are read where they are.  dW takes them written out in order.
//
// bf16 operands, fp32 sums, one rounding.  A workgroup a tile of results; the
// tiles of ragged groups are found on the device, so the host knows nothing
// of the routing and waits for nothing.
//
// Bound by the products.  On several boxes: 32768 rows of 16 experts, 2048 -> 4096, 476 to 521 us forward, 465 to 504 dx, 469
// to 504 dW, 1.06 to 1.18 PFLOP/s, the matrix pipes at work in 55 to 59% of the cycles; the library's dense product of that
// size 385 to 394 us, 1.39 to 1.43.  One expert with 4096 rows, 16384 -> 4096: 390 to 439 us, 1.25 to 1.41, the library's 344 to 352,
// 1.56 to 1.60.  16384 rows of 8 experts, 768 -> 2048, 55 to 73 us, 0.71 to 0.94, the library's 52 to 54.  The differences are the
// loop's own (of one expert), the groups' part tiles, the last round's idle CUs and, of shorter sums, the tiles' starts and ends.
#include <algorithm>
#include <cmath>

#include "bs_host.h"
#include "gemm_common.h"
#include "rownorm.h"

namespace bs {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kForward = 0, kDx = 1, kDw = 2;
constexpr int kRowBytes = kBK * 2;              // a row of a K-step of an operand whose K is contiguous
constexpr uint32_t kNoRow = 0xfffffff0u;        // an offset behind every operand: reads zeros

struct ExpertGemm {
    const int32_t *offsets, *order;             // order: null, or the rows' pairs
    int experts, top_k;
    int64_t rows, tokens;                       // tokens: rows of a gathered operand
    const bf16 *a, *b;
    int64_t a_stride, b_stride, b_expert;       // elements
    void* c;
    int c_f32;                                  // results in 32 bits
    int64_t c_expert;
    int m, n, k;                                // of one expert's product; m or k of the rows is -1
    int tiles_m, tiles_n, panel;
    int rows_of_tiles;                          // as many as there may be
    int act;
    float act_k;
    int stream;                                 // results past the caches' size, stored around them
};

// ---------------------------------------------------------------------------
// LDS tiles of a K-step of 64.  K contiguous: rows of 128 bytes, the 16-byte
// chunk c of row r at c ^ r % 8, so the 16 lanes that a fragment read serves at a
// time meet all 64 banks.  K down the rows: T columns a row, the chunk u of
// row k at u ^ col_turn(k): 32 lanes of a transposing read take two chunks of
// eight rows, k % 4 + 8 (k / 8 % 2), which lie 16 chunks or (T = 64) 8 apart.
// ---------------------------------------------------------------------------
template <int T>
__device__ __forceinline__ int col_turn(int k)
{
    static_assert(T % 64 == 0 && (T & (T - 1)) == 0, "whole loads of rows, chunks that a turn stays among");
    return T == 64 ? 2 * ((k >> 1 & 1) + 2 * (k >> 3 & 1)) : 2 * ((k & 3) + 4 * (k >> 3 & 1));
}

template <int T, bool ALONG_K>
__device__ __forceinline__ bf16x8 read_fragment(const char* tile, int r0, int k0, int lane)
{
    if constexpr (ALONG_K) {
        const int r = r0 + (lane & 15), c = k0 / 8 + (lane >> 4);
        return *reinterpret_cast<const bf16x8*>(tile + r * kRowBytes + ((c ^ (r & 7)) * 16));
    } else {
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const int j = lane & 15, k = k0 + 8 * (lane >> 4) + (j >> 2), u = r0 / 8 + ((j & 3) >> 1);
        const char* at = tile + k * (T * 2) + ((u ^ col_turn<T>(k)) * 16) + (j & 1) * 8;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 4 * (T * 2)));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

__device__ __forceinline__ i32x4 rsrc_words(const void* p, int64_t bytes)
{
    const uint64_t a = (uint64_t)p;
    const uint32_t n = (uint32_t)max((int64_t)0, min(bytes, (int64_t)kNoRow));
    return i32x4{(int)uniform_u32((uint32_t)a), (int)uniform_u32((uint32_t)(a >> 32) & 0xffffu), (int)uniform_u32(n), 0x00020000};
}
// 16 bytes a lane from `rsrc` at voff + soff straight into LDS, 1 KiB from `lds` on; behind the operand's end zeros
__device__ __forceinline__ void load_lds16(i32x4 rsrc, uint32_t lds, uint32_t voff, uint32_t soff)
{
    // (one wait state between the write of m0 and its use)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc), "s"(soff));
}
__device__ __forceinline__ void wait_for_loads() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier_only()
{
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// LDS written by some lanes of a wave and read by others of it, or the other way round
__device__ __forceinline__ void wave_order()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A tile's expert: the tile'th tile of `size` rows in the order of the experts, or of the rows of no expert, those before the
// first one's and then those behind the last one's
struct Group {
    int expert;                 // -1: none
    int64_t first, end;         // the expert's rows, or those before or behind all of them
    int64_t tile;               // of these rows
};
__device__ __forceinline__ int group_bound(const ExpertGemm& g, int e)
{
    return (int)max((int64_t)0, min((int64_t)g.offsets[e], g.rows));
}
// the sum over this lane and those below it: four steps inside rows of 16 lanes, two across them
__device__ __forceinline__ int wave_scan(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);     // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);     // last lane of rows 0, 2 into rows 1, 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);     // last lane of row 1 into rows 2, 3
    return v;
}
// How `size` rows a tile lie over the experts
struct Groups {
    int from, to, sum;          // of lane e's expert e < 64, and the tiles of those up to it
    int lead;                   // rows before the first expert's
    int64_t all;                // tiles, with those of the rows of no expert
    __device__ __forceinline__ void load(const ExpertGemm& g, int e, int size)
    {
        from = group_bound(g, min(e, g.experts)), to = max(from, group_bound(g, min(e + 1, g.experts)));
        sum = wave_scan((int)((uint32_t)(to - from + size - 1) / (uint32_t)size));      // (64 experts' tiles are below 2^31)
    }
    __device__ __forceinline__ Groups(const ExpertGemm& g, int size)
    {
        const int lane = threadIdx.x & 63;
        all = (g.rows - group_bound(g, g.experts) + size - 1) / size;
        for (int e = 64; e < g.experts; e += 64) {
            load(g, e + lane, size);
            all += __builtin_amdgcn_readlane(sum, 63);
        }
        load(g, lane, size);
        lead = __builtin_amdgcn_readlane(from, 0);
        all += __builtin_amdgcn_readlane(sum, 63) + (lead + (int64_t)size - 1) / size;
    }
    // (once)
    __device__ __forceinline__ Group find(const ExpertGemm& g, int tile, int size) const
    {
        Groups now = *this;
        int64_t before = 0;     // (the tiles of offsets that overlap add up past 2^31)
        for (int e0 = 0; e0 < g.experts; e0 += 64) {
            if (e0) now.load(g, e0 + (threadIdx.x & 63), size);
            const uint64_t past = __ballot(before + now.sum > tile);
            if (past) {
                const int at = __builtin_ctzll(past), from_ = __builtin_amdgcn_readlane(now.from, at), to_ = __builtin_amdgcn_readlane(now.to, at);
                const int tiles = (int)((uint32_t)(to_ - from_ + size - 1) / (uint32_t)size);
                return {e0 + at, from_, to_, tile - before - (__builtin_amdgcn_readlane(now.sum, at) - tiles)};
            }
            before += __builtin_amdgcn_readlane(now.sum, 63);
        }
        const int64_t rest = tile - before, front = (lead + (int64_t)size - 1) / size;
        if (rest < front) return {-1, 0, lead, rest};
        return {-1, (int64_t)group_bound(g, g.experts), g.rows, rest - front};
    }
};

// The expert with the rank'th most rows, of up to 8: dW's longest sums begin first and its shortest fill the end (16384 rows of
// 8 experts 768 -> 2048 70.5 -> 62.2 us).  More experts' shorter sums even out by themselves (of 16 no change or 33 -> 36 us,
// of 64 107 -> 125).
__device__ __forceinline__ int by_length(const ExpertGemm& g, int rank)
{
    if (g.experts > 8) return rank;
    const int lane = threadIdx.x & 63, e = min(lane, g.experts - 1);
    const int from = group_bound(g, e), rows = lane < g.experts ? max(0, group_bound(g, e + 1) - from) : -1;
    int before = 0;
    for (int i = 0; i < g.experts; i++) {
        const int other = __builtin_amdgcn_readlane(rows, i);
        before += other > rows || (other == rows && i < lane);
    }
    return __builtin_ctzll(__ballot(lane < g.experts && before == rank));
}

// the operand's row of row r, or -1
template <bool GATHER>
__device__ __forceinline__ int64_t source_row(const ExpertGemm& g, int64_t r)
{
    if constexpr (!GATHER) return r;
    const int pair = g.order[r], t = pair / g.top_k;
    return pair >= 0 && t < g.tokens ? t : -1;
}

__device__ __forceinline__ float activated(float z, int act, float k)
{
    if (act == BS_ACT_NONE) return z;
    const uint32_t b = f32_to_bf16(z);
    const uint32_t r = bf16_to_f32(b) <= 0.f ? 0u : b;      // (NaN kept, as torch's)
    return bf16_to_f32(act == BS_ACT_RELU ? r : relu2_sq_bits(r, k));
}

// four results of a row from column `col` on; `row`: the row's first element
template <int KIND>
__device__ __forceinline__ void store_four(const ExpertGemm& g, int64_t row, int64_t col, const f32x4& v)
{
    if (col >= g.n) return;
    const int nv = (int)min((int64_t)4, g.n - col);
    if (KIND == kDx && g.c_f32) {
        float* to = static_cast<float*>(g.c) + row + col;
        if (g.n % 4 == 0) {
            *reinterpret_cast<f32x4*>(to) = v;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (e < nv) to[e] = v[e];
        }
        return;
    }
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = f32_to_bf16(KIND == kForward ? activated(v[e], g.act, g.act_k) : v[e]);
    uint16_t* to = static_cast<uint16_t*>(g.c) + row + col;
    if (g.n % 4 == 0) {
        *reinterpret_cast<uint2*>(to) = uint2{o[0] | o[1] << 16, o[2] | o[3] << 16};
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (e < nv) to[e] = (uint16_t)o[e];
    }
}

// The results from (c_row, c_col) on of `grp`, rows up to c_rows: WGM x WGN waves, each 16 IM x 16 JN of them.  AHEAD:
// fragments are read ahead of the barrier, for a workgroup that has a CU to itself.
template <int KIND, bool GATHER, int WGM, int WGN, int IM, int JN, int STAGES, bool AHEAD>
__device__ __forceinline__ void gemm_tile(const ExpertGemm& g, const Group& grp, int64_t c_row, int64_t c_rows, int64_t c_col, int64_t k_total, char* s_mem)
{
    constexpr int WAVES = WGM * WGN, TM = 16 * IM * WGM, TN = 16 * JN * WGN;
    constexpr bool A_ALONG = KIND != kDw, B_ALONG = KIND == kForward;
    static_assert(!GATHER || KIND == kForward, "x is gathered by the forward product alone");
    constexpr int A_BYTES = TM * kRowBytes, B_BYTES = TN * kRowBytes, STAGE = A_BYTES + B_BYTES;
    constexpr int LA = TM / 8 / WAVES, LB = TN / 8 / WAVES;     // loads of a wave, 1 KiB each
    static_assert(LA * 8 * WAVES == TM && LB * 8 * WAVES == TN, "a stage is whole loads of every wave");
    static_assert(!AHEAD || STAGES == 2, "two stages in turn");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = wave / WGN, wn = wave % WGN;
    if (c_row >= c_rows || c_col >= g.n) return;

    // where this lane's parts of a stage come from
    uint32_t a_off[LA], b_off[LB];
    const int chunk = (lane & 7) ^ (lane >> 3);
    const bf16* b_base = g.b + (KIND == kDw ? 0 : max(0, grp.expert) * g.b_expert);
    const int64_t a_row_bytes = g.a_stride * 2, b_row_bytes = g.b_stride * 2;
    // K down the rows: this lane's row of a load and its chunk of columns
    auto along_m = [&](int i, int loads, auto t, int& k, int& unit) {
        constexpr int T = decltype(t)::value;
        k = (wave * loads + i) * (512 / T) + lane / (T / 8);
        unit = (lane % (T / 8)) ^ col_turn<T>(k);
    };
    i32x4 ra = {}, rb = {};
    if constexpr (A_ALONG) {
        const bf16* base = GATHER ? g.a : g.a + c_row * g.a_stride;
        ra = rsrc_words(base, GATHER ? ((g.tokens - 1) * g.a_stride + g.k + 7) / 8 * 16 : (int64_t)kNoRow);
#pragma unroll
        for (int i = 0; i < LA; i++) {
            const int64_t r = (wave * LA + i) * 8 + (lane >> 3);
            const int64_t at = c_row + r < c_rows && k_total ? (GATHER ? source_row<GATHER>(g, c_row + r) : r) : -1;
            a_off[i] = at < 0 ? kNoRow : (uint32_t)(at * a_row_bytes) + chunk * 16;
        }
    }
    if constexpr (B_ALONG) {
        rb = rsrc_words(b_base, (int64_t)g.n * b_row_bytes);
#pragma unroll
        for (int i = 0; i < LB; i++) {
            const int64_t r = c_col + (wave * LB + i) * 8 + (lane >> 3);
            b_off[i] = r < g.n ? (uint32_t)(r * b_row_bytes) + chunk * 16 : kNoRow;
        }
    }
    if constexpr (!A_ALONG) {
#pragma unroll
        for (int i = 0; i < LA; i++) {
            int k, unit;
            along_m(i, LA, IC<TM>{}, k, unit);
            a_off[i] = (uint32_t)(k * a_row_bytes) + (uint32_t)(c_row * 2) + unit * 16;
        }
    }
    if constexpr (!B_ALONG) {
#pragma unroll
        for (int i = 0; i < LB; i++) {
            int k, unit;
            along_m(i, LB, IC<TN>{}, k, unit);
            b_off[i] = (uint32_t)(k * b_row_bytes) + (uint32_t)(c_col * 2) + unit * 16;
        }
    }
    const int steps = (int)((k_total + kBK - 1) / kBK);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_mem;
    // the q-th of this wave's loads of a step: first those of A
    constexpr int LOADS = LA + LB;
    i32x4 step_a = ra, step_b = rb;
    auto load_one = [&](int q, int step, int stage) {
        const uint32_t lds = lds0 + stage * STAGE;
        if (q < LA) {
            const uint32_t to = lds + (wave * LA + q) * 1024;
            if constexpr (A_ALONG) {
                load_lds16(ra, to, chunk * 8 + step * kBK < g.k ? a_off[q] : kNoRow, (uint32_t)step * kRowBytes);
            } else {
                // (the rows that are left bound the operand: those behind them are zeros)
                const int64_t at = grp.first + (int64_t)step * kBK, left = grp.end - at;
                if (q == 0) step_a = rsrc_words(g.a + at * g.a_stride, (left - 1) * a_row_bytes + (g.m + 7) / 8 * 16);
                load_lds16(step_a, to, a_off[q], 0);
            }
        } else {
            const int i = q - LA;
            const uint32_t to = lds + A_BYTES + (wave * LB + i) * 1024;
            if constexpr (B_ALONG) {
                load_lds16(rb, to, chunk * 8 + step * kBK < g.k ? b_off[i] : kNoRow, (uint32_t)step * kRowBytes);
            } else {
                const int64_t at = (KIND == kDw ? grp.first : 0) + (int64_t)step * kBK, end = KIND == kDw ? grp.end : g.k;
                if (i == 0) step_b = rsrc_words(b_base + at * g.b_stride, (end - at - 1) * b_row_bytes + (g.n + 7) / 8 * 16);
                load_lds16(step_b, to, b_off[i], 0);
            }
        }
    };
    auto load_all = [&](int step, int stage) {
#pragma unroll
        for (int q = 0; q < LOADS; q++) load_one(q, step, stage);
    };

    // A step is two halves of 32 of K.  A fragment of A is read again, for the next half, as soon as its last product is
    // under way, those of B into a second set.  The one barrier of a step stands a quarter into its second half: by then
    // all of the step's stage is in registers, so that it is loaded again, and the next step's stage has come, a whole
    // step after its loads.
    constexpr int MEET = IM / 4;
    static_assert(!AHEAD || LOADS <= 2 * IM - MEET, "a place in the loop for each load");
    bf16x8 fa[IM], fb[2][JN];
    auto read_a = [&](int stage, int i, int k0) { fa[i] = read_fragment<TM, A_ALONG>(s_mem + stage * STAGE, wm * 16 * IM + 16 * i, k0, lane); };
    auto read_b = [&](int stage, int j, int k0) {
        fb[k0 / 32][j] = read_fragment<TN, B_ALONG>(s_mem + stage * STAGE + A_BYTES, wn * 16 * JN + 16 * j, k0, lane);
    };
    f32x4 acc[IM][JN];
#pragma unroll
    for (int i = 0; i < IM; i++)
#pragma unroll
        for (int j = 0; j < JN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (!AHEAD) {
#pragma unroll
        for (int i = 0; i < STAGES - 1; i++)
            if (i < steps) load_all(i, i);
        for (int step = 0, stage = 0; step < steps; step++) {
            // this step's stage has come and the last one's has been read, in every wave
            if (step + STAGES - 2 < steps)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * (LA + LB)) : "memory");
            else
                wait_for_loads();
            barrier_only();
            if (step + STAGES - 1 < steps) {
                const int last = stage == 0 ? STAGES - 1 : stage - 1;
                load_all(step + STAGES - 1, last);
            }
#pragma unroll
            for (int k0 = 0; k0 < kBK; k0 += 32) {
#pragma unroll
                for (int i = 0; i < IM; i++) read_a(stage, i, k0);
#pragma unroll
                for (int j = 0; j < JN; j++) read_b(stage, j, k0);
#pragma unroll
                for (int i = 0; i < IM; i++)
#pragma unroll
                    for (int j = 0; j < JN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[k0 / 32][j], fa[i], acc[i][j], 0, 0, 0);
            }
            stage = stage == STAGES - 1 ? 0 : stage + 1;
        }
    }
    if (AHEAD && steps) {
        load_all(0, 0);
        if (steps > 1) {
            load_all(1, 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LA + LB) : "memory");
        } else {
            wait_for_loads();
        }
        barrier_only();
#pragma unroll
        for (int i = 0; i < IM; i++) read_a(0, i, 0);
#pragma unroll
        for (int j = 0; j < JN; j++) read_b(0, j, 0);
    }
    for (int step = 0; AHEAD && step < steps; step++) {
        const int stage = step & 1;
#pragma unroll
        for (int i = 0; i < IM; i++) {
#pragma unroll
            for (int j = i; j < JN; j += IM) read_b(stage, j, 32);
#pragma unroll
            for (int j = 0; j < JN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[0][j], fa[i], acc[i][j], 0, 0, 0);
            read_a(stage, i, 32);
            __builtin_amdgcn_sched_barrier(0);
            // (the last of the loads that began in the step before)
            if (step > 0 && step + 1 < steps && IM - MEET + i < LOADS) load_one(IM - MEET + i, step + 1, stage ^ 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        // (behind the last step the next stage holds what it held: read, not used)
#pragma unroll
        for (int i = 0; i < IM; i++) {
            if (i == MEET) {
                wait_for_loads();
                barrier_only();
            }
#pragma unroll
            for (int j = i - MEET; j < JN && j >= 0; j += IM - MEET) read_b(stage ^ 1, j, 0);
#pragma unroll
            for (int j = 0; j < JN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[1][j], fa[i], acc[i][j], 0, 0, 0);
            if (i >= MEET) read_a(stage ^ 1, i, 0);
            if (i == MEET)
#pragma unroll
                for (int o = 0; o < MEET; o++) read_a(stage ^ 1, o, 0);
            __builtin_amdgcn_sched_barrier(0);
            // (a load at a time: more at once hold up the products behind them)
            if (step + 2 < steps && i >= MEET && i - MEET < LOADS) load_one(i - MEET, step + 2, stage);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // a lane has row lane % 16 and columns 4 (lane / 16) on of each block
    const int64_t c0 = KIND == kDw ? (int64_t)grp.expert * g.c_expert : 0;
    // Out as whole rows of the wave's columns through LDS, 16 rows at a time: stored from the lanes that hold them, 8 bytes
    // of 16 rows each, the results take a seventh of 16384 x 768 -> 2048's time (82 us instead of 72).
    auto store_rows = [&](auto wide) {
        constexpr int SIZE = decltype(wide)::value;                                     // bytes of a result
        constexpr int ROW = 16 * JN * SIZE, CHUNKS = ROW / 16, ROWS = 64 / CHUNKS;      // of a row; rows of a store
        static_assert(WAVES * 16 * ROW <= STAGES * STAGE, "LDS budget");
        char* const out = s_mem + wave * (16 * ROW);
        if (steps) {
            wait_for_loads();
            barrier_only();     // (the stages have been read)
        }
#pragma unroll
        for (int i = 0; i < IM; i++) {
            const int r = lane & 15;
            auto at_chunk = [&](int row, int c) { return out + row * ROW + ((c ^ (row & (CHUNKS - 1))) * 16); };
#pragma unroll
            for (int j = 0; j < JN; j++) {
                if constexpr (SIZE == 4) {
                    *reinterpret_cast<f32x4*>(at_chunk(r, 4 * j + (lane >> 4))) = acc[i][j];
                } else {
                    uint32_t o[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) o[e] = f32_to_bf16(KIND == kForward ? activated(acc[i][j][e], g.act, g.act_k) : acc[i][j][e]);
                    *reinterpret_cast<uint2*>(at_chunk(r, 2 * j + (lane >> 5)) + (lane >> 4 & 1) * 8) = uint2{o[0] | o[1] << 16, o[2] | o[3] << 16};
                }
            }
            wave_order();
#pragma unroll
            for (int u = 0; u < 16 / ROWS; u++) {
                const int row = u * ROWS + lane / CHUNKS, c = lane % CHUNKS;
                const uint4 v = *reinterpret_cast<const uint4*>(at_chunk(row, c));
                const int64_t at = c_row + (wm * IM + i) * 16 + row, col = c_col + wn * 16 * JN + c * (16 / SIZE);
                if (at >= c_rows || col >= g.n) continue;
                char* const to = static_cast<char*>(g.c) + (c0 + at * g.n + col) * SIZE;
                if (g.stream)
                    st16<true>(to, v);
                else
                    st16<false>(to, v);
            }
            wave_order();
        }
    };
    if (KIND == kDx && g.c_f32 && g.n % 4 == 0) return store_rows(IC<4>{});
    if (!(KIND == kDx && g.c_f32) && g.n % 8 == 0) return store_rows(IC<2>{});
#pragma unroll
    for (int i = 0; i < IM; i++) {
        const int64_t r = c_row + (wm * IM + i) * 16 + (lane & 15);
        if (r >= c_rows) continue;
#pragma unroll
        for (int j = 0; j < JN; j++) store_four<KIND>(g, c0 + r * g.n, c_col + (wn * JN + j) * 16 + 4 * (lane >> 4), acc[i][j]);
    }
}

// id of `all` tiles, `tiles_n` to a row of them: in panels of g.panel rows
__device__ __forceinline__ void panel_tile(const ExpertGemm& g, int id, int rows, int& tm, int& tn)
{
    const int panel = id / (g.panel * g.tiles_n), in_panel = id - panel * g.panel * g.tiles_n;
    const int high = min(g.panel, rows - panel * g.panel);
    tm = panel * g.panel + in_panel % high, tn = in_panel / high;
}
// Workgroups go round the XCDs in turn: of `at_once`, as many as are resident, each XCD takes a run
__device__ __forceinline__ int xcd_run(int id, int all, int at_once)
{
    const int group = id / at_once * at_once;
    return group + at_once <= all ? group + (id - group) % kXcds * (at_once / kXcds) + (id - group) / kXcds : id;
}

template <int KIND, bool GATHER, int WGM, int WGN, int IM, int JN, int STAGES, bool AHEAD>
__global__ __launch_bounds__(64 * WGM * WGN) void expert_gemm_kernel(ExpertGemm g)
{
    constexpr int TM = 16 * IM * WGM, TN = 16 * JN * WGN, LDS = STAGES * (TM + TN) * kRowBytes;
    static_assert(LDS <= 160 * 1024, "LDS budget");
    constexpr int AT_ONCE = kCus * (160 * 1024 / LDS);
    __shared__ __attribute__((aligned(16))) char s_mem[LDS];
    int tm, tn;
    if constexpr (KIND == kDw) {
        panel_tile(g, xcd_run((int)blockIdx.x, (int)gridDim.x, AT_ONCE), g.rows_of_tiles, tm, tn);
        const int e = by_length(g, tm / g.tiles_m), from = group_bound(g, e);
        const Group grp = {e, from, max(from, group_bound(g, e + 1)), tm % g.tiles_m};
        gemm_tile<KIND, GATHER, WGM, WGN, IM, JN, STAGES, AHEAD>(g, grp, grp.tile * TM, g.m, (int64_t)tn * TN, grp.end - grp.first, s_mem);
    } else {
        const Groups groups(g, TM);
        const int rows = AHEAD ? (int)min((int64_t)g.rows_of_tiles, groups.all) : g.rows_of_tiles, all = rows * g.tiles_n;
        // What is left of the last round: up to a quarter of one in quarters of tiles, up to half in halves, so that it takes
        // no whole round (16384 rows of 8 experts 768 -> 2048 gathered 73 -> 65 us on one box, 32768 of 16 2048 -> 4096 484 -> 476).
        const int left = AHEAD ? all % AT_ONCE : 0, parts = left == 0 || left > AT_ONCE / 2 ? 1 : left > AT_ONCE / 4 ? 2 : 4;
        const int id = (int)blockIdx.x, whole = parts == 1 ? all : all - left;
        const int tile = id < whole ? xcd_run(id, whole, AT_ONCE) : whole + (id - whole) / parts, part = id < whole ? 0 : (id - whole) % parts;
        if (tile >= all) return;
        panel_tile(g, tile, rows, tm, tn);
        const Group grp = groups.find(g, tm, TM);
        const int64_t c_row = grp.first + grp.tile * TM, c_col = (int64_t)tn * TN, k = grp.expert < 0 ? 0 : g.k;
        if constexpr (AHEAD) {
            if (id >= whole && parts == 4)
                return gemm_tile<KIND, GATHER, WGM, WGN, IM / 2, JN / 2, STAGES, AHEAD>(g, grp, c_row + part / 2 * (TM / 2), grp.end, c_col + part % 2 * (TN / 2), k, s_mem);
            if (id >= whole && parts == 2)
                return gemm_tile<KIND, GATHER, WGM, WGN, IM, JN / 2, STAGES, AHEAD>(g, grp, c_row, grp.end, c_col + part * (TN / 2), k, s_mem);
        }
        gemm_tile<KIND, GATHER, WGM, WGN, IM, JN, STAGES, AHEAD>(g, grp, c_row, grp.end, c_col, k, s_mem);
    }
}

// ---------------------------------------------------------------------------
// Forward for few rows an expert: bound by reading the experts' weights.  A
// workgroup has 16 columns and up to 32 rows, each of its eight waves an eighth
// of K, whose operands go from memory straight into registers, eight steps of
// 32 of K at once; the waves' sums meet in LDS, in order.
// ---------------------------------------------------------------------------
constexpr int kFewRows = 32, kFewCols = 16, kFewAhead = 8;

template <bool GATHER, int MR>
__device__ __forceinline__ void few_products(const ExpertGemm& g, const Group& grp, int64_t c_row, int64_t c_rows, int64_t c_col, f32x4 (*s_sum)[2][64])
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int steps = grp.expert < 0 ? 0 : (g.k + 31) / 32, from = steps * wave / 8, to = steps * (wave + 1) / 8;
    const int k_lane = (lane >> 4) * 8;
    const bf16* w = nullptr;
    if (c_col + (lane & 15) < g.n) w = g.b + max(0, grp.expert) * g.b_expert + (c_col + (lane & 15)) * g.b_stride + k_lane;
    const bf16* x[MR];
#pragma unroll
    for (int m = 0; m < MR; m++) {
        const int64_t r = c_row + 16 * m + (lane & 15), at = r < c_rows && steps ? source_row<GATHER>(g, r) : -1;
        x[m] = at < 0 ? nullptr : g.a + at * g.a_stride + k_lane;
    }
    f32x4 acc[MR];
#pragma unroll
    for (int m = 0; m < MR; m++) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s0 = from; s0 < to; s0 += kFewAhead) {
        bf16x8 fw[kFewAhead], fx[MR][kFewAhead];
#pragma unroll
        for (int u = 0; u < kFewAhead; u++) {
            const int k = (s0 + u) * 32;
            const bool in = s0 + u < to && k + k_lane < g.k;
            fw[u] = w && in ? *reinterpret_cast<const bf16x8*>(w + k) : bf16x8{};
#pragma unroll
            for (int m = 0; m < MR; m++) fx[m][u] = x[m] && in ? *reinterpret_cast<const bf16x8*>(x[m] + k) : bf16x8{};
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < kFewAhead; u++)
#pragma unroll
            for (int m = 0; m < MR; m++) acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[u], fx[m][u], acc[m], 0, 0, 0);
    }
#pragma unroll
    for (int m = 0; m < MR; m++) s_sum[wave][m][lane] = acc[m];
    __syncthreads();
    if (wave >= MR) return;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; i++) sum += s_sum[i][wave][lane];
    const int64_t r = c_row + 16 * wave + (lane & 15);
    if (r < c_rows) store_four<kForward>(g, r * g.n, c_col + 4 * (lane >> 4), sum);
}

template <bool GATHER>
__global__ __launch_bounds__(512) void expert_few_kernel(ExpertGemm g)
{
    __shared__ __attribute__((aligned(16))) f32x4 s_sum[8][2][64];
    const int tn = (int)blockIdx.x % g.tiles_n, tm = (int)blockIdx.x / g.tiles_n;
    const Group grp = Groups(g, kFewRows).find(g, tm, kFewRows);
    const int64_t c_row = grp.first + grp.tile * kFewRows, c_rows = min(grp.end, c_row + kFewRows);
    if (c_row >= c_rows) return;
    if (c_rows - c_row <= 16)
        few_products<GATHER, 1>(g, grp, c_row, c_rows, (int64_t)tn * kFewCols, s_sum);
    else
        few_products<GATHER, 2>(g, grp, c_row, c_rows, (int64_t)tn * kFewCols, s_sum);
}

template <int KIND, bool GATHER, int WGM, int WGN, int IM, int JN, int STAGES, bool AHEAD>
static int launch_gemm(ExpertGemm g, const char* what, hipStream_t st)
{
    constexpr int TM = 16 * IM * WGM, TN = 16 * JN * WGN;
    g.tiles_n = (g.n + TN - 1) / TN;
    g.tiles_m = KIND == kDw ? (g.m + TM - 1) / TM : 0;
    // (parts of tiles: one at most for each expert that has rows, and one each of the rows before and behind them)
    const int64_t tiles_m = KIND == kDw ? (int64_t)g.experts * g.tiles_m : g.rows / TM + std::min<int64_t>(g.experts + 2, g.rows);
    g.panel = 8;
    // (32768 rows of 16 experts 2048 -> 4096 510 us without, 489 with; dW of 64 experts 1024 -> 2048 147 and 110)
    g.stream = use_nontemporal((KIND == kDw ? (int64_t)g.experts * g.m : g.rows) * g.n * (KIND == kDx && g.c_f32 ? 4 : 2));
    // (AHEAD: and the parts of the last round's tiles)
    const int64_t blocks = tiles_m * g.tiles_n + (AHEAD && KIND != kDw ? 3 * kCus / 4 : 0);
    g.rows_of_tiles = (int)tiles_m;
    if (blocks >= (1ll << 32) / (64 * WGM * WGN)) return set_error(BS_ERR_INVALID, "%s: more tiles than a launch's 2^32 threads hold", what);
    hipLaunchKernelGGL((expert_gemm_kernel<KIND, GATHER, WGM, WGN, IM, JN, STAGES, AHEAD>), dim3((uint32_t)blocks), dim3(64 * WGM * WGN), 0, st, g);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? BS_OK : set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}

template <bool GATHER>
static int launch_few(ExpertGemm g, const char* what, hipStream_t st)
{
    g.tiles_n = (g.n + kFewCols - 1) / kFewCols;
    const int64_t tiles_m = g.rows / kFewRows + std::min<int64_t>(g.experts + 2, g.rows);
    hipLaunchKernelGGL(expert_few_kernel<GATHER>, dim3((uint32_t)(tiles_m * g.tiles_n)), dim3(512), 0, st, g);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? BS_OK : set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}

// What a product takes on tiles of one size, in us: rounds of as many as are
// resident at once, each its steps and a start and an end, or reading the
// weights (of 2 to 64 rows an expert: 4.1 TB/s, on larger tiles 3.2 to 3.9).  The
// host knows how many rows there are, not how they lie: half a tile is left over for each expert, of less than three quarters
// of a tile one in 20 has two (one alone has them all: 4096 rows 16384 -> 4096 425 us, 538 on the tile for half a tile more), and
// the longest of dW's sums has 1.4 times the mean's steps.
static double tile_time(const ExpertGemm& g, int kind, int tm, int tn, int at_once, double step)
{
    const double columns = (g.n + tn - 1) / tn;
    if (kind == kDw) {
        const double tiles = (double)g.experts * ((g.m + tm - 1) / tm) * columns, time = (double)g.rows / g.experts / kBK * step;
        return std::max(1.0, tiles / at_once) * (time + 5.0) + 0.4 * time;
    }
    const double experts = (double)std::min<int64_t>(g.experts, g.rows), each = (double)g.rows / experts / tm;
    const double tiles = experts * columns * (experts == 1 ? std::ceil(each) : each <= 0.25 ? 1.0 : each < 0.75 ? 1.05 * std::max(1.0, each + 0.5) : each + 0.5);
    const double weights = experts * g.n * g.k * 2 / (tm == 64 ? 4.1e6 : 3.6e6);
    // (the last round in parts of the largest tiles: its steps take 0.35 and 0.65 of a tile's)
    const double rounds = std::floor(tiles / at_once), left = tiles / at_once - rounds, steps = (double)g.k / kBK * step;
    const double last = left == 0.0 ? 0.0 : steps * (tm < 256 || left > 0.5 ? 1.0 : left > 0.25 ? 0.65 : 0.35) + 5.0;
    return std::max(weights, rounds * (steps + 5.0) + last);
}

// Forward for up to two rows an expert: expert_few_kernel (8 rows of 64 experts of 4096 -> 1024 13.2 us, on tiles of 64 x 64
// 20.9; 64 rows 50 and 65; 32 rows of 8 experts of 4096 -> 2048 24.3 and 22.0).  Else the tile whose time is least by
// tile_time (measured on one box in us, forward / dx / dW, x gathered in forward):
//   rows, experts, in -> out           64 x 64       128 x 128     192 x 128   256 x 256
//   16384,  8,  768 -> 2048         119 / 91 / 95    78 / 65 / 72   73 / 72 / -   65 / 55 / 74
//   16384,  8, 2048 ->  768          92 / 102 / 93   68 / 66 / 68   73 / 59 / -   56 / 68 / 73
//   32768, 16, 2048 -> 4096         976 / 929 / 996 621 / 570 / 572 559 / 532 / - 486 / 489 / 504
//   16384,  4,  512 -> 1024          49 / 38 / 40    34 / 31 / 63   30 / 26 / -   36 / 27 / 116
//     512,  8, 2048 -> 2048          22 / 22 / 41    27 / 24 / 21   31 / 30 / -   42 / 42 / 23
//    2048, 64, 4096 -> 1024         132 / 116 / 278  171 / 122 / 124     -         138 / 127 / 126
//    2048, 256, 2048 ->  512        122 / 137 / 280  156 / 131 / 123     -         141 / 150 / 129
//    8192, 64, 4096 -> 1024         192 / 194 / 347  174 / 159 / 165     -         217 / 164 / 158
template <int KIND, bool GATHER>
static int launch_kind(const ExpertGemm& g, const char* what, hipStream_t st)
{
    if constexpr (KIND == kForward)
        if (g.rows <= 2 * std::min<int64_t>(g.experts, g.rows)) return launch_few<GATHER>(g, what, st);
    const double small = tile_time(g, KIND, 64, 64, kCus * 2, 0.45), middle = tile_time(g, KIND, 128, 128, kCus * 2, 0.95),
                 wide = tile_time(g, KIND, 192, 128, kCus * 2, 1.3), large = tile_time(g, KIND, 256, 256, kCus, 1.55);
    const double best = std::min(std::min(small, middle), KIND == kDw ? large : std::min(wide, large));
    // (of equals, bound by the weights, the smallest)
    if (best == small) return launch_gemm<KIND, GATHER, 2, 2, 2, 2, 4, false>(g, what, st);
    if (best == middle) return launch_gemm<KIND, GATHER, 2, 2, 4, 4, 2, false>(g, what, st);
    if constexpr (KIND != kDw)
        if (best == wide) return launch_gemm<KIND, GATHER, 2, 2, 6, 4, 2, false>(g, what, st);
    return launch_gemm<KIND, GATHER, 2, 4, 8, 4, 2, true>(g, what, st);
}

static int experts_check(const bs_experts* x, int64_t in, int64_t out, const char* what)
{
    if (x == nullptr) return set_error(BS_ERR_INVALID, "%s: null arguments", what);
    if (x->experts < 1 || x->experts > 1024) return set_error(BS_ERR_INVALID, "%s: experts must be in 1..1024, got %d", what, x->experts);
    if (x->rows < 0 || x->rows >= (1ll << 31) || x->tokens < 0 || x->tokens >= (1ll << 31))
        return set_error(BS_ERR_INVALID, "%s: rows and tokens must be in 0..2^31-1", what);
    if (x->top_k < 1) return set_error(BS_ERR_INVALID, "%s: top_k must be positive, got %d", what, x->top_k);
    if (in < 1 || out < 1 || in > 65536 || out > 65536 || in * out >= (1ll << 30))
        return set_error(BS_ERR_INVALID, "%s: in and out must be in 1..65536 and in*out below 2^30, got %lld, %lld", what, (long long)in, (long long)out);
    if (x->offsets == nullptr || (((uintptr_t)x->offsets | (uintptr_t)x->order) & 3u))
        return set_error(BS_ERR_INVALID, "%s: null or misaligned offsets or order", what);
    return BS_OK;
}

// rows of `cols` at a stride that 16-byte loads take
static bool loads_ok(const void* p, int64_t stride, int64_t cols) { return ((uintptr_t)p & 15u) == 0 && stride % 8 == 0 && stride >= (cols + 7) / 8 * 8; }

static int operand_check(const char* what, const char* name, const void* p, int64_t rows, int64_t stride, int64_t cols, bool gathered)
{
    if (rows == 0) return BS_OK;
    if (p == nullptr) return set_error(BS_ERR_INVALID, "%s: null %s", what, name);
    if (!loads_ok(p, stride, cols) || stride >= (1ll << 22))
        return set_error(BS_ERR_INVALID, "%s: %s needs rows of whole 16-byte chunks at 16-byte addresses, less than 2^22 elements apart", what, name);
    if (gathered && rows * stride * 2 >= (int64_t)kNoRow)
        return set_error(BS_ERR_INVALID, "%s: gathered rows span 4 GiB or more", what);
    return BS_OK;
}

static ExpertGemm gemm_args(const bs_experts& x, bool gather)
{
    ExpertGemm g{};
    g.offsets = x.offsets, g.order = gather ? x.order : nullptr, g.experts = x.experts, g.top_k = x.top_k, g.rows = x.rows, g.tokens = x.tokens;
    return g;
}

// ---------------------------------------------------------------------------
// rows padded with zeros to whole 16-byte chunks
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void pad_rows_kernel(const uint16_t* x, int64_t rows, int64_t cols, int64_t stride, uint16_t* out, int64_t width)
{
    const int64_t per_row = width / 8, all = rows * per_row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per_row, c = (i - r * per_row) * 8;
        const Raw<bf16> v = load_raw(reinterpret_cast<const bf16*>(x) + r * stride + c, (int)max((int64_t)0, min((int64_t)8, cols - c)));
        *reinterpret_cast<uint4*>(out + i * 8) = uint4{v.w[0], v.w[1], v.w[2], v.w[3]};
    }
}

}  // namespace bs

using namespace bs;

extern "C" int bs_expert_linear(const bs_experts* experts, const void* x, int64_t x_stride, const void* W, int64_t w_stride, int64_t in,
                                int64_t out, int act, float act_k, void* y, void* stream)
{
    clear_error();
    const char* what = "bs_expert_linear";
    if (const int rc = experts_check(experts, in, out, what); rc != BS_OK) return rc;
    if (act < BS_ACT_NONE || act > BS_ACT_RELU2) return set_error(BS_ERR_INVALID, "%s: unknown activation %d", what, act);
    if (experts->rows == 0) return BS_OK;
    const bool gather = experts->order != nullptr;
    if (const int rc = operand_check(what, "x", x, gather ? experts->tokens : experts->rows, x_stride, in, gather); rc != BS_OK) return rc;
    if (const int rc = operand_check(what, "W", W, out, w_stride, in, false); rc != BS_OK) return rc;
    if (out * w_stride * 2 >= (int64_t)kNoRow) return set_error(BS_ERR_INVALID, "%s: an expert's W spans 4 GiB or more", what);
    if (y == nullptr || ((uintptr_t)y & 15u)) return set_error(BS_ERR_INVALID, "%s: null or misaligned y", what);
    ExpertGemm g = gemm_args(*experts, gather);
    g.a = static_cast<const bf16*>(x), g.a_stride = x_stride, g.b = static_cast<const bf16*>(W), g.b_stride = w_stride, g.b_expert = out * w_stride;
    g.c = y, g.m = -1, g.n = (int)out, g.k = (int)in, g.act = act, g.act_k = act_k;
    return gather ? launch_kind<kForward, true>(g, what, (hipStream_t)stream) : launch_kind<kForward, false>(g, what, (hipStream_t)stream);
}

extern "C" int bs_expert_linear_dx(const bs_experts* experts, const void* dy, int64_t dy_stride, const void* W, int64_t w_stride, int64_t in,
                                   int64_t out, void* dx, int dx_type, void* stream)
{
    clear_error();
    const char* what = "bs_expert_linear_dx";
    if (const int rc = experts_check(experts, in, out, what); rc != BS_OK) return rc;
    if (experts->rows == 0) return BS_OK;
    if (experts->order) return set_error(BS_ERR_INVALID, "%s: dx is rows in the experts' order, so order must be null", what);
    if (dx_type != BS_DT_BF16 && dx_type != BS_DT_F32) return set_error(BS_ERR_INVALID, "%s: dx dtype %d must be bf16 or fp32", what, dx_type);
    if (const int rc = operand_check(what, "dy", dy, experts->rows, dy_stride, out, false); rc != BS_OK) return rc;
    if (const int rc = operand_check(what, "W", W, out, w_stride, in, false); rc != BS_OK) return rc;
    if (dx == nullptr || ((uintptr_t)dx & 15u)) return set_error(BS_ERR_INVALID, "%s: null or misaligned dx", what);
    ExpertGemm g = gemm_args(*experts, false);
    g.a = static_cast<const bf16*>(dy), g.a_stride = dy_stride, g.b = static_cast<const bf16*>(W), g.b_stride = w_stride, g.b_expert = out * w_stride;
    g.c = dx, g.c_f32 = dx_type == BS_DT_F32, g.m = -1, g.n = (int)in, g.k = (int)out;
    return launch_kind<kDx, false>(g, what, (hipStream_t)stream);
}

extern "C" int bs_expert_linear_dw(const bs_experts* experts, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, int64_t in,
                                   int64_t out, void* dW, void* stream)
{
    clear_error();
    const char* what = "bs_expert_linear_dw";
    if (const int rc = experts_check(experts, in, out, what); rc != BS_OK) return rc;
    if (experts->order) return set_error(BS_ERR_INVALID, "%s: x is rows in the experts' order, so order must be null", what);
    if (const int rc = operand_check(what, "dy", dy, experts->rows, dy_stride, out, false); rc != BS_OK) return rc;
    if (const int rc = operand_check(what, "x", x, experts->rows, x_stride, in, false); rc != BS_OK) return rc;
    if (dW == nullptr || ((uintptr_t)dW & 15u)) return set_error(BS_ERR_INVALID, "%s: null or misaligned dW", what);
    ExpertGemm g = gemm_args(*experts, false);
    g.a = static_cast<const bf16*>(dy), g.a_stride = dy_stride, g.b = static_cast<const bf16*>(x), g.b_stride = x_stride;
    g.c = dW, g.c_expert = in * out, g.m = (int)out, g.n = (int)in, g.k = -1;
    return launch_kind<kDw, false>(g, what, (hipStream_t)stream);
}

extern "C" int bs_pad_rows(const void* x, int64_t rows, int64_t cols, int64_t stride, void* out, int64_t width, void* stream)
{
    clear_error();
    const char* what = "bs_pad_rows";
    if (rows < 0 || cols < 0 || width < cols || width % 8 || stride < 0 || (width && rows >= (1ll << 40) / width))
        return set_error(BS_ERR_INVALID, "%s: width must be a multiple of 8, at least cols, and rows*width below 2^40", what);
    if (rows == 0 || width == 0) return BS_OK;
    if ((cols && x == nullptr) || out == nullptr || ((uintptr_t)x & 1u) || ((uintptr_t)out & 15u))
        return set_error(BS_ERR_INVALID, "%s: null or misaligned pointer", what);
    const int64_t chunks = rows * (width / 8);
    hipLaunchKernelGGL(pad_rows_kernel, dim3((uint32_t)std::min<int64_t>((chunks + 255) / 256, 4096)), dim3(256), 0, (hipStream_t)stream,
                       static_cast<const uint16_t*>(x), rows, cols, stride, static_cast<uint16_t*>(out), width);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? BS_OK : set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}
