// Products of ragged groups of rows with their experts' weights
// (bitsparse_amd/experts.py).  Expert e has the rows offsets[e] up to
// offsets[e + 1]:
//   forward  y[r, n]     = sum over d of x[src r, d] W[e][n, d]
//   dx       dx[r, d]    = sum over n of dy[r, n] W[e][n, d]
//   dW       dW[e][n, d] = sum over the expert's r of dy[r, n] x[src r, d]
// src r is r, or the row's token, so that gathered rows are never written.
//
// bf16 operands, fp32 sums, one rounding.  A workgroup a tile of results; the
// tiles of ragged groups are found on the device, so the host knows nothing
// of the routing and waits for nothing.
#include <algorithm>

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
    bf16* c;
    int64_t c_expert;
    int m, n, k;                                // of one expert's product; m or k of the rows is -1
    int tiles_m, tiles_n;
    int act;
    float act_k;
};

// ---------------------------------------------------------------------------
// LDS tiles of a K-step of 64.  K contiguous: rows of 128 bytes, the 16-byte
// chunk c of row r at c ^ r % 8, so the 16 lanes that a fragment read serves at a
// time meet all 64 banks.  K down the rows: T columns a row, the chunk u of
// row k at u ^ 2 (k % 4 + 4 (k / 8 % 2)): 32 lanes of a transposing read take
// half of eight rows.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int col_turn(int k) { return 2 * ((k & 3) + 4 * (k >> 3 & 1)); }

template <int T, bool ALONG_K>
__device__ __forceinline__ bf16x8 read_fragment(const char* tile, int r0, int k0, int lane)
{
    if constexpr (ALONG_K) {
        const int r = r0 + (lane & 15), c = k0 / 8 + (lane >> 4);
        return *reinterpret_cast<const bf16x8*>(tile + r * kRowBytes + ((c ^ (r & 7)) * 16));
    } else {
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const int j = lane & 15, k = k0 + 8 * (lane >> 4) + (j >> 2), u = r0 / 8 + ((j & 3) >> 1);
        const char* at = tile + k * (T * 2) + ((u ^ col_turn(k)) * 16) + (j & 1) * 8;
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

// A tile's expert: the tile'th tile of `size` rows in the order of the experts, or behind the last expert's
struct Group {
    int expert;                 // -1: behind
    int64_t first, end;         // the expert's rows
    int64_t tile;               // of the expert, or of the rows behind
};
__device__ __forceinline__ int group_bound(const ExpertGemm& g, int e)
{
    return (int)max((int64_t)0, min((int64_t)g.offsets[e], g.rows));
}
__device__ __forceinline__ Group find_group(const ExpertGemm& g, int tile, int size)
{
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int e0 = 0; e0 < g.experts; e0 += 64) {
        const int e = e0 + lane;
        const int from = group_bound(g, min(e, g.experts)), to = max(from, group_bound(g, min(e + 1, g.experts)));
        const int tiles = (to - from + size - 1) / size;
        int sum = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(sum, d);
            sum += lane >= d ? o : 0;
        }
        const uint64_t past = __ballot(before + sum > tile);
        if (past) {
            const int at = __builtin_ctzll(past);
            const int mine = before + sum - tiles;
            return {e0 + at, (int64_t)(int)uniform_u32((uint32_t)__shfl(from, at)), (int64_t)(int)uniform_u32((uint32_t)__shfl(to, at)),
                    (int64_t)(tile - (int)uniform_u32((uint32_t)__shfl(mine, at)))};
        }
        before += (int)uniform_u32((uint32_t)__shfl(sum, 63));
    }
    return {-1, (int64_t)group_bound(g, g.experts), g.rows, (int64_t)(tile - before)};
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

// WGM x WGN waves, each 16 IM x 16 JN results
template <int KIND, bool GATHER, int WGM, int WGN, int IM, int JN>
__global__ __launch_bounds__(64 * WGM * WGN) void expert_gemm_kernel(ExpertGemm g)
{
    constexpr int WAVES = WGM * WGN, TM = 16 * IM * WGM, TN = 16 * JN * WGN;
    constexpr bool A_ALONG = KIND != kDw, B_ALONG = KIND == kForward;
    constexpr bool GA = GATHER && KIND == kForward, GB = GATHER && KIND == kDw;
    constexpr int A_BYTES = TM * kRowBytes, B_BYTES = TN * kRowBytes, STAGE = A_BYTES + B_BYTES;
    constexpr int LA = TM / 8 / WAVES, LB = TN / 8 / WAVES;     // loads of a wave, 1 KiB each
    static_assert(LA * 8 * WAVES == TM && LB * 8 * WAVES == TN, "a stage is whole loads of every wave");
    static_assert(2 * STAGE <= 160 * 1024, "LDS budget");
    __shared__ __attribute__((aligned(16))) char s_mem[2 * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = wave / WGN, wn = wave % WGN;

    const int tn = (int)blockIdx.x % g.tiles_n, tm = (int)blockIdx.x / g.tiles_n;
    Group grp;
    int64_t c_row, c_rows, k_total;
    if constexpr (KIND == kDw) {
        const int e = tm / g.tiles_m;
        const int from = group_bound(g, e);
        grp = {e, from, max(from, group_bound(g, e + 1)), tm % g.tiles_m};
        c_row = grp.tile * TM, c_rows = g.m, k_total = grp.end - grp.first;
    } else {
        grp = find_group(g, tm, TM);
        c_row = grp.first + grp.tile * TM, c_rows = grp.end, k_total = grp.expert < 0 ? 0 : g.k;
    }
    if (c_row >= c_rows) return;
    const int64_t c_col = (int64_t)tn * TN;

    // where this lane's parts of a stage come from
    uint32_t a_off[LA], b_off[LB];
    const int chunk = (lane & 7) ^ (lane >> 3);
    const bf16* b_base = g.b + (KIND == kDw ? 0 : max(0, grp.expert) * g.b_expert);
    const int64_t a_row_bytes = g.a_stride * 2, b_row_bytes = g.b_stride * 2;
    // K down the rows: this lane's row of a load and its chunk of columns
    auto along_m = [&](int i, int loads, int t, int& k, int& unit) {
        k = (wave * loads + i) * (512 / t) + lane / (t / 8);
        unit = (lane % (t / 8)) ^ col_turn(k);
    };
    i32x4 ra, rb;
    if constexpr (A_ALONG) {
        const bf16* base = GA ? g.a : g.a + c_row * g.a_stride;
        ra = rsrc_words(base, GA ? ((g.tokens - 1) * g.a_stride + g.k + 7) / 8 * 16 : (int64_t)kNoRow);
#pragma unroll
        for (int i = 0; i < LA; i++) {
            const int64_t r = (wave * LA + i) * 8 + (lane >> 3);
            const int64_t at = c_row + r < c_rows && k_total ? (GA ? source_row<GA>(g, c_row + r) : r) : -1;
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
    const int steps = (int)((k_total + kBK - 1) / kBK);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_mem;
    auto load = [&](int step, int stage) {
        const uint32_t lds = lds0 + stage * STAGE;
        const bool in_k = chunk * 8 + step * kBK < g.k;        // of an operand with K along its rows
        if constexpr (A_ALONG) {
#pragma unroll
            for (int i = 0; i < LA; i++)
                load_lds16(ra, lds + (wave * LA + i) * 1024, in_k ? a_off[i] : kNoRow, (uint32_t)step * kRowBytes);
        } else {
            // (the rows that are left bound the operand: those behind them are zeros)
            const int64_t at = grp.first + (int64_t)step * kBK, left = grp.end - at;
            const i32x4 r = rsrc_words(g.a + at * g.a_stride, (left - 1) * a_row_bytes + (g.m + 7) / 8 * 16);
#pragma unroll
            for (int i = 0; i < LA; i++) {
                int k, unit;
                along_m(i, LA, TM, k, unit);
                load_lds16(r, lds + (wave * LA + i) * 1024, (uint32_t)(k * a_row_bytes) + (uint32_t)(c_row * 2) + unit * 16, 0);
            }
        }
        if constexpr (B_ALONG) {
#pragma unroll
            for (int i = 0; i < LB; i++)
                load_lds16(rb, lds + A_BYTES + (wave * LB + i) * 1024, in_k ? b_off[i] : kNoRow, (uint32_t)step * kRowBytes);
        } else {
            const int64_t at = (KIND == kDw ? grp.first : 0) + (int64_t)step * kBK, end = KIND == kDw ? grp.end : g.k;
            const bf16* base = GB ? g.b : b_base + at * g.b_stride;
            const i32x4 r = rsrc_words(base, ((GB ? g.tokens : end - at) - 1) * b_row_bytes + (g.n + 7) / 8 * 16);
#pragma unroll
            for (int i = 0; i < LB; i++) {
                int k, unit;
                along_m(i, LB, TN, k, unit);
                int64_t src = k;
                if constexpr (GB) src = at + k < end ? source_row<GB>(g, at + k) : -1;
                load_lds16(r, lds + A_BYTES + (wave * LB + i) * 1024,
                           src < 0 ? kNoRow : (uint32_t)(src * b_row_bytes) + (uint32_t)(c_col * 2) + unit * 16, 0);
            }
        }
    };

    f32x4 acc[IM][JN];
#pragma unroll
    for (int i = 0; i < IM; i++)
#pragma unroll
        for (int j = 0; j < JN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (steps) load(0, 0);
    for (int step = 0; step < steps; step++) {
        // this step's parts are there and the other stage has been read, in every wave
        wait_for_loads();
        barrier_only();
        if (step + 1 < steps) load(step + 1, (step + 1) & 1);
        const char* ta = s_mem + (step & 1) * STAGE;
#pragma unroll
        for (int k0 = 0; k0 < kBK; k0 += 32) {
            bf16x8 fa[IM], fb[JN];
#pragma unroll
            for (int i = 0; i < IM; i++) fa[i] = read_fragment<TM, A_ALONG>(ta, wm * 16 * IM + 16 * i, k0, lane);
#pragma unroll
            for (int j = 0; j < JN; j++) fb[j] = read_fragment<TN, B_ALONG>(ta + A_BYTES, wn * 16 * JN + 16 * j, k0, lane);
#pragma unroll
            for (int i = 0; i < IM; i++)
#pragma unroll
                for (int j = 0; j < JN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa[i], acc[i][j], 0, 0, 0);
        }
    }

    // a lane has row lane % 16 and columns 4 (lane / 16) on of each block
    bf16* c = g.c + (KIND == kDw ? grp.expert * g.c_expert : 0);
    const bool wide = g.n % 4 == 0;
#pragma unroll
    for (int i = 0; i < IM; i++) {
        const int64_t r = c_row + (wm * IM + i) * 16 + (lane & 15);
        if (r >= c_rows) continue;
#pragma unroll
        for (int j = 0; j < JN; j++) {
            const int64_t col = c_col + (wn * JN + j) * 16 + 4 * (lane >> 4);
            if (col >= g.n) continue;
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = f32_to_bf16(KIND == kForward ? activated(acc[i][j][e], g.act, g.act_k) : acc[i][j][e]);
            uint16_t* to = reinterpret_cast<uint16_t*>(c) + r * g.n + col;
            if (wide) {
                *reinterpret_cast<uint2*>(to) = uint2{o[0] | o[1] << 16, o[2] | o[3] << 16};
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (col + e < g.n) to[e] = (uint16_t)o[e];
            }
        }
    }
}

template <int KIND, bool GATHER, int WGM, int WGN, int IM, int JN>
static int launch_gemm(ExpertGemm g, const char* what, hipStream_t st)
{
    constexpr int TM = 16 * IM * WGM, TN = 16 * JN * WGN;
    g.tiles_n = (g.n + TN - 1) / TN;
    g.tiles_m = KIND == kDw ? (g.m + TM - 1) / TM : 0;
    // every expert's last tile may be a part of one, and so may that of the rows behind them
    const int64_t tiles_m = KIND == kDw ? (int64_t)g.experts * g.tiles_m : g.rows / TM + g.experts + 2;
    if (tiles_m * g.tiles_n >= (1ll << 31)) return set_error(BS_ERR_INVALID, "%s: too many tiles", what);
    hipLaunchKernelGGL((expert_gemm_kernel<KIND, GATHER, WGM, WGN, IM, JN>), dim3((uint32_t)(tiles_m * g.tiles_n)), dim3(64 * WGM * WGN), 0, st, g);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? BS_OK : set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}

template <int KIND, bool GATHER>
static int launch_kind(const ExpertGemm& g, const char* what, hipStream_t st)
{
    return launch_gemm<KIND, GATHER, 2, 2, 4, 4>(g, what, st);
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
    if (y == nullptr || ((uintptr_t)y & 7u)) return set_error(BS_ERR_INVALID, "%s: null or misaligned y", what);
    ExpertGemm g = gemm_args(*experts, gather);
    g.a = static_cast<const bf16*>(x), g.a_stride = x_stride, g.b = static_cast<const bf16*>(W), g.b_stride = w_stride, g.b_expert = out * w_stride;
    g.c = static_cast<bf16*>(y), g.m = -1, g.n = (int)out, g.k = (int)in, g.act = act, g.act_k = act_k;
    return gather ? launch_kind<kForward, true>(g, what, (hipStream_t)stream) : launch_kind<kForward, false>(g, what, (hipStream_t)stream);
}

extern "C" int bs_expert_linear_dx(const bs_experts* experts, const void* dy, int64_t dy_stride, const void* W, int64_t w_stride, int64_t in,
                                   int64_t out, void* dx, void* stream)
{
    clear_error();
    const char* what = "bs_expert_linear_dx";
    if (const int rc = experts_check(experts, in, out, what); rc != BS_OK) return rc;
    if (experts->rows == 0) return BS_OK;
    const bool gather = experts->order != nullptr;
    (void)gather;
    if (const int rc = operand_check(what, "dy", dy, experts->rows, dy_stride, out, false); rc != BS_OK) return rc;
    if (const int rc = operand_check(what, "W", W, out, w_stride, in, false); rc != BS_OK) return rc;
    if (dx == nullptr || ((uintptr_t)dx & 7u)) return set_error(BS_ERR_INVALID, "%s: null or misaligned dx", what);
    ExpertGemm g = gemm_args(*experts, false);
    g.a = static_cast<const bf16*>(dy), g.a_stride = dy_stride, g.b = static_cast<const bf16*>(W), g.b_stride = w_stride, g.b_expert = out * w_stride;
    g.c = static_cast<bf16*>(dx), g.m = -1, g.n = (int)in, g.k = (int)out;
    return launch_kind<kDx, false>(g, what, (hipStream_t)stream);
}

extern "C" int bs_expert_linear_dw(const bs_experts* experts, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, int64_t in,
                                   int64_t out, void* dW, void* stream)
{
    clear_error();
    const char* what = "bs_expert_linear_dw";
    if (const int rc = experts_check(experts, in, out, what); rc != BS_OK) return rc;
    const bool gather = experts->order != nullptr;
    if (const int rc = operand_check(what, "dy", dy, experts->rows, dy_stride, out, false); rc != BS_OK) return rc;
    if (const int rc = operand_check(what, "x", x, experts->rows == 0 ? 0 : gather ? experts->tokens : experts->rows, x_stride, in, gather); rc != BS_OK) return rc;
    if (dW == nullptr || ((uintptr_t)dW & 7u)) return set_error(BS_ERR_INVALID, "%s: null or misaligned dW", what);
    ExpertGemm g = gemm_args(*experts, gather);
    g.a = static_cast<const bf16*>(dy), g.a_stride = dy_stride, g.b = static_cast<const bf16*>(x), g.b_stride = x_stride;
    g.c = static_cast<bf16*>(dW), g.c_expert = in * out, g.m = (int)out, g.n = (int)in, g.k = -1;
    return gather ? launch_kind<kDw, true>(g, what, (hipStream_t)stream) : launch_kind<kDw, false>(g, what, (hipStream_t)stream);
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
