// Orthogonalising updates by Newton-Schulz products (bitsparse_amd/muon.py).
//
// For matrices U [m, n], m <= n (a taller one is taken as its transpose):
//   X_0     = U / (||U||_F + eps)
//   A_k     = X_k X_k^T                        gram      m^2 n   operations (half of a symmetric product)
//   B_k     = a I + b A_k + c A_k^2            poly      m^3
//   X_{k+1} = B_k X_k                          step      2 m^2 n
// (up to 256 rows X_{k+1} = a X_k + A_k (b X_k + c A_k X_k) instead: ns_narrow_kernel)
// and of the last X either itself in bf16 or, for an optimiser, the update of
// the weights.  U is the gradient or, with a momentum, M' = mu M + (1 - mu) G
// and U = (1 - mu) G + mu M' (Nesterov) or M'.
//
// The products run on the matrix cores with fp16 operands and fp32 sums.  X,
// A and B are held as fp16 times 2^12: ||X_0|| <= 1 keeps every singular
// value of the iteration below 1.21 and so every element of X, A and B below
// 3.5 (other coefficients: refused where they leave fp16's range), and elements down to 2^-26 keep all 11 bits.
// On gradients of full rank the result is 1.0-2.4e-3 from the exact one so (bf16
// operands, three bits shorter: 1.0-2.0e-2), where rounding it to bf16 costs
// 1.7e-3.  With t tokens, fewer than rows, the rounding noise in the directions
// without a gradient is raised by a = 3.44 a step, to about 0.16 / sqrt(t).
//
// Where the result goes into fp32 weights that is not enough: there each of X,
// A and B is held as two fp16 numbers, the value and what is left of it (22
// bits), and a product is three, high x high + high x low + low x high, one
// after the other into the same sums: 2e-6 from the exact result, as products
// of fp32 operands come, at the matrix cores' fp16 rate.
//
// All buffers are padded with zeros to whole tiles, which the products keep
// (B's padding only meets X's zero rows), so the main loop has no bounds.  A
// matrix [R, C] lies as C / 32 panels of R rows: every tile that a product
// loads for a step of 32 of K is then one run of memory (P's and gram's) or
// runs of 2 KiB (X's columns in step), where rows of 64 bytes out of a row-major
// matrix cost half of each cache line (4096 x 16384: gram 318 us instead of 355).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "bs_device.h"
#include "bs_host.h"
#include "rownorm.h"

namespace bs {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float kHeld = 4096.f;         // fp16 value = true value * kHeld
constexpr int kPanel = 32;              // columns of a panel; K of a main-loop step
constexpr int kNsBatch = 64;            // matrices of a launch
constexpr int kNsParts = 1024;          // most partial sums of squares of a matrix
constexpr int kNsCus = 256, kNsXcds = 8;

// (constants of a plain type: an unnamed one in a kernel's name differs between its host and device sides)
constexpr int kGram = 0, kPoly = 1, kStep = 2, kLast = 3;

struct NsMatrix {
    const void* g;
    void* m;
    void* w;                            // weights, or the result
    int64_t g_stride, m_stride, w_stride;
    int tall;                           // given as [n, m]
    float rate;                         // of its update
};
struct NsMatrices {
    NsMatrix at[kNsBatch];
};
// what a product's kernel is given of them: 4 KiB that only the last one reads
struct NsNone {
};
template <int KIND>
using NsGiven = std::conditional_t<KIND == kLast, NsMatrices, NsNone>;

// ---------------------------------------------------------------------------
// U, its norm and X_0
// ---------------------------------------------------------------------------
struct NsPrep {
    int64_t m, n, pitch, np;
    int g_f32, m_f32, momentum, nesterov, parts, precise;
    float mu, fresh, eps;               // fresh: 1 - mu
    double* parts_at;                   // [count][kNsParts]
    _Float16* x;                        // [count] matrices, precise: and the low parts behind all of them
    int64_t low;                        // elements from a value to its low part
};

__device__ __forceinline__ void ns_chunk(const void* p, int f32, int64_t i, int nv, float (&v)[8])
{
    if (f32) {
        const Raw<float> r = load_raw(static_cast<const float*>(p) + i, nv);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = raw_get(r, e);
    } else {
        const Raw<bf16> r = load_raw(static_cast<const bf16*>(p) + i, nv);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = raw_get(r, e);
    }
}

// 8 elements of U; with a momentum M' comes from (update) M or is read
__device__ __forceinline__ void ns_u(const NsPrep& a, const NsMatrix& t, int64_t r, int64_t c, int nv, bool update, float (&u)[8])
{
    ns_chunk(t.g, a.g_f32, r * t.g_stride + c, nv, u);
    if (!a.momentum) return;
    float m[8];
    ns_chunk(t.m, a.m_f32, r * t.m_stride + c, nv, m);
    if (update) {
#pragma unroll
        for (int e = 0; e < 8; e++) m[e] = a.mu * m[e] + a.fresh * u[e];
        if (a.m_f32) {
            store_raw(static_cast<float*>(t.m) + r * t.m_stride + c, to_raw<float>(m), nv);
        } else {
            const Raw<bf16> o = to_raw<bf16>(m);
            store_raw(static_cast<bf16*>(t.m) + r * t.m_stride + c, o, nv);
#pragma unroll
            for (int e = 0; e < 8; e++) m[e] = raw_get(o, e);       // U is of M' as stored
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) u[e] = a.nesterov ? a.fresh * u[e] + a.mu * m[e] : m[e];
}

// The momentum's update and partial sums of squares of U (in 64 bits: any
// gradient that fp32 holds has a norm).  blockIdx.y: the matrix.  Memory
// bound: 8 elements a load, four chunks of a thread in flight.
__global__ __launch_bounds__(256) void ns_norm_kernel(NsPrep a, NsMatrices mats)
{
    const NsMatrix t = mats.at[blockIdx.y];
    const uint32_t rows = (uint32_t)(t.tall ? a.n : a.m), cols = (uint32_t)(t.tall ? a.m : a.n);
    const uint32_t per_row = (cols + 7) / 8, total = rows * per_row;    // (< 2^30)
    const uint32_t step = gridDim.x * 256;
    double s = 0.0;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < total; i += 4 * step) {
        float u[4][8];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t at = i + k * step, r = at / per_row, c = (at - r * per_row) * 8;
            const int nv = at < total ? (int)min(8u, cols - c) : 0;
            ns_u(a, t, r, c, nv, true, u[k]);
#pragma unroll
            for (int e = 0; e < 8; e++) u[k][e] = e < nv ? u[k][e] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) s += (double)u[k][e] * (double)u[k][e];
    }
    __shared__ double s_part[256];
    s_part[threadIdx.x] = s;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) s_part[threadIdx.x] += s_part[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) a.parts_at[(int64_t)blockIdx.y * kNsParts + blockIdx.x] = s_part[0];
}

// where element (r, c) of a matrix lies
__device__ __forceinline__ int64_t panel_at(int64_t pitch, int64_t r, int64_t c)
{
    return ((c / kPanel) * pitch + r) * kPanel + c % kPanel;
}

__device__ __forceinline__ f16x8 ns_low(const float (&v)[8], f16x8 high)
{
    f16x8 l;
#pragma unroll
    for (int e = 0; e < 8; e++) l[e] = (_Float16)(v[e] - (float)high[e]);
    return l;
}

// X_0 in 64 x 64 tiles of [mp, np], zeros outside [m, n]; a taller matrix is
// turned through LDS.  Every workgroup adds the partial sums itself, in order.
__global__ __launch_bounds__(256) void ns_scale_kernel(NsPrep a, NsMatrices mats)
{
    const NsMatrix t = mats.at[blockIdx.z];
    __shared__ float s_t[64][68];
    __shared__ double s_q[256];
    const int64_t i0 = (int64_t)blockIdx.y * 64, j0 = (int64_t)blockIdx.x * 64;
    const int64_t rows = t.tall ? a.n : a.m, cols = t.tall ? a.m : a.n;
    float u[2][8];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int r = k * 32 + (int)threadIdx.x / 8, c = (int)threadIdx.x % 8 * 8;
        const int64_t gr = (t.tall ? j0 : i0) + r, gc = (t.tall ? i0 : j0) + c;
        const int nv = gr < rows ? (int)max((int64_t)0, min((int64_t)8, cols - gc)) : 0;
        ns_u(a, t, nv ? gr : 0, nv ? gc : 0, nv, false, u[k]);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            u[k][e] = e < nv ? u[k][e] : 0.f;
            if (t.tall) s_t[c + e][r] = u[k][e];
        }
    }
    double sq = 0.0;
    for (int i = threadIdx.x; i < a.parts; i += 256) sq += a.parts_at[(int64_t)blockIdx.z * kNsParts + i];
    s_q[threadIdx.x] = sq;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) s_q[threadIdx.x] += s_q[threadIdx.x + w];
        __syncthreads();
    }
    // (a norm past fp32's range, of elements inside it: of U 2^-40 instead)
    const double norm64 = sqrt(s_q[0]);
    const float down = norm64 > 1e38 ? 0x1p-40f : 1.f, norm = (float)(norm64 * (double)down) + a.eps * down;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int r = k * 32 + (int)threadIdx.x / 8, c = (int)threadIdx.x % 8 * 8;
        float v[8];
        f16x8 h;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[e] = (t.tall ? s_t[r][c + e] : u[k][e]) * down / norm * kHeld;
            h[e] = (_Float16)v[e];
        }
        _Float16* out = a.x + (int64_t)blockIdx.z * a.pitch * a.np + panel_at(a.pitch, i0 + r, j0 + c);
        *reinterpret_cast<f16x8*>(out) = h;
        if (a.precise) *reinterpret_cast<f16x8*>(out + a.low) = ns_low(v, h);
    }
}

// ---------------------------------------------------------------------------
// the products: C[i, j] = sum_k P[i, k] Q[j, k] (gram, poly) or
// sum_k P[i, k] Q[k, j] (step, last)
// ---------------------------------------------------------------------------
struct NsGemm {
    const _Float16 *p, *q;              // [count] matrices
    int64_t p_size, q_size, out_size;   // elements of one matrix
    int64_t p_low, q_low, out_low;      // precise: elements from a value to its low part
    int pitch;                          // rows from panel to panel
    int k_steps;                        // of one pass over K
    int passes;                         // 1, or 3 (precise)
    int tiles_m, tiles_n;               // of one matrix's product
    int tiles;                          // of all matrices, those left out by symmetry not counted
    int whole;                          // tiles that one workgroup does; the others' steps are
    int sharers;                        // dealt out evenly to this many workgroups,
    int lanes;                          // a group of tiles to each of this many sets of them
    float* part;                        // [sharers][2][tile]: their sums
    _Float16* out;
    float a, b, c;                      // poly
    // last
    int64_t m, n;
    int w_f32, update;
    float keep;
};

constexpr int kScratch = 16 * 36 * 4;  // bytes of LDS for a wave's results on their way out

// WGM x WGN waves, each a block of 32 IM x 32 JN; STAGES of the K loop in LDS
template <int WGM_, int WGN_, int IM_, int JN_, int STAGES_>
struct NsCfg {
    static constexpr int WGM = WGM_, WGN = WGN_, IM = IM_, JN = JN_, STAGES = STAGES_;
    static constexpr int WAVES = WGM * WGN, THREADS = 64 * WAVES;
    static constexpr int TM = 32 * IM * WGM, TN = 32 * JN * WGN;
    static constexpr int P_BYTES = TM * kPanel * 2, Q_BYTES = TN * kPanel * 2;
    static constexpr int STAGE = P_BYTES + Q_BYTES;
    static constexpr int LOADS = 4;                             // of a wave for a stage: 2 KiB of P, 2 of Q
    static constexpr int LDS = STAGES * STAGE + WAVES * kScratch;
    static_assert(TM == TN, "square tiles: half of a symmetric product is its lower triangle of tiles");
    static_assert(LDS <= 160 * 1024, "LDS budget");
    static_assert(P_BYTES == WAVES * 2048, "a stage is one pair of loads of P and one of Q of every wave");
    static_assert(STAGES >= 3, "a stage that is read, the one whose first fragments are read ahead, one that is loaded");
};
using NsLarge = NsCfg<2, 4, 4, 2, 4>;       // 256 x 256
using NsMiddle = NsCfg<2, 2, 2, 2, 4>;      // 128 x 128

// N runs of 1 KiB, one behind the other, from `rsrc` at voff + soff (16 bytes a
// lane) straight into LDS at `lds`
template <int N>
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, uint32_t lds, uint32_t voff, uint32_t soff)
{
    // (one wait state between the write of m0 and its use; the offset counts on both sides)
    static_assert(N == 2 || N == 4, "pairs of runs");
    if constexpr (N == 2)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds\n\t"
                     "buffer_load_dwordx4 %1, %2, %3 offen offset:1024 lds" ::"s"(lds), "v"(voff), "s"(rsrc), "s"(soff));
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds\n\t"
                     "buffer_load_dwordx4 %1, %2, %3 offen offset:1024 lds\n\t"
                     "buffer_load_dwordx4 %1, %2, %3 offen offset:2048 lds\n\t"
                     "buffer_load_dwordx4 %1, %2, %3 offen offset:3072 lds" ::"s"(lds), "v"(voff), "s"(rsrc), "s"(soff));
}
__device__ __forceinline__ i32x4 ns_rsrc(const void* p, uint32_t bytes)
{
    const uint64_t a = (uint64_t)p;
    return i32x4{(int)uniform_u32((uint32_t)a), (int)uniform_u32((uint32_t)(a >> 32) & 0xffffu), (int)uniform_u32(bytes), 0x00020000};
}
template <int N>
__device__ __forceinline__ void wait_loads()
{
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// (the builtin alone orders no memory access of the compiler's)
__device__ __forceinline__ void ns_barrier()
{
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_all() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

struct NsTile {
    int batch, ti, tj;
};
template <bool SYM>
__device__ __forceinline__ NsTile ns_tile(const NsGemm& g, int tile)
{
    const int per = SYM ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
    NsTile t;
    t.batch = tile / per;
    tile -= t.batch * per;
    if constexpr (SYM) {        // those with tj <= ti: 8 A^2 + 2 A in the first A groups of four rows, column by column
        int a = (int)sqrtf((float)tile * 0.125f);
        while (8 * (a + 1) * (a + 1) + 2 * (a + 1) <= tile) a++;
        while (8 * a * a + 2 * a > tile) a--;
        tile -= 8 * a * a + 2 * a;
        const int rows = min(4, g.tiles_m - 4 * a), whole = rows * (4 * a + 1);       // columns 0 .. 4 a have all rows
        if (tile < whole) {
            t.ti = 4 * a + tile % rows;
            t.tj = tile / rows;
        } else {
            tile -= whole;
            int c = 1;
            for (; tile >= rows - c; c++) tile -= rows - c;
            t.tj = 4 * a + c;
            t.ti = t.tj + tile;
        }
    } else {                    // four rows of tiles at a time: neighbours share rows of P and columns of Q
        const int group = tile / (4 * g.tiles_n), first = 4 * group, rows = min(4, g.tiles_m - first);
        tile -= group * 4 * g.tiles_n;
        t.ti = first + tile % rows;
        t.tj = tile / rows;
    }
    return t;
}

// A block of 32 x 32 results: four 16 x 16 products, q = 2 (row half) + column
// half, a lane holding row lane % 16, columns 4 (lane / 16) + e of each.
struct NsBlock {
    f32x4 q[4];
};
__device__ __forceinline__ int ns_row(int q, int lane) { return 16 * (q >> 1) + (lane & 15); }
__device__ __forceinline__ int ns_col(int q, int lane) { return 16 * (q & 1) + 4 * (lane >> 4); }

// A's values where poly's results of a block go (p is A).
struct NsOld {
    f16x4 high[4], low[4];
};
__device__ __forceinline__ NsOld ns_old(const NsGemm& g, int batch, int r0, int c0)
{
    const int lane = threadIdx.x & 63;
    const _Float16* at = g.p + batch * g.p_size + ((int64_t)(c0 / kPanel) * g.pitch + r0) * kPanel;
    NsOld o = {};
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int in = ns_row(q, lane) * kPanel + ns_col(q, lane);
        o.high[q] = *reinterpret_cast<const f16x4*>(at + in);
        if (g.passes > 1) o.low[q] = *reinterpret_cast<const f16x4*>(at + g.p_low + in);
    }
    return o;
}

// Results of a block at (r0, c0) of matrix `batch`.  `scratch`: kScratch bytes
// of LDS of this wave's own.  `mirror`: also as the block at (c0, r0) of a
// symmetric result, turned by transposing reads.
template <int KIND>
__device__ __forceinline__ void ns_finish(const NsGemm& g, const NsGiven<KIND>& mats, int batch, int r0, int c0, bool mirror,
                                          const NsBlock& acc, char* scratch, const NsOld& old)
{
    const int lane = threadIdx.x & 63;
    if constexpr (KIND == kLast) {      // the weights, in their own orientation: 8 elements of a row a lane
        const NsMatrix mat = mats.at[batch];
        float* s = reinterpret_cast<float*>(scratch);
        const int64_t rows = mat.tall ? g.n : g.m, cols = mat.tall ? g.m : g.n;
#pragma unroll
        for (int u = 0; u < 2; u++) {   // 16 rows of the block, or (tall) 16 columns
#pragma unroll
            for (int v = 0; v < 2; v++) {
                if (mat.tall) {
#pragma unroll
                    for (int e = 0; e < 4; e++) s[(4 * (lane >> 4) + e) * 36 + 16 * v + (lane & 15)] = acc.q[2 * v + u][e];
                } else {
                    *reinterpret_cast<f32x4*>(s + (lane & 15) * 36 + 16 * v + 4 * (lane >> 4)) = acc.q[2 * u + v];
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            const int64_t wr = (mat.tall ? c0 : r0) + 16 * u + (lane >> 2), wc = (mat.tall ? r0 : c0) + 8 * (lane & 3);
            const int nv = wr < rows ? (int)max((int64_t)0, min((int64_t)8, cols - wc)) : 0;
            const int64_t at = nv ? wr * mat.w_stride + wc : 0;
            float o[8], w[8];
            if (g.update) ns_chunk(mat.w, g.w_f32, at, nv, w);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                o[e] = s[(lane >> 2) * 36 + 8 * (lane & 3) + e] * (1.f / (kHeld * kHeld));
                if (g.update) o[e] = g.keep * w[e] - mat.rate * o[e];
            }
            if (g.w_f32)
                store_raw(static_cast<float*>(mat.w) + at, to_raw<float>(o), nv);
            else
                store_raw(static_cast<bf16*>(mat.w) + at, to_raw<bf16>(o), nv);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    } else {
        _Float16* out = g.out + batch * g.out_size;
        const int64_t at = ((int64_t)(c0 / kPanel) * g.pitch + r0) * kPanel, turned = ((int64_t)(r0 / kPanel) * g.pitch + c0) * kPanel;
        const bool precise = g.passes > 1;
        f16x4 high[4], low[4];
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float x = acc.q[q][e] * ((KIND == kPoly ? g.c : 1.f) / kHeld);
                if constexpr (KIND == kPoly)
                    x += g.b * ((float)old.high[q][e] + (float)old.low[q][e]) + (r0 + ns_row(q, lane) == c0 + ns_col(q, lane) + e ? g.a * kHeld : 0.f);
                high[q][e] = (_Float16)x;
                low[q][e] = (_Float16)(x - (float)high[q][e]);
            }
        // Out as whole rows, 1 KiB a store, through LDS: 16-byte chunk c of row r lies at c ^ (r / 4 & 3).  (Stored from the
        // lanes that hold them, 8 bytes of a row each, the results take four times the requests to L2.)
        auto emit = [&](const f16x4 (&v)[4], _Float16* to) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int r = ns_row(q, lane), c = ns_col(q, lane);
                *reinterpret_cast<f16x4*>(scratch + r * 64 + (c / 8 ^ (r >> 2 & 3)) * 16 + c % 8 * 2) = v[q];
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int r = 16 * u + (lane >> 2);
                *reinterpret_cast<f16x8*>(to + u * 512 + lane * 8) = *reinterpret_cast<const f16x8*>(scratch + r * 64 + ((lane & 3) ^ (r >> 2 & 3)) * 16);
            }
        };
        for (int part = 0; part < (precise ? 2 : 1); part++) {
            _Float16* to = out + (part ? g.out_low : 0);
            emit(part ? low : high, to + at);
            if (mirror) {       // row by column: a transposing read gives 16 lanes a column each of four rows
                typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
                f16x4 v[4];
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int j = lane & 15, r = ns_col(q, lane) + (j >> 2), c = 16 * (q >> 1) + 4 * (j & 3);
                    v[q] = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4*)(scratch + r * 64 + (c / 8 ^ (r >> 2 & 3)) * 16 + c % 8 * 2)));
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                emit(v, to + turned);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
}

// where a sharer's sums of its first (0) or second tile lie: 16 bytes a lane, block after block of its wave
template <class Cfg>
__device__ __forceinline__ float* ns_part(const NsGemm& g, int sharer, int second)
{
    return g.part + ((int64_t)(2 * sharer + second) * Cfg::WAVES + ((int)threadIdx.x >> 6)) * (Cfg::IM * Cfg::JN * 1024) +
           ((int)threadIdx.x & 63) * 4;
}

// A stage's tiles in LDS: rows of 64 bytes, of P (and a symmetric Q) K along
// them, the 16-byte chunk c of row r at c ^ t(r / 4 & 3) with t = 0, 2, 3, 1:
// the 16 lanes that a fragment read serves at a time (0-3, 12-15, 20-23, 24-27
// and so on) then meet all 64 banks.  Of step's Q panels of 32 columns, K down
// the rows, the halves of rows 8-15 and 24-31 changed over: 32 lanes of a
// transposing read take half of eight rows.
__device__ __forceinline__ int ns_turn(int r) { return 0x78 >> (2 * (r >> 2 & 3)) & 3; }
__device__ __forceinline__ uint32_t ns_voff_rows(int lane) { return (uint32_t)((lane & ~3) | ((lane & 3) ^ ns_turn(lane >> 2))) * 16u; }
__device__ __forceinline__ uint32_t ns_voff_cols(int lane) { return (uint32_t)((lane & ~3) | ((lane & 3) ^ 2 * (lane >> 5))) * 16u; }
// 16 rows from r0 on, 32 of K: a lane has row lane % 16, 8 of K from 8 (lane / 16) on
__device__ __forceinline__ f16x8 ns_row_frag(const char* t, int r0, int lane)
{
    const int r = r0 + (lane & 15);
    return *reinterpret_cast<const f16x8*>(t + r * 64 + ((lane >> 4) ^ ns_turn(r)) * 16);
}
// the same of 16 columns; within 16 lanes lane j points at row k0 + j / 4, columns 4 (j % 4) on, and gets column j of four rows
__device__ __forceinline__ f16x8 ns_col_frag(const char* t, int c0, int lane)
{
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int j = lane & 15, k = 8 * (lane >> 4) + (j >> 2), half = (c0 >> 4 & 1) ^ (lane >> 4 & 1);
    const char* at = t + (c0 & ~31) * 64 + k * 64 + half * 32 + (j & 3) * 8;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 256));
    return __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Few tiles: 64 x 64 a workgroup, each of its four waves the whole tile over a
// quarter of K, with loads of its own and no barrier until their sums meet.
// Such a product is bound by latency: a wave has five steps of loads in flight
// (with all of a CU's LDS, as much as its share of L2 delivers), and the
// products take a quarter of the steps one after the other that they take in
// workgroups that split the tile instead (gram of 1001 x 2731, 136 tiles: 12.8
// us against 18.2 with its shares; of 256 x 1024, 10 tiles: 7.5 against 9.9).
constexpr int kFewTile = 64, kFewStages = 5, kFewStage = 2 * kFewTile * kPanel * 2;
template <int KIND>
__global__ __launch_bounds__(256) void ns_few_kernel(NsGemm g, NsGiven<KIND> mats)
{
    __shared__ __attribute__((aligned(16))) char s_mem[4 * kFewStages * kFewStage];
    static_assert(sizeof(s_mem) <= 160 * 1024 && 12 * 4096 + 4 * kScratch <= (int)sizeof(s_mem), "LDS budget");
    constexpr bool kSym = KIND == kGram || KIND == kPoly;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    int id = (int)blockIdx.x;
    {
        const int group = id / kNsCus * kNsCus, here = min(kNsCus, (int)gridDim.x - group);
        if (here == kNsCus) id = group + (id - group) % kNsXcds * (kNsCus / kNsXcds) + (id - group) / kNsXcds;
    }
    NsTile t = ns_tile<kSym>(g, id);
    t = {(int)uniform_u32((uint32_t)t.batch), (int)uniform_u32((uint32_t)t.ti), (int)uniform_u32((uint32_t)t.tj)};
    const int k_total = g.k_steps * g.passes, from = k_total * wave / 4, to = k_total * (wave + 1) / 4;
    const _Float16* p = g.p + t.batch * g.p_size + (int64_t)t.ti * kFewTile * kPanel;
    const _Float16* q = g.q + t.batch * g.q_size + (kSym ? (int64_t)t.tj * kFewTile * kPanel : (int64_t)t.tj * kFewTile * g.pitch);
    const bool low = g.passes > 1;
    const int64_t p_room = ((int64_t)(g.k_steps - 1) * g.pitch + kFewTile) * kPanel + (low ? g.p_low : 0);
    const int64_t q_room = (kSym ? ((int64_t)(g.k_steps - 1) * g.pitch + kFewTile) * kPanel : (int64_t)kFewTile * g.pitch) + (low ? g.q_low : 0);
    const i32x4 rp = ns_rsrc(p, (uint32_t)(p_room * 2)), rq = ns_rsrc(q, (uint32_t)(q_room * 2));
    char* const ring = s_mem + wave * (kFewStages * kFewStage);
    const uint32_t ring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_mem + (uint32_t)wave * (kFewStages * kFewStage);
    const uint32_t voff_rows = ns_voff_rows(lane), voff_cols = ns_voff_cols(lane);
    auto load = [&](int step, int stage) {
        const int pass = step < g.k_steps ? 0 : step < 2 * g.k_steps ? 1 : 2;
        const uint32_t k = (uint32_t)(step - pass * g.k_steps), lds = ring0 + stage * kFewStage;
        load_to_lds<4>(rp, lds, voff_rows, k * (uint32_t)g.pitch * 64u + (pass == 2 ? (uint32_t)g.p_low * 2u : 0u));
        const uint32_t q_off = k * (kSym ? (uint32_t)g.pitch * 64u : 2048u) + (pass == 1 ? (uint32_t)g.q_low * 2u : 0u);
        if constexpr (kSym) {
            load_to_lds<4>(rq, lds + kFewStage / 2, voff_rows, q_off);
        } else {
            load_to_lds<2>(rq, lds + kFewStage / 2, voff_cols, q_off);
            load_to_lds<2>(rq, lds + kFewStage / 2 + 2048, voff_cols, q_off + (uint32_t)g.pitch * 64u);
        }
    };
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // this wave's block of the result; what poly adds to it comes with the first loads
    const int r0 = t.ti * kFewTile + 32 * (wave >> 1), c0 = t.tj * kFewTile + 32 * (wave & 1);
    NsOld old;
    if constexpr (KIND == kPoly) old = ns_old(g, t.batch, r0, c0);
    f16x8 fp[4], fq[4];
    auto read = [&](int stage) {
        const char* tp = ring + stage * kFewStage;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            fp[i] = ns_row_frag(tp, 16 * i, lane);
            fq[i] = kSym ? ns_row_frag(tp + kFewStage / 2, 16 * i, lane) : ns_col_frag(tp + kFewStage / 2, 16 * i, lane);
        }
    };
#pragma unroll
    for (int s = 0; s < kFewStages; s++)
        if (from + s < to) load(from + s, s);
    int stage = 0;
    for (int step = from; step < to; step++) {
        // this step's tiles are there (eight loads a step; the last steps wait for all)
        if (step + kFewStages <= to)
            wait_loads<8 * (kFewStages - 1)>();
        else
            wait_loads<0>();
        read(stage);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fq[j], fp[i], acc[i][j], 0, 0, 0);
        // (the fragments are in registers: the stage may be loaded again)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (step + kFewStages < to) load(step + kFewStages, stage);
        stage = stage == kFewStages - 1 ? 0 : stage + 1;
    }
    // The waves' sums: block w of the tile to wave w, added in the waves' order.
    wait_all();
    __syncthreads();
    f32x4* const meet = reinterpret_cast<f32x4*>(s_mem);      // [block][the other waves][4][64]
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int block = 2 * i + j;
            if (block == wave) continue;
#pragma unroll
            for (int q = 0; q < 4; q++)
                meet[((block * 3 + (wave < block ? wave : wave - 1)) * 4 + q) * 64 + lane] = acc[2 * i + (q >> 1)][2 * j + (q & 1)];
        }
    __syncthreads();
    NsBlock sum;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int a = q >> 1, b = q & 1;
        const f32x4 mine = wave == 0 ? acc[a][b] : wave == 1 ? acc[a][2 + b] : wave == 2 ? acc[2 + a][b] : acc[2 + a][2 + b];
        sum.q[q] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; w++) sum.q[q] += w == wave ? mine : meet[((wave * 3 + (w < wave ? w : w - 1)) * 4 + q) * 64 + lane];
    }
    ns_finish<KIND>(g, mats, t.batch, r0, c0, kSym && t.ti != t.tj, sum, s_mem + 12 * 4096 + wave * kScratch, old);
}

// Symmetric products of few tiles: 32 x 32 a workgroup, an eighth of K to each
// of its waves, whose operands go from memory into registers in the matrix
// instructions' own order, without LDS, four steps of loads at once.  With
// g.sharers workgroups a tile (long K) their sums meet in ns_fine_join_kernel.
// Gram of 256 x 1024: 5.2 us (64 x 64 tiles: 7.5), of 256 x 16384: 10.8 + 3.9
// (128 x 128 tiles with shares: 41 + 5); bound by latency.
constexpr int kFineTile = 32;
template <int KIND, bool LOW>
__global__ __launch_bounds__(512) void ns_fine_kernel(NsGemm g)
{
    constexpr int kParts = LOW ? 2 : 1, kAhead = 4 / kParts;
    __shared__ __attribute__((aligned(16))) f32x4 s_sum[8][4][64];
    __shared__ __attribute__((aligned(16))) char s_out[kScratch];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int id = (int)blockIdx.x, eighth = 8 * (id % g.sharers) + wave;
    NsTile t = ns_tile<true>(g, id / g.sharers);
    t = {(int)uniform_u32((uint32_t)t.batch), (int)uniform_u32((uint32_t)t.ti), (int)uniform_u32((uint32_t)t.tj)};
    const int from = (int)((int64_t)g.k_steps * eighth / (8 * g.sharers)), to = (int)((int64_t)g.k_steps * (eighth + 1) / (8 * g.sharers));
    const int r0 = t.ti * kFineTile, c0 = t.tj * kFineTile;
    const _Float16* const p = g.p + t.batch * g.p_size + (lane & 15) * kPanel + (lane >> 4) * 8;
    NsOld old;
    if constexpr (KIND == kPoly)
        if (wave == 0) old = ns_old(g, t.batch, r0, c0);
    f32x4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // steps k on, all their loads before the first product; of the last ones those past the end with nothing for Q
    auto steps = [&](int k, auto n, auto last) {
        constexpr int kN = decltype(n)::value;
        f16x8 fp[kN][kParts][2], fq[kN][kParts][2];
#pragma unroll
        for (int s = 0; s < kN; s++) {
            const _Float16* const at = p + (int64_t)(decltype(last)::value ? min(k + s, to - 1) : k + s) * g.pitch * kPanel;
#pragma unroll
            for (int part = 0; part < kParts; part++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    fp[s][part][i] = *reinterpret_cast<const f16x8*>(at + (part ? g.p_low : 0) + (r0 + 16 * i) * kPanel);
                    fq[s][part][i] = *reinterpret_cast<const f16x8*>(at + (part ? g.p_low : 0) + (c0 + 16 * i) * kPanel);
                }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < kN; s++) {
            if (decltype(last)::value && k + s >= to)
#pragma unroll
                for (int part = 0; part < kParts; part++) fq[s][part][0] = fq[s][part][1] = f16x8{};
#pragma unroll
            for (int pass = 0; pass < 2 * kParts - 1; pass++)
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fq[s][pass == 1][j], fp[s][pass / 2][i], acc[i][j], 0, 0, 0);
        }
    };
    typedef std::integral_constant<int, kAhead> All;
    typedef std::integral_constant<int, kAhead / 2> Half;
    int k = from;
    for (; k + kAhead <= to; k += kAhead) steps(k, All{}, std::false_type{});
    if (k + kAhead / 2 < to)
        steps(k, All{}, std::true_type{});
    else if (k < to)
        steps(k, Half{}, std::true_type{});
#pragma unroll
    for (int q = 0; q < 4; q++) s_sum[wave][q][lane] = acc[q >> 1][q & 1];
    __syncthreads();
    if (wave < 4) {         // a quarter of the block each, the waves' sums in order
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 8; w++) sum += s_sum[w][wave][lane];
        if (g.sharers > 1)
            *reinterpret_cast<f32x4*>(g.part + (int64_t)id * 1024 + wave * 256 + lane * 4) = sum;
        else
            s_sum[0][wave][lane] = sum;
    }
    if (g.sharers > 1) return;
    __syncthreads();
    if (wave) return;
    NsBlock sum;
#pragma unroll
    for (int q = 0; q < 4; q++) sum.q[q] = s_sum[0][q][lane];
    ns_finish<KIND>(g, {}, t.batch, r0, c0, t.ti != t.tj, sum, s_out, old);
}

// A gram's tiles of more than one workgroup: their sums added in order.
__global__ __launch_bounds__(64) void ns_fine_join_kernel(NsGemm g)
{
    __shared__ __attribute__((aligned(16))) char s_out[kScratch];
    const int lane = threadIdx.x & 63;
    const NsTile t = ns_tile<true>(g, (int)blockIdx.x);
    const float* part = g.part + (int64_t)blockIdx.x * g.sharers * 1024 + lane * 4;
    NsBlock sum;
#pragma unroll
    for (int q = 0; q < 4; q++) sum.q[q] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int i = 0; i < g.sharers; i++)
#pragma unroll
        for (int q = 0; q < 4; q++) sum.q[q] += *reinterpret_cast<const f32x4*>(part + (int64_t)i * 1024 + q * 256);
    ns_finish<kGram>(g, {}, t.batch, t.ti * kFineTile, t.tj * kFineTile, t.ti != t.tj, sum, s_out, NsOld{});
}

// Matrices of up to 256 rows: X' = a X + A (b X + c A X), so poly and step are
// two products with the same A and need no B.  A workgroup has 32 columns and
// all rows, a wave 32 of those.  Its rows of A come from memory into registers
// in the matrix instructions' own order, all at once, and serve both products;
// X and then Z = b X + c A X are in LDS for all waves.  Z always has its low
// part: near a singular value of 1, a X + A Z = 3.4 - 2.7 loses two bits.
// 256 x 1024: 7 us where the kernels poly and step take 5.2 each, 64 x 1024: 3.6;
// both bound by the chain of one load, two products and a barrier between.
template <int KIND, int GROUPS, bool LOW>
__global__ __launch_bounds__(128 * GROUPS) void ns_narrow_kernel(NsGemm g, NsGiven<KIND> mats)
{
    constexpr int kWaves = 2 * GROUPS, kSteps = 2 * GROUPS, kParts = LOW ? 2 : 1, kPart = kSteps * 2048;
    __shared__ __attribute__((aligned(16))) char s_x[kParts * kPart], s_z[2 * kPart], s_out[kWaves * kScratch];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int batch = (int)blockIdx.x / g.tiles_n, r0 = 32 * wave, c0 = (int)blockIdx.x % g.tiles_n * kPanel;
    // a step of X, 32 rows of this panel, to each wave; the low part behind it
    const _Float16* q = g.q + batch * g.q_size + (int64_t)c0 * g.pitch;
    const i32x4 rq = ns_rsrc(q, (uint32_t)(((int64_t)kPanel * g.pitch + (LOW ? g.q_low : 0)) * 2));
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_x + (uint32_t)wave * 2048u;
#pragma unroll
    for (int part = 0; part < kParts; part++)
        load_to_lds<2>(rq, lds + part * kPart, ns_voff_cols(lane), (uint32_t)wave * 2048u + (part ? (uint32_t)g.q_low * 2u : 0u));
    f16x8 rows[kParts][kSteps][2];
    {
        const _Float16* const a = g.p + batch * g.p_size + (r0 + (lane & 15)) * kPanel + (lane >> 4) * 8;
#pragma unroll
        for (int k = 0; k < kSteps; k++)
#pragma unroll
            for (int part = 0; part < kParts; part++)
#pragma unroll
                for (int i = 0; i < 2; i++)
                    rows[part][k][i] = *reinterpret_cast<const f16x8*>(a + (part ? g.p_low : 0) + ((int64_t)k * g.pitch + 16 * i) * kPanel);
    }
    auto product = [&](const char* with, auto passes, f32x4 (&acc)[2][2]) {     // high high, high low, low high
#pragma unroll
        for (int pass = 0; pass < decltype(passes)::value; pass++)
#pragma unroll
            for (int k = 0; k < kSteps; k++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const f16x8 x = ns_col_frag(with + (pass == 1 ? kPart : 0) + k * 2048, 16 * j, lane);
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, rows[pass / 2][k][i], acc[i][j], 0, 0, 0);
                }
    };
    wait_all();
    __syncthreads();
    f32x4 acc[2][2], sum[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    product(s_x, std::integral_constant<int, LOW ? 3 : 1>{}, acc);
    // where a lane's results lie in a step's rows, their halves changed over as ns_voff_cols puts them
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int r = 16 * i + (lane & 15), at = wave * 2048 + r * 64 + (j ^ (r >> 3 & 1)) * 32 + (lane >> 4) * 8;
            const f16x4 x = *reinterpret_cast<const f16x4*>(s_x + at);
            f16x4 x_low = {}, z, z_low;
            if constexpr (LOW) x_low = *reinterpret_cast<const f16x4*>(s_x + kPart + at);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float held = (float)x[e] + (float)x_low[e], to = g.b * held + g.c * (1.f / kHeld) * acc[i][j][e];
                z[e] = (_Float16)to;
                z_low[e] = (_Float16)(to - (float)z[e]);
                sum[i][j][e] = g.a * kHeld * held;
            }
            *reinterpret_cast<f16x4*>(s_z + at) = z;
            *reinterpret_cast<f16x4*>(s_z + kPart + at) = z_low;
        }
    __syncthreads();
    product(s_z, std::integral_constant<int, LOW ? 3 : 2>{}, sum);
    ns_finish<KIND>(g, mats, batch, r0, c0, false, NsBlock{{sum[0][0], sum[0][1], sum[1][0], sum[1][1]}}, s_out + wave * kScratch, NsOld{});
}

// Each workgroup goes through whole tiles and then through its share of the
// others', one unbroken sequence of K steps: the loads run STAGES - 1 steps
// ahead, over the ends of tiles too, so that only a tile's results interrupt
// the products.  Bound by power: with random values the chip runs these
// products at about 1.8 GHz, with zeros at 2.3, and the matrix pipes are busy
// for 63 to 65% of the cycles; step of 4096 x 16384 takes 420 us with a
// gradient's values and 490 with normal ones, 1.1 to 1.3 PFLOP/s (the library's
// product of that shape 505 us with normal ones).
template <class Cfg, int KIND>
__global__ __launch_bounds__(Cfg::THREADS) void ns_gemm_kernel(NsGemm g, NsGiven<KIND> mats)
{
    __shared__ __attribute__((aligned(16))) char s_mem[Cfg::LDS];
    constexpr bool kSym = KIND == kGram || KIND == kPoly;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = wave / Cfg::WGN, wn = wave % Cfg::WGN;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_mem;
    char* scratch = s_mem + Cfg::STAGES * Cfg::STAGE + wave * kScratch;

    // Workgroups go round the XCDs in turn: each XCD takes a contiguous part of every 256.
    int id = (int)blockIdx.x;
    {
        const int group = id / kNsCus * kNsCus, here = min(kNsCus, (int)gridDim.x - group);
        if (here == kNsCus) id = group + (id - group) % kNsXcds * (kNsCus / kNsXcds) + (id - group) / kNsXcds;
    }
    const int k_total = g.k_steps * g.passes;
    const int wholes = id < g.whole ? (g.whole - id - 1) / (int)gridDim.x + 1 : 0;
    // Its share of the rest.  Lane l has the tiles l, l + lanes, ... behind the whole ones, its sharers' steps one after the
    // other in them: those at one place in every lane are at the same K of neighbouring tiles at the same time and share
    // what they load.  (The divisions leave their uniform results in vector registers.)
    int share_from = 0, share_to = 0, share_tile = 0;           // steps of the tiles from share_tile on
    if (id < g.sharers) {
        const int64_t all = (int64_t)(g.tiles - g.whole) / g.lanes * k_total, w = id / g.lanes, sharers = g.sharers / g.lanes;
        const int64_t from = all * w / sharers, to = all * (w + 1) / sharers, first = from / k_total;
        share_tile = (int)uniform_u32((uint32_t)first);
        share_from = (int)uniform_u32((uint32_t)(from - first * k_total));
        share_to = (int)uniform_u32((uint32_t)(to - first * k_total));
    }
    const int pieces = wholes + (share_to > share_from) + (share_to > k_total);
    const int64_t steps = (int64_t)wholes * k_total + (share_to - share_from);
    struct Piece {
        NsTile t;
        int from, to;
    };
    auto piece = [&](int i) {
        Piece p;
        const bool whole = i < wholes;
        const int second = i - wholes;
        p.t = ns_tile<kSym>(g, whole ? id + i * (int)gridDim.x : g.whole + (share_tile + second) * g.lanes + id % g.lanes);
        p.t = {(int)uniform_u32((uint32_t)p.t.batch), (int)uniform_u32((uint32_t)p.t.ti), (int)uniform_u32((uint32_t)p.t.tj)};
        p.from = whole || second ? 0 : share_from;
        p.to = whole ? k_total : second ? share_to - k_total : min(share_to, k_total);
        return p;
    };

    const uint32_t voff_rows = ns_voff_rows(lane), voff_cols = ns_voff_cols(lane);

    // This wave's loads, step by step: 2 KiB of P, then of Q (of step's, a panel).  Passes (precise): high high, high low, low high.
    const uint32_t p_wave = (uint32_t)wave * 2048u;
    const uint32_t q_wave = kSym ? p_wave : (uint32_t)wave * (uint32_t)g.pitch * 64u;
    const uint32_t p_step = (uint32_t)g.pitch * 64u, q_step = kSym ? p_step : 2048u;
    // (what lies between a tile's first element and its last: of P and a symmetric Q over all panels, of step's Q over its own)
    const bool low = g.passes > 1;
    const int64_t p_room = ((int64_t)(g.k_steps - 1) * g.pitch + Cfg::TM) * kPanel + (low ? g.p_low : 0);
    const int64_t q_room = (kSym ? ((int64_t)(g.k_steps - 1) * g.pitch + Cfg::TN) * kPanel : (int64_t)Cfg::TN * g.pitch) + (low ? g.q_low : 0);
    i32x4 rp, rq;
    int next_piece = 0, left_in_piece = 0, left_in_pass = 0, pass = 0;
    uint32_t p_off = 0, q_off = 0, lds_at = lds0 + p_wave;
    auto start_pass = [&](int k) {
        left_in_pass = g.k_steps - k;
        p_off = (uint32_t)k * p_step + p_wave + (pass == 2 ? (uint32_t)g.p_low * 2u : 0u);
        q_off = (uint32_t)k * q_step + q_wave + (pass == 1 ? (uint32_t)g.q_low * 2u : 0u);
    };
    auto start_piece = [&] {
        const Piece i = piece(next_piece++);
        const _Float16* p = g.p + i.t.batch * g.p_size + (int64_t)i.t.ti * Cfg::TM * kPanel;
        const _Float16* q = g.q + i.t.batch * g.q_size + (kSym ? (int64_t)i.t.tj * Cfg::TN * kPanel : (int64_t)i.t.tj * Cfg::TN * g.pitch);
        rp = ns_rsrc(p, (uint32_t)(p_room * 2));
        rq = ns_rsrc(q, (uint32_t)(q_room * 2));
        left_in_piece = i.to - i.from;
        pass = i.from >= 2 * g.k_steps ? 2 : i.from >= g.k_steps ? 1 : 0;
        start_pass(i.from - pass * g.k_steps);
    };
    auto load_p = [&] { load_to_lds<2>(rp, lds_at, voff_rows, p_off); };
    auto load_q = [&] {
        load_to_lds<2>(rq, lds_at + Cfg::P_BYTES, kSym ? voff_rows : voff_cols, q_off);
        lds_at = lds_at == lds0 + p_wave + (Cfg::STAGES - 1) * Cfg::STAGE ? lds0 + p_wave : lds_at + Cfg::STAGE;
        p_off += p_step;
        q_off += q_step;
        left_in_piece--;
        if (--left_in_pass == 0 || left_in_piece == 0) {
            if (left_in_piece) {
                pass++;
                start_pass(0);
            } else if (next_piece < pieces) {
                start_piece();
            }
        }
    };

    // A step's products go over the first half of its columns and then over the second.  A fragment is read again for the
    // next time as soon as its last product is under way, half a step to a whole one ahead: the next step's rows and first
    // columns during the second half, ahead of the barrier between the steps, so that the products go on through it.  A
    // barrier so vouches for the stage after the one that begins.
    constexpr int NI = 2 * Cfg::IM, NJ = 2 * Cfg::JN;
    f16x8 fp[NI], fq[NJ];
    auto read_p = [&](int stage, int i) { fp[i] = ns_row_frag(s_mem + stage * Cfg::STAGE, wm * 32 * Cfg::IM + 16 * i, lane); };
    auto read_q = [&](int stage, int j) {
        const char* t = s_mem + stage * Cfg::STAGE + Cfg::P_BYTES;
        const int c0 = wn * 32 * Cfg::JN + 16 * j;
        fq[j] = kSym ? ns_row_frag(t, c0, lane) : ns_col_frag(t, c0, lane);
    };
    constexpr int kAhead = Cfg::STAGES - 1;
    if (pieces == 0) return;
    start_piece();
#pragma unroll
    for (int s = 0; s < kAhead; s++)
        if (s < steps) {
            load_p();
            load_q();
        }
    if (kAhead <= steps)
        wait_loads<(kAhead - 1) * Cfg::LOADS>();
    else
        wait_loads<0>();
    ns_barrier();
#pragma unroll
    for (int j = 0; j < NJ / 2; j++) read_q(0, j);
#pragma unroll
    for (int i = 0; i < NI; i++) read_p(0, i);

    int stage = 0;
    int64_t to_load = steps - kAhead;               // steps whose loads are not issued yet (or less than none)
    for (int n = 0; n < pieces; n++) {
        const Piece here = piece(n);
        f32x4 acc[NI][NJ];
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
            for (int j = 0; j < NJ; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int step = here.from; step < here.to; step++, to_load--) {
            // The next step's tiles are there, and the stage that is loaded now has been read, in every wave (its last
            // fragments went into products before this; those under way are of this step's stage).
            if (to_load >= 0)
                wait_loads<(kAhead - 2) * Cfg::LOADS>();
            else
                wait_loads<0>();
            ns_barrier();
            const int next = stage == kAhead ? 0 : stage + 1;
            // Reads, products and loads in turn: eight waves that all read first would wait for one another.
            // (behind the last step the next stage holds what it held: read, not used)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < NI; i++) {
                    // first half: the columns of the second; second half: the next step's first columns
                    if (i < NJ / 2) read_q(h ? next : stage, h ? i : NJ / 2 + i);
#pragma unroll
                    for (int j = h * NJ / 2; j < (h + 1) * NJ / 2; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fq[j], fp[i], acc[i][j], 0, 0, 0);
                    if (h) read_p(next, i);
                    __builtin_amdgcn_sched_barrier(0);
                    if (to_load > 0 && i == NI / 2 - 1) {
                        if (h)
                            load_q();
                        else
                            load_p();
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            stage = next;
        }
        if (n >= wholes) {
            float* part = ns_part<Cfg>(g, id, n - wholes);
#pragma unroll
            for (int i = 0; i < Cfg::IM; i++)
#pragma unroll
                for (int j = 0; j < Cfg::JN; j++)
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        *reinterpret_cast<f32x4*>(part + ((i * Cfg::JN + j) * 4 + q) * 256) = acc[2 * i + (q >> 1)][2 * j + (q & 1)];
        } else {
#pragma unroll
            for (int i = 0; i < Cfg::IM; i++)
#pragma unroll
                for (int j = 0; j < Cfg::JN; j++) {
                    const int r0 = here.t.ti * Cfg::TM + (wm * Cfg::IM + i) * 32, c0 = here.t.tj * Cfg::TN + (wn * Cfg::JN + j) * 32;
                    NsOld old;
                    if constexpr (KIND == kPoly) old = ns_old(g, here.t.batch, r0, c0);
                    ns_finish<KIND>(g, mats, here.t.batch, r0, c0, kSym && here.t.ti != here.t.tj,
                                    NsBlock{{acc[2 * i][2 * j], acc[2 * i][2 * j + 1], acc[2 * i + 1][2 * j], acc[2 * i + 1][2 * j + 1]}}, scratch, old);
                }
        }
    }
}

// The shared tiles: their sharers' sums added in order, then as a tile with a
// workgroup of its own.  A wave a block of 32 x 32.
template <class Cfg, int KIND>
__global__ __launch_bounds__(256) void ns_join_kernel(NsGemm g, NsGiven<KIND> mats)
{
    __shared__ __attribute__((aligned(16))) char s_mem[4 * kScratch];
    constexpr int kBlocks = Cfg::WAVES * Cfg::IM * Cfg::JN;
    static_assert(kBlocks % 4 == 0, "four blocks of a tile to a workgroup");
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int shared = (int)blockIdx.x / (kBlocks / 4), block = (int)blockIdx.x % (kBlocks / 4) * 4 + wave;
    const int of_wave = block / (Cfg::IM * Cfg::JN), i = block % (Cfg::IM * Cfg::JN) / Cfg::JN, j = block % Cfg::JN;
    constexpr bool kSym = KIND == kGram || KIND == kPoly;
    const NsTile t = ns_tile<kSym>(g, g.whole + shared);
    const int r0 = t.ti * Cfg::TM + (of_wave / Cfg::WGN * Cfg::IM + i) * 32, c0 = t.tj * Cfg::TN + (of_wave % Cfg::WGN * Cfg::JN + j) * 32;
    NsOld old;
    if constexpr (KIND == kPoly) old = ns_old(g, t.batch, r0, c0);
    const int64_t k_total = (int64_t)g.k_steps * g.passes, all = (g.tiles - g.whole) / g.lanes * k_total;
    const int64_t from = shared / g.lanes * k_total, to = from + k_total;      // of its lane's steps
    const int sharers = g.sharers / g.lanes;
    // the sharer of step s is the last w with all w / sharers <= s
    auto sharer = [&](int64_t s) { return (int)(((s + 1) * sharers - 1) / all); };
    NsBlock acc = {};
    const int last = sharer(to - 1);
    for (int w = sharer(from); w <= last; w++) {
        const int second = all * w / sharers < from;            // it began with the tile before
        const float* part = g.part + ((int64_t)(2 * (w * g.lanes + shared % g.lanes) + second) * Cfg::WAVES + of_wave) * (Cfg::IM * Cfg::JN * 1024) + (i * Cfg::JN + j) * 1024 + lane * 4;
#pragma unroll
        for (int q = 0; q < 4; q++) acc.q[q] += *reinterpret_cast<const f32x4*>(part + q * 256);
    }
    ns_finish<KIND>(g, mats, t.batch, r0, c0, kSym && t.ti != t.tj, acc, s_mem + wave * kScratch, old);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// One product of all matrices on tiles of one size: how many of them get a
// workgroup of their own, and its time in microseconds as the choice sees it.
struct NsProduct {
    int tile;
    int64_t tiles, whole, sharers, lanes, groups;     // (sharers: workgroups in all; of a split gram, a tile's)
    double time;
};
struct NsPlan {
    NsProduct gram, poly, step;
    bool narrow;                        // poly inside of step
    int64_t mp, np;
    // Panels are 2 KiB further apart than their rows need: at one step of step all workgroups load the same 32 rows of
    // their panels, which a power of two would put on the same few memory channels.
    int64_t pitch() const { return mp + kPanel; }
    int64_t size(int64_t cols) const { return pitch() * cols; }     // elements of a matrix with so many columns
    int64_t x_bytes, a_bytes, parts_bytes, share_bytes, total;
};

// What a product takes on tiles of a size, in microseconds: a K step of 32 with
// few workgroups on the chip and with `per_cu` on every CU, and what comes with
// every round of tiles (first loads, results).  Measured with each size alone on
// products of 256 x 1024 to 4096 x 16384 and batches of them.
struct NsTileRate {
    int tile, per_cu;
    double alone, full, round;
};
constexpr NsTileRate kNsRates[] = {{256, 1, 0.6, 0.85, 5.0}, {128, 2, 0.25, 0.70, 3.0}, {kFewTile, 1, 0.08, 0.145, 1.7}};
constexpr double kNsLaunch = 4.0;

static NsProduct ns_product(const NsTileRate& r, int64_t rows, int64_t cols, bool sym, int64_t k, int64_t count, int passes)
{
    NsProduct p{};
    const int64_t tm = rows / r.tile, tn = cols / r.tile, steps = k / kPanel * passes, slots = (int64_t)kNsCus * r.per_cu;
    p.tile = r.tile;
    p.tiles = (sym ? tm * (tm + 1) / 2 : tm * tn) * count;
    p.whole = p.tiles;
    p.groups = r.tile == kFewTile ? p.tiles : std::min(p.tiles, slots);
    const int64_t rounds = (p.tiles + slots - 1) / slots, rest = p.tiles % slots;
    auto time = [&](int64_t tiles, double k_steps) {
        return (r.alone + (r.full - r.alone) * std::min(1.0, (double)tiles / (double)slots)) * k_steps + r.round;
    };
    p.time = kNsLaunch + (double)(rounds - 1) * time(slots, (double)steps) + time(rounds > 1 ? slots : p.tiles, (double)steps);
    // A last round that does not fill the chip is dealt out in shares of its steps instead, where the steps saved are
    // worth the sums' way through memory (at about 4 TB/s, one after the other for a tile) and one more kernel (step of
    // two matrices of 2048 x 5500 in 22 bits, 352 tiles for 256 CUs: 340 us in two rounds, 251 + 19 with shares).
    if (rest > 0 && r.tile != kFewTile) {
        int64_t lanes = 8;
        while (rest % lanes) lanes /= 2;
        for (const int64_t most : {slots, 4 * rest, 2 * rest}) {
            const int64_t sharers = std::min({slots, rest * steps, most});      // (all multiples of lanes)
            const double share = (double)(rest * steps) / (double)sharers, parts = (double)sharers / (double)rest + 1.0;
            const double bytes = 5.0 * r.tile * r.tile * (double)(sharers + rest);     // read, and a part of the writing
            const double shared = kNsLaunch + (double)(rounds - 1) * time(slots, (double)steps) + time(sharers, share) + 3.0 +
                                  0.5 * parts + bytes / 4e6;
            if (shared < p.time)
                p.whole = p.tiles - rest, p.sharers = sharers, p.lanes = lanes, p.groups = p.whole ? slots : sharers, p.time = shared;
        }
    }
    return p;
}

// A symmetric product in 32 x 32 tiles; a gram's with as many workgroups a tile
// as its K is worth, whose sums lie where the next X will (`room` bytes; poly's
// K is too short for more than one).  Up to 512 rows, as every row is read
// rows / 32 times: orthogonalize of 512 x 2048 takes 105 us against 130 without
// these tiles (22 bits 141 against 181), of 768 x 3072 177 against 178 (323
// against 314).  Rates as above: microseconds a step of K, a tile, a join.
constexpr int64_t kFineRows = 512;
constexpr double kFineStep = 0.035, kFineFull = 0.05, kFineRound = 1.2, kFineJoin = 0.8, kFinePart = 0.05;
static NsProduct ns_fine(int64_t rows, int64_t k, int64_t count, int passes, int64_t room)
{
    NsProduct best{};
    const int64_t n = rows / kFineTile, steps = k / kPanel;
    const double step_bytes = passes > 1 ? 2.0 : 1.0;
    for (int64_t split = 1; split == 1 || (split * best.tiles <= kNsCus && 16 * split <= steps && split * best.tiles * kFineTile * kFineTile * 4 <= room); split *= 2) {
        NsProduct p{};
        p.tile = kFineTile, p.tiles = n * (n + 1) / 2 * count, p.whole = p.groups = p.tiles, p.sharers = split;
        const double fill = (double)(p.tiles * split) / (double)kNsCus, each = (double)steps / (double)split * step_bytes;
        p.time = kNsLaunch + kFineRound + each * std::max(kFineStep, kFineFull * std::ceil(fill)) + (split > 1 ? kNsLaunch + kFineJoin + kFinePart * (double)split : 0.0);
        if (split == 1 || p.time < best.time) best = p;
    }
    return best;
}

// poly and step in one kernel, 32 columns of the result to a workgroup: its own
// chain of loads and products, and a share of a full chip's time (measured
// on 1 workgroup to 12 a CU; operands of 22 bits take about 2 and 3 times as long).
constexpr int64_t kNarrow = 256;        // most rows
static NsProduct ns_narrow(int64_t mp, int64_t np, int64_t count, int passes)
{
    NsProduct p{};
    const double groups = (double)mp / 64.0;
    p.tiles = np / kPanel * count, p.whole = p.groups = p.tiles;
    p.time = kNsLaunch + 0.5 + 0.75 * groups * (passes > 1 ? 2.0 : 1.0) +
             (double)p.tiles * (0.001 * groups + 0.00033 * groups * groups) * (passes > 1 ? 3.2 : 1.0);
    return p;
}

// The tile of each product that its estimate is shortest on.  Padding: whole
// tiles of the largest size used.
static NsPlan ns_plan(int64_t m, int64_t n, int64_t count, bool precise)
{
    NsPlan best{};
    auto up = [](int64_t v, int64_t t) { return (v + t - 1) / t * t; };
    const int passes = precise ? 3 : 1, passes_held = precise ? 2 : 1;
    double best_time = 0;
    for (const NsTileRate& most : kNsRates) {
        NsPlan p{};
        p.mp = up(m, most.tile), p.np = up(n, most.tile);
        auto pick = [&](int64_t rows, int64_t cols, bool sym, int64_t k) {
            NsProduct b{};
            for (const NsTileRate& r : kNsRates) {
                if (r.tile > most.tile) continue;       // (the sizes divide one another)
                const NsProduct q = ns_product(r, rows, cols, sym, k, count, passes);
                if (b.tile == 0 || q.time < b.time) b = q;
            }
            if (sym && rows <= kFineRows) {
                const NsProduct q = ns_fine(rows, k, count, passes, p.size(p.np) * 2 * count * passes_held);
                if (q.time < b.time) b = q;
            }
            return b;
        };
        p.gram = pick(p.mp, p.mp, true, p.np);
        p.poly = pick(p.mp, p.mp, true, p.mp);
        p.step = pick(p.mp, p.np, false, p.mp);
        const NsProduct both = ns_narrow(p.mp, p.np, count, passes);
        if (p.mp <= kNarrow && both.time < p.poly.time + p.step.time) p.narrow = true, p.poly = NsProduct{}, p.step = both;
        const double time = p.gram.time + p.poly.time + p.step.time;
        if (best.mp == 0 || time < best_time) best = p, best_time = time;
    }
    NsPlan& p = best;
    p.x_bytes = p.size(p.np) * 2 * count * (precise ? 2 : 1);
    p.a_bytes = p.size(p.mp) * 2 * count * (precise ? 2 : 1);
    p.parts_bytes = (kNsParts * 8 * count + 255) / 256 * 256;
    for (const NsProduct& q : {p.gram, p.poly, p.step}) if (q.tile > kFewTile) p.share_bytes = std::max(p.share_bytes, q.sharers * 2 * q.tile * q.tile * 4);
    p.total = 2 * p.x_bytes + 2 * p.a_bytes + p.parts_bytes + p.share_bytes;
    return p;
}

template <int KIND>
static NsGiven<KIND> ns_given(const NsMatrices& mats)
{
    if constexpr (KIND == kLast)
        return mats;
    else
        return {};
}

template <class Cfg, int KIND>
static void ns_launch_cfg(const NsGemm& g, const NsProduct& p, const NsMatrices& mats, hipStream_t st)
{
    hipLaunchKernelGGL(HIP_KERNEL_NAME(ns_gemm_kernel<Cfg, KIND>), dim3((uint32_t)p.groups), dim3(Cfg::THREADS), 0, st, g, ns_given<KIND>(mats));
    if (p.sharers)
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ns_join_kernel<Cfg, KIND>), dim3((uint32_t)(p.tiles - p.whole) * (Cfg::WAVES * Cfg::IM * Cfg::JN / 4)),
                           dim3(256), 0, st, g, ns_given<KIND>(mats));
}

template <int KIND>
static void ns_launch(NsGemm g, const NsPlan& plan, const NsProduct& p, const NsMatrices& mats, hipStream_t st)
{
    g.tiles = (int)p.tiles, g.whole = (int)p.whole, g.sharers = (int)p.sharers, g.lanes = (int)p.lanes;
    g.tiles_m = (int)(plan.mp / p.tile);
    g.tiles_n = (int)((KIND == kGram || KIND == kPoly ? plan.mp : plan.np) / p.tile);
    if constexpr (KIND == kGram || KIND == kPoly)
        if (p.tile == kFineTile) {
            auto* kernel = g.passes > 1 ? ns_fine_kernel<KIND, true> : ns_fine_kernel<KIND, false>;
            hipLaunchKernelGGL(kernel, dim3((uint32_t)(p.tiles * p.sharers)), dim3(512), 0, st, g);
            if (KIND == kGram && p.sharers > 1) hipLaunchKernelGGL(ns_fine_join_kernel, dim3((uint32_t)p.tiles), dim3(64), 0, st, g);
            return;
        }
    if (p.tile == 256)
        ns_launch_cfg<NsLarge, KIND>(g, p, mats, st);
    else if (p.tile == 128)
        ns_launch_cfg<NsMiddle, KIND>(g, p, mats, st);
    else
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ns_few_kernel<KIND>), dim3((uint32_t)p.tiles), dim3(256), 0, st, g, ns_given<KIND>(mats));
}

template <int KIND, bool LOW>
static void ns_launch_narrow(NsGemm g, const NsPlan& plan, const NsMatrices& mats, hipStream_t st)
{
    g.tiles_n = (int)(plan.np / kPanel);
    const int groups = (int)(plan.mp / 64);
    auto* kernel = groups == 1 ? ns_narrow_kernel<KIND, 1, LOW> : groups == 2 ? ns_narrow_kernel<KIND, 2, LOW>
                   : groups == 3 ? ns_narrow_kernel<KIND, 3, LOW> : ns_narrow_kernel<KIND, 4, LOW>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)plan.step.tiles), dim3(128 * groups), 0, st, g, ns_given<KIND>(mats));
}

struct NsWork {
    _Float16 *x[2], *a, *b;
};

static void ns_products(const NsPlan& p, const NsWork& w, NsGemm g, const NsMatrices& mats, int64_t count, int steps, hipStream_t st)
{
    const int64_t x_size = p.size(p.np), a_size = p.size(p.mp);
    for (int k = 0; k < steps; k++) {
        _Float16 *x = w.x[k & 1], *y = w.x[(k + 1) & 1];
        NsGemm gram = g;
        gram.p = gram.q = x, gram.p_size = gram.q_size = x_size, gram.p_low = gram.q_low = x_size * count;
        gram.pitch = (int)p.pitch(), gram.k_steps = (int)(p.np / kPanel);
        gram.out = w.a, gram.out_size = a_size, gram.out_low = a_size * count;
        if (p.gram.tile == kFineTile) gram.part = reinterpret_cast<float*>(y);
        ns_launch<kGram>(gram, p, p.gram, mats, st);
        NsGemm poly = gram;
        poly.part = g.part;
        poly.p = poly.q = w.a, poly.p_size = poly.q_size = a_size, poly.p_low = poly.q_low = a_size * count;
        poly.k_steps = (int)(p.mp / kPanel);
        poly.out = w.b;
        if (!p.narrow) ns_launch<kPoly>(poly, p, p.poly, mats, st);
        NsGemm step = poly;
        step.p = p.narrow ? w.a : w.b, step.q = x, step.q_size = x_size, step.q_low = x_size * count;
        step.out = y, step.out_size = x_size, step.out_low = x_size * count;
        if (p.narrow && g.passes == 1)
            k + 1 < steps ? ns_launch_narrow<kStep, false>(step, p, mats, st) : ns_launch_narrow<kLast, false>(step, p, mats, st);
        else if (p.narrow)
            k + 1 < steps ? ns_launch_narrow<kStep, true>(step, p, mats, st) : ns_launch_narrow<kLast, true>(step, p, mats, st);
        else
            k + 1 < steps ? ns_launch<kStep>(step, p, p.step, mats, st) : ns_launch<kLast>(step, p, p.step, mats, st);
    }
}

// Matrices that go through the products together: no more than 64, and no more
// than 1 GiB holds two X, A and B of (or one), which also keeps every offset
// inside a buffer under 2^32 bytes.  Few large matrices fill the chip: of 8
// of 4096 x 16384 each takes 3.74 ms together (2.7 GiB) and 3.86 in threes, of
// 64 of 2048 x 8192 0.51 together (5.2 GiB) and 0.54 in tens (1.1).
constexpr int64_t kNsScratch = int64_t(1) << 30;
static int64_t ns_together(int64_t m, int64_t n, int64_t count, bool precise)
{
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    const int64_t one = 4 * (up(m) + kPanel) * (up(n) + up(m)) * (precise ? 2 : 1);
    return std::min({count, (int64_t)kNsBatch, std::max<int64_t>(1, kNsScratch / one)});
}

// More than go together go in as many groups as they need, even to one matrix,
// each with the plan of its own size: 72 of 768 x 3072 take 2.89 ms as 36 and
// 36 (3.30 as 64 and 8).
struct NsGroups {
    int64_t most, groups, small, larger;        // `larger` groups of small + 1, the others of small
    NsGroups(int64_t m, int64_t n, int64_t count, bool precise)
    {
        most = ns_together(m, n, count, precise);
        groups = (count + most - 1) / most;
        small = count / groups;
        larger = count % groups;
    }
};

// Whether all X but the last, A, B and Z stay where fp16 holds them.  Their elements are no larger than their
// largest singular values: from s <= 1 on, q(s^2) of B, s q(s^2) of the next X and s (b + c s^2) of the narrow kernel's Z,
// with q(t) = a + b t + c t^2; extremes lie at the ends or where a derivative is 0.
static bool ns_in_range(double a, double b, double c, int steps)
{
    constexpr double kMost = 15.0;      // (65504 / kHeld = 15.99, less the products' own errors)
    if (!std::isfinite(a + b + c)) return false;
    double s = 1.0;
    for (int k = 0; k < steps; k++) {
        const double end = s * s, root = std::sqrt(std::max(0.0, 9.0 * b * b - 20.0 * a * c));
        double most_b = 0.0, most_x = 0.0, most_z = 0.0;
        for (double t : {0.0, end, -b / (2.0 * c), (-3.0 * b + root) / (10.0 * c), (-3.0 * b - root) / (10.0 * c), -a / (3.0 * b), -b / (3.0 * c)}) {
            if (!(t >= 0.0 && t <= end)) continue;      // (nor where a divisor is 0)
            const double q = std::fabs(a + b * t + c * t * t);
            most_b = std::max(most_b, q);
            most_x = std::max(most_x, std::sqrt(t) * q);
            most_z = std::max(most_z, std::sqrt(t) * std::fabs(b + c * t));
        }
        if (end > kMost || most_b > kMost || most_z > kMost || (k + 1 < steps && most_x > kMost)) return false;
        s = most_x;
    }
    return true;
}

}  // namespace bs

using namespace bs;

extern "C" int64_t bs_newton_schulz_workspace_bytes(int64_t rows, int64_t cols, int64_t count, int precise)
{
    if (rows <= 0 || cols <= 0 || count <= 0 || rows > 65536 || cols > 65536) return 0;
    const int64_t m = std::min(rows, cols), n = std::max(rows, cols);
    const NsGroups g(m, n, count, precise != 0);
    int64_t total = ns_plan(m, n, g.most, precise != 0).total;      // (what any number of matrices needs)
    if (g.groups > 1) total = std::max(total, ns_plan(m, n, g.small, precise != 0).total);
    if (g.groups > 1 && g.larger) total = std::max(total, ns_plan(m, n, g.small + 1, precise != 0).total);
    return total;
}

extern "C" int bs_newton_schulz(const bs_matrix* matrices, int64_t count, int64_t rows, int64_t cols,
                                const bs_newton_schulz_rule* rule, void* workspace, int64_t workspace_bytes, void* stream)
{
    clear_error();
    const char* what = "bs_newton_schulz";
    if (count < 0 || (count > 0 && matrices == nullptr) || rule == nullptr)
        return set_error(BS_ERR_INVALID, "%s: null arguments or a negative count", what);
    const int64_t m = std::min(rows, cols), n = std::max(rows, cols);
    if (m <= 0 || n > 65536) return set_error(BS_ERR_INVALID, "%s: matrices of 1..65536 rows and columns, got %lld x %lld", what, (long long)rows, (long long)cols);
    if (m * n >= (int64_t(1) << 29)) return set_error(BS_ERR_INVALID, "%s: rows*cols must be < 2^29", what);
    const bs_newton_schulz_rule& r = *rule;
    if (r.steps < 1 || r.steps > 100) return set_error(BS_ERR_INVALID, "%s: steps must be in 1..100, got %d", what, r.steps);
    // (the bounds on X start from ||X_0|| <= 1)
    if (!(r.eps >= 0.f)) return set_error(BS_ERR_INVALID, "%s: eps must not be negative, got %g", what, r.eps);
    if (!ns_in_range(r.a, r.b, r.c, r.steps))
        return set_error(BS_ERR_INVALID, "%s: the coefficients %g, %g, %g take values past 15, out of the operands' range", what, r.a, r.b, r.c);
    auto known = [](int t) { return t == BS_DT_BF16 || t == BS_DT_F32; };
    if (!known(r.grad_type) || !known(r.out_type) || (r.momentum && !known(r.momentum_type)))
        return set_error(BS_ERR_INVALID, "%s: dtypes must be bf16 or fp32", what);
    auto mask = [](int t) { return t == BS_DT_F32 ? 3u : 1u; };
    for (int64_t i = 0; i < count; i++) {
        const bs_matrix& t = matrices[i];
        const int64_t c = t.transposed ? rows : cols;
        if (t.grad == nullptr || t.out == nullptr || (r.momentum && t.momentum == nullptr))
            return set_error(BS_ERR_INVALID, "%s: null matrix", what);
        if (((uintptr_t)t.grad & mask(r.grad_type)) || ((uintptr_t)t.out & mask(r.out_type)) ||
            (r.momentum && ((uintptr_t)t.momentum & mask(r.momentum_type))))
            return set_error(BS_ERR_INVALID, "%s: a matrix is misaligned for its type", what);
        if (t.grad_stride < 0 || t.out_stride < c || (r.momentum && t.momentum_stride < c))
            return set_error(BS_ERR_INVALID, "%s: rows of a matrix that is written overlap", what);
    }
    if (count == 0) return BS_OK;
    const bool precise = r.precise != 0;
    if (workspace == nullptr || ((uintptr_t)workspace & 255u) || workspace_bytes < bs_newton_schulz_workspace_bytes(rows, cols, count, precise))
        return set_error(BS_ERR_INVALID, "%s: workspace too small or misaligned", what);
    const hipStream_t st = (hipStream_t)stream;
    const NsGroups groups(m, n, count, precise);
    NsPlan p{};
    int64_t first = 0, here = 0;
    for (int64_t group = 0; group < groups.groups; group++, first += here) {
        const int64_t size = groups.small + (group < groups.larger);
        if (size != here) p = ns_plan(m, n, size, precise);
        here = size;
        NsMatrices mats{};
        for (int64_t i = 0; i < here; i++) {
            const bs_matrix& t = matrices[first + i];
            const bool tall = (t.transposed ? cols : rows) > (t.transposed ? rows : cols);
            mats.at[i] = {t.grad, t.momentum, t.out, t.grad_stride, t.momentum_stride, t.out_stride, tall, t.rate};
        }
        char* ws = static_cast<char*>(workspace);
        NsPrep a{};
        a.m = m, a.n = n, a.np = p.np;
        a.g_f32 = r.grad_type == BS_DT_F32, a.m_f32 = r.momentum_type == BS_DT_F32, a.momentum = r.momentum, a.nesterov = r.nesterov;
        a.mu = r.mu, a.fresh = r.fresh, a.eps = r.eps, a.precise = precise, a.low = p.size(p.np) * here, a.pitch = p.pitch();
        // about 4096 elements or more to a workgroup, and no more of them than 8 a CU over all matrices
        a.parts = (int)std::max<int64_t>(1, std::min({(int64_t)kNsParts, (m * n + 8191) / 8192, (8 * kNsCus + here - 1) / here}));
        a.parts_at = reinterpret_cast<double*>(ws);
        NsWork w;
        char* at = ws + p.parts_bytes;
        w.x[0] = reinterpret_cast<_Float16*>(at);
        w.x[1] = reinterpret_cast<_Float16*>(at + p.x_bytes);
        w.a = reinterpret_cast<_Float16*>(at + 2 * p.x_bytes);
        w.b = reinterpret_cast<_Float16*>(at + 2 * p.x_bytes + p.a_bytes);
        a.x = w.x[0];
        hipLaunchKernelGGL(ns_norm_kernel, dim3(a.parts, (uint32_t)here), dim3(256), 0, st, a, mats);
        hipLaunchKernelGGL(ns_scale_kernel, dim3((uint32_t)(p.np / 64), (uint32_t)(p.mp / 64), (uint32_t)here), dim3(256), 0, st, a, mats);
        NsGemm g{};
        g.passes = precise ? 3 : 1, g.a = r.a, g.b = r.b, g.c = r.c;
        g.part = reinterpret_cast<float*>(at + 2 * p.x_bytes + 2 * p.a_bytes);
        g.m = m, g.n = n, g.w_f32 = r.out_type == BS_DT_F32, g.update = r.update, g.keep = r.keep;
        ns_products(p, w, g, mats, here, r.steps, st);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
    }
    return BS_OK;
}
