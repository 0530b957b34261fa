// Orthogonalising updates by Newton-Schulz products (bitsparse_amd/muon.py).
//
// For matrices U [m, n], m <= n (a taller one is taken as its transpose):
//   X_0     = U / (||U||_F + eps)
//   A_k     = X_k X_k^T                        gram      m^2 n   operations (half of a symmetric product)
//   B_k     = a I + b A_k + c A_k^2            poly      m^3
//   X_{k+1} = B_k X_k                          step      2 m^2 n
// and of the last X either itself in bf16 or, for an optimiser, the update of
// the weights.  U is the gradient or, with a momentum, M' = mu M + (1 - mu) G
// and U = (1 - mu) G + mu M' (Nesterov) or M'.
//
// The products run on the matrix cores with fp16 operands and fp32 sums.  X,
// A and B are held as fp16 times 2^12: ||X_0|| <= 1 keeps every singular
// value of the iteration below 1.21 and so every element of X, A and B below
// 3.5, far inside fp16's range, and elements down to 2^-26 keep all 11 bits.
// bf16 operands, three bits shorter, measure 1.0-2.0e-2 from the exact
// result on gradients, fp16 ones 1.0-2.4e-3, less than the 1.7e-3 that
// rounding the result itself to bf16 costs.
//
// All buffers are padded with zeros to whole tiles, which the products keep
// (B's padding only meets X's zero rows), so the main loop has no bounds.
#include <algorithm>
#include <type_traits>

#include "bs_device.h"
#include "bs_host.h"

namespace bs {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float kHeld = 4096.f;         // fp16 value = true value * kHeld
constexpr int kStepK = 64;              // K of a main-loop step
constexpr int kNsBatch = 64;            // matrices of a launch
constexpr int kNsParts = 64;            // partial sums of squares of a matrix

enum : int { kGram = 0, kPoly, kStep, kLast };

struct NsMatrix {
    const void* g;
    void* m;
    void* w;                            // weights, or the result
    int64_t g_stride, m_stride, w_stride;
    int tall;                           // given as [n, m]
};
struct NsMatrices {
    NsMatrix at[kNsBatch];
};

// ---------------------------------------------------------------------------
// U, its norm and X_0
// ---------------------------------------------------------------------------
struct NsPrep {
    int64_t m, n, mp, np;
    int g_f32, m_f32, momentum, nesterov;
    float mu, eps;
    double* parts;                      // [count][kNsParts]
    _Float16* x;                        // [count][mp][np]
};

__device__ __forceinline__ float ns_load(const void* p, int f32, int64_t i)
{
    return f32 ? static_cast<const float*>(p)[i] : (float)static_cast<const __bf16*>(p)[i];
}
__device__ __forceinline__ void ns_store(void* p, int f32, int64_t i, float v)
{
    if (f32)
        static_cast<float*>(p)[i] = v;
    else
        static_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_bf16(v);
}
// M' as its type holds it, and U
__device__ __forceinline__ float ns_update(const NsPrep& a, float g, float m) { return a.nesterov ? (1.f - a.mu) * g + a.mu * m : m; }

// The momentum's update and partial sums of squares of U (in 64 bits: any
// gradient that fp32 holds has a norm).  blockIdx.y: the matrix.
__global__ __launch_bounds__(256) void ns_norm_kernel(NsPrep a, NsMatrices mats)
{
    const NsMatrix t = mats.at[blockIdx.y];
    const int64_t rows = t.tall ? a.n : a.m, cols = t.tall ? a.m : a.n, total = rows * cols;
    double s = 0.0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / cols, c = i - r * cols;
        float u = ns_load(t.g, a.g_f32, r * t.g_stride + c);
        if (a.momentum) {
            const int64_t at = r * t.m_stride + c;
            const float m = a.mu * ns_load(t.m, a.m_f32, at) + (1.f - a.mu) * u;
            ns_store(t.m, a.m_f32, at, m);
            u = ns_update(a, u, a.m_f32 ? m : (float)(__bf16)m);
        }
        s += (double)u * (double)u;
    }
    __shared__ double s_part[256];
    s_part[threadIdx.x] = s;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) s_part[threadIdx.x] += s_part[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) a.parts[(int64_t)blockIdx.y * kNsParts + blockIdx.x] = s_part[0];
}

// X_0 in 64 x 64 tiles of [mp, np], zeros outside [m, n].
__global__ __launch_bounds__(256) void ns_scale_kernel(NsPrep a, NsMatrices mats, int parts)
{
    const NsMatrix t = mats.at[blockIdx.z];
    __shared__ float s_t[64][65];
    double q = 0.0;
    for (int i = 0; i < parts; i++) q += a.parts[(int64_t)blockIdx.z * kNsParts + i];
    const float norm = (float)sqrt(q) + a.eps;
    const int64_t i0 = (int64_t)blockIdx.y * 64, j0 = (int64_t)blockIdx.x * 64;
    const int c = threadIdx.x & 63, r4 = threadIdx.x >> 6;
    for (int r = r4; r < 64; r += 4) {
        const int64_t gr = (t.tall ? j0 : i0) + r, gc = (t.tall ? i0 : j0) + c;
        float u = 0.f;
        if (gr < (t.tall ? a.n : a.m) && gc < (t.tall ? a.m : a.n)) {
            u = ns_load(t.g, a.g_f32, gr * t.g_stride + gc);
            if (a.momentum) u = ns_update(a, u, ns_load(t.m, a.m_f32, gr * t.m_stride + gc));
        }
        if (t.tall)
            s_t[c][r] = u;
        else
            s_t[r][c] = u;
    }
    __syncthreads();
    for (int r = r4; r < 64; r += 4)
        a.x[((int64_t)blockIdx.z * a.mp + i0 + r) * a.np + j0 + c] = (_Float16)(s_t[r][c] / norm * kHeld);
}

// ---------------------------------------------------------------------------
// the products: C[i, j] = sum_k P[i, k] Q[j, k] (gram, poly) or
// sum_k P[i, k] Q[k, j] (step, last)
// ---------------------------------------------------------------------------
struct NsGemm {
    const _Float16 *p, *q;              // [count] matrices
    int64_t p_size, q_size, out_size;   // elements of one matrix
    int ldp, ldq, ldo;
    int k_steps;
    int tiles_m, tiles_n;               // of the whole product
    int count;
    _Float16* out;
    float a, b, c;                      // poly
    // last
    int64_t m, n;
    int w_f32, update;
    float keep, rate;
};

// WGM x WGN waves, each a block of 32 IM x 32 JN
template <int WGM_, int WGN_, int IM_, int JN_>
struct NsCfg {
    static constexpr int WGM = WGM_, WGN = WGN_, IM = IM_, JN = JN_;
    static constexpr int THREADS = 64 * WGM * WGN;
    static constexpr int TM = 32 * IM * WGM, TN = 32 * JN * WGN;
    static constexpr int P_BYTES = TM * kStepK * 2, Q_BYTES = TN * kStepK * 2;
    static constexpr int STAGE = P_BYTES + Q_BYTES;
    static constexpr int PITCH = TN + 8;                        // of the result's tile in LDS
    static constexpr int LDS = 2 * STAGE > TM * PITCH * 2 ? 2 * STAGE : TM * PITCH * 2;
    static_assert(LDS <= 160 * 1024, "LDS budget");
    static_assert(P_BYTES / 1024 % (WGM * WGN) == 0 && Q_BYTES / 1024 % (WGM * WGN) == 0, "whole loads for every wave");
};
using NsLarge = NsCfg<2, 4, 4, 2>;      // 256 x 256
using NsMiddle = NsCfg<2, 2, 2, 2>;     // 128 x 128
using NsSmall = NsCfg<2, 2, 1, 1>;      // 64 x 64

// 16 bytes a lane from `rsrc` at voff + soff straight into LDS at `lds` + 16 lane
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, uint32_t lds, uint32_t voff, uint32_t soff)
{
    // (one wait state between the write of m0 and its use)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc), "s"(soff)
                 : "memory", "m0");
}
__device__ __forceinline__ i32x4 ns_rsrc(const void* p, uint32_t bytes)
{
    const uint64_t a = (uint64_t)p;
    return i32x4{(int)uniform_u32((uint32_t)a), (int)uniform_u32((uint32_t)(a >> 32) & 0xffffu), (int)bytes, 0x00020000};
}

template <class Cfg, int KIND>
__global__ __launch_bounds__(Cfg::THREADS) void ns_gemm_kernel(NsGemm g, NsMatrices mats)
{
    __shared__ __attribute__((aligned(16))) char s_mem[Cfg::LDS];
    constexpr bool kSym = KIND == kGram || KIND == kPoly;
    constexpr int kWaves = Cfg::WGM * Cfg::WGN;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = wave / Cfg::WGN, wn = wave % Cfg::WGN;

    // the tile: of a symmetric product only those with tj <= ti
    const int per = kSym ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
    const int batch = (int)blockIdx.x / per, tile = (int)blockIdx.x % per;
    int ti, tj;
    if constexpr (kSym) {
        ti = (int)((sqrtf(8.f * (float)tile + 1.f) - 1.f) * 0.5f);
        while ((ti + 1) * (ti + 2) / 2 <= tile) ti++;
        while (ti * (ti + 1) / 2 > tile) ti--;
        tj = tile - ti * (ti + 1) / 2;
    } else {
        ti = tile % g.tiles_m;
        tj = tile / g.tiles_m;
    }

    const _Float16* p = g.p + batch * g.p_size + (int64_t)ti * Cfg::TM * g.ldp;
    const _Float16* q = g.q + batch * g.q_size + (kSym ? (int64_t)tj * Cfg::TN * g.ldq : (int64_t)tj * Cfg::TN);
    const i32x4 rp = ns_rsrc(p, (uint32_t)(Cfg::TM * (int64_t)g.ldp * 2));
    // (rows of Q: the tile's, or all K up to the tile's last column)
    const i32x4 rq = ns_rsrc(q, kSym ? (uint32_t)(Cfg::TN * (int64_t)g.ldq * 2)
                                     : (uint32_t)(((int64_t)(g.k_steps * kStepK - 1) * g.ldq + Cfg::TN) * 2));
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_mem;

    // Loads.  An [R, 64] tile with K along the row: rows of 128 bytes, the 16-byte chunk c of row r at c ^ (r & 7), so
    // that eight lanes reading one chunk of eight rows meet all banks.  A [64, TN] tile with K down the rows: chunk c of
    // row k at c ^ 2 (k & 3), so that the four rows a transposing read takes lie in different bank groups.
    auto load_rows = [&](i32x4 rsrc, uint32_t lds, int rows, int ld, int k0) {
        for (int s = 0; s < rows / 8 / kWaves; s++) {
            const int slot = s * kWaves + wave;                     // 1 KiB: 8 rows
            const int r = slot * 8 + (lane >> 3), c = (lane & 7) ^ (r & 7);
            load_to_lds(rsrc, lds + slot * 1024, (uint32_t)(r * ld + c * 8) * 2u, (uint32_t)k0 * 2u);
        }
    };
    auto load_cols = [&](i32x4 rsrc, uint32_t lds, int ld, int k0) {
        constexpr int kChunks = Cfg::TN / 8;                        // of a row
        for (int s = 0; s < Cfg::Q_BYTES / 1024 / kWaves; s++) {
            const int at = (s * kWaves + wave) * 64 + lane;
            const int k = at / kChunks, c = (at % kChunks) ^ (2 * (k & 3));
            load_to_lds(rsrc, lds + (s * kWaves + wave) * 1024, (uint32_t)(k * ld + c * 8) * 2u, (uint32_t)k0 * (uint32_t)ld * 2u);
        }
    };
    auto load = [&](int step) {
        const uint32_t at = lds0 + (step & 1) * Cfg::STAGE;
        load_rows(rp, at, Cfg::TM, g.ldp, step * kStepK);
        if constexpr (kSym)
            load_rows(rq, at + Cfg::P_BYTES, Cfg::TN, g.ldq, step * kStepK);
        else
            load_cols(rq, at + Cfg::P_BYTES, g.ldq, step * kStepK);
    };

    f32x16 acc[Cfg::IM][Cfg::JN];
#pragma unroll
    for (int i = 0; i < Cfg::IM; i++)
#pragma unroll
        for (int j = 0; j < Cfg::JN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;

    auto row_frag = [&](const char* t, int r0, int slice) -> f16x8 {
        const int r = r0 + (lane & 31), c = (2 * slice + (lane >> 5)) ^ (r & 7);
        return *reinterpret_cast<const f16x8*>(t + r * 128 + c * 16);
    };
    // within 16 lanes lane j points at row k0 + j / 4, columns 4 (j % 4) on, and gets column j of four rows
    auto col_frag = [&](const char* t, int c0, int slice) -> f16x8 {
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const int j = lane & 15, col = c0 + (lane & 16) + 4 * (j & 3);
        s16x4 h[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int k = 16 * slice + 8 * (lane >> 5) + 4 * u + (j >> 2);
            const int chunk = (col >> 3) ^ (2 * (k & 3));
            h[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(t + k * (Cfg::TN * 2) + chunk * 16 + (col & 7) * 2));
        }
        return __builtin_bit_cast(f16x8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
    };

    load(0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    for (int step = 0; step < g.k_steps; step++) {
        if (step + 1 < g.k_steps) load(step + 1);
        const char* tp = s_mem + (step & 1) * Cfg::STAGE;
        const char* tq = tp + Cfg::P_BYTES;
#pragma unroll
        for (int s = 0; s < kStepK / 16; s++) {
            f16x8 fp[Cfg::IM], fq[Cfg::JN];
#pragma unroll
            for (int i = 0; i < Cfg::IM; i++) fp[i] = row_frag(tp, wm * 32 * Cfg::IM + 32 * i, s);
#pragma unroll
            for (int j = 0; j < Cfg::JN; j++)
                fq[j] = kSym ? row_frag(tq, wn * 32 * Cfg::JN + 32 * j, s) : col_frag(tq, wn * 32 * Cfg::JN + 32 * j, s);
#pragma unroll
            for (int i = 0; i < Cfg::IM; i++)
#pragma unroll
                for (int j = 0; j < Cfg::JN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fq[j], fp[i], acc[i][j], 0, 0, 0);
        }
        // this step's reads are done and the next step's tiles are there, in every wave
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
    }

    // Results: lane holds row i = lane % 32 of a block, columns 8 q + 4 (lane / 32) + e in register 4 q + e.  Through LDS
    // as a row-major tile (the main loop's last barrier has passed).
    _Float16* tile_s = reinterpret_cast<_Float16*>(s_mem);
    const float scale = KIND == kLast ? 1.f / kHeld : KIND == kPoly ? g.c / kHeld : 1.f / kHeld;
#pragma unroll
    for (int i = 0; i < Cfg::IM; i++)
#pragma unroll
        for (int j = 0; j < Cfg::JN; j++) {
            const int r = (wm * Cfg::IM + i) * 32 + (lane & 31);
#pragma unroll
            for (int qd = 0; qd < 4; qd++) {
                const int c = (wn * Cfg::JN + j) * 32 + 8 * qd + 4 * (lane >> 5);
                f16x4 v;
                f16x4 old = {};
                const int gi = ti * Cfg::TM + r, gj = tj * Cfg::TN + c;
                if constexpr (KIND == kPoly)        // p is A
                    old = *reinterpret_cast<const f16x4*>(g.p + batch * g.p_size + (int64_t)gi * g.ldp + gj);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float x = acc[i][j][4 * qd + e] * scale;
                    if constexpr (KIND == kPoly) x += g.b * (float)old[e] + (gi == gj + e ? g.a * kHeld : 0.f);
                    v[e] = (_Float16)x;
                }
                *reinterpret_cast<f16x4*>(tile_s + r * Cfg::PITCH + c) = v;
            }
        }
    __syncthreads();

    if constexpr (KIND != kLast) {
        _Float16* out = g.out + batch * g.out_size;
        for (int t = threadIdx.x; t < Cfg::TM * Cfg::TN / 8; t += Cfg::THREADS) {
            const int r = t / (Cfg::TN / 8), c = t % (Cfg::TN / 8) * 8;
            *reinterpret_cast<f16x8*>(out + (int64_t)(ti * Cfg::TM + r) * g.ldo + tj * Cfg::TN + c) =
                *reinterpret_cast<const f16x8*>(tile_s + r * Cfg::PITCH + c);
        }
        if (kSym && ti != tj) {
            for (int t = threadIdx.x; t < Cfg::TM * Cfg::TN / 8; t += Cfg::THREADS) {
                const int r = t / (Cfg::TM / 8), c = t % (Cfg::TM / 8) * 8;     // row r, columns c on of the transpose
                f16x8 v;
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = tile_s[(c + e) * Cfg::PITCH + r];
                *reinterpret_cast<f16x8*>(out + (int64_t)(tj * Cfg::TN + r) * g.ldo + ti * Cfg::TM + c) = v;
            }
        }
    } else {
        const NsMatrix mat = mats.at[batch];
        const int64_t rows = mat.tall ? g.n : g.m, cols = mat.tall ? g.m : g.n;
        const int64_t r0 = mat.tall ? (int64_t)tj * Cfg::TN : (int64_t)ti * Cfg::TM;
        const int64_t c0 = mat.tall ? (int64_t)ti * Cfg::TM : (int64_t)tj * Cfg::TN;
        const int width = mat.tall ? Cfg::TM : Cfg::TN;
        for (int t = threadIdx.x; t < Cfg::TM * Cfg::TN; t += Cfg::THREADS) {
            const int r = t / width, c = t % width;
            if (r0 + r >= rows || c0 + c >= cols) continue;
            const float o = (float)(mat.tall ? tile_s[c * Cfg::PITCH + r] : tile_s[r * Cfg::PITCH + c]) * (1.f / kHeld);
            const int64_t at = (r0 + r) * mat.w_stride + c0 + c;
            ns_store(mat.w, g.w_f32, at, g.update ? g.keep * ns_load(mat.w, g.w_f32, at) - g.rate * o : o);
        }
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
struct NsPlan {
    int tile;                   // 256, 128 or 64
    int64_t mp, np;
    int64_t x_bytes, a_bytes, parts_bytes, total;   // of `count` matrices
};

// The largest tile whose products still give every CU work, and of those whose
// padding does not undo the gain.
static NsPlan ns_plan(int64_t m, int64_t n, int64_t count)
{
    NsPlan p{};
    auto up = [](int64_t v, int64_t t) { return (v + t - 1) / t * t; };
    double best = 0;
    for (const int t : {256, 128, 64}) {
        const int64_t mp = up(m, t), np = up(n, t), tm = mp / t, tn = np / t;
        // time of the three products in tile steps over the CUs: a tile step of 256, 128, 64 takes about 1, 0.34, 0.13
        const double cost = t == 256 ? 1.0 : t == 128 ? 0.34 : 0.13;
        const int64_t slots = t == 256 ? 256 : t == 128 ? 512 : 1024;
        auto rounds = [&](int64_t tiles) { return (double)((tiles * count + slots - 1) / slots) * (double)slots / 256.0; };
        const double time = cost * (rounds(tm * (tm + 1) / 2) * (double)(np + mp) + rounds(tm * tn) * (double)mp);
        if (p.tile == 0 || time < best) p.tile = t, p.mp = mp, p.np = np, best = time;
    }
    p.x_bytes = p.mp * p.np * 2 * count;
    p.a_bytes = p.mp * p.mp * 2 * count;
    p.parts_bytes = (kNsParts * 8 * count + 255) / 256 * 256;
    p.total = 2 * p.x_bytes + 2 * p.a_bytes + p.parts_bytes;
    return p;
}

template <class Cfg, int KIND>
static hipError_t ns_launch(const NsGemm& g, const NsMatrices& mats, hipStream_t st)
{
    const int per = KIND == kGram || KIND == kPoly ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(ns_gemm_kernel<Cfg, KIND>), dim3((uint32_t)(per * g.count)), dim3(Cfg::THREADS), 0, st, g, mats);
    return hipGetLastError();
}

struct NsWork {
    _Float16 *x[2], *a, *b;
};

template <class Cfg>
static hipError_t ns_products(const NsPlan& p, const NsWork& w, NsGemm g, const NsMatrices& mats, int steps, hipStream_t st)
{
    g.tiles_m = (int)(p.mp / Cfg::TM);
    g.tiles_n = (int)(p.np / Cfg::TN);
    hipError_t e = hipSuccess;
    for (int k = 0; k < steps && e == hipSuccess; k++) {
        _Float16 *x = w.x[k & 1], *y = w.x[(k + 1) & 1];
        NsGemm gram = g;
        gram.p = gram.q = x, gram.p_size = gram.q_size = p.mp * p.np, gram.ldp = gram.ldq = (int)p.np;
        gram.out = w.a, gram.out_size = p.mp * p.mp, gram.ldo = (int)p.mp, gram.k_steps = (int)(p.np / kStepK);
        e = ns_launch<Cfg, kGram>(gram, mats, st);
        if (e != hipSuccess) break;
        NsGemm poly = gram;
        poly.p = poly.q = w.a, poly.p_size = poly.q_size = p.mp * p.mp, poly.ldp = poly.ldq = (int)p.mp;
        poly.out = w.b, poly.k_steps = (int)(p.mp / kStepK);
        e = ns_launch<Cfg, kPoly>(poly, mats, st);
        if (e != hipSuccess) break;
        NsGemm step = poly;
        step.p = w.b, step.q = x, step.q_size = p.mp * p.np, step.ldq = (int)p.np;
        step.out = y, step.out_size = p.mp * p.np, step.ldo = (int)p.np;
        e = k + 1 < steps ? ns_launch<Cfg, kStep>(step, mats, st) : ns_launch<Cfg, kLast>(step, mats, st);
    }
    return e;
}

}  // namespace bs

using namespace bs;

extern "C" int64_t bs_newton_schulz_workspace_bytes(int64_t rows, int64_t cols, int64_t count)
{
    if (rows <= 0 || cols <= 0 || count <= 0 || rows > 65536 || cols > 65536) return 0;
    return ns_plan(std::min(rows, cols), std::max(rows, cols), std::min<int64_t>(count, kNsBatch)).total;
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
    if (m * n >= (int64_t(1) << 30)) return set_error(BS_ERR_INVALID, "%s: rows*cols must be < 2^30", what);
    const bs_newton_schulz_rule& r = *rule;
    if (r.steps < 1 || r.steps > 100) return set_error(BS_ERR_INVALID, "%s: steps must be in 1..100, got %d", what, r.steps);
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
    if (workspace == nullptr || ((uintptr_t)workspace & 255u) || workspace_bytes < bs_newton_schulz_workspace_bytes(rows, cols, count))
        return set_error(BS_ERR_INVALID, "%s: workspace too small or misaligned", what);
    const hipStream_t st = (hipStream_t)stream;
    for (int64_t first = 0; first < count; first += kNsBatch) {
        const int64_t here = std::min<int64_t>(count - first, kNsBatch);
        const NsPlan p = ns_plan(m, n, std::min<int64_t>(count, kNsBatch));
        NsMatrices mats{};
        for (int64_t i = 0; i < here; i++) {
            const bs_matrix& t = matrices[first + i];
            const bool tall = (t.transposed ? cols : rows) > (t.transposed ? rows : cols);
            mats.at[i] = {t.grad, t.momentum, t.out, t.grad_stride, t.momentum_stride, t.out_stride, tall};
        }
        char* ws = static_cast<char*>(workspace);
        NsPrep a{};
        a.m = m, a.n = n, a.mp = p.mp, a.np = p.np;
        a.g_f32 = r.grad_type == BS_DT_F32, a.m_f32 = r.momentum_type == BS_DT_F32, a.momentum = r.momentum, a.nesterov = r.nesterov;
        a.mu = r.mu, a.eps = r.eps;
        a.parts = reinterpret_cast<double*>(ws);
        NsWork w;
        w.x[0] = reinterpret_cast<_Float16*>(ws + p.parts_bytes);
        w.x[1] = reinterpret_cast<_Float16*>(ws + p.parts_bytes + p.x_bytes);
        w.a = reinterpret_cast<_Float16*>(ws + p.parts_bytes + 2 * p.x_bytes);
        w.b = reinterpret_cast<_Float16*>(ws + p.parts_bytes + 2 * p.x_bytes + p.a_bytes);
        a.x = w.x[0];
        const int parts = (int)std::min<int64_t>(kNsParts, (m * n + 4095) / 4096);
        hipLaunchKernelGGL(ns_norm_kernel, dim3(parts, (uint32_t)here), dim3(256), 0, st, a, mats);
        hipLaunchKernelGGL(ns_scale_kernel, dim3((uint32_t)(p.np / 64), (uint32_t)(p.mp / 64), (uint32_t)here), dim3(256), 0, st, a, mats, parts);
        hipError_t e = hipGetLastError();
        if (e == hipSuccess) {
            NsGemm g{};
            g.count = (int)here, g.a = r.a, g.b = r.b, g.c = r.c;
            g.m = m, g.n = n, g.w_f32 = r.out_type == BS_DT_F32, g.update = r.update, g.keep = r.keep, g.rate = r.rate;
            e = p.tile == 256 ? ns_products<NsLarge>(p, w, g, mats, r.steps, st)
                : p.tile == 128 ? ns_products<NsMiddle>(p, w, g, mats, r.steps, st)
                                : ns_products<NsSmall>(p, w, g, mats, r.steps, st);
        }
        if (e != hipSuccess) return set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
    }
    return BS_OK;
}
