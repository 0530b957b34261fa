// What the forward and backward row kernels of the step between two blocks
// share: how a row lies on the lanes, loads and stores of its 8-element
// chunks in either type, sums over a row.
//
// A row of D elements is D / 8 chunks.  ceil(D / 512) waves hold a row, a
// chunk a lane, and a workgroup holds as many rows as its eight waves make
// (longer rows: 16 waves, and two or four chunks a lane).  The whole row then
// stays with its lanes between the passes that its statistics take, and it is
// read once; with one chunk a lane all of it is in registers.
#pragma once

#include "bs_device.h"

namespace bs {

constexpr int kMaxRowCols = 32768;

typedef __bf16 bf16;

// 8 elements as loaded
template <typename T>
struct Raw {
    uint32_t w[2 * sizeof(T)];
};

template <typename T>
__device__ __forceinline__ float raw_get(const Raw<T>& r, int e)
{
    if constexpr (sizeof(T) == 2)
        return __uint_as_float(e & 1 ? r.w[e >> 1] & 0xffff0000u : r.w[e >> 1] << 16);
    else
        return __uint_as_float(r.w[e]);
}

// 8 elements at any address that their type allows; those from `nv` on are 0
// and not read.  WHOLE: nv is 0 or 8 everywhere (rows of a multiple of 8).
// The last chunk of another row moves as 4, 2 and 1 elements.
template <bool WHOLE = false, typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* p, int nv)
{
    Raw<T> r;
    if (nv >= 8) {
        __builtin_memcpy(&r, p, sizeof(r));
        return r;
    }
    constexpr int W = 2 * (int)sizeof(T);       // words
    typedef uint32_t half_t __attribute__((ext_vector_type(W / 2), aligned(2)));
    typedef uint32_t quarter_t __attribute__((ext_vector_type(W / 4), aligned(2)));
    half_t four = 0;
    quarter_t two = 0;
    uint32_t one = 0;
    if (!WHOLE && nv > 0) {
        if (nv & 4) {
            four = *reinterpret_cast<const half_t*>(p);
            p += 4;
        }
        if (nv & 2) {
            two = *reinterpret_cast<const quarter_t*>(p);
            p += 2;
        }
        if (nv & 1) one = sizeof(T) == 2 ? *reinterpret_cast<const uint16_t*>(p) : *reinterpret_cast<const uint32_t*>(p);
    }
#pragma unroll
    for (int i = 0; i < W / 2; i++) r.w[i] = four[i];
#pragma unroll
    for (int i = 0; i < W / 4; i++) {           // behind the four, or first
        r.w[W / 2 + i] = nv & 4 ? two[i] : 0u;
        r.w[i] = nv & 4 ? r.w[i] : two[i];
        r.w[W - W / 4 + i] = 0u;
    }
    constexpr int S = W / 4;                    // words of two elements
    const int pairs = nv >> 1;
    r.w[0] |= pairs == 0 ? one : 0u;
    r.w[S] |= pairs == 1 ? one : 0u;
    r.w[2 * S] |= pairs == 2 ? one : 0u;
    r.w[3 * S] |= pairs == 3 ? one : 0u;
    return r;
}

template <typename T>
__device__ __forceinline__ Raw<T> to_raw(const float (&v)[8])
{
    Raw<T> r;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; i++) r.w[i] = f32_to_bf16(v[2 * i]) | (f32_to_bf16(v[2 * i + 1]) << 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) r.w[i] = __float_as_uint(v[i]);
    }
    return r;
}

template <bool WHOLE = false, typename T>
__device__ __forceinline__ void store_raw(T* p, const Raw<T>& r, int nv)
{
    if (nv >= 8) {
        __builtin_memcpy(p, &r, sizeof(r));
        return;
    }
    if (WHOLE || nv <= 0) return;
    constexpr int W = 2 * (int)sizeof(T);
    typedef uint32_t half_t __attribute__((ext_vector_type(W / 2), aligned(2)));
    typedef uint32_t quarter_t __attribute__((ext_vector_type(W / 4), aligned(2)));
    half_t four;
    quarter_t two;
#pragma unroll
    for (int i = 0; i < W / 2; i++) four[i] = r.w[i];
    // (masks, not selections: those between elements of an array become its address)
    const uint32_t far = nv & 4 ? ~0u : 0u, mid = nv & 2 ? ~0u : 0u;
#pragma unroll
    for (int i = 0; i < W / 4; i++) two[i] = (r.w[W / 2 + i] & far) | (r.w[i] & ~far);
    const uint32_t one = (((r.w[W - W / 4] & far) | (r.w[W / 4] & ~far)) & mid) | (two[0] & ~mid);
    if (nv & 4) {
        *reinterpret_cast<half_t*>(p) = four;
        p += 4;
    }
    if (nv & 2) {
        *reinterpret_cast<quarter_t*>(p) = two;
        p += 2;
    }
    if (nv & 1) {
        if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint16_t*>(p) = (uint16_t)one;
        else
            *reinterpret_cast<uint32_t*>(p) = one;
    }
}

// A learned vector (or one number for all columns), in either type; null: `other` everywhere.
struct RowParam {
    const void* p;
    int f32;        // fp32, or bf16
    int one;        // one number
};

__device__ __forceinline__ float param_one(const RowParam& a, int64_t i)
{
    return a.f32 ? static_cast<const float*>(a.p)[i] : (float)static_cast<const bf16*>(a.p)[i];
}
__device__ __forceinline__ void param_chunk(const RowParam& a, int64_t col, int nv, float other, float (&v)[8])
{
    if (a.p == nullptr || a.one || nv <= 0) {
        const float s = a.p == nullptr || nv <= 0 ? other : param_one(a, 0);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = s;
    } else if (a.f32) {
        const Raw<float> r = load_raw(static_cast<const float*>(a.p) + col, nv);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = raw_get(r, e);
    } else {
        const Raw<bf16> r = load_raw(static_cast<const bf16*>(a.p) + col, nv);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = raw_get(r, e);
    }
}
__device__ __forceinline__ void param_store(void* p, int f32, int64_t i, float v)
{
    if (f32)
        static_cast<float*>(p)[i] = v;
    else
        static_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_bf16(v);
}

// Sum over the 64 lanes of a wave, the same value in every lane: four steps
// inside rows of 16 lanes, two across them, read back from the last lane.
__device__ __forceinline__ float wave_sum_f32(float v)
{
#define BS_DPP_ADD(ctrl, rows)                                                                                     \
    v += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), ctrl, rows, 0xf, false))
    BS_DPP_ADD(0xb1, 0xf);      // lane ^ 1
    BS_DPP_ADD(0x4e, 0xf);      // lane ^ 2
    BS_DPP_ADD(0x141, 0xf);     // mirror in 8
    BS_DPP_ADD(0x140, 0xf);     // mirror in 16
    BS_DPP_ADD(0x142, 0xa);     // last lane of rows 0, 2 into rows 1, 3
    BS_DPP_ADD(0x143, 0xc);     // last lane of row 1 into rows 2, 3
#undef BS_DPP_ADD
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}

// How a thread's chunks lie in its row.
template <int C>
struct RowPlace {
    int waves;              // of a row
    int sub;                // which of the workgroup's rows
    int wave, lane_in_row;  // this thread's
    int in_row[C];          // elements of its chunks inside the row
    int64_t col[C];
    float n_wave;           // elements of the row in this wave
    float inv_cols;
    __device__ __forceinline__ RowPlace(int64_t cols, int waves_)
    {
        waves = waves_;
        const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        sub = w / waves;
        wave = w - sub * waves;
        lane_in_row = wave * 64 + ((int)threadIdx.x & 63);
        n_wave = n_of(wave, cols);
        inv_cols = 1.0f / (float)cols;
#pragma unroll
        for (int k = 0; k < C; k++) {
            const int c = (k * 64 * waves + lane_in_row) * 8;
            col[k] = c;
            in_row[k] = max(0, min(8, (int)cols - c));
        }
    }
    // elements of the row in wave i
    __device__ __forceinline__ float n_of(int i, int64_t cols) const
    {
        int n = 0;
#pragma unroll
        for (int k = 0; k < C; k++) n += max(0, min(512, (int)cols - (k * waves + i) * 512));
        return (float)n;
    }
};

// 1 / sqrt(v) within about half a unit of the last place: one Newton step on
// the instruction's value, whose residual 1 - v r^2 is exact to its last bit
// by fused products (the correctly rounded root and division cost more and
// round twice).  0 and infinity have no residual and keep inf and 0.
__device__ __forceinline__ float row_rstd(float v)
{
    const float r = rsqrtf(v), h = v * r;
    const float e = fmaf(-h, r, 1.f) - fmaf(v, r, -h) * r;
    return fabsf(e) < 0.5f ? fmaf(0.5f * r, e, r) : r;
}

// LDS for the sums of rows over their waves: two buffers in turn, so that one
// barrier a sum is enough (a thread that writes a buffer again has passed the
// barrier that came after everybody's reads of it).
struct RowSums {
    float4 part[2][16];
};

// Mean (0 for an RMS norm) and mean of squared deviations of a row.  A layer
// norm's deviations are from each wave's own mean first; the waves' are joined
// by n (mean_w - mean)^2, so nothing is lost where the mean is large.
template <int C>
__device__ __forceinline__ void row_moments(const float (&v)[C][8], const int (&nv)[C], const RowPlace<C>& at, int64_t cols, bool layer,
                                            RowSums& s, int& turn, float& mean, float& var)
{
    float mw = 0.f;
    if (layer) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < C; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) t += v[k][e];
        mw = wave_sum_f32(t) / fmaxf(at.n_wave, 1.f);
    }
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < C; k++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float d = v[k][e] - mw;
            q += e < nv[k] ? d * d : 0.f;
        }
    q = wave_sum_f32(q);
    if (at.waves > 1) {
        const float4* part = s.part[turn] + at.sub * at.waves;
        if ((threadIdx.x & 63) == 0) s.part[turn][at.sub * at.waves + at.wave] = float4{mw, q, 0.f, 0.f};
        __syncthreads();
        float m = 0.f;
        if (layer) {
            for (int i = 0; i < at.waves; i++) m += part[i].x * at.n_of(i, cols);
            m *= at.inv_cols;
        }
        q = 0.f;
        for (int i = 0; i < at.waves; i++) {
            const float4 p = part[i];
            const float d = p.x - m;
            q += layer ? p.y + at.n_of(i, cols) * d * d : p.y;
        }
        mw = m;
        turn ^= 1;
    }
    mean = mw;
    var = q * at.inv_cols;
}

// Sums of up to three values over a row, the same in all its threads.
template <int N, int C>
__device__ __forceinline__ void row_sums(float (&v)[N], const RowPlace<C>& at, RowSums& s, int& turn)
{
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = wave_sum_f32(v[i]);
    if (at.waves > 1) {
        const float4* part = s.part[turn] + at.sub * at.waves;
        if ((threadIdx.x & 63) == 0)
            s.part[turn][at.sub * at.waves + at.wave] = float4{v[0], N > 1 ? v[N > 1 ? 1 : 0] : 0.f, N > 2 ? v[N > 2 ? 2 : 0] : 0.f, 0.f};
        __syncthreads();
        float t[3] = {0.f, 0.f, 0.f};
        for (int i = 0; i < at.waves; i++) {
            const float4 p = part[i];
            t[0] += p.x;
            t[1] += p.y;
            t[2] += p.z;
        }
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = t[i];
        turn ^= 1;
    }
}

// Workgroups of a row kernel: chunks of a lane, waves of a row, rows of a
// workgroup at a time, threads.  `wide`: the longest rows of one chunk a lane.
struct RowLaunch {
    int chunks, waves, rows, threads;
};
inline RowLaunch row_launch(int64_t cols, int64_t wide)
{
    const int most = wide > 4096 ? 16 : 8;
    const int c = cols <= wide ? 1 : cols <= 2 * wide ? 2 : 4;
    const int w = (int)((cols + 512 * c - 1) / (512 * c));
    const int r = w <= most / 2 ? 8 / w > 0 ? 8 / w : 1 : 1;
    return {c, w, r, 64 * w * r};
}

}  // namespace bs
