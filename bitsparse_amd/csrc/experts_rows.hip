// The experts' rows back into tokens: the weighted sum over a token's choices,
// its gradients, and the step between the two products of an expert's backward.
//
//   out[t] = sum over j of w[t, j] y[place[t, j]]        (32-bit sums in the order of j)
//   dy[place[t, j]] = w[t, j] dout[t];  dw[t, j] = <dout[t], y[place[t, j]]>
//
// over the places that are rows of an expert; dy is 0 in all other rows.
//
// Bound by memory: y, dout and the results once.  A workgroup a token.  16384
// tokens, 4 choices, 4096 wide: the sum 143 us, 4.7 TB/s; its gradients, with
// dout held by the caches over a token's choices, 239 us, 5.1 TB/s (a copy
// reaches 4.9); 32 tokens, 8 choices: 4.6 us, latency.  Narrow rows leave most of a
// workgroup's threads without a chunk, and the workgroups' number counts: 16384 tokens, 2 choices, 64 and 256
// wide 17 us for 6 and 25 MB, 1024 wide 23 us for 101.
#include <algorithm>

#include "bs_host.h"
#include "rownorm.h"

namespace bs {

constexpr int kMaxChoices = 64;
constexpr int kTailBlocks = 64;     // workgroups that clear the rows of no expert
constexpr int64_t kSlice = 1 << 22; // workgroups of a launch, which has fewer than 2^32 threads

struct CombineArgs {
    int64_t tokens, rows, cols;
    int top_k;
    const void* y;
    int64_t y_stride;
    const float* weights;       // null: 1
    const int32_t *place, *first, *used;        // rows *first (null: 0) up to *used (null: all) belong to an expert
    bf16* out;
    // backward
    const bf16* g;
    int64_t g_stride;
    bf16* dy;
    float* dw;
};

// the rows that belong to an expert
struct ExpertRows {
    int from, to;
    __device__ __forceinline__ explicit ExpertRows(const CombineArgs& a)
        : from(a.first ? max(0, *a.first) : 0), to(a.used ? (int)min(a.rows, (int64_t)max(0, *a.used)) : (int)a.rows)
    {
    }
    __device__ __forceinline__ bool have(int p) const { return p >= from && p < to; }
};
// 0 into dy's other rows, by kTailBlocks workgroups
template <bool WHOLE>
__device__ __forceinline__ void clear_others(const CombineArgs& a, const ExpertRows& of, int64_t block)
{
    const int64_t front = min((int64_t)of.from, a.rows);
    for (int64_t i = block; i < front + (a.rows - of.to); i += kTailBlocks) {
        const int64_t r = i < front ? i : of.to + (i - front);
        for (int64_t c = threadIdx.x * 8; c < a.cols; c += 2048)
            store_raw<WHOLE>(a.dy + r * a.cols + c, Raw<bf16>{}, (int)min((int64_t)8, a.cols - c));
    }
}

template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a)
{
    const ExpertRows of(a);
    const int64_t t = blockIdx.x;
    const int32_t* place = a.place + t * a.top_k;
    for (int64_t c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 8; c < a.cols; c += (int64_t)gridDim.y * 2048) {
        const int nv = (int)min((int64_t)8, a.cols - c);
        float acc[8] = {};
        for (int j = 0; j < a.top_k; j++) {
            const int p = place[j];
            if (!of.have(p)) continue;
            const float w = a.weights ? a.weights[t * a.top_k + j] : 1.f;
            const Raw<T> y = load_raw<WHOLE>(static_cast<const T*>(a.y) + p * a.y_stride + c, nv);
#pragma unroll
            for (int e = 0; e < 8; e++) acc[e] = fmaf(w, raw_get(y, e), acc[e]);
        }
        store_raw<WHOLE>(a.out + t * a.cols + c, to_raw<bf16>(acc), nv);
    }
}

// dy alone, or (no weights) each token's row to its places: 8192 tokens, 2 choices, 768 wide 9.4 us
template <bool WHOLE>
__global__ __launch_bounds__(256) void spread_kernel(CombineArgs a)
{
    const int64_t chunks = (a.cols + 7) / 8;
    const ExpertRows of(a);
    if ((int64_t)blockIdx.x >= a.tokens) return clear_others<WHOLE>(a, of, blockIdx.x - a.tokens);
    const int64_t t = blockIdx.x;
    // (choices one after the other in a thread's chunks: a short row's threads are all at work)
    for (int64_t i = threadIdx.x; i < chunks * a.top_k; i += 256) {
        const int64_t j = i / chunks, c = (i - j * chunks) * 8;
        const int p = a.place[t * a.top_k + j];
        if (!of.have(p)) continue;
        const int nv = (int)min((int64_t)8, a.cols - c);
        const Raw<bf16> g = load_raw<WHOLE>(a.g + t * a.g_stride + c, nv);
        if (a.weights == nullptr) {
            store_raw<WHOLE>(a.dy + p * a.cols + c, g, nv);
            continue;
        }
        const float w = a.weights[t * a.top_k + j];
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = w * raw_get(g, e);
        store_raw<WHOLE>(a.dy + p * a.cols + c, to_raw<bf16>(o), nv);
    }
}

// dw, and dy where it is asked for
template <bool WHOLE>
__global__ __launch_bounds__(256) void combine_backward_kernel(CombineArgs a)
{
    __shared__ float s_dot[4][kMaxChoices];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const ExpertRows of(a);
    if ((int64_t)blockIdx.x >= a.tokens) {
        if (a.dy) clear_others<WHOLE>(a, of, blockIdx.x - a.tokens);
        return;
    }
    const int64_t t = blockIdx.x;
    for (int j = 0; j < a.top_k; j++) {
        const int p = a.place[t * a.top_k + j];
        const bool there = of.have(p);
        const float w = a.weights ? a.weights[t * a.top_k + j] : 1.f;
        float dot = 0.f;
        if (there)
            for (int64_t c = threadIdx.x * 8; c < a.cols; c += 2048) {
                const int nv = (int)min((int64_t)8, a.cols - c);
                const Raw<bf16> g = load_raw<WHOLE>(a.g + t * a.g_stride + c, nv);
                if (a.dy) {
                    float o[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) o[e] = w * raw_get(g, e);
                    store_raw<WHOLE>(a.dy + p * a.cols + c, to_raw<bf16>(o), nv);
                }
                const Raw<bf16> y = load_raw<WHOLE>(static_cast<const bf16*>(a.y) + p * a.y_stride + c, nv);
#pragma unroll
                for (int e = 0; e < 8; e++) dot = fmaf(raw_get(g, e), raw_get(y, e), dot);
            }
        dot = wave_sum_f32(dot);
        if (lane == 0) s_dot[wave][j] = dot;
    }
    __syncthreads();
    if ((int)threadIdx.x < a.top_k)
        a.dw[t * a.top_k + threadIdx.x] = (s_dot[0][threadIdx.x] + s_dot[1][threadIdx.x]) + (s_dot[2][threadIdx.x] + s_dot[3][threadIdx.x]);
}

// The backward of y = sum w act(z) W2^T between its products, a workgroup a
// row.  g = dout W2 (of the row's token), r = the saved activation relu(z);
// h = r or bf16(bf16(r r) k):
//   dw = <g, h>;  dz = w g [r > 0] or w g 2 k r;  and w h, W2's right operand
struct ActGradArgs {
    int64_t first, cols, pairs;     // first: a launch's first row
    int square;
    float k;
    const float* weights;
    const int32_t *order, *used;
    bf16 *g, *r;                // in: g, r; out: dz, w h
    float* dw;
};

template <bool WHOLE>
__global__ __launch_bounds__(256) void experts_act_grad_kernel(ActGradArgs a)
{
    __shared__ float s_dot[4];
    const int64_t row = a.first + blockIdx.x;
    const int pair = row < *a.used ? a.order[row] : -1;
    const bool there = pair >= 0 && pair < a.pairs;
    const float w = there ? a.weights[pair] : 0.f;
    float dot = 0.f;
    for (int64_t c = threadIdx.x * 8; c < a.cols; c += 2048) {
        const int nv = (int)min((int64_t)8, a.cols - c);
        const Raw<bf16> g = load_raw<WHOLE>(a.g + row * a.cols + c, nv), r = load_raw<WHOLE>(a.r + row * a.cols + c, nv);
        float dz[8], wh[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float x = raw_get(r, e), ge = raw_get(g, e);
            const float h = a.square ? bf16_to_f32(relu2_sq_bits(__float_as_uint(x) >> 16, a.k)) : x;
            // (select, not a product: a gradient of infinity where nothing came through is 0)
            dz[e] = !there || x == 0.f ? 0.f : a.square ? w * ge * (2.f * a.k * x) : w * ge;
            wh[e] = there ? w * h : 0.f;
            dot += h == 0.f ? 0.f : ge * h;
        }
        store_raw<WHOLE>(a.g + row * a.cols + c, to_raw<bf16>(dz), nv);
        store_raw<WHOLE>(a.r + row * a.cols + c, to_raw<bf16>(wh), nv);
    }
    if (a.dw == nullptr) return;
    dot = wave_sum_f32(dot);
    if ((threadIdx.x & 63) == 0) s_dot[threadIdx.x >> 6] = dot;
    __syncthreads();
    if (threadIdx.x == 0 && there) a.dw[pair] = (s_dot[0] + s_dot[1]) + (s_dot[2] + s_dot[3]);
}

static int combine_check(const char* what, int64_t tokens, int top_k, int64_t rows, int64_t cols)
{
    if (tokens < 0 || rows < 0 || cols < 0 || top_k < 1 || top_k > kMaxChoices || tokens >= (1ll << 31) - kTailBlocks || rows >= (1ll << 31) ||
        (cols && std::max(tokens, rows) >= (1ll << 40) / cols))
        return set_error(BS_ERR_INVALID, "%s: top_k must be in 1..%d, tokens and rows below 2^31, rows*cols below 2^40, got %lld, %d, %lld x %lld",
                         what, kMaxChoices, (long long)tokens, top_k, (long long)rows, (long long)cols);
    return BS_OK;
}

// (the plan's tokens, choices and rows, as the two calls without a plan have them)
static int combine_plan_check(const char* what, const bs_experts* x)
{
    if (x == nullptr) return set_error(BS_ERR_INVALID, "%s: null arguments", what);
    if (x->experts < 1 || x->experts > 1024) return set_error(BS_ERR_INVALID, "%s: experts must be in 1..1024, got %d", what, x->experts);
    if (x->offsets == nullptr || ((uintptr_t)x->offsets & 3u)) return set_error(BS_ERR_INVALID, "%s: null or misaligned offsets", what);
    return BS_OK;
}

static int combine(const char* what, const void* y, int y_type, int64_t y_stride, const float* weights, const int32_t* place, const int32_t* first,
                   const int32_t* used, int64_t tokens, int top_k, int64_t rows, int64_t cols, void* out, void* stream)
{
    if (const int rc = combine_check(what, tokens, top_k, rows, cols); rc != BS_OK) return rc;
    if (tokens == 0 || cols == 0) return BS_OK;
    if ((rows && y == nullptr) || place == nullptr || out == nullptr) return set_error(BS_ERR_INVALID, "%s: null pointer", what);
    if (y_type != BS_DT_BF16 && y_type != BS_DT_F32) return set_error(BS_ERR_INVALID, "%s: y dtype %d must be bf16 or fp32", what, y_type);
    if (y_stride < 0) return set_error(BS_ERR_INVALID, "%s: negative row stride", what);
    if (((uintptr_t)y & (y_type == BS_DT_F32 ? 3u : 1u)) || ((uintptr_t)out & 1u) || (((uintptr_t)weights | (uintptr_t)place) & 3u))
        return set_error(BS_ERR_INVALID, "%s: misaligned pointer", what);
    CombineArgs a{};
    a.rows = rows, a.cols = cols, a.top_k = top_k, a.y = y, a.y_stride = y_stride, a.first = first, a.used = used;
    const bool whole = cols % 8 == 0;
    auto* kernel = y_type == BS_DT_F32 ? (whole ? combine_kernel<float, true> : combine_kernel<float, false>)
                                       : (whole ? combine_kernel<bf16, true> : combine_kernel<bf16, false>);
    const uint32_t parts = (uint32_t)std::min<int64_t>((cols + 2047) / 2048, 65535);
    for (int64_t t = 0; t < tokens; t += kSlice) {
        a.tokens = std::min(kSlice, tokens - t);
        a.weights = weights ? weights + t * top_k : nullptr, a.place = place + t * top_k, a.out = static_cast<bf16*>(out) + t * cols;
        hipLaunchKernelGGL(kernel, dim3((uint32_t)a.tokens, parts), dim3(256), 0, (hipStream_t)stream, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
    }
    return BS_OK;
}

static int combine_backward(const char* what, const void* g, int64_t g_stride, const void* y, int64_t y_stride, const float* weights,
                            const int32_t* place, const int32_t* first, const int32_t* used, int64_t tokens, int top_k, int64_t rows, int64_t cols,
                            void* dy, float* dw, void* stream)
{
    if (const int rc = combine_check(what, tokens, top_k, rows, cols); rc != BS_OK) return rc;
    if ((dy == nullptr && dw == nullptr) || (tokens == 0 && rows == 0)) return BS_OK;
    if ((tokens && cols && g == nullptr) || (tokens && place == nullptr) || (dy && used == nullptr) || (dw && rows && cols && y == nullptr))
        return set_error(BS_ERR_INVALID, "%s: null pointer", what);
    if (g_stride < 0 || y_stride < 0) return set_error(BS_ERR_INVALID, "%s: negative row stride", what);
    if ((((uintptr_t)g | (uintptr_t)y | (uintptr_t)dy) & 1u) || (((uintptr_t)weights | (uintptr_t)place | (uintptr_t)used | (uintptr_t)dw) & 3u))
        return set_error(BS_ERR_INVALID, "%s: misaligned pointer", what);
    CombineArgs a{};
    a.rows = rows, a.cols = cols, a.top_k = top_k, a.y = y, a.y_stride = y_stride;
    a.first = first, a.used = used, a.g_stride = g_stride, a.dy = static_cast<bf16*>(dy);
    auto* kernel = dw ? (cols % 8 == 0 ? combine_backward_kernel<true> : combine_backward_kernel<false>)
                      : (cols % 8 == 0 ? spread_kernel<true> : spread_kernel<false>);
    // (no tokens: the rows of no expert alone)
    for (int64_t t = 0; t == 0 || t < tokens; t += kSlice) {
        a.tokens = std::min(kSlice, tokens - t);
        const int64_t blocks = a.tokens + (dy && t + kSlice >= tokens ? kTailBlocks : 0);
        if (blocks == 0) break;
        a.weights = weights ? weights + t * top_k : nullptr, a.place = place + t * top_k, a.g = static_cast<const bf16*>(g) + t * g_stride;
        a.dw = dw ? dw + t * top_k : nullptr;
        hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(256), 0, (hipStream_t)stream, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
    }
    return BS_OK;
}

}  // namespace bs

using namespace bs;

extern "C" int bs_expert_combine(const void* y, int y_type, int64_t y_stride, const float* weights, const int32_t* place, int64_t tokens, int top_k,
                                 int64_t rows, int64_t cols, void* out, void* stream)
{
    clear_error();
    return combine("bs_expert_combine", y, y_type, y_stride, weights, place, nullptr, nullptr, tokens, top_k, rows, cols, out, stream);
}

extern "C" int bs_expert_combine_plan(const bs_experts* experts, const void* y, int y_type, int64_t y_stride, const float* weights, const int32_t* place,
                                      int64_t cols, void* out, void* stream)
{
    clear_error();
    const char* what = "bs_expert_combine_plan";
    if (const int rc = combine_plan_check(what, experts); rc != BS_OK) return rc;
    return combine(what, y, y_type, y_stride, weights, place, experts->offsets, experts->offsets + experts->experts, experts->tokens, experts->top_k,
                   experts->rows, cols, out, stream);
}

extern "C" int bs_expert_combine_backward(const void* g, int64_t g_stride, const void* y, int64_t y_stride, const float* weights,
                                          const int32_t* place, const int32_t* used, int64_t tokens, int top_k, int64_t rows, int64_t cols,
                                          void* dy, float* dw, void* stream)
{
    clear_error();
    return combine_backward("bs_expert_combine_backward", g, g_stride, y, y_stride, weights, place, nullptr, used, tokens, top_k, rows, cols, dy, dw, stream);
}

extern "C" int bs_expert_combine_plan_backward(const bs_experts* experts, const void* g, int64_t g_stride, const void* y, int64_t y_stride,
                                               const float* weights, const int32_t* place, int64_t cols, void* dy, float* dw, void* stream)
{
    clear_error();
    const char* what = "bs_expert_combine_plan_backward";
    if (const int rc = combine_plan_check(what, experts); rc != BS_OK) return rc;
    return combine_backward(what, g, g_stride, y, y_stride, weights, place, experts->offsets, experts->offsets + experts->experts, experts->tokens,
                            experts->top_k, experts->rows, cols, dy, dw, stream);
}

extern "C" int bs_experts_act_grad(void* g, void* r, int64_t rows, int64_t cols, int square, float k, const float* weights,
                                   const int32_t* order, const int32_t* used, int64_t pairs, float* dw, void* stream)
{
    clear_error();
    const char* what = "bs_experts_act_grad";
    if (rows < 0 || cols < 0 || rows >= (1ll << 31) || (cols && rows >= (1ll << 40) / cols) || pairs < 0)
        return set_error(BS_ERR_INVALID, "%s: rows must be below 2^31 and rows*cols below 2^40, got %lld x %lld", what, (long long)rows, (long long)cols);
    if (rows == 0) return BS_OK;
    if ((cols && (g == nullptr || r == nullptr)) || weights == nullptr || order == nullptr || used == nullptr)
        return set_error(BS_ERR_INVALID, "%s: null pointer", what);
    if ((((uintptr_t)g | (uintptr_t)r) & 1u) || (((uintptr_t)weights | (uintptr_t)order | (uintptr_t)used | (uintptr_t)dw) & 3u))
        return set_error(BS_ERR_INVALID, "%s: misaligned pointer", what);
    ActGradArgs a{0, cols, pairs, square, k, weights, order, used, static_cast<bf16*>(g), static_cast<bf16*>(r), dw};
    auto* kernel = cols % 8 == 0 ? experts_act_grad_kernel<true> : experts_act_grad_kernel<false>;
    for (; a.first < rows; a.first += kSlice) {
        hipLaunchKernelGGL(kernel, dim3((uint32_t)std::min(kSlice, rows - a.first)), dim3(256), 0, (hipStream_t)stream, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
    }
    return BS_OK;
}
