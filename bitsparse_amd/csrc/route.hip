// Routing of tokens to experts, its gradient, and the order of the routed
// (token, choice) pairs by expert (bitsparse_amd/experts.py).
//
//   s = softmax(l) or 1 / (1 + exp(-l));  c = s + bias
//   the `top_groups` groups whose `group_best` largest c have the largest sum
//   the top_k largest c of those groups; w = scale s / sum(s) or scale s
//
// The choice is made between 64-bit values, as what lies next to each other in
// 32 bits would be ordered by its roundings; equal values go by index.  A wave
// a token, an expert a lane and a round.
//
//   dw -> ds = (scale / S) (dw - <dw, s> / S) or scale dw, 0 elsewhere
//   softmax: dl = s (ds - <ds, s>);  sigmoid: dl = s (1 - s) ds
#include <algorithm>

#include "bs_host.h"
#include "rownorm.h"

namespace bs {

constexpr int kMaxExperts = 1024, kMaxTopK = 64;

struct RouteArgs {
    int64_t tokens;
    int experts, top_k;
    const void* logits;
    int64_t stride;
    int f32;
    const float* bias;
    int sigmoid, groups, top_groups, group_best, renorm;
    float scale;
    float* weights;
    int32_t* chosen;
    // backward
    const float* d_weights;
    void* d_logits;
};

__device__ __forceinline__ float route_logit(const RouteArgs& a, int64_t row, int e)
{
    const int64_t i = row * a.stride + e;
    return a.f32 ? static_cast<const float*>(a.logits)[i] : (float)static_cast<const bf16*>(a.logits)[i];
}

// 64-bit values as integers in the same order; NaN above all, 0: none
__device__ __forceinline__ uint64_t order_key(double v)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    if (v != v) return ~0ull;
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double key_value(uint64_t k)
{
    return __builtin_bit_cast(double, k >> 63 ? k & ~(1ull << 63) : ~k);
}

struct Best {
    uint64_t key;
    int at;
};
__device__ __forceinline__ Best better(const Best& a, const Best& b)
{
    return b.key > a.key || (b.key == a.key && b.at < a.at) ? b : a;
}
// the best over the wave, in every lane
__device__ __forceinline__ Best wave_best(Best v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        Best o;
        o.key = (uint64_t)(uint32_t)__shfl_xor((int)(v.key >> 32), d) << 32 | (uint32_t)__shfl_xor((int)v.key, d);
        o.at = __shfl_xor(v.at, d);
        v = better(v, o);
    }
    return v;
}
__device__ __forceinline__ double wave_max_f64(double v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = fmax(v, __shfl_xor(v, d));
    return v;
}
__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// V: experts of a lane
template <int V>
__global__ __launch_bounds__(256) void route_forward_kernel(RouteArgs a)
{
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.tokens) return;
    double s[V];
    uint64_t key[V];
    double top = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = lane + 64 * i;
        s[i] = e < a.experts ? (double)route_logit(a, row, e) : -INFINITY;
        top = s[i] != s[i] ? s[i] : top != top ? top : fmax(top, s[i]);
    }
    bool there[V];
#pragma unroll
    for (int i = 0; i < V; i++) there[i] = lane + 64 * i < a.experts && s[i] != -INFINITY;
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < V; i++) s[i] = 1.0 / (1.0 + exp(-s[i]));
    } else {
        const bool nan = __any(top != top);
        top = wave_max_f64(nan ? 0.0 : top);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            s[i] = there[i] ? exp(s[i] - top) : 0.0;
            sum += s[i];
        }
        sum = wave_sum_f64(sum);
#pragma unroll
        for (int i = 0; i < V; i++) s[i] /= sum;
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = lane + 64 * i;
        double c = s[i];
        if (a.bias && e < a.experts) c += (double)a.bias[e];
        key[i] = there[i] && c != -INFINITY ? order_key(c) : 0;
    }
    if (a.top_groups < a.groups) {
        // group g's score to lane g
        const int size = a.experts / a.groups;
        Best mine = {0, lane};
        for (int g = 0; g < a.groups; g++) {
            Best first = {0, 1 << 30}, second = {0, 1 << 30};
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int e = lane + 64 * i;
                if (e / size == g && key[i]) first = better(first, Best{key[i], e});
            }
            first = wave_best(first);
            double score = first.key == ~0ull ? NAN : key_value(first.key);
            if (a.group_best == 2) {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const int e = lane + 64 * i;
                    if (e / size == g && key[i] && e != first.at) second = better(second, Best{key[i], e});
                }
                second = wave_best(second);
                if (second.key) score += second.key == ~0ull ? NAN : key_value(second.key);
            }
            if (lane == g) mine.key = first.key ? order_key(score) : 0;
        }
        uint64_t kept = 0;
        for (int j = 0; j < a.top_groups; j++) {
            const Best b = wave_best(mine);
            if (b.key) kept |= 1ull << b.at;
            if (lane == b.at) mine.key = 0;
        }
#pragma unroll
        for (int i = 0; i < V; i++)
            if (!(kept >> min(63, (lane + 64 * i) / size) & 1)) key[i] = 0;
    }
    double total = 0.0, own = 0.0;
    int chosen = -1;
    for (int j = 0; j < a.top_k; j++) {
        Best b = {0, 1 << 30};
#pragma unroll
        for (int i = 0; i < V; i++)
            if (key[i]) b = better(b, Best{key[i], lane + 64 * i});
        b = wave_best(b);
        double v = 0.0;
        if (b.key) {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (lane + 64 * i == b.at) {
                    key[i] = 0;
                    v = s[i];
                }
            v = __shfl(v, b.at & 63);
        }
        total += v;
        if (lane == j) {
            own = v;
            chosen = b.key ? b.at : -1;
        }
    }
    if (lane < a.top_k) {
        double w = own;
        if (a.renorm) w = total == 0.0 ? 0.0 : w / total;
        a.weights[row * a.top_k + lane] = (float)(w * (double)a.scale);
        a.chosen[row * a.top_k + lane] = chosen;
    }
}

template <int V>
__global__ __launch_bounds__(256) void route_backward_kernel(RouteArgs a)
{
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.tokens) return;
    float s[V], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = lane + 64 * i;
        s[i] = e < a.experts ? route_logit(a, row, e) : -INFINITY;
        top = fmaxf(top, s[i]);
    }
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < V; i++) s[i] = 1.f / (1.f + expf(-s[i]));
    } else {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < V; i++) {
            s[i] = s[i] == -INFINITY ? 0.f : expf(s[i] - top);
            sum += s[i];
        }
        sum = wave_sum_f32(sum);
#pragma unroll
        for (int i = 0; i < V; i++) s[i] = sum == 0.f ? 0.f : s[i] / sum;
    }
    // lane j: the j-th choice, its score and gradient
    int e = -1;
    float g = 0.f, sc = 0.f;
    if (lane < a.top_k) {
        e = a.chosen[row * a.top_k + lane];
        if (e >= a.experts) e = -1;
        g = e >= 0 ? a.d_weights[row * a.top_k + lane] * a.scale : 0.f;
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float v = __shfl(s[i], e & 63);
        if (e >> 6 == i) sc = v;
    }
    if (a.renorm) {
        const float total = wave_sum_f32(sc), dot = wave_sum_f32(g * sc);
        g = total == 0.f || e < 0 ? 0.f : (g - dot / total) / total;
    }
    const float dot = a.sigmoid ? 0.f : wave_sum_f32(g * sc);
    float ds[V];
#pragma unroll
    for (int i = 0; i < V; i++) ds[i] = 0.f;
    for (int j = 0; j < a.top_k; j++) {
        const int at = __shfl(e, j);
        const float v = __shfl(g, j);
#pragma unroll
        for (int i = 0; i < V; i++)
            if (at == lane + 64 * i) ds[i] += v;
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int x = lane + 64 * i;
        if (x >= a.experts) continue;
        const float d = a.sigmoid ? s[i] * (1.f - s[i]) * ds[i] : s[i] * (ds[i] - dot);
        param_store(a.d_logits, a.f32, row * a.experts + x, d);
    }
}

// ---------------------------------------------------------------------------
// The pairs by expert: a counting sort that keeps equal ones in order, without
// atomics.  A workgroup an expert, each reads all ids: once to count its own
// and those of lower experts, once to place its own; a wave has a run of them,
// so their order needs no more than the waves' counts.
// ---------------------------------------------------------------------------
struct PlanArgs {
    const int32_t* chosen;
    int32_t pairs;
    int experts;
    int32_t *offsets, *order, *place;
};

__global__ __launch_bounds__(1024) void expert_plan_kernel(PlanArgs a)
{
    __shared__ int s_own[16], s_lower[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int mine = (int)blockIdx.x;
    const int64_t run = (((int64_t)a.pairs + 15) / 16 + 63) / 64 * 64;
    const int64_t from = wave * run, to = min((int64_t)a.pairs, from + run);
    int own = 0, lower = 0;
    for (int64_t i = from + lane; i < to; i += 64) {
        const int e = a.chosen[i];
        own += e == mine;
        lower += e >= 0 && e < mine;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        own += __shfl_xor(own, d);
        lower += __shfl_xor(lower, d);
    }
    if (lane == 0) {
        s_own[wave] = own;
        s_lower[wave] = lower;
    }
    __syncthreads();
    int first = 0, before = 0, all = 0;
    for (int w = 0; w < 16; w++) {
        first += s_lower[w];
        before += w < wave ? s_own[w] : 0;
        all += s_own[w];
    }
    if (threadIdx.x == 0) a.offsets[mine] = first;
    if (mine == a.experts - 1) {
        if (threadIdx.x == 0) a.offsets[a.experts] = first + all;
        for (int64_t r = first + all + (int)threadIdx.x; r < a.pairs; r += 1024) a.order[r] = -1;
    }
    int row = first + before;
    for (int64_t i0 = from; i0 < to; i0 += 64) {
        const int64_t i = i0 + lane;
        const int e = i < to ? a.chosen[i] : -1;
        const uint64_t hit = __ballot(i < to && e == mine);
        if (i < to && e == mine) {
            const int r = row + (int)popc_below(hit);
            a.order[r] = (int)i;
            a.place[i] = r;
        } else if (i < to && mine == 0 && (e < 0 || e >= a.experts)) {
            a.place[i] = -1;
        }
        row += __popcll(hit);
    }
}

static int route_check(const bs_route* r, const char* what)
{
    if (r == nullptr) return set_error(BS_ERR_INVALID, "%s: null arguments", what);
    if (r->experts < 1 || r->experts > kMaxExperts) return set_error(BS_ERR_INVALID, "%s: experts must be in 1..%d, got %d", what, kMaxExperts, r->experts);
    if (r->top_k < 1 || r->top_k > std::min(kMaxTopK, r->experts))
        return set_error(BS_ERR_INVALID, "%s: top_k must be in 1..%d (at most experts), got %d", what, kMaxTopK, r->top_k);
    if (r->tokens < 0 || r->tokens * r->top_k >= (1ll << 31)) return set_error(BS_ERR_INVALID, "%s: tokens*top_k must be in 0..2^31-1", what);
    if (r->logits_type != BS_DT_BF16 && r->logits_type != BS_DT_F32) return set_error(BS_ERR_INVALID, "%s: logits dtype %d must be bf16 or fp32", what, r->logits_type);
    if (r->score != BS_SCORE_SOFTMAX && r->score != BS_SCORE_SIGMOID) return set_error(BS_ERR_INVALID, "%s: unknown score %d", what, r->score);
    if (r->groups < 1 || r->groups > 64 || r->experts % r->groups) return set_error(BS_ERR_INVALID, "%s: groups must be in 1..64 and divide experts, got %d", what, r->groups);
    if (r->top_groups < 1 || r->top_groups > r->groups) return set_error(BS_ERR_INVALID, "%s: top_groups must be in 1..groups, got %d", what, r->top_groups);
    if (r->group_best != 1 && r->group_best != 2) return set_error(BS_ERR_INVALID, "%s: group_best must be 1 or 2, got %d", what, r->group_best);
    if (r->top_k > r->top_groups * (r->experts / r->groups)) return set_error(BS_ERR_INVALID, "%s: top_k %d is more than %d groups hold", what, r->top_k, r->top_groups);
    if (r->logits_stride < 0) return set_error(BS_ERR_INVALID, "%s: negative row stride", what);
    if (r->tokens && r->logits == nullptr) return set_error(BS_ERR_INVALID, "%s: null logits", what);
    if ((uintptr_t)r->logits & (r->logits_type == BS_DT_F32 ? 3u : 1u)) return set_error(BS_ERR_INVALID, "%s: logits misaligned for their type", what);
    if ((uintptr_t)r->bias & 3u) return set_error(BS_ERR_INVALID, "%s: bias misaligned", what);
    return BS_OK;
}

static RouteArgs route_args(const bs_route& r)
{
    RouteArgs a{};
    a.tokens = r.tokens, a.experts = r.experts, a.top_k = r.top_k, a.logits = r.logits, a.stride = r.logits_stride;
    a.f32 = r.logits_type == BS_DT_F32, a.bias = r.bias, a.sigmoid = r.score == BS_SCORE_SIGMOID, a.groups = r.groups;
    a.top_groups = r.top_groups, a.group_best = r.group_best, a.renorm = r.renormalize, a.scale = r.scale;
    return a;
}

}  // namespace bs

using namespace bs;

extern "C" int bs_route_forward(const bs_route* route, float* weights, int32_t* chosen, void* stream)
{
    clear_error();
    const char* what = "bs_route_forward";
    if (const int rc = route_check(route, what); rc != BS_OK) return rc;
    if (route->tokens == 0) return BS_OK;
    if (weights == nullptr || chosen == nullptr || (((uintptr_t)weights | (uintptr_t)chosen) & 3u))
        return set_error(BS_ERR_INVALID, "%s: null or misaligned result", what);
    RouteArgs a = route_args(*route);
    a.weights = weights, a.chosen = chosen;
    const int v = (a.experts + 63) / 64;
    auto* kernel = v <= 1 ? route_forward_kernel<1> : v <= 2 ? route_forward_kernel<2> : v <= 4 ? route_forward_kernel<4>
                   : v <= 8 ? route_forward_kernel<8> : route_forward_kernel<16>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)((a.tokens + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? BS_OK : set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}

extern "C" int bs_route_backward(const bs_route* route, const int32_t* chosen, const float* d_weights, void* d_logits, void* stream)
{
    clear_error();
    const char* what = "bs_route_backward";
    if (const int rc = route_check(route, what); rc != BS_OK) return rc;
    if (route->tokens == 0) return BS_OK;
    if (chosen == nullptr || d_weights == nullptr || d_logits == nullptr || (((uintptr_t)chosen | (uintptr_t)d_weights) & 3u) ||
        ((uintptr_t)d_logits & (route->logits_type == BS_DT_F32 ? 3u : 1u)))
        return set_error(BS_ERR_INVALID, "%s: null or misaligned operand", what);
    RouteArgs a = route_args(*route);
    a.chosen = const_cast<int32_t*>(chosen), a.d_weights = d_weights, a.d_logits = d_logits;
    const int v = (a.experts + 63) / 64;
    auto* kernel = v <= 1 ? route_backward_kernel<1> : v <= 2 ? route_backward_kernel<2> : v <= 4 ? route_backward_kernel<4>
                   : v <= 8 ? route_backward_kernel<8> : route_backward_kernel<16>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)((a.tokens + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? BS_OK : set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}

extern "C" int bs_expert_plan(const int32_t* chosen, int64_t pairs, int experts, int32_t* offsets, int32_t* order, int32_t* place,
                              void* stream)
{
    clear_error();
    const char* what = "bs_expert_plan";
    if (experts < 1 || experts > kMaxExperts) return set_error(BS_ERR_INVALID, "%s: experts must be in 1..%d, got %d", what, kMaxExperts, experts);
    if (pairs < 0 || pairs >= (1ll << 31)) return set_error(BS_ERR_INVALID, "%s: pairs must be in 0..2^31-1", what);
    if (offsets == nullptr || (pairs && (chosen == nullptr || order == nullptr || place == nullptr)))
        return set_error(BS_ERR_INVALID, "%s: null pointer", what);
    if (((uintptr_t)chosen | (uintptr_t)offsets | (uintptr_t)order | (uintptr_t)place) & 3u) return set_error(BS_ERR_INVALID, "%s: misaligned pointer", what);
    const PlanArgs a{chosen, (int32_t)pairs, experts, offsets, order, place};
    hipLaunchKernelGGL(expert_plan_kernel, dim3((uint32_t)experts), dim3(1024), 0, (hipStream_t)stream, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? BS_OK : set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}
