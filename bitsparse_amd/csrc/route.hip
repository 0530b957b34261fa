// Routing of tokens to experts, its gradient, and the order of the routed
// (token, choice) pairs by expert (bitsparse_amd/experts.py).
//
//   s = softmax(l) or 1 / (1 + exp(-l));  c = s + bias
//   the `top_groups` groups whose `group_best` largest c have the largest sum
//   the top_k largest c of those groups; w = scale s / sum(s) or scale s
//
// The choice is made between 64-bit values, as what lies next to each other in
// 32 bits would be ordered by its roundings; equal values go by index.  Where
// c has the order of the logits it is between those.
//
// Bound by the choice's own instructions, some 1300 a wave of four tokens with
// 256 experts: 32768 tokens, 8 of 256 experts in 4 of 8 groups, sigmoid and
// bias: forward 33 us, backward 23 us (67 MB: 14 us at a copy's rate); 8192 tokens, 2
// of 8: 4.0 and 3.6 us; one token of 64 experts 4.2 us, latency.
//
//   dw -> ds = (scale / S) (dw - <dw, s> / S) or scale dw, 0 elsewhere
//   softmax: dl = s (ds - <ds, s>);  sigmoid: dl = s (1 - s) ds
#include <algorithm>
#include <type_traits>

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
    int by_logit;               // the order of c is that of the logits
    float scale;
    float* weights;
    int32_t* chosen;
    // backward
    const float* d_weights;
    void* d_logits;
};

// L lanes have a token, 64 / L tokens a wave; lane l of them has the V experts
// from V l on.
template <int L>
struct Lanes {
    // x of the lane 1, 2, 4 (mirrored in 8), 8 (mirrored in 16), 16, 32 away: enough for what is the same on both sides so far
    template <int D>
    static __device__ __forceinline__ uint32_t other(uint32_t x)
    {
        if constexpr (D == 1) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true);
        if constexpr (D == 2) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true);
        if constexpr (D == 4) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xf, 0xf, true);
        if constexpr (D == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xf, 0xf, true);
        if constexpr (D >= 16) return (uint32_t)__shfl_xor((int)x, D);
    }
    template <int D>
    static __device__ __forceinline__ float other(float x) { return __uint_as_float(other<D>(__float_as_uint(x))); }
    template <int D>
    static __device__ __forceinline__ double other(double x)
    {
        const uint64_t b = __builtin_bit_cast(uint64_t, x);
        return __builtin_bit_cast(double, (uint64_t)other<D>((uint32_t)(b >> 32)) << 32 | other<D>((uint32_t)b));
    }
    // v joined over the token's lanes, the same in all of them
    template <int D = 1, typename T, typename F>
    static __device__ __forceinline__ T all(T v, F&& join)
    {
        if constexpr (D < L) {
            v = join(v, other<D>(v));
            return all<2 * D>(v, join);
        }
        return v;
    }
};

// V logits of a row from its element e0 on, -infinity behind its end
template <int V, typename T>
__device__ __forceinline__ void load_logits(const T* row, int e0, int experts, float (&v)[V])
{
    if constexpr (V % 8 == 0) {
#pragma unroll
        for (int c = 0; c < V; c += 8) {
            const int nv = max(0, min(8, experts - e0 - c));
            const Raw<T> r = load_raw(row + e0 + c, nv);
#pragma unroll
            for (int i = 0; i < 8; i++) v[c + i] = i < nv ? raw_get(r, i) : -INFINITY;
        }
    } else if (V == 4 && e0 + 4 <= experts) {
        uint32_t w[sizeof(T)];
        __builtin_memcpy(w, row + e0, sizeof(w));
#pragma unroll
        for (int i = 0; i < V; i++)
            v[i] = sizeof(T) == 4 ? __uint_as_float(w[i % (int)sizeof(T)]) : __uint_as_float(i & 1 ? w[i / 2 % (int)sizeof(T)] & 0xffff0000u : w[i / 2 % (int)sizeof(T)] << 16);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = e0 + i < experts ? (float)row[e0 + i] : -INFINITY;
    }
}
template <int V>
__device__ __forceinline__ void load_logits(const RouteArgs& a, int64_t row, int e0, float (&v)[V])
{
    if (a.f32)
        load_logits(static_cast<const float*>(a.logits) + row * a.stride, e0, a.experts, v);
    else
        load_logits(static_cast<const bf16*>(a.logits) + row * a.stride, e0, a.experts, v);
}

// LDS written by some lanes of a wave and read by others of it
__device__ __forceinline__ void wave_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The groups that stay, a bit each, from their scores in LDS: fewer than
// top_groups come before each.  worst: the least score that stays, next: the
// largest that does not (over the lane's groups).
template <int L, typename T>
__device__ __forceinline__ uint64_t route_groups(const RouteArgs& a, const T* s_score, int l, T& worst, T& next)
{
    uint32_t low = 0, high = 0;
    worst = INFINITY, next = -INFINITY;
    for (int g = l; g < a.groups; g += L) {
        const T mine = s_score[g];
        int before = 0;
        for (int h = 0; h < a.groups; h++) {
            const T v = s_score[h];
            before += v > mine || (v == mine && h < g);
        }
        if (before < a.top_groups && mine != (T)-INFINITY) {
            (g < 32 ? low : high) |= 1u << (g & 31);
            worst = mine < worst ? mine : worst;
        } else {
            next = mine > next ? mine : next;
        }
    }
    const auto either = [](uint32_t x, uint32_t y) { return x | y; };
    return (uint64_t)Lanes<L>::all(high, either) << 32 | Lanes<L>::all(low, either);
}
// whether expert e's group stays
__device__ __forceinline__ bool group_kept(uint64_t kept, int e, uint32_t part)
{
    return kept >> ((uint32_t)e * part >> 22 & 63) & 1;     // part: 2^22 / size rounded up, e / size = e part >> 22 for e, size <= 1024
}

// The choice between 64-bit values c, -infinity where there is no expert (any
// more): choice j in lane j % L's place j / L.
template <int L, int V, int SLOTS>
__device__ __forceinline__ void route_exact(const RouteArgs& a, double (&c)[V], int lane, double* s_score, int (&id)[SLOTS])
{
    typedef double T;
    typedef Lanes<L> Ln;
    constexpr T kNone = -INFINITY;
    const int l = lane % L, sub = lane / L, e0 = l * V;
    const auto larger = [](T x, T y) { return x > y ? x : y; };
    if (a.top_groups < a.groups) {
        const int size = a.experts / a.groups;
        // the best and the second best
        struct Pair {
            T x, y;
        };
        auto add = [](Pair p, T v) {
            const bool more = v > p.x;
            return Pair{more ? v : p.x, more ? p.x : v > p.y ? v : p.y};
        };
        auto score = [&](Pair p) { return a.group_best == 1 || p.y == kNone ? p.x : p.x + p.y; };
        const int span = size / V;          // lanes of a group, where it has whole lanes
        if (span * V == size && (span & (span - 1)) == 0 && span <= 16) {
            Pair p = {kNone, kNone};
#pragma unroll
            for (int i = 0; i < V; i++) p = add(p, c[i]);
            auto meet = [&](auto d) {
                constexpr int D = decltype(d)::value;
                if (span > D) p = add(add(p, Ln::template other<D>(p.x)), Ln::template other<D>(p.y));
            };
            meet(std::integral_constant<int, 1>{});
            meet(std::integral_constant<int, 2>{});
            meet(std::integral_constant<int, 4>{});
            meet(std::integral_constant<int, 8>{});
            if (l % span == 0 && l / span < a.groups) s_score[l / span] = score(p);
        } else {
            for (int g = 0; g < a.groups; g++) {
                Pair p = {kNone, kNone};
#pragma unroll
                for (int i = 0; i < V; i++) p = add(p, e0 + i >= g * size && e0 + i < (g + 1) * size ? c[i] : kNone);
                const T best = Ln::all(p.x, larger);
                // (one lane gives its best up, the first of those that have it)
                const uint64_t have = __ballot(p.x == best) >> (sub * L) & (L == 64 ? ~0ull : (1ull << (L & 63)) - 1);
                const bool first = l == __builtin_ctzll(have);
                const T second = Ln::all(first ? p.y : p.x, larger);
                if (l == 0) s_score[g] = score(Pair{best, second});
            }
        }
        wave_fence();
        T worst, next;
        const uint64_t kept = route_groups<L>(a, s_score, l, worst, next);
        wave_fence();
        const uint32_t part = ((1u << 22) + size - 1) / size;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (!group_kept(kept, e0 + i, part)) c[i] = kNone;
    }
#pragma unroll
    for (int s = 0; s < SLOTS; s++) {
        id[s] = -1;
        for (int j = 0; j < L && s * L + j < a.top_k; j++) {
            T best = c[0];
#pragma unroll
            for (int i = 1; i < V; i++) best = larger(best, c[i]);
            uint32_t at = ~0u;
#pragma unroll
            for (int i = V - 1; i >= 0; i--) at = c[i] == best ? e0 + i : at;
            const T most = Ln::all(best, larger);
            at = Ln::all(best == most ? at : ~0u, [](uint32_t x, uint32_t y) { return min(x, y); });
#pragma unroll
            for (int i = 0; i < V; i++) c[i] = at == (uint32_t)(e0 + i) ? kNone : c[i];
            if (l == j) id[s] = most == kNone ? -1 : (int)at;
        }
    }
}

// The same between 32-bit values, none of them -0, cut to 28 bits, the place in the lane in the
// other four: their order as integers (0: none) is that of the values, and among equal ones
// that of the places.  A lane's are sorted once, so that a choice is the largest of the lanes' first
// ones.  True where what decides lies closer together than `near` and the cut (of values up to `size`):
// the choice is then not sure.
__device__ __forceinline__ uint32_t place_key(float v, int place)
{
    const uint32_t b = __float_as_uint(v);
    return v == -INFINITY ? 0u : ((b >> 31 ? ~b : b | 1u << 31) & ~15u) | (uint32_t)(15 - place);
}
__device__ __forceinline__ float key_value(uint32_t k)
{
    k &= ~15u;
    return k == 0 ? -INFINITY : __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}

template <int L, int V, int SLOTS>
__device__ __forceinline__ bool route_fast(const RouteArgs& a, const float (&c)[V], int lane, float* s_score, float near, float size, int (&id)[SLOTS])
{
    static_assert(V <= 16, "four bits of place");
    typedef Lanes<L> Ln;
    const int l = lane % L, e0 = l * V;
    const auto larger = [](uint32_t x, uint32_t y) { return max(x, y); };
    const auto apart = [&](float x, float y, float times) { return near < 0.f || x - y > times * (near + 0x1p-18f * fabsf(x)); };
    uint32_t k[V];
#pragma unroll
    for (int i = 0; i < V; i++) k[i] = place_key(c[i], i);
    bool unsure = false;
    if (a.top_groups < a.groups) {
        const int experts = a.experts / a.groups, span = experts / V;
        // (no whole lanes, or no power of two of them: every token in 64 bits; 32768 tokens of 160 experts in 8 groups 72 us, 96 in
        // 8 42, of 128 in 8 on this path 22)
        if (span * V != experts || (span & (span - 1)) != 0 || span > 16) return true;
        uint32_t x = 0, y = 0;          // the best and the second best
        auto add = [&](uint32_t v) {
            y = max(y, min(x, v));
            x = max(x, v);
        };
#pragma unroll
        for (int i = 0; i < V; i++) add(k[i]);
        auto meet = [&](auto d) {
            constexpr int D = decltype(d)::value;
            if (span > D) {
                const uint32_t ox = Ln::template other<D>(x), oy = Ln::template other<D>(y);
                add(ox);
                add(oy);
            }
        };
        meet(std::integral_constant<int, 1>{});
        meet(std::integral_constant<int, 2>{});
        meet(std::integral_constant<int, 4>{});
        meet(std::integral_constant<int, 8>{});
        const float vx = key_value(x), vy = key_value(y);
        if (l % span == 0 && l / span < a.groups) s_score[l / span] = a.group_best == 1 || y == 0 ? vx : vx + vy;
        wave_fence();
        float worst, next;
        const uint64_t kept = route_groups<L>(a, s_score, l, worst, next);
        wave_fence();
        worst = Ln::all(worst, [](float p, float q) { return p < q ? p : q; });
        next = Ln::all(next, [](float p, float q) { return p > q ? p : q; });
        // (a sum of two that cancel is cut as they are)
        unsure = next != -INFINITY && !(near < 0.f || worst - next > 4.f * near + 0x1p-17f * fmaxf(size, fabsf(worst)));
        const bool mine = kept >> (l / span & 63) & 1;
#pragma unroll
        for (int i = 0; i < V; i++) k[i] = mine ? k[i] : 0u;
    }
    // (merging networks of pairs, fours, ...: the largest first)
#pragma unroll
    for (int p = 1; p < V; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < V; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; i++)
                    if (i + j + q < V && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const uint32_t hi = max(k[i + j], k[i + j + q]), lo = min(k[i + j], k[i + j + q]);
                        k[i + j] = hi, k[i + j + q] = lo;
                    }
    float last = 0.f;
#pragma unroll
    for (int s = 0; s < SLOTS; s++) {
        id[s] = -1;
        for (int j = 0; j < L && s * L + j < a.top_k; j++) {
            // (of the lanes with the largest value the lowest index)
            const uint32_t most = Ln::all(k[0] & ~15u, larger);
            const uint32_t at = Ln::all((k[0] & ~15u) == most ? (uint32_t)e0 + 15 - (k[0] & 15) : ~0u, [](uint32_t x, uint32_t y) { return min(x, y); });
            const float value = key_value(most);
            if (s + j > 0) unsure |= most != 0 && !apart(last, value, 1.f);
            last = value;
            if (l == j) id[s] = most == 0 ? -1 : (int)at;
            const bool mine = at - (uint32_t)e0 < (uint32_t)V;
#pragma unroll
            for (int i = 0; i < V; i++) k[i] = mine ? (i + 1 < V ? k[i + 1 < V ? i + 1 : i] : 0u) : k[i];
        }
    }
    const uint32_t left = Ln::all(k[0] & ~15u, larger);         // the first that is left out
    return unsure || (left != 0 && !apart(last, key_value(left), 1.f));
}

// First the fast choice, then where it is not sure the exact one (32768 tokens,
// 8 of 256 experts in 4 of 8 groups, by sigmoid and bias: 47 us if all were exact).
template <int L, int V>
__global__ __launch_bounds__(256) void route_forward_kernel(RouteArgs a)
{
    constexpr int TOKENS = 64 / L, SLOTS = (kMaxTopK + L - 1) / L;
    __shared__ double s_score[4][TOKENS][64];
    typedef Lanes<L> Ln;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % L, sub = lane / L;
    const int64_t token = ((int64_t)blockIdx.x * 4 + wave) * TOKENS + sub, row = min(token, a.tokens - 1);
    const auto sum_of = [](auto x, auto y) { return x + y; };
    const int e0 = l * V;
    float lg[V], bias[V];
    load_logits(a, row, e0, lg);
    if (a.bias)
        load_logits(a.bias, e0, a.experts, bias);
    else
#pragma unroll
        for (int i = 0; i < V; i++) bias[i] = 0.f;

    // softmax: the largest logit and the sum of exponentials over it (a NaN makes the sum NaN)
    float top = -INFINITY, sum = 0.f, c[V];
    if (!a.sigmoid) {
#pragma unroll
        for (int i = 0; i < V; i++) top = fmaxf(top, lg[i]);
        top = Ln::all(top, [](float x, float y) { return fmaxf(x, y); });
#pragma unroll
        for (int i = 0; i < V; i++) {
            c[i] = lg[i] == -INFINITY ? 0.f : expf(lg[i] - top);
            sum += c[i];
        }
        sum = Ln::all(sum, sum_of);
        const float part = 1.f / sum;
#pragma unroll
        for (int i = 0; i < V; i++) c[i] *= part;
    } else if (!a.by_logit) {
        // (the instructions' own precision, 2^-23: l's product with log2(e) is off by |l| 2^-24, s by a quarter of e^-|l| of that)
#pragma unroll
        for (int i = 0; i < V; i++) c[i] = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * lg[i]));
    }
    float most_bias = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++) {
        // (a logit of -0 becomes +0: they are equal, their bits are not; a score is never -0)
        c[i] = a.by_logit ? lg[i] + 0.f : lg[i] == -INFINITY ? -INFINITY : c[i] + bias[i];
        c[i] = c[i] != c[i] ? INFINITY : c[i];
        most_bias = fmaxf(most_bias, bias[i] == -INFINITY ? 0.f : fabsf(bias[i]));
    }
    // What two scores together may be off by: a sigmoid's, at most 1, six roundings of 2^-24, a softmax's, at most 1 / sum, as
    // many and those of a sum over lanes and their experts, 22 more; the biased one's another of both.  A bf16 logit is its key.
    float near = -1.f, size = 0.f;
    if (!a.by_logit) {
        most_bias = Ln::all(most_bias, [](float x, float y) { return fmaxf(x, y); });
        near = (a.sigmoid ? 0x1p-20f : 0x1p-18f / sum) + 0x1p-22f * most_bias;
        size = (a.sigmoid ? 1.f : 1.f / sum) + most_bias;
    } else if (a.f32) {
        near = 0.f;
    }
    int id[SLOTS];
    if (__any(route_fast<L, V>(a, c, lane, reinterpret_cast<float*>(s_score[wave][sub]), near, size, id))) {
        double d[V];
        if (a.by_logit) {
#pragma unroll
            for (int i = 0; i < V; i++) d[i] = c[i];
        } else if (a.sigmoid) {
#pragma unroll
            for (int i = 0; i < V; i++) d[i] = 1.0 / (1.0 + exp(-(double)lg[i]));
        } else {
            double total = 0.0;
#pragma unroll
            for (int i = 0; i < V; i++) {
                d[i] = lg[i] == -INFINITY ? 0.0 : exp((double)lg[i] - (double)top);
                total += d[i];
            }
            total = Ln::all(total, sum_of);
#pragma unroll
            for (int i = 0; i < V; i++) d[i] /= total;
        }
#pragma unroll
        for (int i = 0; i < V; i++) {
            if (!a.by_logit) d[i] = lg[i] == -INFINITY ? -INFINITY : d[i] + (double)bias[i];
            d[i] = d[i] != d[i] ? (double)INFINITY : d[i];
        }
        wave_fence();
        route_exact<L, V>(a, d, lane, s_score[wave][sub], id);
    }
    float w[SLOTS], total = 0.f;
#pragma unroll
    for (int s = 0; s < SLOTS; s++) {
        w[s] = 0.f;
        if (s * L >= a.top_k) continue;
        // the logit again; the difference's rounding, which the exponential turns into as much of its value, is put back (of none
        // where it is 0: the difference may be past fp32's range)
        const int64_t at = row * a.stride + max(0, id[s]);
        const float of = a.f32 ? static_cast<const float*>(a.logits)[at] : (float)static_cast<const bf16*>(a.logits)[at];
        const float d = of - top, back = d - of, lost = (of - (d - back)) - (top + back), e = expf(a.sigmoid ? -of : d);
        w[s] = id[s] < 0 ? 0.f : a.sigmoid ? 1.f / (1.f + e) : fmaf(e, e == 0.f ? 0.f : lost, e) / sum;
        total += w[s];
    }
    if (a.renorm) total = Ln::all(total, sum_of);
#pragma unroll
    for (int s = 0; s < SLOTS; s++) {
        const int j = s * L + l;
        if (j >= a.top_k || token >= a.tokens) continue;
        a.weights[token * a.top_k + j] = a.scale * (!a.renorm ? w[s] : total == 0.f ? 0.f : w[s] / total);
        a.chosen[token * a.top_k + j] = id[s];
    }
}

template <int L, int V>
__global__ __launch_bounds__(256) void route_backward_kernel(RouteArgs a)
{
    constexpr int TOKENS = 64 / L, SLOTS = (kMaxTopK + L - 1) / L;
    typedef Lanes<L> Ln;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % L, sub = lane / L;
    const int64_t token = ((int64_t)blockIdx.x * 4 + wave) * TOKENS + sub, row = min(token, a.tokens - 1);
    const auto sum_of = [](float x, float y) { return x + y; };
    const int e0 = l * V;
    float s[V];
    load_logits(a, row, e0, s);
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < V; i++) s[i] = __builtin_amdgcn_rcpf(1.f + expf(-s[i]));      // (within a unit of the last place)
    } else {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < V; i++) top = fmaxf(top, s[i]);
        top = Ln::all(top, [](float x, float y) { return fmaxf(x, y); });
#pragma unroll
        for (int i = 0; i < V; i++) {
            s[i] = s[i] == -INFINITY ? 0.f : expf(s[i] - top);
            sum += s[i];
        }
        sum = Ln::all(sum, sum_of);
        const float part = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int i = 0; i < V; i++) s[i] *= part;
    }
    // lane l has the choices l, l + L, ...: experts, scores, gradients
    int e[SLOTS];
    float g[SLOTS], sc[SLOTS], total = 0.f, dot = 0.f;
#pragma unroll
    for (int t = 0; t < SLOTS; t++) {
        const int j = t * L + l;
        e[t] = j < a.top_k ? a.chosen[row * a.top_k + j] : -1;
        if (e[t] >= a.experts) e[t] = -1;
        g[t] = e[t] >= 0 ? a.d_weights[row * a.top_k + j] * a.scale : 0.f;
        sc[t] = 0.f;
        if (t * L < a.top_k) {
            const int from = (sub * L + max(0, e[t]) / V) & 63;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float v = __shfl(s[i], from);
                if (e[t] >= 0 && e[t] % V == i) sc[t] = v;
            }
        }
        total += sc[t];
        dot += e[t] >= 0 ? g[t] * sc[t] : 0.f;
    }
    dot = Ln::all(dot, sum_of);
    if (a.renorm) {
        total = Ln::all(total, sum_of);
        const float part = total == 0.f ? 0.f : 1.f / total, mean = dot * part;
#pragma unroll
        for (int t = 0; t < SLOTS; t++) g[t] = e[t] < 0 ? 0.f : (g[t] - mean) * part;
        dot = 0.f;              // of the renormalised weights' gradient with s
    }
    float ds[V];
#pragma unroll
    for (int i = 0; i < V; i++) ds[i] = 0.f;
#pragma unroll
    for (int t = 0; t < SLOTS; t++)
        for (int j = 0; j < L && t * L + j < a.top_k; j++) {
            const int at = __shfl(e[t], sub * L + j);
            const float v = __shfl(g[t], sub * L + j);
#pragma unroll
            for (int i = 0; i < V; i++) ds[i] += at == e0 + i ? v : 0.f;
        }
    if (token >= a.tokens) return;
    float d[V];
#pragma unroll
    for (int i = 0; i < V; i++) d[i] = a.sigmoid ? s[i] * (1.f - s[i]) * ds[i] : s[i] * (ds[i] - dot);
    const int64_t at = token * a.experts + e0;
    if constexpr (V % 8 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 8) {
            float o[8];
#pragma unroll
            for (int k = 0; k < 8; k++) o[k] = d[i + k];
            const int nv = max(0, min(8, a.experts - e0 - i));
            if (a.f32)
                store_raw(static_cast<float*>(a.d_logits) + at + i, to_raw<float>(o), nv);
            else
                store_raw(static_cast<bf16*>(a.d_logits) + at + i, to_raw<bf16>(o), nv);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (e0 + i < a.experts) param_store(a.d_logits, a.f32, at + i, d[i]);
    }
}

// ---------------------------------------------------------------------------
// The pairs by expert: a counting sort that keeps equal ones in order, without
// atomics.  A block of pairs is a run of each of 16 waves; a wave counts 64 of
// them at a time, the lanes with the same expert told by a ballot for each bit of it.
// One block does it all by itself; of more, each writes its counts and a
// second kernel adds those of the blocks before it.  Bound by latency, and by a
// wave's run past some 65536 pairs: 262144 pairs, 256 experts 5.8 + 11.0 us, 1048576 in all 49, 16384 pairs of 8 3.4 + 5.6, 8 pairs of 64 3.6
// (a workgroup an expert, each reading all ids: 150, 13 and 3.9).
// ---------------------------------------------------------------------------
constexpr int kPlanBlock = 1024;        // pairs of a block, at least, where there are several
constexpr int kPlanBlocks = 64;         // most blocks
constexpr int kPlanAhead = 4;           // loads of a wave at a time

struct PlanArgs {
    const int32_t* chosen;
    int64_t pairs, run;         // run: pairs of a wave, a multiple of 64
    int experts, bits, blocks;
    int32_t *offsets, *order, *place;
    int32_t* counts;            // [blocks, experts], of several blocks
};

// the lanes whose expert is this lane's
__device__ __forceinline__ uint64_t same_expert(uint32_t e, int bits)
{
    uint64_t same = ~0ull;
    for (int b = 0; b < bits; b++) {
        const bool one = e >> b & 1;
        const uint64_t ones = __ballot(one);
        same &= one ? ones : ~ones;
    }
    return same;
}

// COUNT: the first of two kernels
template <bool COUNT>
__global__ __launch_bounds__(1024) void expert_plan_kernel(PlanArgs a)
{
    extern __shared__ int s_mem[];
    int* const s_count = s_mem;                         // [16][experts]
    int* const s_total = s_mem + 16 * a.experts;        // [experts]
    __shared__ int s_wave[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), E = a.experts;
    for (int i = tid; i < 16 * E; i += 1024) s_count[i] = 0;
    __syncthreads();
    const int64_t from = ((int64_t)blockIdx.x * 16 + wave) * a.run, to = min(a.pairs, from + a.run);
    int* const mine = s_count + wave * E;
    // f(pair, its expert, or E for all that are none of the experts')
    auto each = [&](auto f) {
        for (int64_t i0 = from; i0 < to; i0 += 64 * kPlanAhead) {
            uint32_t e[kPlanAhead];
#pragma unroll
            for (int u = 0; u < kPlanAhead; u++) {
                const int64_t i = i0 + 64 * u + lane;
                e[u] = i < to ? (uint32_t)a.chosen[i] : ~0u;
            }
#pragma unroll
            for (int u = 0; u < kPlanAhead; u++)
                if (i0 + 64 * u < to) f(i0 + 64 * u + lane, min(e[u], (uint32_t)E));
        }
    };
    each([&](int64_t, uint32_t e) {
        const uint64_t same = same_expert(e, a.bits);
        if (e < (uint32_t)E && popc_below(same) == 0) mine[e] += __popcll(same);
        wave_fence();
    });
    __syncthreads();
    // each wave's counts become the rows of the waves before it
    for (int e = tid; e < E; e += 1024) {
        int sum = 0;
        for (int w = 0; w < 16; w++) {
            const int n = s_count[w * E + e];
            s_count[w * E + e] = sum;
            sum += n;
        }
        if (COUNT)
            a.counts[(int64_t)blockIdx.x * E + e] = sum;
        else
            s_total[e] = sum;
    }
    if (COUNT) return;
    __syncthreads();
    // the experts' first rows
    int all = 0, before = 0;            // of expert `tid`, in all blocks and in those before this one
    if (a.blocks > 1) {
        // (as many threads to an expert as there are; sums of whole numbers, in any order)
        int* const s_all = s_mem + 17 * E;
        for (int i = tid; i < E; i += 1024) s_total[i] = s_all[i] = 0;
        __syncthreads();
        const int parts = min(1024 / E, a.blocks), part = tid / E, e = tid - part * E;
        if (part < parts) {
            int n_all = 0, n_before = 0;
#pragma unroll 8
            for (int b = part; b < a.blocks; b += parts) {
                const int n = a.counts[(int64_t)b * E + e];
                n_all += n;
                n_before += b < (int)blockIdx.x ? n : 0;
            }
            atomicAdd(&s_all[e], n_all);
            atomicAdd(&s_total[e], n_before);
        }
        __syncthreads();
        if (tid < E) all = s_all[tid], before = s_total[tid];
        __syncthreads();
    } else if (tid < E) {
        all = s_total[tid];
    }
    int sum = all;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(sum, d);
        sum += lane >= d ? o : 0;
    }
    if (lane == 63) s_wave[wave] = sum;
    __syncthreads();
    int used = 0;
    for (int w = 0; w < 16; w++) {
        const int n = s_wave[w];
        sum += w < wave ? n : 0;
        used += n;
    }
    if (tid < E) {
        s_total[tid] = sum - all + before;
        if (blockIdx.x == 0) a.offsets[tid] = sum - all;
    }
    if (blockIdx.x == 0 && tid == 0) a.offsets[E] = used;
    for (int64_t r = used + (int64_t)blockIdx.x * 1024 + tid; r < a.pairs; r += (int64_t)a.blocks * 1024) a.order[r] = -1;
    __syncthreads();
    each([&](int64_t i, uint32_t e) {
        const uint64_t same = same_expert(e, a.bits);
        int r = -1;
        if (e < (uint32_t)E) {
            const int rank = (int)popc_below(same);
            r = s_total[e] + mine[e] + rank;
            wave_fence();
            if (rank == 0) mine[e] += __popcll(same);
            a.order[r] = (int)i;
        }
        wave_fence();
        if (i < to) a.place[i] = r;
    });
}

static int route_check(const bs_route* r, const char* what)
{
    if (r == nullptr) return set_error(BS_ERR_INVALID, "%s: null arguments", what);
    if (r->experts < 1 || r->experts > kMaxExperts) return set_error(BS_ERR_INVALID, "%s: experts must be in 1..%d, got %d", what, kMaxExperts, r->experts);
    if (r->top_k < 1 || r->top_k > std::min(kMaxTopK, r->experts))
        return set_error(BS_ERR_INVALID, "%s: top_k must be in 1..%d (at most experts), got %d", what, kMaxTopK, r->top_k);
    if (r->tokens < 0 || r->tokens >= (1ll << 31) || r->tokens * r->top_k >= (1ll << 31)) return set_error(BS_ERR_INVALID, "%s: tokens*top_k must be in 0..2^31-1", what);
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
    a.by_logit = r.bias == nullptr && (r.top_groups == r.groups || r.group_best == 1);
    return a;
}

// (a launch has fewer than 2^32 threads)
template <typename K>
static int launch_route(K* kernel, const RouteArgs& all, const char* what, hipStream_t st)
{
    const int tokens = all.experts <= 256 ? 16 : 4;     // of a workgroup
    const int64_t slice = (int64_t)tokens << 23, size = all.f32 ? 4 : 2;
    for (int64_t t = 0; t < all.tokens; t += slice) {
        RouteArgs a = all;
        a.tokens = std::min(slice, all.tokens - t);
        a.logits = static_cast<const char*>(all.logits) + t * all.stride * size;
        a.chosen += t * all.top_k;
        if (all.weights) a.weights += t * all.top_k;
        if (all.d_weights) a.d_weights += t * all.top_k, a.d_logits = static_cast<char*>(all.d_logits) + t * all.experts * size;
        hipLaunchKernelGGL(kernel, dim3((uint32_t)((a.tokens + tokens - 1) / tokens)), dim3(256), 0, st, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
    }
    return BS_OK;
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
    const int E = a.experts;
    auto* kernel = E <= 16 ? route_forward_kernel<16, 1> : E <= 64 ? route_forward_kernel<16, 4> : E <= 128 ? route_forward_kernel<16, 8>
                   : E <= 256 ? route_forward_kernel<16, 16> : E <= 512 ? route_forward_kernel<64, 8> : route_forward_kernel<64, 16>;
    return launch_route(kernel, a, what, (hipStream_t)stream);
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
    const int E = a.experts;
    auto* kernel = E <= 16 ? route_backward_kernel<16, 1> : E <= 64 ? route_backward_kernel<16, 4> : E <= 128 ? route_backward_kernel<16, 8>
                   : E <= 256 ? route_backward_kernel<16, 16> : E <= 512 ? route_backward_kernel<64, 8> : route_backward_kernel<64, 16>;
    return launch_route(kernel, a, what, (hipStream_t)stream);
}

static int64_t plan_blocks(int64_t pairs)
{
    return pairs <= 4 * kPlanBlock ? 1 : std::min<int64_t>((pairs + kPlanBlock - 1) / kPlanBlock, kPlanBlocks);
}

extern "C" int64_t bs_expert_plan_workspace_bytes(int64_t pairs, int experts)
{
    if (pairs <= 0 || pairs >= (1ll << 31) || experts < 1 || experts > kMaxExperts) return 0;
    const int64_t blocks = plan_blocks(pairs);
    return blocks > 1 ? blocks * experts * 4 : 0;
}

extern "C" int bs_expert_plan(const int32_t* chosen, int64_t pairs, int experts, int32_t* offsets, int32_t* order, int32_t* place,
                              void* workspace, int64_t workspace_bytes, void* stream)
{
    clear_error();
    const char* what = "bs_expert_plan";
    if (experts < 1 || experts > kMaxExperts) return set_error(BS_ERR_INVALID, "%s: experts must be in 1..%d, got %d", what, kMaxExperts, experts);
    if (pairs < 0 || pairs >= (1ll << 31)) return set_error(BS_ERR_INVALID, "%s: pairs must be in 0..2^31-1", what);
    if (offsets == nullptr || (pairs && (chosen == nullptr || order == nullptr || place == nullptr)))
        return set_error(BS_ERR_INVALID, "%s: null pointer", what);
    if (((uintptr_t)chosen | (uintptr_t)offsets | (uintptr_t)order | (uintptr_t)place) & 3u) return set_error(BS_ERR_INVALID, "%s: misaligned pointer", what);
    const int64_t blocks = plan_blocks(pairs), run = ((pairs + blocks * 16 - 1) / (blocks * 16) + 63) / 64 * 64;
    const int64_t need = bs_expert_plan_workspace_bytes(pairs, experts);
    if (need && (workspace == nullptr || workspace_bytes < need || ((uintptr_t)workspace & 3u)))
        return set_error(BS_ERR_INVALID, "%s: workspace too small or misaligned", what);
    int bits = 0;
    while (experts >> bits) bits++;         // (ids up to and with `experts`)
    const PlanArgs a{chosen, pairs, run, experts, bits, (int)blocks, offsets, order, place, static_cast<int32_t*>(workspace)};
    const uint32_t lds = 18u * experts * 4;
    const hipStream_t st = (hipStream_t)stream;
    if (blocks > 1) hipLaunchKernelGGL(expert_plan_kernel<true>, dim3((uint32_t)blocks), dim3(1024), lds, st, a);
    hipLaunchKernelGGL(expert_plan_kernel<false>, dim3((uint32_t)blocks), dim3(1024), lds, st, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? BS_OK : set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}
