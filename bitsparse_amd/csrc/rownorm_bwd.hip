// The step between two MLP blocks, backward: every gradient of
//   p = norm_post(y) or y;  x' = scale x + gate p;  h = norm_pre(x')
// in one pass over the rows and a small one over partial column sums.
//
// With n = the standardised row, r = 1 / deviation and mu() the row's mean
// (the first mu() only for a layer norm):
//   dn = dh w_pre;   G  = dx' + r (dn - mu(dn) - n mu(dn n))
//   dx = scale G;    dp = gate G
//   dm = dp w_post;  dy = r_y (dm - mu(dm) - n_y mu(dm n_y))
// and over rows dw_pre = sum dh n, db_pre = sum dh, dscale = sum G x,
// dw_post = sum dp n_y, db_post = sum dp, dgate = sum G p.  A gate that is
// the same in every row comes out of those sums: with A = sum G n_y and
// B = sum G, dw_post = gate A, db_post = gate B and dgate = w_post A +
// b_post B, so five sums a column serve all six vectors.
//
// Bound by memory: dx', dh, x', y (and x for dscale; y not where no gradient is formed of it) read once, dx and dy
// written once, a row with its lanes throughout.  Each workgroup keeps its
// column sums over all its rows and writes one row of partial sums; the second
// kernel adds those in order.  No atomics: the same bits at every call.
// 16384 x 4096 in bf16: 182 us, 5.2 TB/s (a copy reaches 5.15); 8192 x 768,
// which stays in the last level cache: 23 us, 3.8 TB/s.  With a dropout, whose
// bits are formed again, 199 us where the same step without takes 144.  Up to 4096 elements
// row, sums and vectors are in registers.  Past that they do not all fit (the
// join's spill 40 to 90 registers a lane up to 8192 elements, 630 to 960 up to
// 16384, 1200 to 1600 beyond): 8192 x 8192 297 us, 3.2 TB/s; 4096 x 16384 1.49
// ms, 0.63 TB/s; 2048 x 32768 1.94 ms.
#include <algorithm>
#include <type_traits>

#include "bs_host.h"
#include "rownorm.h"
#include "rownorm_host.h"

namespace bs {

enum : int { kSumA = 0, kSumB, kSumW2, kSumB2, kSumScale, kColSums };

struct JoinBwd {
    int64_t rows, cols;
    const void *x, *x1, *y, *gx, *gh;
    int64_t x_stride, x1_stride, y_stride, gx_stride, gh_stride;
    RowParam w_post, b_post, w_pre, gate, scale;
    const void* row_gate;
    int row_gate_f32, gate_per;
    int64_t gate_stride;
    float scale_value;
    int post, pre;
    const float *stats_post, *stats_pre;
    void *dx, *dy, *d_row_gate;
    int want;               // bit i: column sum i
    int one_scale, one_gate;    // gradients of a scale or gate that is one number
    float* part;            // [blocks, sums wanted, cols]
    float* part_one;        // [blocks, 2]
    int waves, rows_here;       // of a row, of a workgroup at a time
    DropRule drop;
};

// JOIN: there is a y.  DROP: p was dropped out of, by the same factors here.  C chunks a lane; HOLD: the vectors fit the registers; AHEAD: and the next row's loads.
// WHOLE: rows of a multiple of 8 elements.
// PLAIN: RMS norms (or none), no gate that differs from row to row, no sums for biases: a third fewer instructions, which
// two waves a SIMD do not hide behind the loads (16384 x 4096: 182 against 232 us).
template <typename XT, typename YT, bool JOIN, bool DROP, int C, int MAXT, bool HOLD, bool AHEAD, bool PLAIN, bool WHOLE>
__global__ __launch_bounds__(MAXT) void join_backward_kernel(JoinBwd a)
{
    __shared__ RowSums s_sums;
    __shared__ float s_join[C == 1 ? 4096 : 1];         // a sum of every row of the workgroup
    const RowPlace<C> at(a.cols, a.waves);
    int turn = 0;
    const bool per_row = !PLAIN && a.gate_per == BS_PER_ROW, per_element = !PLAIN && a.gate_per == BS_PER_ELEMENT;
    const bool layer_post = !PLAIN && a.post == BS_NORM_LAYER, layer_pre = !PLAIN && a.pre == BS_NORM_LAYER;
    void* const d_row_gate = PLAIN ? nullptr : a.d_row_gate;
    const DropKey key = DROP ? drop_key(a.drop) : DropKey{};

    // the next row's loads are in flight while this row's sums meet
    struct Row {
        Raw<XT> gx[C], x1[C], x[C];
        Raw<YT> gh[C], y[C];
        float2 st_pre, st_post;
    };
    Row next;
    auto load = [&](Row& o, int64_t row) {
        const bool mine = row < a.rows;
        o.st_pre = a.gh && mine ? *reinterpret_cast<const float2*>(a.stats_pre + 2 * row) : float2{0.f, 1.f};
        if constexpr (JOIN) o.st_post = a.post && mine ? *reinterpret_cast<const float2*>(a.stats_post + 2 * row) : float2{0.f, 1.f};
#pragma unroll
        for (int k = 0; k < C; k++) {
            const int nv = mine ? at.in_row[k] : 0, nv_gx = a.gx ? nv : 0, nv_gh = a.gh ? nv : 0;
            o.gx[k] = load_raw<WHOLE>(static_cast<const XT*>(a.gx) + row * a.gx_stride + at.col[k], nv_gx);
            o.gh[k] = load_raw<WHOLE>(static_cast<const YT*>(a.gh) + row * a.gh_stride + at.col[k], nv_gh);
            o.x1[k] = load_raw<WHOLE>(static_cast<const XT*>(a.x1) + row * a.x1_stride + at.col[k], nv_gh);
            if constexpr (JOIN) {
                o.y[k] = load_raw<WHOLE>(static_cast<const YT*>(a.y) + row * a.y_stride + at.col[k], a.y ? nv : 0);
                o.x[k] = load_raw<WHOLE>(static_cast<const XT*>(a.x) + row * a.x_stride + at.col[k], a.x ? nv : 0);
            }
        }
    };
    const int64_t step = (int64_t)gridDim.x * a.rows_here;
    int64_t row = (int64_t)blockIdx.x * a.rows_here + at.sub;
    load(next, row);

    float acc[kColSums][C][8];
#pragma unroll
    for (int i = 0; i < kColSums; i++)
#pragma unroll
        for (int k = 0; k < C; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) acc[i][k][e] = 0.f;
    float sc[C][8], gw[C][8], w2[C][8];       // scale, gate * weight_post, weight_pre
    auto vectors_pre = [&](int k) { param_chunk(a.w_pre, at.col[k], at.in_row[k], 1.f, w2[k]); };
    auto vectors_post = [&](int k) {
        param_chunk(a.scale, at.col[k], at.in_row[k], a.scale_value, sc[k]);
        float g[8];
        param_chunk(a.gate, at.col[k], at.in_row[k], 1.f, g);
        param_chunk(a.w_post, at.col[k], at.in_row[k], 1.f, gw[k]);
#pragma unroll
        for (int e = 0; e < 8; e++) gw[k][e] *= g[e];
    };
    if constexpr (HOLD) {
#pragma unroll
        for (int k = 0; k < C; k++) {
            vectors_pre(k);
            if constexpr (JOIN) vectors_post(k);
        }
    }

    // (as many rounds for every row of a workgroup: they meet at barriers)
    for (int64_t first = (int64_t)blockIdx.x * a.rows_here; first < a.rows; first += step, row += step) {
        const bool mine = row < a.rows;
        int nv[C];
#pragma unroll
        for (int k = 0; k < C; k++) nv[k] = mine ? at.in_row[k] : 0;
        Row now = next;
        if constexpr (AHEAD) {
            load(next, row + step);
        }
        float G[C][8];
        if (a.gh) {
            const float2 st = {PLAIN ? 0.f : now.st_pre.x, now.st_pre.y};
            float dn[C][8], n[C][8], s[2] = {0.f, 0.f};
#pragma unroll
            for (int k = 0; k < C; k++) {
                if constexpr (!HOLD) vectors_pre(k);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float gh = raw_get(now.gh[k], e);
                    n[k][e] = (raw_get(now.x1[k], e) - st.x) * st.y;
                    dn[k][e] = gh * w2[k][e];
                    if (!PLAIN) s[0] += dn[k][e];
                    s[1] += dn[k][e] * n[k][e];
                    acc[kSumW2][k][e] += gh * n[k][e];
                    if (!PLAIN) acc[kSumB2][k][e] += gh;
                }
            }
            row_sums(s, at, s_sums, turn);
            const float m0 = layer_pre ? s[0] * at.inv_cols : 0.f, m1 = s[1] * at.inv_cols;
#pragma unroll
            for (int k = 0; k < C; k++)
#pragma unroll
                for (int e = 0; e < 8; e++) G[k][e] = raw_get(now.gx[k], e) + st.y * (dn[k][e] - m0 - n[k][e] * m1);
        } else {
#pragma unroll
            for (int k = 0; k < C; k++)
#pragma unroll
                for (int e = 0; e < 8; e++) G[k][e] = raw_get(now.gx[k], e);
        }
        if constexpr (!JOIN) {
            if (a.dx)
#pragma unroll
                for (int k = 0; k < C; k++)
                    store_raw<WHOLE>(static_cast<XT*>(a.dx) + row * a.cols + at.col[k], to_raw<XT>(G[k]), nv[k]);
        } else {
            const float2 st = {PLAIN ? 0.f : now.st_post.x, now.st_post.y};
            const float rg = per_row && mine ? param_one(RowParam{a.row_gate, a.row_gate_f32, 0}, row * a.gate_stride) : 1.f;
            float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < C; k++) {
                if constexpr (!HOLD) vectors_post(k);
                float o[8], ge[8], b1[8];
                if (per_element)
                    param_chunk(RowParam{a.row_gate, a.row_gate_f32, 0}, row * a.gate_stride + at.col[k], nv[k], 0.f, ge);
                if (d_row_gate) param_chunk(a.b_post, at.col[k], nv[k], 0.f, b1);
                std::conditional_t<DROP, DropMask, DropNothing> drop(a.drop, key, (uint32_t)(at.col[k] >> 3), (uint32_t)row);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    // (past the row's end x' and the gradients are 0, and so is G but for a layer norm's mean)
                    const float g0 = PLAIN || e < nv[k] ? G[k][e] : 0.f;
                    o[e] = sc[k][e] * g0;
                    acc[kSumScale][k][e] += g0 * raw_get(now.x[k], e);
                    float n = (raw_get(now.y[k], e) - st.x) * st.y;
                    float gg = PLAIN ? g0 : per_element ? g0 * ge[e] : rg * g0;    // G of the gate's part that is not a vector
                    // (a dropped element passes nothing, whatever it and its gradient are; gp: G as the gate's gradient has it)
                    gg = drop.of(a.drop, e, gg);
                    const float gp = drop.of(a.drop, e, g0);
                    if (DROP && !a.post) n = drop.kept(a.drop, e) ? n : 0.f;
                    acc[kSumA][k][e] += gg * n;
                    if (!PLAIN) acc[kSumB][k][e] += gg;
                    const float dm = gg * gw[k][e];
                    if (!PLAIN) s[0] += dm;
                    s[1] += dm * n;
                    G[k][e] = dm;
                    if (d_row_gate) {
                        ge[e] = gp * (n * gw[k][e] + b1[e]);      // (such a gate is no vector: gw is weight_post)
                        s[2] += ge[e];
                    }
                }
                if (a.dx) store_raw<WHOLE>(static_cast<XT*>(a.dx) + row * a.cols + at.col[k], to_raw<XT>(o), nv[k]);
                if (d_row_gate && per_element) {
                    if (a.row_gate_f32)
                        store_raw<WHOLE>(static_cast<float*>(d_row_gate) + row * a.cols + at.col[k], to_raw<float>(ge), nv[k]);
                    else
                        store_raw<WHOLE>(static_cast<bf16*>(d_row_gate) + row * a.cols + at.col[k], to_raw<bf16>(ge), nv[k]);
                }
            }
            if (a.post || (per_row && d_row_gate)) row_sums(s, at, s_sums, turn);
            if (per_row && d_row_gate && mine && at.lane_in_row == 0) param_store(d_row_gate, a.row_gate_f32, row, s[2]);
            if (a.dy) {
                const float m0 = layer_post ? s[0] * at.inv_cols : 0.f, m1 = s[1] * at.inv_cols;
#pragma unroll
                for (int k = 0; k < C; k++) {
                    float o[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        // (without a norm dp alone: y may hold what 0 times makes a NaN)
                        const float n = (raw_get(now.y[k], e) - st.x) * st.y;
                        o[e] = a.post ? st.y * (G[k][e] - m0 - n * m1) : G[k][e];
                    }
                    store_raw<WHOLE>(static_cast<YT*>(a.dy) + row * a.cols + at.col[k], to_raw<YT>(o), nv[k]);
                }
            }
        }
        if constexpr (!AHEAD) load(next, row + step);
    }

    // one number for all columns: this workgroup's part of its gradient
    if (a.one_scale || a.one_gate) {
        float t[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < C; k++) {
            float b1[8], w1[8];
            param_chunk(a.b_post, at.col[k], at.in_row[k], 0.f, b1);
            param_chunk(a.w_post, at.col[k], at.in_row[k], 1.f, w1);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (e >= at.in_row[k]) continue;
                t[0] += acc[kSumScale][k][e];
                t[1] += w1[e] * acc[kSumA][k][e] + (a.b_post.p ? b1[e] * acc[kSumB][k][e] : 0.f);    // (B may be infinite)
            }
        }
        const int wave = (int)threadIdx.x >> 6, waves = (int)blockDim.x >> 6;
        t[0] = wave_sum_f32(t[0]);
        t[1] = wave_sum_f32(t[1]);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s_sums.part[0][wave] = float4{t[0], t[1], 0.f, 0.f};
        __syncthreads();
        if (threadIdx.x < 2) {
            float s = 0.f;
            for (int i = 0; i < waves; i++) s += threadIdx.x ? s_sums.part[0][i].y : s_sums.part[0][i].x;
            a.part_one[2 * (int64_t)blockIdx.x + threadIdx.x] = s;
        }
    }
    const int n_sums = __builtin_popcount(a.want);
    int slot = 0;
#pragma unroll
    for (int i = 0; i < kColSums; i++) {
        if (!(a.want >> i & 1)) continue;
        float* out = a.part + ((int64_t)blockIdx.x * n_sums + slot++) * a.cols;
        if (C == 1 && a.rows_here > 1) {
            // the workgroup's rows into one
            __syncthreads();
            const int pitch = 512 * a.waves;
#pragma unroll
            for (int e = 0; e < 8; e++) s_join[at.sub * pitch + e * (pitch / 8) + at.lane_in_row] = acc[i][0][e];
            __syncthreads();
            for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
                float t = 0.f;
                for (int r = 0; r < a.rows_here; r++) t += s_join[r * pitch + c % 8 * (pitch / 8) + c / 8];
                out[c] = t;
            }
        } else {
#pragma unroll
            for (int k = 0; k < C; k++) store_raw(out + at.col[k], to_raw<float>(acc[i][k]), at.in_row[k]);
        }
    }
}

// ---------------------------------------------------------------------------
// the partial sums, in order, into the vectors' gradients
// ---------------------------------------------------------------------------
struct JoinFinish {
    const float *part, *part_one;
    int64_t blocks, cols;
    int want, col_blocks, fixed_gate;       // fixed_gate: the gate is a vector (or absent), not in the sums
    RowParam w_post, b_post, gate;
    void *d_w_post, *d_b_post, *d_w_pre, *d_b_pre, *d_gate, *d_scale;
    int f32_w_post, f32_b_post, f32_w_pre, f32_b_pre, f32_gate, f32_scale, one_gate, one_scale;
};

constexpr int kFinishThreads = 1024;
constexpr int kFinishLanes = kFinishThreads / 64;

__global__ __launch_bounds__(kFinishThreads) void join_finish_kernel(JoinFinish a)
{
    __shared__ float s_part[kColSums][kFinishLanes][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if ((int)blockIdx.x >= a.col_blocks) {      // the gradients of single numbers
        float t[2] = {0.f, 0.f};
        for (int64_t p = threadIdx.x; p < a.blocks; p += kFinishThreads) {
            t[0] += a.part_one[2 * p];
            t[1] += a.part_one[2 * p + 1];
        }
        t[0] = wave_sum_f32(t[0]);
        t[1] = wave_sum_f32(t[1]);
        if (lane == 0) {
            s_part[0][wave][0] = t[0];
            s_part[0][wave][1] = t[1];
        }
        __syncthreads();
        if (threadIdx.x < 2) {
            float s = 0.f;
            for (int i = 0; i < kFinishLanes; i++) s += s_part[0][i][threadIdx.x];
            if (threadIdx.x == 0 && a.one_scale) param_store(a.d_scale, a.f32_scale, 0, s);
            if (threadIdx.x == 1 && a.one_gate) param_store(a.d_gate, a.f32_gate, 0, s);
        }
        return;
    }
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    const int n_sums = __builtin_popcount(a.want);
    const int64_t stride = (int64_t)n_sums * a.cols;
    int slot = 0;
#pragma unroll
    for (int i = 0; i < kColSums; i++) {
        float t = 0.f;
        if (a.want >> i & 1) {
            if (c < a.cols) {
                const float* p = a.part + (int64_t)slot * a.cols + c;
                int64_t b = wave;
                for (; b + 7 * kFinishLanes < a.blocks; b += 8 * kFinishLanes) {    // eight loads in flight
                    float v[8];
#pragma unroll
                    for (int u = 0; u < 8; u++) v[u] = p[(b + u * kFinishLanes) * stride];
#pragma unroll
                    for (int u = 0; u < 8; u++) t += v[u];
                }
                for (; b < a.blocks; b += kFinishLanes) t += p[b * stride];
            }
            slot++;
        }
        s_part[i][wave][lane] = t;
    }
    __syncthreads();
    if (wave != 0 || c >= a.cols) return;
    float s[kColSums];
#pragma unroll
    for (int i = 0; i < kColSums; i++) {
        s[i] = 0.f;
#pragma unroll
        for (int w = 0; w < kFinishLanes; w++) s[i] += s_part[i][w][lane];
    }
    const float g = a.fixed_gate && a.gate.p ? param_one(a.gate, a.gate.one ? 0 : c) : 1.f;
    if (a.d_w_post) param_store(a.d_w_post, a.f32_w_post, c, g * s[kSumA]);
    if (a.d_b_post) param_store(a.d_b_post, a.f32_b_post, c, g * s[kSumB]);
    if (a.d_gate && !a.one_gate) {
        const float w = a.w_post.p ? param_one(a.w_post, c) : 1.f, b = a.b_post.p ? param_one(a.b_post, c) : 0.f;
        param_store(a.d_gate, a.f32_gate, c, w * s[kSumA] + b * s[kSumB]);
    }
    if (a.d_w_pre) param_store(a.d_w_pre, a.f32_w_pre, c, s[kSumW2]);
    if (a.d_b_pre) param_store(a.d_b_pre, a.f32_b_pre, c, s[kSumB2]);
    if (a.d_scale && !a.one_scale) param_store(a.d_scale, a.f32_scale, c, s[kSumScale]);
}

// Workgroups of the first kernel: all that are resident at once (8 waves a
// CU), and no fewer than four rounds of rows to each, so that the partial sums
// stay a small part of the bytes moved.  Twice as many take 40 us instead of 34
// at 8192 x 768 and 85 instead of 72 at 3005 x 2501; two or eight rounds as long.
constexpr int kBwdThreads = 512, kBwdRounds = 4;        // threads of a CU
static int64_t backward_blocks(int64_t rows, const RowLaunch& l)
{
    const int64_t most = 256ll * std::max(1, kBwdThreads / l.threads);
    return std::max<int64_t>(1, std::min((rows + kBwdRounds * l.rows - 1) / (kBwdRounds * l.rows), most));
}
// Sixteen waves would leave 128 registers a lane, fewer than the sums take: rows past 4096 have two chunks a lane.
static RowLaunch backward_launch(int64_t cols) { return row_launch(cols, cols <= 16384 ? 4096 : 8192); }

template <typename XT, typename YT, bool JOIN, bool DROP>
static void launch_backward(const JoinBwd& a, const RowLaunch& l, int64_t blocks, hipStream_t st)
{
    const dim3 grid((uint32_t)blocks), block(l.threads);
    // (the gradient of a gate that is one number takes the bias's sum where there is a bias)
    const bool plain = a.post != BS_NORM_LAYER && a.pre != BS_NORM_LAYER && a.gate_per <= BS_PER_CHANNEL &&
                       !(a.want & (1 << kSumB | 1 << kSumB2)) && !(a.one_gate && a.b_post.p);
    const bool whole = a.cols % 8 == 0;
    auto* kernel = l.chunks == 1 ? (plain ? whole ? join_backward_kernel<XT, YT, JOIN, DROP, 1, 512, true, true, true, true>
                                                  : join_backward_kernel<XT, YT, JOIN, DROP, 1, 512, true, true, true, false>
                                          : whole ? join_backward_kernel<XT, YT, JOIN, DROP, 1, 512, true, true, false, true>
                                                  : join_backward_kernel<XT, YT, JOIN, DROP, 1, 512, true, true, false, false>)
                   : l.chunks == 2    ? join_backward_kernel<XT, YT, JOIN, DROP, 2, 512, false, false, false, false>
                   : l.threads <= 512 ? join_backward_kernel<XT, YT, JOIN, DROP, 4, 512, false, false, false, false>
                                      : join_backward_kernel<XT, YT, JOIN, DROP, 4, 1024, false, false, false, false>;
    hipLaunchKernelGGL(kernel, grid, block, 0, st, a);
}

}  // namespace bs

using namespace bs;

extern "C" int64_t bs_join_backward_workspace_bytes(int64_t rows, int64_t cols)
{
    if (rows <= 0 || cols <= 0 || cols > kMaxRowCols) return 0;
    return backward_blocks(rows, backward_launch(cols)) * (kColSums * cols + 2) * 4;
}

namespace bs {

static int join_backward(const char* what, const bs_join* args, const bs_join_grads* grads, const bs_drop* drop, void* workspace,
                         int64_t workspace_bytes, void* stream)
{
    clear_error();
    if (const int rc = join_check(args, what); rc != BS_OK) return rc;
    if (grads == nullptr) return set_error(BS_ERR_INVALID, "%s: null arguments", what);
    const bs_join& j = *args;
    const bs_join_grads& g = *grads;
    DropRule rule{};
    if (drop)
        if (const int rc = join_drop_check(j, drop, what, &rule); rc != BS_OK) return rc;
    if (j.rows == 0) return set_error(BS_ERR_INVALID, "%s: no rows", what);
    const bool join = j.y != nullptr;
    const bool fixed_gate = j.gate_per <= BS_PER_CHANNEL;
    if (!join && (g.grad_x1 || g.d_y)) return set_error(BS_ERR_INVALID, "%s: grad_x1 and d_y need y", what);
    if (j.norm_pre == BS_NORM_NONE && g.grad_h) return set_error(BS_ERR_INVALID, "%s: grad_h without norm_pre", what);
    if (g.grad_x1 == nullptr && g.grad_h == nullptr) return set_error(BS_ERR_INVALID, "%s: no gradient given", what);
    if (g.grad_x1_stride < 0 || g.grad_h_stride < 0) return set_error(BS_ERR_INVALID, "%s: negative row stride", what);
    if ((g.grad_h && (j.stats_pre == nullptr || (join && g.x1 == nullptr))) || (j.norm_post && j.stats_post == nullptr))
        return set_error(BS_ERR_INVALID, "%s: the forward's x1 or statistics are missing", what);
    const unsigned xm = j.x_type == BS_DT_F32 ? 3u : 1u, ym = j.y_type == BS_DT_F32 ? 3u : 1u;
    if ((((uintptr_t)g.x1 | (uintptr_t)g.grad_x1 | (uintptr_t)g.d_x) & xm) || (((uintptr_t)g.grad_h | (uintptr_t)g.d_y) & ym))
        return set_error(BS_ERR_INVALID, "%s: a gradient or x1 misaligned for its type", what);
    const struct { const void* d; const bs_vector* of; const char* name; } vectors[] = {
        {g.d_gate, &j.gate, "d_gate"}, {g.d_scale, &j.scale, "d_scale"}, {g.d_weight_post, &j.weight_post, "d_weight_post"},
        {g.d_bias_post, &j.bias_post, "d_bias_post"}, {g.d_weight_pre, &j.weight_pre, "d_weight_pre"},
        {g.d_bias_pre, &j.bias_pre, "d_bias_pre"}};
    for (const auto& v : vectors) {
        if (v.d == nullptr) continue;
        if (v.of->data == nullptr) return set_error(BS_ERR_INVALID, "%s: %s of an absent vector", what, v.name);
        if ((uintptr_t)v.d & (v.of->type == BS_DT_F32 ? 3u : 1u))
            return set_error(BS_ERR_INVALID, "%s: %s misaligned for its type", what, v.name);
    }
    const int64_t need = bs_join_backward_workspace_bytes(j.rows, j.cols);
    if (workspace == nullptr || workspace_bytes < need || ((uintptr_t)workspace & 15u))
        return set_error(BS_ERR_INVALID, "%s: workspace too small or misaligned", what);

    const RowLaunch l = backward_launch(j.cols);
    const int64_t blocks = backward_blocks(j.rows, l);
    JoinBwd a{};
    a.rows = j.rows, a.cols = j.cols;
    a.x = g.d_scale ? j.x : nullptr, a.x_stride = j.x_stride;
    a.x1 = join ? g.x1 : j.x, a.x1_stride = join ? j.cols : j.x_stride;
    a.y = g.d_gate || (j.norm_post && (g.d_y || g.d_weight_post)) ? j.y : nullptr, a.y_stride = j.y_stride;
    a.gx = g.grad_x1, a.gx_stride = g.grad_x1_stride, a.gh = g.grad_h, a.gh_stride = g.grad_h_stride;
    a.w_post = row_param(j.weight_post, 0), a.b_post = g.d_gate ? row_param(j.bias_post, 0) : RowParam{nullptr, 0, 0}, a.w_pre = row_param(j.weight_pre, 0);
    a.gate = fixed_gate ? row_param(j.gate, j.gate_per) : RowParam{nullptr, 0, 0};
    a.scale = row_param(j.scale, j.scale_per), a.scale_value = j.scale_value;
    a.row_gate = fixed_gate ? nullptr : j.gate.data, a.row_gate_f32 = j.gate.type == BS_DT_F32;
    a.gate_per = j.gate_per, a.gate_stride = j.gate_stride;
    a.post = j.norm_post, a.pre = j.norm_pre, a.stats_post = j.stats_post, a.stats_pre = j.stats_pre;
    a.dx = g.d_x, a.dy = g.d_y, a.d_row_gate = fixed_gate ? nullptr : g.d_gate;
    a.one_scale = g.d_scale && j.scale_per == BS_PER_TENSOR;
    a.one_gate = g.d_gate && j.gate_per == BS_PER_TENSOR;
    const bool gate_sum = g.d_gate && j.gate_per == BS_PER_CHANNEL;
    if (g.d_weight_post || gate_sum) a.want |= 1 << kSumA;
    if (g.d_bias_post || (gate_sum && j.bias_post.data)) a.want |= 1 << kSumB;
    if (g.d_weight_pre) a.want |= 1 << kSumW2;
    if (g.d_bias_pre) a.want |= 1 << kSumB2;
    if (g.d_scale && !a.one_scale) a.want |= 1 << kSumScale;
    a.part = static_cast<float*>(workspace);
    a.part_one = a.part + blocks * kColSums * j.cols;
    a.waves = l.waves, a.rows_here = l.rows;
    const hipStream_t st = (hipStream_t)stream;
    const bool xb = j.x_type == BS_DT_BF16, yb = j.y_type == BS_DT_BF16;
    a.drop = rule;
    if (drop)
        (xb ? launch_backward<bf16, bf16, true, true> : yb ? launch_backward<float, bf16, true, true> : launch_backward<float, float, true, true>)(a, l, blocks, st);
    else if (join)
        (xb ? launch_backward<bf16, bf16, true, false> : yb ? launch_backward<float, bf16, true, false> : launch_backward<float, float, true, false>)(a, l, blocks, st);
    else
        (xb ? launch_backward<bf16, bf16, false, false> : yb ? launch_backward<float, bf16, false, false> : launch_backward<float, float, false, false>)(a, l, blocks, st);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));

    if (a.want == 0 && !a.one_scale && !a.one_gate) return BS_OK;
    JoinFinish f{};
    f.part = a.part, f.part_one = a.part_one, f.blocks = blocks, f.cols = j.cols, f.want = a.want;
    f.col_blocks = a.want ? (int)((j.cols + 63) / 64) : 0;
    f.fixed_gate = fixed_gate;
    f.w_post = a.w_post, f.b_post = a.b_post, f.gate = a.gate;
    f.d_w_post = g.d_weight_post, f.f32_w_post = j.weight_post.type == BS_DT_F32;
    f.d_b_post = g.d_bias_post, f.f32_b_post = j.bias_post.type == BS_DT_F32;
    f.d_w_pre = g.d_weight_pre, f.f32_w_pre = j.weight_pre.type == BS_DT_F32;
    f.d_b_pre = g.d_bias_pre, f.f32_b_pre = j.bias_pre.type == BS_DT_F32;
    f.d_gate = fixed_gate ? g.d_gate : nullptr, f.f32_gate = j.gate.type == BS_DT_F32, f.one_gate = a.one_gate;
    f.d_scale = g.d_scale, f.f32_scale = j.scale.type == BS_DT_F32, f.one_scale = a.one_scale;
    const uint32_t ones = a.one_scale || a.one_gate ? 1u : 0u;
    hipLaunchKernelGGL(join_finish_kernel, dim3((uint32_t)f.col_blocks + ones), dim3(kFinishThreads), 0, st, f);
    e = hipGetLastError();
    return e == hipSuccess ? BS_OK : set_error(BS_ERR_HIP, "%s finish launch: %s", what, hipGetErrorString(e));
}

}  // namespace bs

extern "C" int bs_join_backward(const bs_join* args, const bs_join_grads* grads, void* workspace, int64_t workspace_bytes,
                                void* stream)
{
    return join_backward("bs_join_backward", args, grads, nullptr, workspace, workspace_bytes, stream);
}

extern "C" int bs_join_drop_backward(const bs_join* args, const bs_join_grads* grads, const bs_drop* drop, void* workspace,
                                     int64_t workspace_bytes, void* stream)
{
    if (drop == nullptr) return set_error(BS_ERR_INVALID, "bs_join_drop_backward: null drop");
    return join_backward("bs_join_drop_backward", args, grads, drop, workspace, workspace_bytes, stream);
}
