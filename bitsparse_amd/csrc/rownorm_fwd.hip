// The step between two MLP blocks, forward: norm of the block's output, gate,
// scaled residual and the next block's norm in one pass over the rows.
//
//   p = norm_post(y) or y;  x' = scale x + gate p;  h = norm_pre(x')
//
// Bound by memory: x and y are read and x' and h written once, all four with
// the row's own lanes between the two statistics (rownorm.h).  The next row's
// loads are in flight while this row's sums meet.  Up to 8192 elements the
// vectors are held in registers over the rows that a workgroup goes through.
// 16384 x 4096 in bf16: 101 us, 5.3 TB/s (a copy reaches 5.15), the norm alone
// 46 us, 5.8 TB/s; 32 x 4096: 5.6 us, latency.  Past 8192 elements the join
// spills registers (70 to 100 a lane, 220 to 380 past 16384): 4096 x 16384 202
// us, 2.7 TB/s; 2048 x 32768 387 us.
#include <algorithm>

#include "bs_host.h"
#include "rownorm.h"
#include "rownorm_host.h"

namespace bs {

struct JoinFwd {
    int64_t rows, cols;
    const void *x, *y;
    int64_t x_stride, y_stride;
    RowParam w_post, b_post, w_pre, b_pre, gate, scale;     // gate: per tensor or channel
    const void* row_gate;       // per row or element
    int row_gate_f32, gate_per;
    int64_t gate_stride;
    float scale_value;
    int post, pre;              // BS_NORM_*
    float eps_post, eps_pre;
    float *stats_post, *stats_pre;
    void *x1, *h;
    int waves, rows_here;       // of a row, of a workgroup at a time
};

// JOIN: there is a y.  C chunks a lane; HOLD: the vectors fit the registers;
// WHOLE: rows of a multiple of 8 elements.
template <typename XT, typename YT, bool JOIN, int C, int MAXT, bool HOLD, bool WHOLE>
__global__ __launch_bounds__(MAXT) void join_forward_kernel(JoinFwd a)
{
    __shared__ RowSums s_sums;
    const RowPlace<C> at(a.cols, a.waves);
    int turn = 0;
    const bool per_row = a.gate_per == BS_PER_ROW, per_element = a.gate_per == BS_PER_ELEMENT;

    const int64_t step = (int64_t)gridDim.x * a.rows_here;
    int64_t row = (int64_t)blockIdx.x * a.rows_here + at.sub;
    Raw<XT> xr[C];
    Raw<YT> yr[C];
    int nv[C], nv_next[C];
    auto load = [&](int64_t r) {
#pragma unroll
        for (int k = 0; k < C; k++) {
            nv_next[k] = r < a.rows ? at.in_row[k] : 0;
            xr[k] = load_raw<WHOLE>(static_cast<const XT*>(a.x) + r * a.x_stride + at.col[k], nv_next[k]);
            if constexpr (JOIN) yr[k] = load_raw<WHOLE>(static_cast<const YT*>(a.y) + r * a.y_stride + at.col[k], nv_next[k]);
        }
    };
    load(row);

    float sc[C][8], gv[C][8], w1[C][8], b1[C][8], w2[C][8], b2[C][8];
    auto vectors = [&](int k) {
        if constexpr (JOIN) {
            param_chunk(a.scale, at.col[k], at.in_row[k], a.scale_value, sc[k]);
            param_chunk(a.gate, at.col[k], at.in_row[k], 1.f, gv[k]);
            param_chunk(a.w_post, at.col[k], at.in_row[k], 1.f, w1[k]);
            param_chunk(a.b_post, at.col[k], at.in_row[k], 0.f, b1[k]);
        }
        if (a.pre) {
            param_chunk(a.w_pre, at.col[k], at.in_row[k], 1.f, w2[k]);
            param_chunk(a.b_pre, at.col[k], at.in_row[k], 0.f, b2[k]);
        }
    };
    if constexpr (HOLD) {
#pragma unroll
        for (int k = 0; k < C; k++) vectors(k);
    }

    // The first row and the vectors are waited for here (vmcnt 0): the wait would else stand at the head of the loop and be
    // for the next row's loads too (join of 16384 x 4096 111 instead of 101 us, norm alone 52 instead of 46).
    __builtin_amdgcn_s_waitcnt(0x0f70);
    // (as many rounds for every row of a workgroup: they meet at barriers)
    for (int64_t first = (int64_t)blockIdx.x * a.rows_here; first < a.rows; first += step, row += step) {
        float v[C][8], y[C][8];
#pragma unroll
        for (int k = 0; k < C; k++) {
            nv[k] = nv_next[k];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[k][e] = raw_get(xr[k], e);
                if constexpr (JOIN) y[k][e] = raw_get(yr[k], e);
            }
        }
        const bool mine = row < a.rows;
        load(row + step);

        if constexpr (JOIN) {
            float mean = 0.f, rstd = 1.f;
            if (a.post) {
                float var;
                row_moments(y, nv, at, a.cols, a.post == BS_NORM_LAYER, s_sums, turn, mean, var);
                rstd = row_rstd(var + a.eps_post);
                if (a.stats_post && mine && at.lane_in_row == 0)
                    *reinterpret_cast<float2*>(a.stats_post + 2 * row) = float2{mean, rstd};
            }
            const float rg = per_row && mine ? param_one(RowParam{a.row_gate, a.row_gate_f32, 0}, row * a.gate_stride) : 1.f;
#pragma unroll
            for (int k = 0; k < C; k++) {
                if constexpr (!HOLD) vectors(k);
                float g[8];
                if (per_element)
                    param_chunk(RowParam{a.row_gate, a.row_gate_f32, 0}, row * a.gate_stride + at.col[k], nv[k], 0.f, g);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    // (p whole before its gate: an infinite gate times two terms of different signs would be NaN, and times
                    // an absent bias's 0; rstd last: with RMS norms of 16-bit x, y and vectors p and the sum are the only
                    // roundings in 32 bits)
                    const float gate = gv[k][e] * (per_element ? g[e] : rg);
                    const float p = fmaf((y[k][e] - mean) * w1[k][e], rstd, b1[k][e]);
                    v[k][e] = fmaf(gate, p, sc[k][e] * v[k][e]);
                }
                const Raw<XT> o = to_raw<XT>(v[k]);
                store_raw<WHOLE>(static_cast<XT*>(a.x1) + row * a.cols + at.col[k], o, nv[k]);
#pragma unroll
                for (int e = 0; e < 8; e++) v[k][e] = e < nv[k] ? raw_get(o, e) : 0.f;   // as stored
            }
        }
        if (a.pre) {
            float mean, var;
            row_moments(v, nv, at, a.cols, a.pre == BS_NORM_LAYER, s_sums, turn, mean, var);
            const float rstd = row_rstd(var + a.eps_pre);
            if (a.stats_pre && mine && at.lane_in_row == 0)
                *reinterpret_cast<float2*>(a.stats_pre + 2 * row) = float2{mean, rstd};
#pragma unroll
            for (int k = 0; k < C; k++) {
                if constexpr (!HOLD) vectors(k);
                float h[8];
#pragma unroll
                for (int e = 0; e < 8; e++) h[e] = fmaf((v[k][e] - mean) * w2[k][e], rstd, b2[k][e]);
                store_raw<WHOLE>(static_cast<YT*>(a.h) + row * a.cols + at.col[k], to_raw<YT>(h), nv[k]);
            }
        }
    }
}

template <typename XT, typename YT, bool JOIN>
static int launch_forward(const JoinFwd& a, const RowLaunch& l, hipStream_t st)
{
    // as many workgroups as are resident at once (16 waves a CU: 106 us at 16384 x 4096; 32 take 112, 8 take 140), each
    // taking every so manieth row
    const int64_t need = (a.rows + l.rows - 1) / l.rows;
    const int64_t most = 256ll * std::max(1, 1024 / l.threads);
    const dim3 grid((uint32_t)std::min(need, most)), block(l.threads);
    const bool whole = a.cols % 8 == 0;
    auto* kernel = l.chunks == 1 ? (l.threads <= 512 ? whole ? join_forward_kernel<XT, YT, JOIN, 1, 512, true, true>
                                                             : join_forward_kernel<XT, YT, JOIN, 1, 512, true, false>
                                                     : join_forward_kernel<XT, YT, JOIN, 1, 1024, true, false>)
                   : l.chunks == 2 ? join_forward_kernel<XT, YT, JOIN, 2, 1024, false, false>
                                   : join_forward_kernel<XT, YT, JOIN, 4, 1024, false, false>;
    hipLaunchKernelGGL(kernel, grid, block, 0, st, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? BS_OK : set_error(BS_ERR_HIP, "bs_join_forward launch: %s", hipGetErrorString(e));
}

// ---------------------------------------------------------------------------
// checks of what both directions take
// ---------------------------------------------------------------------------
static bool type_ok(int t) { return t == BS_DT_BF16 || t == BS_DT_F32; }
static bool aligned_to_type(const void* p, int t) { return ((uintptr_t)p & (t == BS_DT_F32 ? 3u : 1u)) == 0; }

int join_check(const bs_join* a, const char* what)
{
    if (a == nullptr) return set_error(BS_ERR_INVALID, "%s: null arguments", what);
    if (a->rows < 0 || a->cols <= 0 || a->cols > kMaxRowCols)
        return set_error(BS_ERR_INVALID, "%s: rows must be >= 0 and cols in 1..%d, got %lld x %lld", what, kMaxRowCols,
                         (long long)a->rows, (long long)a->cols);
    if ((uint64_t)a->rows >= (1ull << 40) / (uint64_t)a->cols)
        return set_error(BS_ERR_INVALID, "%s: rows*cols must be < 2^40", what);
    if (!type_ok(a->x_type) || !type_ok(a->y_type) || (a->x_type == BS_DT_BF16 && a->y_type == BS_DT_F32))
        return set_error(BS_ERR_INVALID, "%s: dtypes (x %d, y or h %d) must be bf16/bf16, fp32/bf16 or fp32/fp32", what,
                         a->x_type, a->y_type);
    for (const int n : {a->norm_post, a->norm_pre})
        if (n < BS_NORM_NONE || n > BS_NORM_LAYER) return set_error(BS_ERR_INVALID, "%s: unknown norm %d", what, n);
    const bool join = a->y != nullptr;
    if (!join && a->norm_pre == BS_NORM_NONE) return set_error(BS_ERR_INVALID, "%s: neither y nor norm_pre", what);
    if (!join && (a->norm_post != BS_NORM_NONE || a->gate.data || a->scale.data))
        return set_error(BS_ERR_INVALID, "%s: norm_post, gate and scale need y", what);
    if (a->rows > 0 && a->x == nullptr) return set_error(BS_ERR_INVALID, "%s: null x", what);
    if (a->x_stride < 0 || (join && a->y_stride < 0) || a->gate_stride < 0)
        return set_error(BS_ERR_INVALID, "%s: negative row stride", what);
    if (!aligned_to_type(a->x, a->x_type) || !aligned_to_type(a->y, a->y_type))
        return set_error(BS_ERR_INVALID, "%s: x or y misaligned for its type", what);
    for (const bs_vector* v : {&a->weight_post, &a->bias_post, &a->weight_pre, &a->bias_pre, &a->gate, &a->scale})
        if (v->data && (!type_ok(v->type) || !aligned_to_type(v->data, v->type)))
            return set_error(BS_ERR_INVALID, "%s: a vector's dtype %d is unknown or its address misaligned", what, v->type);
    if (a->norm_post == BS_NORM_NONE && (a->weight_post.data || a->bias_post.data))
        return set_error(BS_ERR_INVALID, "%s: weight_post or bias_post without norm_post", what);
    if (a->norm_pre == BS_NORM_NONE && (a->weight_pre.data || a->bias_pre.data))
        return set_error(BS_ERR_INVALID, "%s: weight_pre or bias_pre without norm_pre", what);
    if ((a->gate.data != nullptr) != (a->gate_per != BS_PER_NOTHING) || a->gate_per < 0 || a->gate_per > BS_PER_ELEMENT)
        return set_error(BS_ERR_INVALID, "%s: gate and gate_per %d do not fit", what, a->gate_per);
    if ((a->scale.data != nullptr) != (a->scale_per != BS_PER_NOTHING) || a->scale_per < 0 || a->scale_per > BS_PER_CHANNEL)
        return set_error(BS_ERR_INVALID, "%s: scale and scale_per %d do not fit", what, a->scale_per);
    if (((uintptr_t)a->stats_post | (uintptr_t)a->stats_pre) & 7u)
        return set_error(BS_ERR_INVALID, "%s: stats misaligned", what);
    return BS_OK;
}

RowParam row_param(const bs_vector& v, int per) { return {v.data, v.type == BS_DT_F32, per == BS_PER_TENSOR}; }

}  // namespace bs

using namespace bs;

extern "C" int bs_join_forward(const bs_join* args, void* x1, void* h, void* stream)
{
    clear_error();
    if (const int rc = join_check(args, "bs_join_forward"); rc != BS_OK) return rc;
    const bs_join& j = *args;
    if (j.rows == 0) return BS_OK;
    if ((j.y && x1 == nullptr) || (j.norm_pre && h == nullptr))
        return set_error(BS_ERR_INVALID, "bs_join_forward: null result");
    if (!aligned_to_type(x1, j.x_type) || !aligned_to_type(h, j.y_type))
        return set_error(BS_ERR_INVALID, "bs_join_forward: result misaligned for its type");
    const RowLaunch l = row_launch(j.cols, 8192);
    const bool whole = j.gate_per == BS_PER_TENSOR || j.gate_per == BS_PER_CHANNEL;
    JoinFwd a{};
    a.rows = j.rows, a.cols = j.cols, a.x = j.x, a.y = j.y, a.x_stride = j.x_stride, a.y_stride = j.y_stride;
    a.w_post = row_param(j.weight_post, 0), a.b_post = row_param(j.bias_post, 0);
    a.w_pre = row_param(j.weight_pre, 0), a.b_pre = row_param(j.bias_pre, 0);
    a.gate = whole ? row_param(j.gate, j.gate_per) : RowParam{nullptr, 0, 0};
    a.scale = row_param(j.scale, j.scale_per);
    a.row_gate = whole ? nullptr : j.gate.data, a.row_gate_f32 = j.gate.type == BS_DT_F32;
    a.gate_per = j.gate_per, a.gate_stride = j.gate_stride, a.scale_value = j.scale_value;
    a.post = j.norm_post, a.pre = j.norm_pre, a.eps_post = j.eps_post, a.eps_pre = j.eps_pre;
    a.stats_post = j.stats_post, a.stats_pre = j.stats_pre, a.x1 = x1, a.h = h, a.waves = l.waves, a.rows_here = l.rows;
    const hipStream_t st = (hipStream_t)stream;
    if (j.y == nullptr) {
        if (j.x_type == BS_DT_BF16) return launch_forward<bf16, bf16, false>(a, l, st);
        if (j.y_type == BS_DT_BF16) return launch_forward<float, bf16, false>(a, l, st);
        return launch_forward<float, float, false>(a, l, st);
    }
    if (j.x_type == BS_DT_BF16) return launch_forward<bf16, bf16, true>(a, l, st);
    if (j.y_type == BS_DT_BF16) return launch_forward<float, bf16, true>(a, l, st);
    return launch_forward<float, float, true>(a, l, st);
}
