// Dropout: out = 0 where an element's random half is below the bound, x times
// 65536 / (65536 - bound) elsewhere (philox.h).  Its own backward: the same
// call on the gradient.
//
// Bound by memory, x read once and out written once: the bits (20 64-bit
// products for eight elements, a third of the time by themselves) are formed
// while other waves' loads are on their way.  16384 x 4096: bf16 52 us, 5.1 TB/s, fp32 104 us
// (a copy reaches 4.9 TB/s); 257 x 100: 3.1 us, latency.
#include <algorithm>

#include "bs_host.h"
#include "philox.h"
#include "rownorm.h"

namespace bs {

struct DropArgs {
    const void* x;
    void* out;
    int64_t rows, cols, stride, chunks;     // chunks of all rows
    DropRule rule;
};

template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs a)
{
    const DropKey key = drop_key(a.rule);
    const int64_t per_row = (a.cols + 7) / 8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.chunks; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per_row, chunk = i - row * per_row;
        const int nv = (int)min((int64_t)8, a.cols - chunk * 8);
        const Raw<T> x = load_raw(static_cast<const T*>(a.x) + row * a.stride + chunk * 8, nv);
        const DropMask mask(a.rule, key, (uint32_t)chunk, (uint32_t)row);
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = mask.of(a.rule, e, raw_get(x, e));
        store_raw(static_cast<T*>(a.out) + row * a.cols + chunk * 8, to_raw<T>(o), nv);
    }
}

int drop_rule(const bs_drop* d, const char* what, DropRule* r)
{
    if (d == nullptr) return set_error(BS_ERR_INVALID, "%s: null arguments", what);
    if (d->below < 0 || d->below > 65536) return set_error(BS_ERR_INVALID, "%s: drop.below must be in 0..65536, got %d", what, d->below);
    if ((uintptr_t)d->state & 7u) return set_error(BS_ERR_INVALID, "%s: drop.state misaligned", what);
    r->key0 = (uint32_t)d->seed, r->key1 = (uint32_t)(d->seed >> 32);
    r->offset0 = (uint32_t)d->offset, r->offset1 = (uint32_t)(d->offset >> 32);
    r->at = d->state;
    r->bound = d->below < 65536 ? (uint32_t)d->below << 16 : ~0u, r->mask = d->below < 65536 ? ~0u : 0u;
    r->keep_scale = d->below < 65536 ? (float)(65536.0 / (65536 - d->below)) : 1.f;
    return BS_OK;
}

}  // namespace bs

using namespace bs;

extern "C" int bs_dropout(const bs_drop* drop, const void* x, int type, int64_t rows, int64_t cols, int64_t stride, void* out, void* stream)
{
    clear_error();
    const char* what = "bs_dropout";
    DropArgs a{};
    if (const int rc = drop_rule(drop, what, &a.rule); rc != BS_OK) return rc;
    if (type != BS_DT_BF16 && type != BS_DT_F32) return set_error(BS_ERR_INVALID, "%s: dtype %d must be bf16 or fp32", what, type);
    if (rows < 0 || cols < 0 || rows >= (1ll << 32) || cols >= (1ll << 32) || (cols && rows >= (1ll << 40) / cols))
        return set_error(BS_ERR_INVALID, "%s: rows and cols must be in 0..2^32-1 and rows*cols < 2^40, got %lld x %lld", what,
                         (long long)rows, (long long)cols);
    if (rows == 0 || cols == 0) return BS_OK;
    if (x == nullptr || out == nullptr) return set_error(BS_ERR_INVALID, "%s: null pointer", what);
    if (stride < 0) return set_error(BS_ERR_INVALID, "%s: negative row stride", what);
    if (((uintptr_t)x | (uintptr_t)out) & (type == BS_DT_F32 ? 3u : 1u)) return set_error(BS_ERR_INVALID, "%s: x or out misaligned for its type", what);
    a.x = x, a.out = out, a.rows = rows, a.cols = cols, a.stride = stride;
    a.chunks = rows * ((cols + 7) / 8);
    const dim3 grid((uint32_t)std::min<int64_t>((a.chunks + 255) / 256, 256 * 16)), block(256);
    if (type == BS_DT_BF16)
        hipLaunchKernelGGL(dropout_kernel<bf16>, grid, block, 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(dropout_kernel<float>, grid, block, 0, (hipStream_t)stream, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? BS_OK : set_error(BS_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}
