// Attention of new tokens over a paged cache (kernels.h CacheAttn).
#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace vh {
namespace {

// Keys [lo, hi) that a query at position pos of a request of len tokens sees.
struct Seen {
    int lo, hi;
};
__device__ __forceinline__ Seen keys_seen(const CacheAttn &a, int len, long long pos) {
    long long hi = len;
    if (a.block) hi = pos < 0 ? 0 : min(hi, ((long long)((unsigned)pos / a.block) + 1) * a.block);
    const long long lo = a.window ? max(0ll, hi - a.window) : 0;
    return {(int)lo, (int)hi};
}

template <int KIND>
__device__ __forceinline__ float cache_value(const CacheView &c, bool is_v, size_t row, int d) {
    const void *base = is_v ? c.v : c.k;
    if constexpr (KIND == kCacheF32) return static_cast<const float *>(base)[row * c.width + d];
    if constexpr (KIND == kCacheBf16) return (float)static_cast<const __bf16 *>(base)[row * c.width + d];
    const uint16_t s = (is_v ? c.vd : c.kd)[row * (c.width / 32) + d / 32];
    return (float)static_cast<const int8_t *>(base)[row * c.width + d] * (float)__builtin_bit_cast(_Float16, s);
}

// One wave a query and head: a lane takes a key for the scores, then two dims
// for the sum.
template <int KIND>
__global__ __launch_bounds__(64) void cache_attn_kernel(CacheAttn a) {
    const int lane = threadIdx.x, t = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
    const int g = h / a.group;
    int r = 0;
    auto start = [&](int i) { return min(max(a.starts[i], 0), a.tokens); };
    while (r < a.requests && start(r + 1) <= t) r++;
    if (r == a.requests || start(r) > t) return;
    const int len = (int)min((long long)max(a.lens[r], 0), a.max_pages << a.cache.page_shift);
    const long long pos = (long long)len - (start(r + 1) - start(r)) + (t - start(r));
    const Seen seen = keys_seen(a, len, pos);
    const float *q = a.q + ((size_t)t * a.heads + h) * a.head_dim;
    float m = -INFINITY, l = 0.0f, o[2] = {0.0f, 0.0f};
    const int mask = (1 << a.cache.page_shift) - 1;
    for (int k0 = seen.lo; k0 < seen.hi; k0 += 64) {
        const int key = k0 + lane;
        int page = -1;
        if (key < seen.hi) page = a.table[(size_t)r * a.max_pages + (key >> a.cache.page_shift)];
        const bool live = page >= 0 && page < a.cache.slots >> a.cache.page_shift;
        const size_t row = live ? cache_row(a.cache, (page << a.cache.page_shift) + (key & mask), g) : 0;
        float s = -INFINITY;
        if (live) {
            s = 0.0f;
            for (int d = 0; d < a.head_dim; d++) s += q[d] * cache_value<KIND>(a.cache, false, row, d);
            s *= a.scale_log2;
        }
        const float mn = fmaxf(m, wave_max(s)), ref = mn == -INFINITY ? 0.0f : mn;
        const float corr = exp2f(m - ref), p = exp2f(s - ref);
        m = mn;
        l = l * corr + wave_sum(p);
        // 64 keys are summed before they meet the rest: a chain of roundings over a
        // long context stays short.
        float some[2] = {0.0f, 0.0f};
        for (int j = 0; j < 64; j++) {
            const size_t vrow = (size_t)__shfl((long long)row, j, 64);
            const float pj = __shfl(p, j, 64);
            if (!__shfl((int)live, j, 64)) continue;
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (lane + 64 * u < a.head_dim) some[u] += pj * cache_value<KIND>(a.cache, true, vrow, lane + 64 * u);
        }
#pragma unroll
        for (int u = 0; u < 2; u++) o[u] = o[u] * corr + some[u];
    }
#pragma unroll
    for (int u = 0; u < 2; u++)
        if (lane + 64 * u < a.head_dim)
            a.out[((size_t)t * a.heads + h) * a.head_dim + lane + 64 * u] = l == 0.0f ? 0.0f : o[u] / l;
}

}  // namespace

hipError_t launch_cache_attn(hipStream_t s, const CacheAttn &a) {
    const unsigned grid = (unsigned)((size_t)a.tokens * a.heads);
    if (a.cache.kind == kCacheF32) cache_attn_kernel<kCacheF32><<<grid, 64, 0, s>>>(a);
    else if (a.cache.kind == kCacheBf16) cache_attn_kernel<kCacheBf16><<<grid, 64, 0, s>>>(a);
    else cache_attn_kernel<kCacheQ8><<<grid, 64, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace vh
