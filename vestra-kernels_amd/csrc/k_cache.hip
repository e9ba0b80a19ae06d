// Rotary positions of several axes, and the paged cache of keys and values:
// its writes, its reads as floats, and the tables that say where they go.
//
// All of them move each byte once and compute little: HBM bounds the large
// calls, launch and load latency the small ones.
#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace vh {
namespace {

constexpr int kU = 4;  // row groups that a wave has in flight

// quantize_row_q8_0's value (src/q8_0_dot.rs:38-44): half away from zero, NaN to 0.
__device__ __forceinline__ int q8_of(float v, float inv) {
    const float q = roundf(mul_rn(v, inv));
    return isnan(q) ? 0 : (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// Sine and cosine of a number of turns, to floats.  Whole quarters go off exactly;
// what is left, at most an eighth of a turn, is an angle below pi / 4, where the power
// series to the 15th and 16th power are exact to 2^-54: the results are the
// correctly rounded ones but where a value lies within that of the middle between two
// floats.
__device__ __forceinline__ void turn_sincos(double turns, float &sn, float &cs) {
    const double r = turns - rint(turns), quarters = rint(4.0 * r);
    const double x = (r - 0.25 * quarters) * 6.283185307179586476925286766559, z = x * x;
    double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;  // 15!, 16!
    s = __builtin_fma(s, z, 1.0 / 6227020800.0);
    c = __builtin_fma(c, z, -1.0 / 87178291200.0);
    s = __builtin_fma(s, z, -1.0 / 39916800.0);
    c = __builtin_fma(c, z, 1.0 / 479001600.0);
    s = __builtin_fma(s, z, 1.0 / 362880.0);
    c = __builtin_fma(c, z, -1.0 / 3628800.0);
    s = __builtin_fma(s, z, -1.0 / 5040.0);
    c = __builtin_fma(c, z, 1.0 / 40320.0);
    s = __builtin_fma(s, z, 1.0 / 120.0);
    c = __builtin_fma(c, z, -1.0 / 720.0);
    s = __builtin_fma(s, z, -1.0 / 6.0);
    c = __builtin_fma(c, z, 1.0 / 24.0);
    s = __builtin_fma(s * z, x, x);
    c = __builtin_fma(c, z, -0.5);
    c = __builtin_fma(c, z, 1.0);
    const int q = (int)quarters & 3;
    const float fs = (float)(q & 1 ? c : s), fc = (float)(q & 1 ? s : c);
    sn = q & 2 ? -fs : fs;
    cs = q == 1 || q == 2 ? -fc : fc;
}

// Rows of one token, head_dim floats each, of which Q and K are rotated on the
// way and K and V end in their slot of the cache.
//
// A row takes head_dim / 4 lanes of four consecutive dims, so a wave holds
// 64 / (head_dim / 4) rows of a token at once and kU such groups in flight.  The
// other dim of a rotated pair is anywhere in the row (sections of any length), so
// the group's values pass through LDS of the wave's own: one 16-byte write and
// four reads a lane, no barrier.  The angles of a token are the same for all of
// its heads: the workgroup forms them once, in turns and 64 bits (a position of
// 10^6 leaves nothing of a 32-bit angle), as sine and cosine in LDS.
//
// x0' = x0 c - x1 s, x1' = x1 c + x0 s, products and sums rounded one by one, as
// rope2d's.  KIND: what the cache holds, or -1 for rotation alone.  NT: loads and
// stores that pass by the caches, for calls beyond what those hold.
//
// A small call is a chain of latencies, so the first rows and slots are asked for
// before the angles are formed.  Measured: 16 x 3457 tokens of 12 heads of 64 rotated
// into another tensor 59 us (5.8 TB/s; a streaming copy reaches 6.45); 865 tokens 4.6 us
// and one token 3.9 us, launch included.
template <int KIND, bool NT>
__global__ __launch_bounds__(256) void cache_rows_kernel(CacheRows a) {
    extern __shared__ __attribute__((aligned(16))) float angles[];  // [tokens][pairs][sin, cos]
    __shared__ __attribute__((aligned(16))) float exchange[4][kU][256];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int t0 = blockIdx.x * a.per_group;
    const int nt = min(a.per_group, a.tokens - t0);
    const RopePlan &rope = a.rope;
    const int lanes = a.head_dim >> 2;        // of a row
    const int rows = 64 / lanes;              // of a group
    const int sub = lane / lanes, c = lane - sub * lanes;
    const bool used = sub < rows;
    const int total_rows = a.heads + 2 * a.kv_heads;
    const int groups = (total_rows + rows - 1) / rows;
    const int n = nt * groups;

    f32x4 x[kU];
    int slot[kU];
    auto token_of = [&](int idx) { return min(idx, n - 1) / groups; };
    auto row_of = [&](int idx) {
        idx = min(idx, n - 1);
        return (idx - idx / groups * groups) * rows + sub;
    };
    auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < kU; u++) {
            const size_t t = t0 + token_of(base + 4 * u);
            const int h = min(row_of(base + 4 * u), total_rows - 1);
            const float *src;
            if (h < a.heads) src = a.q + t * a.q_token + (size_t)h * a.q_head;
            else if (h < a.heads + a.kv_heads) src = a.k + t * a.kv_token + (size_t)(h - a.heads) * a.kv_head;
            else src = a.v + t * a.kv_token + (size_t)(h - a.heads - a.kv_heads) * a.kv_head;
            const f32x4 *p = reinterpret_cast<const f32x4 *>(src) + (used ? c : 0);
            x[u] = NT ? __builtin_nontemporal_load(p) : *p;
            if constexpr (KIND >= 0) slot[u] = a.slots[t];
        }
    };
    // Few tokens of many rows are shared by gridDim.y workgroups.
    const int base0 = blockIdx.y * 4 * kU + wave, stride = gridDim.y * 4 * kU;
    if (base0 < n) load(base0);

    // Of this lane's four dims: the pair (or -1), the other dim, and whether it
    // is the first of the two.
    int pair[4], other[4];
    bool first[4];
    const i32x4 codes = rope.pairs ? reinterpret_cast<const i32x4 *>(rope.dims)[used ? c : 0] : i32x4{-1, -1, -1, -1};
#pragma unroll
    for (int e = 0; e < 4; e++) {
        pair[e] = codes[e] >> 9;  // -1 stays
        first[e] = (codes[e] >> 8) & 1;
        other[e] = codes[e] < 0 ? 4 * c + e : codes[e] & 255;
    }
    if (rope.pairs) {
        for (int i = tid; i < nt * rope.pairs; i += 256) {
            const int t = i / rope.pairs, p = i - t * rope.pairs;
            const int axis = (p >= rope.ends[0]) + (p >= rope.ends[1]) + (p >= rope.ends[2]);
            const double position = a.positions[(size_t)(t0 + t) * rope.axes + axis];
            turn_sincos(position * rope.turns[p], angles[2 * i], angles[2 * i + 1]);
        }
        __syncthreads();
    }
    for (int base = base0; base < n; base += stride) {
#pragma unroll
        for (int u = 0; u < kU; u++) {
            if (base + 4 * u >= n) break;
            const int tok = token_of(base + 4 * u), row = row_of(base + 4 * u);
            f32x4 y = x[u];
            if (rope.pairs) {
                float *buf = exchange[wave][u];
                reinterpret_cast<f32x4 *>(buf)[lane] = y;
                wave_sync();
                const float *mine = buf + sub * a.head_dim;
                const bool turned = row < a.heads + a.kv_heads;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float *sc = angles + 2 * (tok * rope.pairs + max(pair[e], 0));
                    const float w = used ? mine[other[e]] : 0.0f;
                    const float s = first[e] ? -sc[0] : sc[0];
                    const float r = add_rn(mul_rn(y[e], sc[1]), mul_rn(w, s));
                    if (turned && pair[e] >= 0) y[e] = r;
                }
                wave_sync();
            }
            const bool live = used && row < total_rows;
            if (row < a.heads && live) {
                f32x4 *p = reinterpret_cast<f32x4 *>(a.q_out + (size_t)(t0 + tok) * a.o_token + (size_t)row * a.o_head) + c;
                if constexpr (NT) __builtin_nontemporal_store(y, p);
                else *p = y;
            }
            if constexpr (KIND >= 0) {
                const bool write = live && row >= a.heads && slot[u] >= 0 && slot[u] < a.cache.slots;
                const bool is_v = row >= a.heads + a.kv_heads;
                const int g = row - a.heads - (is_v ? a.kv_heads : 0);
                const size_t at = cache_row(a.cache, slot[u], g);
                if constexpr (KIND == kCacheF32) {
                    if (write)
                        reinterpret_cast<f32x4 *>(static_cast<float *>(is_v ? a.cache.v : a.cache.k) +
                                                  at * a.cache.width)[c] = y;
                } else if constexpr (KIND == kCacheBf16) {
                    const bf16x4 b = {(__bf16)y[0], (__bf16)y[1], (__bf16)y[2], (__bf16)y[3]};
                    if (write)
                        reinterpret_cast<bf16x4 *>(static_cast<__bf16 *>(is_v ? a.cache.v : a.cache.k) +
                                                   at * a.cache.width)[c] = b;
                } else {
                    // A block of 32 dims is in 8 adjacent lanes (head_dim % 32 == 0).
                    float amax = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; e++) amax = q8_absmax(amax, y[e]);
                    amax = q8_absmax(amax, dpp_f32<0xb1>(amax));
                    amax = q8_absmax(amax, dpp_f32<0x4e>(amax));
                    amax = q8_absmax(amax, dpp_f32<0x141>(amax));
                    float d, inv;
                    q8_scale(amax, d, inv);
                    uint32_t packed = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) packed |= (uint32_t)(q8_of(y[e], inv) & 255) << (8 * e);
                    if (write) {
                        reinterpret_cast<uint32_t *>(static_cast<int8_t *>(is_v ? a.cache.v : a.cache.k) +
                                                     at * a.cache.width)[c] = packed;
                        if ((c & 7) == 0)
                            (is_v ? a.cache.vd : a.cache.kd)[at * (a.cache.width / 32) + (c >> 3)] =
                                __builtin_bit_cast(uint16_t, (_Float16)d);
                    }
                }
            }
        }
        if (base + stride < n) load(base + stride);
    }
}

// The rows of n slots as floats, [n][kv_heads][head_dim]; zeros where a slot is
// none of the cache's.  One token a workgroup, 16 bytes a thread, and stores that pass
// by the caches at any size: 6914 tokens of 12 heads of 64 in bf16 7.9 us (5.4 TB/s)
// against 10.6, 27656 of 8 heads of 128 43.5 against 58.7, none slower.
template <int KIND>
__global__ __launch_bounds__(256) void cache_gather_kernel(CacheView cache, const int *__restrict__ slots,
                                                           float *__restrict__ k_out, float *__restrict__ v_out,
                                                           int tokens, int head_dim) {
    const int lanes = head_dim >> 2, per_token = 2 * cache.kv_heads * lanes;
    for (int t = blockIdx.x; t < tokens; t += gridDim.x) {
        const int slot = slots[t];
        for (int in = threadIdx.x; in < per_token; in += 256) {
            const int row = in / lanes, c = in - row * lanes;
            const bool is_v = row >= cache.kv_heads;
            const int g = is_v ? row - cache.kv_heads : row;
            f32x4 y{0.0f, 0.0f, 0.0f, 0.0f};
            if (slot >= 0 && slot < cache.slots) {
                const size_t at = cache_row(cache, slot, g) * cache.width;
                const void *base = is_v ? cache.v : cache.k;
                if constexpr (KIND == kCacheF32) {
                    y = reinterpret_cast<const f32x4 *>(static_cast<const float *>(base) + at)[c];
                } else if constexpr (KIND == kCacheBf16) {
                    const bf16x4 b = reinterpret_cast<const bf16x4 *>(static_cast<const __bf16 *>(base) + at)[c];
#pragma unroll
                    for (int e = 0; e < 4; e++) y[e] = (float)b[e];
                } else {
                    const uint32_t p = reinterpret_cast<const uint32_t *>(static_cast<const int8_t *>(base) + at)[c];
                    const float d =
                        (float)__builtin_bit_cast(_Float16, (is_v ? cache.vd : cache.kd)[at / 32 + (c >> 3)]);
#pragma unroll
                    for (int e = 0; e < 4; e++) y[e] = (float)(int8_t)(p >> (8 * e)) * d;
                }
            }
            f32x4 *out = reinterpret_cast<f32x4 *>(is_v ? v_out : k_out) +
                         ((size_t)t * cache.kv_heads + g) * lanes + c;
            __builtin_nontemporal_store(y, out);
        }
    }
}

// Block tables and slot maps from the requests' lengths.
//
//     start[r] = sum of added before r            held[r] = ceil(cached / page)
//     first[r] = sum of the fresh pages before r  fresh[r] = ceil((cached + added) / page) - held[r]
//
// and token i of request r is position p = cached + i, in column p / page of the
// request's table row: a page that it holds, or the free list's entry free_start +
// first + p / page - held.  Every workgroup forms both sums over all requests (in
// LDS: 8 bytes a request, which bounds their number) and then takes 1024 tokens,
// each of which finds its request by bisection; so one launch does without a
// second that would wait for the first.  The first token of a fresh page writes the table,
// whose held entries are only read.  Latency bounds it: 6.1 us for 1024 requests with up
// to 300 new tokens each, 5.3 us for 8 with one at most, launch included.
__global__ __launch_bounds__(256) void pages_assign_kernel(PagesAssign a) {
    extern __shared__ int lds[];
    __shared__ long long tmp[4];
    int *start = lds, *first = lds + a.requests + 1;
    const int tid = threadIdx.x;
    const int mask = (1 << a.page_shift) - 1;
    long long tokens = 0, pages = 0, all = 0;
    for (int r0 = 0; r0 < a.requests; r0 += 1024) {  // four in a row a thread
        long long c[4], n[4], s[4], fresh[4], sum = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int r = r0 + 4 * tid + u;
            c[u] = r < a.requests ? max(a.cached[r], 0) : 0;
            n[u] = r < a.requests ? max(a.added[r], 0) : 0;
            sum += n[u];
        }
        long long at = tokens + scan_all<256>(sum, tmp, &all) - sum;
        tokens += all;
        sum = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            // Tokens past the slot map's end are not placed.
            s[u] = min(at, (long long)a.tokens);
            at += n[u];
            n[u] = min(at, (long long)a.tokens) - s[u];
            fresh[u] = ((c[u] + n[u] + mask) >> a.page_shift) - ((c[u] + mask) >> a.page_shift);
            sum += fresh[u];
        }
        at = pages + scan_all<256>(sum, tmp, &all) - sum;
        pages += all;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int r = r0 + 4 * tid + u;
            if (r < a.requests) {
                start[r] = (int)s[u];
                first[r] = (int)min(at, (long long)INT32_MAX);
                if (blockIdx.x == 0) {
                    a.starts[r] = (int)s[u];
                    a.lens[r] = (int)min(c[u] + n[u], (long long)INT32_MAX);
                }
            }
            at += fresh[u];
        }
    }
    const int last = (int)min(tokens, (long long)a.tokens);
    const int free_start = *a.free_start;
    if (tid == 0) {
        start[a.requests] = last;
        if (blockIdx.x == 0) {
            a.starts[a.requests] = last;
            *a.free_next = (int)min((long long)free_start + pages, (long long)INT32_MAX);
        }
    }
    __syncthreads();
    // Four tokens in a row a thread: one bisection, and then steps to the next
    // request that has any.
    const int from = blockIdx.x * 1024 + 4 * tid;
    int r = 0;
    if (from < last) {
        int hi = a.requests;  // start[r] <= from < start[hi]
        while (hi - r > 1) {
            const int mid = (r + hi) >> 1;
            if (start[mid] <= from) r = mid;
            else hi = mid;
        }
    }
    int c = 0, begin = -1;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const int t = from + u;
        if (t >= a.tokens) break;
        int slot = -1;
        if (t < last) {
            while (start[r + 1] <= t) r++;
            if (begin != start[r] || u == 0) {
                begin = start[r];
                c = max(a.cached[r], 0);
            }
            const long long pos = (long long)c + (t - begin);
            const long long col = pos >> a.page_shift, held = ((long long)c + mask) >> a.page_shift;
            if (col < a.max_pages) {
                int *entry = a.table + (size_t)r * a.max_pages + col;
                int page;
                if (col < held) {
                    page = *entry;
                } else {
                    const long long at = (long long)free_start + first[r] + (col - held);
                    page = at >= 0 && at < a.free_pages ? a.free_list[at] : -1;
                    if ((pos & mask) == 0) *entry = page;
                }
                if (page >= 0 && page < (INT32_MAX >> a.page_shift))
                    slot = (page << a.page_shift) + (int)(pos & mask);
            }
        }
        a.slots[t] = slot;
    }
}

}  // namespace

hipError_t launch_cache_rows(hipStream_t s, CacheRows a) {
    if (a.tokens == 0 || a.heads + 2 * a.kv_heads == 0) return hipSuccess;
    // Tokens of a workgroup: one pass of its 4 kU row groups, whose loads and stores
    // then overlap with other workgroups' rather than wait for the next pass (13828
    // tokens of 48 heads of 128: 97.5 us, with six tokens each 113; 55312 of 12 heads of
    // 64 rotated: 59, with 11 tokens 65), but no fewer workgroups than eight a CU (64
    // tokens at 16 each: 23.5 us against 4.3).  Below that a token's row groups are
    // spread as well (865 tokens of 48 heads of 128: 10.4 us against 11.2).
    const int per = 256 / a.head_dim, groups = (a.heads + 2 * a.kv_heads + per - 1) / per;
    a.per_group = std::min((16 + groups - 1) / groups, std::max(1, a.tokens / 2048));
    // (No more workgroups than a launch has threads for; 16 tokens then, at 2^27.)
    a.per_group = std::max(a.per_group, (a.tokens + (1 << 23) - 1) >> 23);
    const dim3 grid((unsigned)((a.tokens + a.per_group - 1) / a.per_group),
                    a.tokens < 2048 ? (groups + 4 * kU - 1) / (4 * kU) : 1);
    const size_t lds = (size_t)a.per_group * a.rope.pairs * 2 * sizeof(float);
    const bool nt = rows_pass_caches(a);
    auto run = [&](auto kernel, auto streaming) {
        if (nt) streaming<<<grid, 256, lds, s>>>(a);
        else kernel<<<grid, 256, lds, s>>>(a);
    };
    if (a.kv_heads == 0) run(cache_rows_kernel<-1, false>, cache_rows_kernel<-1, true>);
    else if (a.cache.kind == kCacheF32) run(cache_rows_kernel<kCacheF32, false>, cache_rows_kernel<kCacheF32, true>);
    else if (a.cache.kind == kCacheBf16) run(cache_rows_kernel<kCacheBf16, false>, cache_rows_kernel<kCacheBf16, true>);
    else run(cache_rows_kernel<kCacheQ8, false>, cache_rows_kernel<kCacheQ8, true>);
    return hipGetLastError();
}

hipError_t launch_cache_gather(hipStream_t s, const CacheView &cache, const int *slots, float *k, float *v,
                               size_t n, size_t head_dim) {
    if (n == 0) return hipSuccess;
    const unsigned grid = (unsigned)std::min<size_t>(n, 1 << 16);
    auto run = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>(cache, slots, k, v, (int)n, (int)head_dim); };
    if (cache.kind == kCacheF32) run(cache_gather_kernel<kCacheF32>);
    else if (cache.kind == kCacheBf16) run(cache_gather_kernel<kCacheBf16>);
    else run(cache_gather_kernel<kCacheQ8>);
    return hipGetLastError();
}

hipError_t launch_pages_assign(hipStream_t s, const PagesAssign &a) {
    const unsigned grid = (unsigned)std::max(1, (a.tokens + 1023) / 1024);
    pages_assign_kernel<<<grid, 256, (size_t)(2 * a.requests + 1) * sizeof(int), s>>>(a);
    return hipGetLastError();
}

}  // namespace vh
