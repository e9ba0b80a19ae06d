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
// rope2d's.  KIND: what the cache holds, or -1 for rotation alone.
template <int KIND>
__global__ __launch_bounds__(256) void cache_rows_kernel(CacheRows a) {
    extern __shared__ __attribute__((aligned(16))) float angles[];  // [tokens][pairs][sin, cos]
    __shared__ __attribute__((aligned(16))) float exchange[4][kU][256];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int t0 = blockIdx.x * a.per_group;
    const int nt = min(a.per_group, a.tokens - t0);
    const RopePlan &rope = a.rope;
    if (rope.pairs) {
        for (int i = tid; i < nt * rope.pairs; i += 256) {
            const int t = i / rope.pairs, p = i - t * rope.pairs;
            const double turns = (double)a.positions[(size_t)(t0 + t) * rope.axes + rope.axis[p]] * rope.turns[p];
            double sn, cs;
            sincospi(2.0 * (turns - rint(turns)), &sn, &cs);
            angles[2 * i] = (float)sn;
            angles[2 * i + 1] = (float)cs;
        }
        __syncthreads();
    }
    const int lanes = a.head_dim >> 2;        // of a row
    const int rows = 64 / lanes;              // of a group
    const int sub = lane / lanes, c = lane - sub * lanes;
    const bool used = sub < rows;
    // Of this lane's four dims: the pair (or -1), the other dim, and whether it
    // is the first of the two.
    int pair[4], other[4];
    bool first[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        pair[e] = -1;
        other[e] = 4 * c + e;
        first[e] = false;
        if (rope.pairs && used) {
            const int code = rope.dims[4 * c + e];
            if (code >= 0) {
                pair[e] = code >> 9;
                first[e] = (code >> 8) & 1;
                other[e] = code & 255;
            }
        }
    }
    const int total_rows = a.heads + 2 * a.kv_heads;
    const int groups = (total_rows + rows - 1) / rows;
    const int n = nt * groups;
    for (int base = wave; base < n; base += 4 * kU) {
        f32x4 x[kU];
        int row[kU], tok[kU];
#pragma unroll
        for (int u = 0; u < kU; u++) {
            const int idx = min(base + 4 * u, n - 1);
            tok[u] = idx / groups;
            row[u] = (idx - tok[u] * groups) * rows + sub;
            const int h = min(row[u], total_rows - 1);
            const float *src;
            if (h < a.heads) src = a.q + (size_t)(t0 + tok[u]) * a.q_token + (size_t)h * a.q_head;
            else if (h < a.heads + a.kv_heads)
                src = a.k + (size_t)(t0 + tok[u]) * a.kv_token + (size_t)(h - a.heads) * a.kv_head;
            else src = a.v + (size_t)(t0 + tok[u]) * a.kv_token + (size_t)(h - a.heads - a.kv_heads) * a.kv_head;
            x[u] = reinterpret_cast<const f32x4 *>(src)[used ? c : 0];
        }
#pragma unroll
        for (int u = 0; u < kU; u++) {
            if (base + 4 * u >= n) break;
            f32x4 y = x[u];
            if (rope.pairs) {
                float *buf = exchange[wave][u];
                reinterpret_cast<f32x4 *>(buf)[lane] = y;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                const float *mine = buf + sub * a.head_dim;
                const bool turned = row[u] < a.heads + a.kv_heads;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float *sc = angles + 2 * (tok[u] * rope.pairs + max(pair[e], 0));
                    const float w = used ? mine[other[e]] : 0.0f;
                    const float s = first[e] ? -sc[0] : sc[0];
                    const float r = add_rn(mul_rn(y[e], sc[1]), mul_rn(w, s));
                    if (turned && pair[e] >= 0) y[e] = r;
                }
            }
            const bool live = used && row[u] < total_rows;
            if (row[u] < a.heads) {
                if (live)
                    reinterpret_cast<f32x4 *>(a.q_out + (size_t)(t0 + tok[u]) * a.o_token +
                                              (size_t)row[u] * a.o_head)[c] = y;
            }
            if constexpr (KIND >= 0) {
                const int slot = a.slots[t0 + tok[u]];
                const bool write = live && row[u] >= a.heads && slot >= 0 && slot < a.cache.slots;
                const bool is_v = row[u] >= a.heads + a.kv_heads;
                const int g = row[u] - a.heads - (is_v ? a.kv_heads : 0);
                const size_t at = cache_row(a.cache, slot, g);
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
    }
}

// The rows of n slots as floats, [n][kv_heads][head_dim]; zeros where a slot is
// none of the cache's.
template <int KIND>
__global__ __launch_bounds__(256) void cache_gather_kernel(CacheView cache, const int *__restrict__ slots,
                                                           float *__restrict__ k_out, float *__restrict__ v_out,
                                                           size_t quads, int head_dim) {
    const int lanes = head_dim >> 2, per_token = 2 * cache.kv_heads * lanes;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < quads; i += (size_t)gridDim.x * 256) {
        const size_t t = i / per_token;
        const int in = (int)(i - t * per_token);
        const int row = in / lanes, c = in - row * lanes;
        const bool is_v = row >= cache.kv_heads;
        const int g = is_v ? row - cache.kv_heads : row;
        const int slot = slots[t];
        f32x4 y{0.0f, 0.0f, 0.0f, 0.0f};
        if (slot >= 0 && slot < cache.slots) {
            const size_t at = cache_row(cache, slot, g);
            const void *base = is_v ? cache.v : cache.k;
            if constexpr (KIND == kCacheF32) {
                y = reinterpret_cast<const f32x4 *>(static_cast<const float *>(base) + at * cache.width)[c];
            } else if constexpr (KIND == kCacheBf16) {
                const bf16x4 b =
                    reinterpret_cast<const bf16x4 *>(static_cast<const __bf16 *>(base) + at * cache.width)[c];
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = (float)b[e];
            } else {
                const uint32_t p =
                    reinterpret_cast<const uint32_t *>(static_cast<const int8_t *>(base) + at * cache.width)[c];
                const float d = (float)__builtin_bit_cast(
                    _Float16, (is_v ? cache.vd : cache.kd)[at * (cache.width / 32) + (c >> 3)]);
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = (float)(int8_t)(p >> (8 * e)) * d;
            }
        }
        reinterpret_cast<f32x4 *>(is_v ? v_out : k_out)[(t * cache.kv_heads + g) * lanes + c] = y;
    }
}

// Inclusive sum over the workgroup's 256 threads (tmp: 4 values of LDS, free on
// return), and the sum of all of them.
__device__ __forceinline__ long long scan256(long long v, long long *tmp, long long *all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long w = __shfl_up(v, o, 64);
        if (lane >= o) v += w;
    }
    if (lane == 63) tmp[wave] = v;
    __syncthreads();
    long long before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if (w < wave) before += tmp[w];
        sum += tmp[w];
    }
    __syncthreads();
    *all = sum;
    return v + before;
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
// whose held entries are only read.
__global__ __launch_bounds__(256) void pages_assign_kernel(PagesAssign a) {
    extern __shared__ int lds[];
    __shared__ long long tmp[4];
    int *start = lds, *first = lds + a.requests + 1;
    const int tid = threadIdx.x;
    const int mask = (1 << a.page_shift) - 1;
    long long tokens = 0, pages = 0, all = 0;
    for (int r0 = 0; r0 < a.requests; r0 += 256) {
        const int r = r0 + tid;
        const bool in = r < a.requests;
        const long long c = in ? max(a.cached[r], 0) : 0, n = in ? max(a.added[r], 0) : 0;
        const long long end = tokens + scan256(n, tmp, &all);
        tokens += all;
        // Tokens past the slot map's end are not placed.
        const long long s = min(end - n, (long long)a.tokens), placed = min(end, (long long)a.tokens) - s;
        const long long held = (c + mask) >> a.page_shift, need = (c + placed + mask) >> a.page_shift;
        const long long upto = pages + scan256(need - held, tmp, &all);
        pages += all;
        if (in) {
            start[r] = (int)s;
            first[r] = (int)min(upto - (need - held), (long long)INT32_MAX);
            if (blockIdx.x == 0) {
                a.starts[r] = (int)s;
                a.lens[r] = (int)min(c + placed, (long long)INT32_MAX);
            }
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
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const int t = blockIdx.x * 1024 + u * 256 + tid;
        if (t >= a.tokens) break;
        int slot = -1;
        if (t < last) {
            int lo = 0, hi = a.requests;  // start[lo] <= t < start[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (start[mid] <= t) lo = mid;
                else hi = mid;
            }
            const long long c = max(a.cached[lo], 0), pos = c + (t - start[lo]);
            const long long col = pos >> a.page_shift, held = (c + mask) >> a.page_shift;
            if (col < a.max_pages) {
                int *entry = a.table + (size_t)lo * a.max_pages + col;
                int page;
                if (col < held) {
                    page = *entry;
                } else {
                    const long long at = (long long)free_start + first[lo] + (col - held);
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
    // Tokens of a workgroup: as many as leave eight workgroups to a CU, so that
    // few share the forming of angles and the small calls still spread.
    a.per_group = std::min(16, std::max(1, a.tokens / 2048));
    const unsigned grid = (unsigned)((a.tokens + a.per_group - 1) / a.per_group);
    const size_t lds = (size_t)a.per_group * a.rope.pairs * 2 * sizeof(float);
    if (a.kv_heads == 0) cache_rows_kernel<-1><<<grid, 256, lds, s>>>(a);
    else if (a.cache.kind == kCacheF32) cache_rows_kernel<kCacheF32><<<grid, 256, lds, s>>>(a);
    else if (a.cache.kind == kCacheBf16) cache_rows_kernel<kCacheBf16><<<grid, 256, lds, s>>>(a);
    else cache_rows_kernel<kCacheQ8><<<grid, 256, lds, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_cache_gather(hipStream_t s, const CacheView &cache, const int *slots, float *k, float *v,
                               size_t n, size_t head_dim) {
    const size_t quads = n * 2 * cache.kv_heads * (head_dim / 4);
    if (quads == 0) return hipSuccess;
    const unsigned grid = (unsigned)std::min<size_t>((quads + 255) / 256, 16384);
    auto run = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>(cache, slots, k, v, quads, (int)head_dim); };
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
