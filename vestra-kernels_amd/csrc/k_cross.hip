// Keys and values of an encoder's states, stored once, and the attention of a decoder's
// queries over them (kernels.h CrossView, CrossAttn), on the f16 matrix cores.
//
// Stored: scaled by a power of two so that the largest magnitude lies in [2^14, 2^15) --
// of K over an image's head, of V over each dim of it -- a value is a half (kCrossF16),
// or two, hi = f16(v) and lo = f16(v - hi), 22 bits and lo's sign (kCrossF32).  Tokens
// that the mask leaves out are not stored, so the attention knows lengths and no mask.
//
// Products: S^T = K . Q^T and O^T += V^T . P^T with Q and P split the same way (Q by an
// exponent of its own row, P held as 2^9 p), lo . lo left out: three products of
// floats, two of halves.  Each is exact in the f32 sums of v_mfma_f32_16x16x32_f16.  A
// stored value is off by at most 2^-25 of the half's scale, so by 2^-40 of the largest
// where it is below 2^-18 of it.
//
// Layout: a block is 32 keys of a head, K and then V, in the order in which a wave wants
// them: 1 KB, 16 bytes a lane, is one operand.  Memory to LDS, LDS to registers and
// memory to registers are all linear.  Operand (c, t) of K: lane (li, lh) has dims 32 c
// + 8 lh .. + 7 of key 16 t + li.  A lane then holds its own query's scores of keys 16 t
// + 4 lh + r, which is the B operand of V^T . P^T if the 32 keys are taken in the order
// (4 lh .. + 3 of tile 0, then of tile 1): operand df of V holds those of dim 16 df + li.
//
// Work is tiles of query rows (tokens times the query heads that share a head of K and
// V), and the key steps of all tiles, end to end, in equal shares of the workgroups.  The
// lengths are on the device: every workgroup forms the partition from them.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "kernels.h"
#include "split_gemm.h"

namespace vh {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// P is held as 2^kPBits p, p up to 2^kMaxSlack where a score passes the running maximum: 2^15 at
// most, and off by at most 2^-25, so a weight by 2^-34 of the largest.  (Of 2 bits less slack
// the maxima are raised more often: 3457 queries against 3457 keys 135.4 us, 138.9.)
constexpr float kPBits = 9.0f, kMaxSlack = 6.0f;  // base 2
// From maxima of this size on a float's distance to the next is no small part of a score's to the
// maximum, and what one fma would leave of its rounding no weight.
constexpr float kFarMax = 0x1p22f;

template <int KIND>
constexpr int kParts = KIND == kCrossF32 ? 2 : 1;

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// max / sum with the lanes 16 and 32 away, on the VALU: a permlane swap of two
// copies of v leaves v in one and the partner's v in the other, in either order.
__device__ __forceinline__ void swap16(float &a, float &b) {
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ void swap32(float &a, float &b) {
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ float max_groups(float v) {
    float a = v, b = v;
    swap16(a, b);
    a = b = fmaxf(a, b);
    swap32(a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float sum_groups(float v) {
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
    return v;
}

// Two floats to two halves, and what these leave of them (the empty asm keeps the
// compiler from converting each again where a half is used).
__device__ __forceinline__ f16x2 cvt_pk_f16(float a, float b) {
    f16x2 h;
    h[0] = (_Float16)a;
    h[1] = (_Float16)b;
    uint32_t u = __builtin_bit_cast(uint32_t, h);
    asm("" : "+v"(u));
    return __builtin_bit_cast(f16x2, u);
}
__device__ __forceinline__ f16x2 residual_pk_f16(f16x2 h, float a, float b) {
    float minus = -1.0f;
    asm("" : "+s"(minus));
    return cvt_pk_f16(__builtin_fmaf((float)h[0], minus, a), __builtin_fmaf((float)h[1], minus, b));
}
__device__ __forceinline__ void split8(f32x4 a, f32x4 b, f16x8 &hi, f16x8 &lo) {
    f16x2 h[4], l[4];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        h[i] = cvt_pk_f16(a[2 * i], a[2 * i + 1]);
        l[i] = residual_pk_f16(h[i], a[2 * i], a[2 * i + 1]);
        h[2 + i] = cvt_pk_f16(b[2 * i], b[2 * i + 1]);
        l[2 + i] = residual_pk_f16(h[2 + i], b[2 * i], b[2 * i + 1]);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        hi[i] = h[i / 2][i % 2];
        lo[i] = l[i / 2][i % 2];
    }
}

__device__ __forceinline__ uint32_t finite_max(uint32_t mx, float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    return max(mx, b < 0x7f800000u ? b : 0u);
}

// ---- storing ------------------------------------------------------------------------

constexpr int kHeadGroup = 2;   // heads of a workgroup of cross_range_kernel (12 of 64, 865 tokens: of 8 8.4 us, of 2 5.2)
constexpr int kMaxChunks = 32;  // of an image's tokens there

// Of a chunk of an image's tokens: the largest finite magnitudes of K of each head and of
// V of each dim, into ranges [images][chunks][heads][1 + D]; behind the workgroups of the
// heads one that finds where the seen tokens go (kept [images][capacity], the tokens in
// order; lens).  Bound by HBM: 16 images of 3457 tokens, 8 heads of 128, 96 us, 4.7 TB/s; a frame of
// 865, 12 of 64, 5.0 us.
template <int D>
__global__ __launch_bounds__(256) void cross_range_kernel(CrossWrite w) {
    __shared__ uint32_t vmax[kHeadGroup * D], kmax[kHeadGroup];
    __shared__ long long tmp[4];
    const int tid = threadIdx.x, chunk = blockIdx.x, img = blockIdx.z;
    const int h0 = blockIdx.y * kHeadGroup, heads = min(kHeadGroup, w.view.kv_heads - h0);
    const int from = chunk * w.chunk, to = min(from + w.chunk, w.tokens);
    const int *seen = w.seen ? w.seen + (size_t)img * w.tokens : nullptr;
    if (heads <= 0) {  // a workgroup of its own
        int n = 0;
        for (int i = tid; i < from; i += 256) n += seen[i] != 0;
        long long before = 0, all = 0;
        scan_all<256>(n, tmp, &before);
        for (int i0 = from; i0 < to; i0 += 256) {
            const int i = i0 + tid;
            const bool there = i < to && seen[i] != 0;
            const long long end = before + scan_all<256>(there, tmp, &all);
            if (there) w.kept[(size_t)img * w.view.tokens + end - 1] = i;
            before += all;
        }
        if (tid == 0 && to == w.tokens) w.view.lens[img] = (int)before;
        return;
    }
    if (!seen && blockIdx.y == 0 && tid == 0 && to == w.tokens) w.view.lens[img] = w.tokens;
    for (int i = tid; i < kHeadGroup * D; i += 256) vmax[i] = 0;
    if (tid < kHeadGroup) kmax[tid] = 0;
    __syncthreads();
    const int per = w.head_dim / 4, columns = heads * per;
    static_assert(kHeadGroup * D / 4 <= 256, "a thread for each column");
    int rows = 1;  // tokens at once
    while (rows * 2 * columns <= 256) rows *= 2;
    const int c = tid % columns, first = tid / columns;
    if (first < rows) {
        const int h = c / per, d = 4 * (c % per);
        const size_t off = (size_t)img * w.kv_image + (h0 + h) * w.kv_head + d;
        uint32_t km = 0, vm[4] = {0, 0, 0, 0};
        // Eight tokens at a time, the last one again past the end: no load waits in a branch.
        for (int t0 = from + first; t0 < to; t0 += 8 * rows) {
            f32x4 k[8], v[8];
            int live[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const int t = min(t0 + u * rows, to - 1);
                k[u] = *reinterpret_cast<const f32x4 *>(w.k + off + t * w.kv_token);
                v[u] = *reinterpret_cast<const f32x4 *>(w.v + off + t * w.kv_token);
                live[u] = seen ? seen[t] : 1;
            }
#pragma unroll
            for (int u = 0; u < 8; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    km = finite_max(km, live[u] ? k[u][i] : 0.0f);
                    vm[i] = finite_max(vm[i], live[u] ? v[u][i] : 0.0f);
                }
        }
        atomicMax(&kmax[h], km);
#pragma unroll
        for (int i = 0; i < 4; i++) atomicMax(&vmax[h * D + d + i], vm[i]);
    }
    __syncthreads();
    uint32_t *out = w.ranges + (((size_t)img * gridDim.x + chunk) * w.view.kv_heads + h0) * (1 + D);
    for (int i = tid; i < heads * (1 + D); i += 256) {
        const int h = i / (1 + D), d = i % (1 + D);
        out[i] = d ? vmax[h * D + d - 1] : kmax[h];
    }
}

template <bool NT>
__device__ __forceinline__ f32x4 ld4(const float *p) {
    const f32x4 *q = reinterpret_cast<const f32x4 *>(p);
    return NT ? __builtin_nontemporal_load(q) : *q;
}

// Four halves of column li of a 4 x 16 tile of halves in LDS, whose row r is in the lanes 4 r
// .. 4 r + 3 of each 16-lane group (lane i gives the address of row i / 4, columns 4 (i %
// 4) .. + 3, and receives column i).
__device__ __forceinline__ f16x4 read_tr(const char *p) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) s16x4 *)p));
}

// 128 keys of an image's head to their blocks, a block a wave; zeros behind the last key.
// Rows are read whole; V^T comes from its rows of halves in LDS by transposing reads.  Bound by HBM: 16
// images of 3457 tokens, 8 heads of 128, to one half 118 us, 5.6 TB/s; a frame of 865 tokens, 12 of
// 64, to two 7.5 us, the ranges, a row and its blocks one after the other.
template <int KIND, int D, bool NT>
__global__ __launch_bounds__(256) void cross_write_kernel(CrossWrite w) {
    constexpr int NP = kParts<KIND>, C = D / 32, DF = D / 16, PLANE = 32 * D * 2;
    constexpr int LPR = D / 4, RPP = 64 / LPR, PASSES = 32 / RPP;  // lanes of a row of V, rows of a pass
    __shared__ __attribute__((aligned(16))) int exps[4 + D];  // of K, then (from 4 on) of V's dims
    __shared__ __attribute__((aligned(16))) char planes[4][NP * PLANE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, lh = lane >> 4;
    const int g = blockIdx.y, img = blockIdx.z, len = w.view.lens[img];
    if ((int)blockIdx.x * 128 >= len && blockIdx.x) return;
    const int block = blockIdx.x * 4 + wave, key0 = block * 32, last = max(len - 1, 0);
    const bool any = (int)blockIdx.x * 128 < len, full = key0 + 32 <= len && w.head_dim == D;
    const int *kept = w.seen ? w.kept + (size_t)img * w.view.tokens : nullptr;
    // Loads are of the nearest key and dims there are; what was not asked for becomes zero.
    auto token = [&](int key) { return kept ? kept[min(key, last)] : min(key, last); };
    const size_t off = (size_t)img * w.kv_image + g * w.kv_head;
    f32x4 k[2][C][2];
    if (any) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const float *row = w.k + off + token(key0 + 16 * t + li) * w.kv_token;
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int e = 0; e < 2; e++) k[t][c][e] = ld4<NT>(row + min(32 * c + 8 * lh + 4 * e, w.head_dim - 4));
        }
    }
    for (int i = tid; i < 1 + D; i += 256) {
        const uint32_t *r = w.ranges + ((size_t)img * w.chunks * w.view.kv_heads + g) * (1 + D) + i;
        uint32_t mx = 0;
        uint32_t some[kMaxChunks];  // all at once
#pragma unroll
        for (int c = 0; c < kMaxChunks; c++) some[c] = r[(size_t)min(c, w.chunks - 1) * w.view.kv_heads * (1 + D)];
#pragma unroll
        for (int c = 0; c < kMaxChunks; c++) mx = max(mx, some[c]);
        const int e = split_exponent(mx);
        exps[i ? 3 + i : 0] = e;
        if (blockIdx.x == 0) {
            if (i == 0) w.view.k_exp[(size_t)img * w.view.kv_heads + g] = e;
            else w.view.v_exp[((size_t)img * w.view.kv_heads + g) * D + i - 1] = e;
        }
    }
    __syncthreads();
    if (!any) return;
    char *out = w.view.at(img, g) + (size_t)block * cross_block_bytes(KIND, D) + lane * 16;
    const int ke = exps[0];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int c = 0; c < C; c++) {
            f32x4 x[2];
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int i = 0; i < 4; i++) x[e][i] = __builtin_ldexpf(k[t][c][e][i], -ke);
            if (!full) {
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (key0 + 16 * t + li >= len || 32 * c + 8 * lh + 4 * e >= w.head_dim)
                        x[e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            f16x8 hi, lo;
            split8(x[0], x[1], hi, lo);
            *reinterpret_cast<f16x8 *>(out + (2 * c + t) * NP * 1024) = hi;
            if constexpr (NP == 2) *reinterpret_cast<f16x8 *>(out + ((2 * c + t) * NP + 1) * 1024) = lo;
        }
    const int vrow = lane / LPR, vd = 4 * (lane % LPR);
    const i32x4 ve = *reinterpret_cast<const i32x4 *>(exps + 4 + vd);
    char *plane = planes[wave];
    f32x4 v[PASSES];
#pragma unroll
    for (int p = 0; p < PASSES; p++)
        v[p] = ld4<NT>(w.v + off + token(key0 + p * RPP + vrow) * w.kv_token + min(vd, w.head_dim - 4));
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
        const int row = p * RPP + vrow;
#pragma unroll
        for (int i = 0; i < 4; i++) v[p][i] = __builtin_ldexpf(v[p][i], -ve[i]);
        if (!full && (key0 + row >= len || vd >= w.head_dim)) v[p] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        f16x2 h[2], l[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            h[i] = cvt_pk_f16(v[p][2 * i], v[p][2 * i + 1]);
            l[i] = residual_pk_f16(h[i], v[p][2 * i], v[p][2 * i + 1]);
        }
        *reinterpret_cast<f16x4 *>(plane + (row * D + vd) * 2) = f16x4{h[0][0], h[0][1], h[1][0], h[1][1]};
        if constexpr (NP == 2)
            *reinterpret_cast<f16x4 *>(plane + PLANE + (row * D + vd) * 2) = f16x4{l[0][0], l[0][1], l[1][0], l[1][1]};
    }
    wave_sync();
    const char *from = plane + ((4 * lh + (li >> 2)) * D + 4 * (li & 3)) * 2;
#pragma unroll
    for (int df = 0; df < DF; df++)
#pragma unroll
        for (int p = 0; p < NP; p++) {
            const f16x4 a = read_tr(from + p * PLANE + df * 32), b = read_tr(from + p * PLANE + 16 * D * 2 + df * 32);
            *reinterpret_cast<f16x8 *>(out + ((2 * C + df) * NP + p) * 1024) =
                __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
}

// What is stored, as floats [images][capacity][heads][head_dim]; zeros behind the last key.  Bound by
// HBM: 16 images of 3457 tokens, 8 heads of 128, from one half 103 us, 6.6 TB/s; a frame 5.2 us.
template <int KIND, int D, bool NT>
__global__ __launch_bounds__(256) void cross_read_kernel(CrossView view, int head_dim, float *k, float *v, int *lens) {
    constexpr int NP = kParts<KIND>, C = D / 32, ROW = 36;  // floats of a row of 32 dims in LDS
    __shared__ __attribute__((aligned(16))) float stage[4][32 * ROW];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, lh = lane >> 4;
    const int g = blockIdx.y, img = blockIdx.z, len = view.lens[img];
    if (lens && tid == 0 && g == 0 && blockIdx.x == 0) lens[img] = len;
    const int block = blockIdx.x * 4 + wave, key0 = block * 32;
    if (key0 >= view.tokens) return;
    const char *in = view.at(img, g) + (size_t)block * cross_block_bytes(KIND, D) + lane * 16;
    // A block behind the last key is not read: its place is, and left out.
    const bool any = key0 < len;
    if (!any) in = view.at(img, g) + lane * 16;
    const int ke = view.k_exp[(size_t)img * view.kv_heads + g];
    const int *ves = view.v_exp + ((size_t)img * view.kv_heads + g) * D;
    auto get = [&](int operand, float (&x)[8]) {
        const f16x8 hi = *reinterpret_cast<const f16x8 *>(in + operand * NP * 1024);
        const f16x8 lo = *reinterpret_cast<const f16x8 *>(in + (operand * NP + NP - 1) * 1024);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)hi[i] + (NP == 2 ? (float)lo[i] : 0.0f);
    };
    auto put = [&](float *to, int key, int d, f32x4 y) {
        if (key >= view.tokens || d >= head_dim) return;
        if (key >= len) y = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        f32x4 *at = reinterpret_cast<f32x4 *>(to + (((size_t)img * view.tokens + key) * view.kv_heads + g) * head_dim + d);
        if (NT) __builtin_nontemporal_store(y, at);
        else *at = y;
    };
    float *mine = stage[wave];
    // 32 dims at a time through LDS, so that rows are written in whole lines.
    auto rows = [&](float *to, int d0) {
        wave_sync();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int key = 8 * i + (lane >> 3), d = 4 * (lane & 7);
            put(to, key0 + key, d0 + d, *reinterpret_cast<const f32x4 *>(mine + key * ROW + d));
        }
        wave_sync();
    };
#pragma unroll
    for (int c = 0; c < C; c++) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            float x[8];
            get(2 * c + t, x);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                f32x4 y;
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = __builtin_ldexpf(x[4 * e + i], ke);
                *reinterpret_cast<f32x4 *>(mine + (16 * t + li) * ROW + 8 * lh + 4 * e) = y;
            }
        }
        rows(k, 32 * c);
    }
#pragma unroll
    for (int c = 0; c < C; c++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float x[8];
            get(2 * C + 2 * c + h, x);
            const int ve = ves[32 * c + 16 * h + li];
#pragma unroll
            for (int j = 0; j < 8; j++)
                mine[(16 * (j / 4) + 4 * lh + j % 4) * ROW + 16 * h + li] = __builtin_ldexpf(x[j], ve);
        }
        rows(v, 32 * c);
    }
}

// ---- the partition --------------------------------------------------------------------

// What a tile costs besides its key steps, in steps: queries fetched, first loads waited
// for, output written.
constexpr int kTileCost = 2;

// A tile of query rows: image, head of K and V, its rows.
struct Tile {
    int img, g, row, rows, len, steps;
};

template <int BM>
__device__ __forceinline__ Tile tile_of(const CrossAttn &a, int img, int len, int index, int step) {
    Tile t;
    t.img = img;
    t.g = index / a.tiles;
    t.row = (index - t.g * a.tiles) * BM;
    t.rows = min(BM, a.queries * a.group - t.row);
    t.len = len;
    t.steps = (len + step - 1) / step;
    return t;
}

// Where a tile's first step is among its units (of one without steps, the last): the share that has
// it is the first to work on the tile, so that no workgroup begins one for its cost alone.
__device__ __forceinline__ int first_unit(int cost) { return min(kTileCost, cost - 1); }

// Steps of a tile of an image, with what it costs itself.
__device__ __forceinline__ int cost_of(const CrossAttn &a, int img, int step) {
    return (a.view.lens[img] + step - 1) / step + kTileCost;
}

// Sums over the images, and in `base` and `where` the image that unit `at(total)` is in
// and the units before it.
template <int THREADS, class F>
__device__ __forceinline__ long long find_image(const CrossAttn &a, int step, F at, int &where, long long &base) {
    __shared__ long long tmp[THREADS / 64], found[2];
    const long long per = (long long)a.tiles * a.view.kv_heads;
    if (a.images == 1) {
        const long long total = per * cost_of(a, 0, step);
        at(total);
        where = 0;
        base = 0;
        return total;
    }
    long long total = 0, all = 0, end = 0, cost = 0;
    for (int i0 = 0; i0 < a.images; i0 += THREADS) {
        const int i = i0 + threadIdx.x;
        cost = i < a.images ? per * cost_of(a, i, step) : 0;
        end = total + scan_all<THREADS>(cost, tmp, &all);
        total += all;
    }
    const long long unit = at(total);
    if (threadIdx.x == 0) found[0] = -1;
    __syncthreads();
    if (a.images <= THREADS) {
        if (end - cost <= unit && unit < end) {
            found[0] = threadIdx.x;
            found[1] = end - cost;
        }
    } else {
        long long before = 0;
        for (int i0 = 0; i0 < a.images; i0 += THREADS) {
            const int i = i0 + threadIdx.x;
            cost = i < a.images ? per * cost_of(a, i, step) : 0;
            end = before + scan_all<THREADS>(cost, tmp, &all);
            before += all;
            if (end - cost <= unit && unit < end) {
                found[0] = i;
                found[1] = end - cost;
            }
        }
    }
    __syncthreads();
    where = (int)found[0];
    base = found[1];
    return total;
}

// ---- parts ------------------------------------------------------------------------------

// Where the last workgroup of a tile joins them (HERE) they are read and written past the L2
// of an XCD (sc1), as the workgroups of a tile may be on several; a launch of its own
// sees them anyway.
template <bool HERE>
struct Parts {
    __amdgpu_buffer_rsrc_t base;
    __device__ __forceinline__ explicit Parts(const CrossAttn &a)
        : base(__builtin_amdgcn_make_buffer_rsrc(a.parts, 0, 0xffffffff, 0x00027000)) {}
    static constexpr int kAgent = HERE ? 16 : 0;
    __device__ __forceinline__ void put(uint32_t at, f32x4 v) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), base, at, 0, kAgent);
    }
    __device__ __forceinline__ void put(uint32_t at, float x, float y) const {
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(x), __float_as_uint(y)}, base, at, 0, kAgent);
    }
    __device__ __forceinline__ f32x4 four(uint32_t at) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(base, at, 0, kAgent));
    }
    __device__ __forceinline__ u32x2 two(uint32_t at) const {
        return __builtin_amdgcn_raw_buffer_load_b64(base, at, 0, kAgent);
    }
};
// Offsets in bytes of row `in` of part x: [2 shares][BM][D] sums, then [2 shares][BM]
// maxima and sums of weights.
template <int BM, int D>
__device__ __forceinline__ uint32_t sums_at(uint32_t x, int in) {
    return (x * BM + in) * (D * 4);
}
template <int BM, int D>
__device__ __forceinline__ uint32_t weights_at(const CrossAttn &a, uint32_t x, int in) {
    return 2u * a.shares * BM * D * 4 + (x * BM + in) * 8;
}

// Exponents of V's dims d .. d + 3.  Asked for before the sums are there, as a row that waited for them
// at its end would wait for memory once more (54 images of 44 tokens, 40 / 10 heads of 100, 9
// queries 34.4 us, so 28.9; one query against 3460 tokens 9.6 and 9.2).
template <int D>
__device__ __forceinline__ i32x4 dim_exponents(const CrossAttn &a, const Tile &t, int d) {
    return *reinterpret_cast<const i32x4 *>(a.view.v_exp + ((size_t)t.img * a.view.kv_heads + t.g) * D + d);
}

// Row `in` of a tile, four dims from d on: the result, or a workgroup's part of it.
template <int BM, int D, bool HERE>
__device__ __forceinline__ void put_row(const CrossAttn &a, const Tile &t, int part, int in, int d, i32x4 e, f32x4 v,
                                        float m, float l) {
    if (in >= t.rows) return;
    if (part < 0) {
        if (d >= a.head_dim) return;
        const int row = t.row + in, token = row / a.group, head = t.g * a.group + row % a.group;
        const float inv = 1.0f / l;
        f32x4 y;
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = l == 0.0f ? 0.0f : __builtin_ldexpf(v[i] * inv, e[i]);
        *reinterpret_cast<f32x4 *>(a.out + t.img * a.q_image + token * a.q_token + head * a.q_head + d) = y;
    } else {
        const Parts<HERE> parts(a);
        parts.put(sums_at<BM, D>(part, in) + 4 * d, v);
        if (d == 0) parts.put(weights_at<BM, D>(a, part, in), m, l);
    }
}

// A row's four dims of a part, or of several: O on the maximum m, and the sum of weights.
struct Sums {
    float m, l;
    f32x4 y;
    __device__ __forceinline__ void join(const Sums &b) {
        const float mn = fmaxf(m, b.m);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        const float fb = b.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(b.m - mn);
        m = mn;
        l = l * f + b.l * fb;
        y = y * f + b.y * fb;
    }
};

// The parts of shares w0 .. w1 (of w0 the one at part0) become the tile's rows first .. to - 1.  Of the
// workgroup's groups of D / 4 lanes (a group holds a row) as many share a row as the rows
// leave: a single query's parts are summed by all of them.
template <int BM, int D, int THREADS, bool HERE>
__device__ void join_parts(const CrossAttn &a, const Tile &t, int w0, int w1, int part0, int first, int to, char *smem) {
    Sums *some = reinterpret_cast<Sums *>(smem);
    const Parts<HERE> parts(a);
    constexpr int LANES = D / 4, GROUPS = THREADS / LANES;
    int rows = 1;  // at once
    while (rows < GROUPS && rows < to - first) rows *= 2;
    const int sharers = GROUPS / rows;
    const int group = threadIdx.x / LANES, d = 4 * (threadIdx.x % LANES);
    const i32x4 e = dim_exponents<D>(a, t, d);
    for (int in = first + group % rows; in < first + (to - first + rows - 1) / rows * rows; in += rows) {
        auto part = [&](int w) {
            const int x = w == w0 ? part0 : 2 * w, row = min(in, to - 1);
            const u32x2 ml = parts.two(weights_at<BM, D>(a, x, row));
            return Sums{__uint_as_float(ml[0]), __uint_as_float(ml[1]), parts.four(sums_at<BM, D>(x, row) + 4 * d)};
        };
        Sums sum{-INFINITY, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
        for (int w = w0 + group / rows; w <= w1; w += 4 * sharers) {
            Sums x[4];
#pragma unroll
            for (int u = 0; u < 4; u++) x[u] = part(min(w + u * sharers, w1));
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (w + u * sharers <= w1) sum.join(x[u]);
        }
        if (sharers > 1) {  // all rows at once
            some[threadIdx.x] = sum;
            __syncthreads();
            if (group < rows)
                for (int i = 1; i < sharers; i++) sum.join(some[threadIdx.x + i * rows * LANES]);
        }
        if (group < rows && in < to) put_row<BM, D, HERE>(a, t, -1, in, d, e, sum.y, sum.m, sum.l);
    }
}

// Walks this workgroup's steps tile by tile: f(tile, first step, steps, part).  Without room
// for parts (a.parts null) every workgroup takes whole tiles.  HERE: of the workgroups that
// hold a part of a tile the one that is done last joins them, in the order of the shares.
// They count in the counter of the tile's first share (of which it is the last tile, so no
// other counts there), zero before and after.
template <int BM, int STEP, int THREADS, int D, bool HERE, class F>
__device__ __forceinline__ void walk(const CrossAttn &a, char *smem, F f) {
    __shared__ int is_last;
    const int w = (blockIdx.x & 7) * (a.shares >> 3) + (blockIdx.x >> 3);  // neighbours on one XCD
    const int per = a.tiles * a.view.kv_heads;
    if (!a.parts) {
        const long long items = (long long)per * a.images;
        for (long long at = w; at < items; at += a.shares) {
            const int img = (int)(at / per);
            const Tile t = tile_of<BM>(a, img, uniform(a.view.lens[img]), (int)(at - (long long)img * per), STEP);
            f(t, 0, t.steps, -1);
        }
        return;
    }
    int img = 0;
    long long base = 0, share = 1;
    const long long total = find_image<THREADS>(a, STEP, [&](long long all) {
        share = max(1ll, (all + a.shares - 1) / a.shares);
        return w * share;
    }, img, base);
    long long at = w * share;
    const long long end = min(at + share, total);
    if (at >= end) return;
    img = uniform(img);
    int len = uniform(a.view.lens[img]), cost = (len + STEP - 1) / STEP + kTileCost;
    int index = uniform((int)((at - base) / cost)), into = uniform((int)((at - base) - (long long)index * cost));
    for (bool first = true; at < end; first = false) {
        const Tile t = tile_of<BM>(a, img, len, index, STEP);
        const int steps = uniform((int)min(end - at, (long long)cost - into));
        const long long begin = at - into;
        if (begin + first_unit(cost) < end) {
            const bool whole = begin + first_unit(cost) >= w * share && into + steps == cost;
            const int from = max(into - kTileCost, 0), to = max(into + steps - kTileCost, 0);
            f(t, from, to - from, whole ? -1 : 2 * w + (first ? 0 : 1));
            if (HERE && !whole) {
                const int w0 = uniform((int)((begin + first_unit(cost)) / share));
                const int w1 = uniform((int)((begin + cost - 1) / share));
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's parts are out
                __syncthreads();
                if (threadIdx.x == 0) {
                    unsigned *counter = a.counters + w0;
                    is_last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                              (unsigned)(w1 - w0);
                    if (is_last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                __syncthreads();
                if (is_last) {
                    join_parts<BM, D, THREADS, true>(a, t, w0, w1, 2 * w0 + (begin > w0 * share ? 1 : 0), 0, t.rows, smem);
                    __syncthreads();
                }
            }
        }
        at += steps;
        into = 0;
        if (++index == per) {
            index = 0;
            if (++img < a.images) {
                len = uniform(a.view.lens[img]);
                cost = (len + STEP - 1) / STEP + kTileCost;
            }
        }
    }
}

// ---- one wave's arithmetic --------------------------------------------------------------

// QT tiles of 16 queries: their operands, running maxima and sums, and O^T: o[df][u][r] =
// O[query 16 u + li][16 df + 4 lh + r].
template <int KIND, int D, int QT>
struct Queries {
    static constexpr int C = D / 32, DF = D / 16, NP = kParts<KIND>;
    f16x8 qh[QT][C], ql[QT][C];
    f32x4 o[DF][QT];
    float m[QT], l[QT], scale[QT];
    bool far;  // whether a lane has a maximum past kFarMax

    // Rows first .. first + 16 QT - 1 of the tile (rows past its end: zeros).
    __device__ __forceinline__ void load(const CrossAttn &a, const Tile &t, int first, int li, int lh) {
        far = false;
        const int ke = a.view.k_exp[(size_t)t.img * a.view.kv_heads + t.g];
#pragma unroll
        for (int u = 0; u < QT; u++) {
            const int in = first + 16 * u + li;
            const bool there = in < t.rows;
            const int row = t.row + (there ? in : 0), token = row / a.group, head = t.g * a.group + row % a.group;
            const float *src = a.q + t.img * a.q_image + token * a.q_token + head * a.q_head;
            f32x4 x[C][2];
            uint32_t mx = 0;
            // Of many rows from the nearest dims there are, so that no load waits in a branch (865 queries of
            // 12 heads of 64 against 865 keys 26.9 us, so 26.3, against 3300 41.3 and 40.4); of few, whose
            // K is in flight, that costs registers (16 images of 5000 tokens, two halves of 128, 109 and 119).
            constexpr bool kAll = QT > 1;
            const f32x4 zero{0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (kAll) {
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        x[c][e] = *reinterpret_cast<const f32x4 *>(src + min(32 * c + 8 * lh + 4 * e, a.head_dim - 4));
            }
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int d = 32 * c + 8 * lh + 4 * e;
                    if constexpr (kAll) x[c][e] = there && d < a.head_dim ? x[c][e] : zero;
                    else x[c][e] = there && d < a.head_dim ? *reinterpret_cast<const f32x4 *>(src + d) : zero;
#pragma unroll
                    for (int i = 0; i < 4; i++) mx = finite_max(mx, x[c][e][i]);
                }
            mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16, 64));
            mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, 64));
            const int e = split_exponent(mx);
#pragma unroll
            for (int c = 0; c < C; c++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[c][0][i] = __builtin_ldexpf(x[c][0][i], -e);
                    x[c][1][i] = __builtin_ldexpf(x[c][1][i], -e);
                }
                split8(x[c][0], x[c][1], qh[u][c], ql[u][c]);
            }
            // Kept off zero and infinity: a masked score (-inf) stays -inf.
            scale[u] = fminf(fmaxf(__builtin_ldexpf(a.scale_log2, ke + e), 0x1p-126f), 0x1p127f);
            m[u] = -INFINITY;
            l[u] = 0.0f;
#pragma unroll
            for (int df = 0; df < DF; df++) o[df][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    // Scores of 32 keys, the small products first; k(operand): NP consecutive operands.
    template <class F>
    __device__ __forceinline__ void scores(f32x4 (&s)[2][QT], F k) const {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int u = 0; u < QT; u++) s[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < C; c++) {
            f16x8 f[2][NP];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int p = 0; p < NP; p++) f[t][p] = k((2 * c + t) * NP + p);
            if constexpr (NP == 2)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int u = 0; u < QT; u++) s[t][u] = mfma16x16x32_f16(f[t][1], qh[u][c], s[t][u]);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int u = 0; u < QT; u++) s[t][u] = mfma16x16x32_f16(f[t][0], ql[u][c], s[t][u]);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int u = 0; u < QT; u++) s[t][u] = mfma16x16x32_f16(f[t][0], qh[u][c], s[t][u]);
        }
    }

    // Keys from `left` on are behind the last.
    __device__ __forceinline__ void mask(f32x4 (&s)[2][QT], int left, int lh) const {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (16 * t + 4 * lh + r >= left)
#pragma unroll
                    for (int u = 0; u < QT; u++) s[t][u][r] = -INFINITY;
    }

    // Brings the maxima up to those of H times 32 keys' scores.  They are only raised where
    // a score passes one by kMaxSlack, so most steps need no correction.
    template <int H>
    __device__ __forceinline__ void raise(const f32x4 (&s)[H][2][QT]) {
        float mx[QT];
        bool over = false;
#pragma unroll
        for (int u = 0; u < QT; u++) {
            float v = s[0][0][u][0];
#pragma unroll
            for (int h = 0; h < H; h++) {
                v = fmaxf(fmaxf(v, s[h][0][u][0]), s[h][0][u][1]);
                v = fmaxf(fmaxf(v, s[h][0][u][2]), s[h][0][u][3]);
                v = fmaxf(fmaxf(v, s[h][1][u][0]), s[h][1][u][1]);
                v = fmaxf(fmaxf(v, s[h][1][u][2]), s[h][1][u][3]);
            }
            mx[u] = v * scale[u];
            over |= mx[u] - m[u] > kMaxSlack;
        }
        if (__any(over)) {
            bool past = false;
#pragma unroll
            for (int u = 0; u < QT; u++) {
                const float mn = fmaxf(m[u], max_groups(mx[u]));
                const float corr = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[u] - mn);
                m[u] = mn;
                past |= mn != -INFINITY && fabsf(mn) >= kFarMax;
                l[u] *= corr;
#pragma unroll
                for (int df = 0; df < DF; df++) o[df][u] *= corr;
            }
            far = __any(past);
        }
    }

    // Where a maximum is past kFarMax the scores become their distances to it, rounded as it was: no
    // more than the weights' range is left of its rounding.
    template <int H>
    __device__ __forceinline__ void near(f32x4 (&s)[H][2][QT], float (&by)[QT], float (&off)[QT]) const {
#pragma clang fp contract(off)
#pragma unroll
        for (int u = 0; u < QT; u++) {
            by[u] = scale[u];
            off[u] = kPBits - (m[u] == -INFINITY ? 0.0f : m[u]);
        }
        if (!far) return;
#pragma unroll
        for (int u = 0; u < QT; u++) {
            const float top = m[u] == -INFINITY ? 0.0f : m[u];
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float at = s[h][t][u][r] * scale[u];
                        s[h][t][u][r] = at - top;
                    }
            by[u] = 1.0f;
            off[u] = kPBits;
        }
    }

    // The scores of 32 keys become their weights, which are summed and split.
    __device__ __forceinline__ void weights(f32x4 (&s)[2][QT], const float (&by)[QT], const float (&off)[QT],
                                            f16x8 (&ph)[QT], f16x8 (&pl)[QT]) {
#pragma unroll
        for (int u = 0; u < QT; u++) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    s[t][u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][u][r], by[u], off[u]));
            l[u] += ((s[0][u][0] + s[0][u][1]) + (s[0][u][2] + s[0][u][3])) +
                    ((s[1][u][0] + s[1][u][1]) + (s[1][u][2] + s[1][u][3]));
            split8(s[0][u], s[1][u], ph[u], pl[u]);
        }
    }

    // O^T += V^T . P^T for 32 keys; v(operand) as in scores.
    template <class F>
    __device__ __forceinline__ void add(const f16x8 (&ph)[QT], const f16x8 (&pl)[QT], F v) {
#pragma unroll
        for (int d0 = 0; d0 < DF; d0 += 2) {
            f16x8 f[2][NP];
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int p = 0; p < NP; p++) f[k][p] = v((d0 + k) * NP + p);
            if constexpr (NP == 2)
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int u = 0; u < QT; u++) o[d0 + k][u] = mfma16x16x32_f16(f[k][1], ph[u], o[d0 + k][u]);
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int u = 0; u < QT; u++) o[d0 + k][u] = mfma16x16x32_f16(f[k][0], pl[u], o[d0 + k][u]);
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int u = 0; u < QT; u++) o[d0 + k][u] = mfma16x16x32_f16(f[k][0], ph[u], o[d0 + k][u]);
        }
    }
};

// ---- few rows: 16 a tile, each of the four waves its own 32 keys of a step ----------------
// No barrier in the loop; blocks from memory to registers, K a step ahead, past the caches.  Bound by
// HBM where the states are long (48 images of 5000 tokens, 32 / 8 heads of 128, in one half: 159 us, 6.2
// TB/s), else by a chain of latencies (one query, 12 heads of 64, 3460 keys 9.2 us).

template <int D>
constexpr int few_wave_bytes() {
    return 16 * D * 4 + 128;  // the wave's O, maxima and sums
}

template <int KIND, int D>
__global__ __launch_bounds__(256, 2) void cross_few_kernel(CrossAttn a) {
    constexpr int BM = 16, STEP = 128, NP = kParts<KIND>, C = D / 32, DF = D / 16;
    constexpr int BLOCK = cross_block_bytes(KIND, D), WAVE = few_wave_bytes<D>();
    __shared__ __attribute__((aligned(16))) char smem[4 * WAVE];
    static_assert(4 * WAVE >= 256 * sizeof(Sums), "room for join_parts");
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lh = lane >> 4;
    const int wave = uniform(tid >> 6);
    walk<BM, STEP, 256, D, true>(a, smem, [&](const Tile &t, int step0, int steps, int part) {
        const char *base = a.view.at(t.img, t.g) + lane * 16;
        auto load = [&](int step, int operand) {
            const size_t at = (size_t)(step * 4 + wave) * BLOCK + operand * 1024;
            return __builtin_nontemporal_load(reinterpret_cast<const f16x8 *>(base + at));
        };
        // K of this step is in registers; V is loaded before the scores are formed, the next K
        // before the weights meet V.  The last step's blocks behind the last key are left out.
        const int mine = steps - ((step0 + steps - 1) * STEP + 32 * wave >= t.len ? 1 : 0);
        f16x8 k[2 * C * NP], v[DF * NP];
        if (mine > 0) {
#pragma unroll
            for (int i = 0; i < 2 * C * NP; i++) k[i] = load(step0, i);
        }
        i32x4 e[D / 64];
#pragma unroll
        for (int i = 0; i < D / 64; i++) e[i] = dim_exponents<D>(a, t, 64 * i + 4 * (tid & 15));
        Queries<KIND, D, 1> w;
        w.load(a, t, 0, li, lh);
        for (int i = 0; i < mine; i++) {
            const int step = step0 + i, left = t.len - (step * 4 + wave) * 32;
#pragma unroll
            for (int x = 0; x < DF * NP; x++) v[x] = load(step, 2 * C * NP + x);
            f32x4 s[1][2][1];
            w.scores(s[0], [&](int x) { return k[x]; });
            const int next = min(step + 1, step0 + mine - 1);
#pragma unroll
            for (int x = 0; x < 2 * C * NP; x++) k[x] = load(next, x);
            if (left < 32) w.mask(s[0], left, lh);
            w.raise(s);
            float by[1], off[1];
            w.near(s, by, off);
            f16x8 ph[1], pl[1];
            w.weights(s[0], by, off, ph, pl);
            w.add(ph, pl, [&](int x) { return v[x]; });
        }
        // The four waves' sums, each on its own maximum, joined by all threads.
        float *o = reinterpret_cast<float *>(smem + wave * WAVE);
#pragma unroll
        for (int df = 0; df < DF; df++) *reinterpret_cast<f32x4 *>(o + li * D + 16 * df + 4 * lh) = w.o[df][0];
        const float l = sum_groups(w.l[0]);
        if (lh == 0) {
            o[16 * D + 2 * li] = w.m[0];
            o[16 * D + 2 * li + 1] = l;
        }
        __syncthreads();
        const int row = tid >> 4;
        float m = -INFINITY, sum = 0.0f, f[4];
#pragma unroll
        for (int x = 0; x < 4; x++) m = fmaxf(m, reinterpret_cast<float *>(smem + x * WAVE)[16 * D + 2 * row]);
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const float *y = reinterpret_cast<float *>(smem + x * WAVE) + 16 * D + 2 * row;
            f[x] = y[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(y[0] - m);
            sum += y[1] * f[x];
        }
#pragma unroll
        for (int i = 0; i < D / 64; i++) {
            const int d = 64 * i + 4 * (tid & 15);
            f32x4 y{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < 4; x++)
                y += *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(smem + x * WAVE) + row * D + d) * f[x];
            put_row<BM, D, true>(a, t, part, row, d, e[i], y, m, sum);
        }
        __syncthreads();
    });
}

// ---- many rows: 128 a tile, 32 a wave, K and V of a step shared in LDS ----------------------
// Bound by the matrix cores and the vector instructions of the softmax at the clock that both leave
// (1.9 to 2 GHz): in halves 49% and 60% of the cycles, 3457 queries of 12 heads of 64 against 20742 keys
// 447 us, 986 TFLOP/s; in two halves 53% and 50%, of 128 62% and 39%, 1030 TFLOP/s (2 x 865
// queries of 32 / 8 heads against 4000 keys 331 us).  The next step's scores between this step's
// weights, an instruction of the one to four or five of the other, take 5% longer (469, 340).

// Blocks of 32 keys a step; two steps in LDS.  (Halves of 64, two blocks, four, and two with three
// workgroups a CU: 865 queries of 12 heads against 1730 keys 33 us, 40, 37, against 3460 42, 41,
// 45, 3457 against 20742 453, 472, 443.)
template <int KIND, int D>
constexpr int kManyHalves = KIND == kCrossF32 && D == 128 ? 1 : 2;

template <int KIND, int D>
__global__ __launch_bounds__(256, 2) void cross_many_kernel(CrossAttn a) {
    constexpr int BM = 128, QT = 2, H = kManyHalves<KIND, D>, STEP = 32 * H, NP = kParts<KIND>, C = D / 32;
    constexpr int BLOCK = cross_block_bytes(KIND, D), BYTES = H * BLOCK;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lh = lane >> 4;
    const int wave = uniform(tid >> 6);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)smem;
    walk<BM, STEP, 256, D, false>(a, smem, [&](const Tile &t, int step0, int steps, int part) {
        const char *base = a.view.at(t.img, t.g);
        auto copy = [&](int step, int buf) {
            const char *from = base + (size_t)step * BYTES;
#pragma unroll
            for (int u = 0; u < BYTES / 4096; u++)
                copy16_to_lds(from + (4 * u + wave) * 1024, lane * 16,
                              uniform(lds0 + buf * BYTES + (4 * u + wave) * 1024));
        };
        if (steps) copy(step0, 0);
        const int first = 16 * QT * wave;
        Queries<KIND, D, QT> w;
        w.load(a, t, first, li, lh);
        for (int i = 0; i < steps; i++) {
            const int buf = i & 1, key = (step0 + i) * STEP;
            split_wait<0>();
            __syncthreads();  // this step's panels are there, the last one's readers done
            if (i + 1 < steps) copy(step0 + i + 1, buf ^ 1);
            const char *panel = smem + buf * BYTES + lane * 16;
            auto operand = [&](int h, int x) { return *reinterpret_cast<const f16x8 *>(panel + h * BLOCK + x * 1024); };
            f32x4 s[H][2][QT];
#pragma unroll
            for (int h = 0; h < H; h++) w.scores(s[h], [&](int x) { return operand(h, x); });
            if (key + STEP > t.len)
#pragma unroll
                for (int h = 0; h < H; h++) w.mask(s[h], t.len - key - 32 * h, lh);
            w.raise(s);
            float by[QT], off[QT];
            w.near(s, by, off);
#pragma unroll
            for (int h = 0; h < H; h++) {
                f16x8 ph[QT], pl[QT];
                w.weights(s[h], by, off, ph, pl);
                w.add(ph, pl, [&](int x) { return operand(h, 2 * C * NP + x); });
            }
        }
        i32x4 e[D / 16];
        if (part < 0) {
#pragma unroll
            for (int df = 0; df < D / 16; df++) e[df] = dim_exponents<D>(a, t, 16 * df + 4 * lh);
        }
#pragma unroll
        for (int u = 0; u < QT; u++) {
            const float l = sum_groups(w.l[u]);
#pragma unroll
            for (int df = 0; df < D / 16; df++)
                put_row<BM, D, false>(a, t, part, first + 16 * u + li, 16 * df + 4 * lh, e[df], w.o[df][u], w.m[u], l);
        }
        __syncthreads();
    });
}

// Rows of a workgroup of cross_join_kernel (865 queries of 12 heads of 64 against 3300 in two
// halves: 45.3 us, with half as many 48.9, with twice 45.8).
template <int D>
constexpr int kJoinRows = 1024 / D;
// Joins the parts of cross_many_kernel, some rows a workgroup: of tile blockIdx.x where there
// are fewer tiles than shares, as most workgroups would find nothing otherwise (84 tiles:
// 6.3 us; by 512 shares 10.9), else of the tile that begins in share blockIdx.x and
// goes on in the next.
template <int BM, int STEP, int D>
__global__ __launch_bounds__(256) void cross_join_kernel(CrossAttn a, bool by_tile) {
    __shared__ __attribute__((aligned(16))) char smem[256 * sizeof(Sums)];
    __shared__ long long tmp[4];
    const int w = blockIdx.x, per = a.tiles * a.view.kv_heads;
    int img = 0, index = 0, len = 0, cost = 0;
    long long base = 0, share = 1, total = 0, begin = 0;
    const auto shared = [&](long long all) { share = max(1ll, (all + a.shares - 1) / a.shares); };
    if (by_tile) {
        img = w / per;
        index = w - img * per;
        if (a.images == 1) {
            total = (long long)per * cost_of(a, 0, STEP);
        } else {
            for (int i0 = 0; i0 < a.images; i0 += 256) {
                const int i = i0 + threadIdx.x;
                long long sum = 0, before = 0;
                const long long c = i < a.images ? (long long)per * cost_of(a, i, STEP) : 0;
                scan_all<256>(c, tmp, &sum);
                scan_all<256>(i < img ? c : 0, tmp, &before);
                total += sum;
                base += before;
            }
        }
        shared(total);
        len = uniform(a.view.lens[img]);
        cost = (len + STEP - 1) / STEP + kTileCost;
        begin = base + (long long)index * cost;
    } else {
        total = find_image<256>(a, STEP, [&](long long all) {
            shared(all);
            return (w + 1) * share - 1;
        }, img, base);
        const long long end = (w + 1) * share;
        if (end >= total) return;
        img = uniform(img);
        len = uniform(a.view.lens[img]);
        cost = (len + STEP - 1) / STEP + kTileCost;
        index = uniform((int)((end - 1 - base) / cost));
        begin = base + (long long)index * cost;
    }
    const int w0 = uniform((int)((begin + first_unit(cost)) / share)), w1 = uniform((int)((begin + cost - 1) / share));
    if (w0 == w1 || (!by_tile && w0 != w)) return;
    const Tile t = tile_of<BM>(a, img, len, index, STEP);
    const int first = blockIdx.y * kJoinRows<D>;
    if (first >= t.rows) return;
    join_parts<BM, D, 256, false>(a, t, w0, w1, 2 * w0 + (begin > w0 * share ? 1 : 0), first,
                                  min(first + kJoinRows<D>, t.rows), smem);
}

constexpr int kShares = 512;
static_assert(kShares <= kAttnCounters, "a counter for each share");

// Whether a call goes to tiles of 16 rows, by the times of both in us: tiles of 128 cost more to
// begin and to join, and do the arithmetic of 128 whatever they hold; of 16 they reach a third
// of its rate.  (Few / many, one image of 3460 tokens, 12 heads of 64: 17 rows in halves 12.4
// / 19, 64 12.4 / 25, 128 14 / 30, of 20000 tokens 64 35 / 35; two halves 64 16 / 27, of 20000
// 32 46 / 40; sixteen of 4096, 32 / 8 heads of 128: 8 queries in halves 70 / 78, in two
// 130 / 125, 16 100 / 82, 200 / 138.)  The tokens are those that the states were made for.
bool few_rows(const CrossAttn &a) {
    const double rows = (double)a.queries * a.group, tiles = std::ceil(rows / 128) * 128;
    const double products = (a.view.kind == kCrossF32 ? 12e-6 : 8e-6) * a.images * a.view.kv_heads * a.view.tokens * a.view.width;
    return 9 + rows * products / (a.view.kind == kCrossF32 ? 180 : 280) < 22 + tiles * products / 850;
}

template <int KIND, int D>
hipError_t run_attn(hipStream_t s, CrossAttn a, bool few) {
    if (few) {
        cross_few_kernel<KIND, D><<<a.shares, 256, 0, s>>>(a);
        return hipGetLastError();
    }
    constexpr int H = kManyHalves<KIND, D>;
    constexpr size_t bytes = 2 * H * cross_block_bytes(KIND, D);
    static std::atomic<uint64_t> done{0};
    hipError_t e = ensure_dynamic_lds(cross_many_kernel<KIND, D>, bytes, done);
    if (e != hipSuccess) return e;
    cross_many_kernel<KIND, D><<<a.shares, 256, bytes, s>>>(a);
    e = hipGetLastError();
    if (e != hipSuccess || !a.parts) return e;
    constexpr int rows = kJoinRows<D>;
    const size_t items = (size_t)a.tiles * a.view.kv_heads * a.images;
    const bool by_tile = items < (size_t)a.shares;
    const dim3 grid(by_tile ? (unsigned)items : a.shares, (std::min(a.queries * a.group, 128) + rows - 1) / rows);
    cross_join_kernel<128, 32 * H, D><<<grid, 256, 0, s>>>(a, by_tile);
    return hipGetLastError();
}

// Whether rows pass by the caches: those of K and V where they are read the second time, and
// what is read back.
constexpr size_t kCrossStreamBytes = (size_t)64 << 20;

template <int KIND, int D>
hipError_t run_write(hipStream_t s, const CrossWrite &w) {
    const unsigned groups = (w.view.kv_heads + kHeadGroup - 1) / kHeadGroup + (w.seen ? 1 : 0), images = w.view.images;
    const size_t bytes = (size_t)w.tokens * w.view.kv_heads * w.head_dim * 8;  // of an image
    cross_range_kernel<D><<<dim3(w.chunks, groups, images), 256, 0, s>>>(w);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 grid(std::max(1, (w.tokens + 127) / 128), w.view.kv_heads, images);
    if (images * bytes >= kCrossStreamBytes) cross_write_kernel<KIND, D, true><<<grid, 256, 0, s>>>(w);
    else cross_write_kernel<KIND, D, false><<<grid, 256, 0, s>>>(w);
    return hipGetLastError();
}

template <int KIND, int D>
hipError_t run_read(hipStream_t s, const CrossView &v, int head_dim, float *k, float *vv, int *lens) {
    const dim3 grid((v.tokens + 127) / 128, v.kv_heads, v.images);
    if (head_dim % 32 == 0 && (size_t)v.images * v.tokens * v.kv_heads * head_dim * 8 >= kCrossStreamBytes)
        cross_read_kernel<KIND, D, true><<<grid, 256, 0, s>>>(v, head_dim, k, vv, lens);
    else
        cross_read_kernel<KIND, D, false><<<grid, 256, 0, s>>>(v, head_dim, k, vv, lens);
    return hipGetLastError();
}

}  // namespace

// Chunks of an image's tokens in cross_range_kernel, of 32 tokens at least.
int cross_chunks(size_t tokens) { return (int)std::min<size_t>(std::max<size_t>((tokens + 31) / 32, 1), kMaxChunks); }

hipError_t launch_cross_write(hipStream_t s, CrossWrite w) {
    w.chunks = cross_chunks(w.tokens);
    w.chunk = (w.tokens + w.chunks - 1) / w.chunks;
    if (w.view.kind == kCrossF32) return w.view.width == 128 ? run_write<kCrossF32, 128>(s, w) : run_write<kCrossF32, 64>(s, w);
    return w.view.width == 128 ? run_write<kCrossF16, 128>(s, w) : run_write<kCrossF16, 64>(s, w);
}

hipError_t launch_cross_read(hipStream_t s, const CrossView &v, size_t head_dim, float *k, float *vv, int *lens) {
    const int hd = (int)head_dim;
    if (v.kind == kCrossF32) return v.width == 128 ? run_read<kCrossF32, 128>(s, v, hd, k, vv, lens) : run_read<kCrossF32, 64>(s, v, hd, k, vv, lens);
    return v.width == 128 ? run_read<kCrossF16, 128>(s, v, hd, k, vv, lens) : run_read<kCrossF16, 64>(s, v, hd, k, vv, lens);
}

size_t cross_attn_floats(const CrossAttn &a) {
    return (size_t)2 * kShares * (few_rows(a) ? 16 : 128) * (a.view.width + 2);
}

hipError_t launch_cross_attn(hipStream_t s, CrossAttn a) {
    const bool few = few_rows(a);
    a.shares = kShares;
    a.tiles = (a.queries * a.group + (few ? 15 : 127)) / (few ? 16 : 128);
    if (a.view.kind == kCrossF32) return a.view.width == 128 ? run_attn<kCrossF32, 128>(s, a, few) : run_attn<kCrossF32, 64>(s, a, few);
    return a.view.width == 128 ? run_attn<kCrossF16, 128>(s, a, few) : run_attn<kCrossF16, 64>(s, a, few);
}

}  // namespace vh
