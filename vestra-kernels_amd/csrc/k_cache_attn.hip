// Attention of new tokens over a paged cache (kernels.h CacheAttn), on the bf16
// matrix cores with the precision of floats.
//
// A float is exactly three bf16 (8 significand bits each, the range of a float), so
//     q . k = sum over i + j <= 2 of q_i . k_j
// is six products with what is dropped below 2^-24 of each term, whatever the range
// of a row; a bf16 key is one part of its own, and so are the values of a Q8_0
// block (integers up to 127), whose scale joins after the product over its 32
// dims: three products there.  Probabilities are split the same way against V's
// parts (a Q8_0 value times its scale has 18 bits: three parts).  The fp32 matrix
// instructions would take 16 times as long a product, 2.7 times as long as six.
//
// Work is cut into tiles of BM query rows (new tokens of one request times the
// query heads that share a head of the cache, so that a tile reads K and V once for
// all of them), and the key steps of all tiles, laid end to end, into equal shares
// of the workgroups: one long stream beside short ones, one query against a long
// cache and a frame against eight earlier ones all fill the chip.  A tile that
// ends up with several workgroups is joined from their partial sums.  Shares follow
// from the lengths alone and parts are joined in order, so the same call gives the same
// bits.  The lengths are on the device: every workgroup forms the partition itself.
//
// Two kernels, by the rows of a request (launch_cache_attn):
//   few rows:  16 query rows a workgroup, whose four waves take 32 keys each of a
//     step of 128, on their own: K and then V through LDS of the
//     wave's own, no barrier in the loop;
//   many rows: 128 query rows, 32 a wave, which share panels of K and V in LDS.
// Either way a lane holds its own query's scores, keys 16 t + 4 lh + r of tile t,
// which is the B operand of O^T += V^T . P^T if the 32 keys of a product are taken in
// the order (4 lh .. 4 lh + 3 of tile 0, then of tile 1); V^T comes from row-major
// planes by transposing LDS reads of the same rows.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"

namespace vh {
namespace {

// Scores may pass the running maximum by this (base 2).  Weights then reach 2^8, and n weighted
// values of a row sum to a finite number below 2^120 / n.  (Eight taken off every exponent, so that
// weights end at one, costs an instruction a score: a 3457-token frame against 20742 keys in
// bf16 634 us against 619.  Taken off the maximum instead, one key's value no longer returns as
// it is.)
constexpr float kMaxSlack = 8.0f;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// v_mfma_f32_16x16x32_bf16.  Lane l supplies A row l % 16 and B column l % 16 at
// k = 8 * (l / 16) .. + 7; D[4 * (l / 16) + r][l % 16] lands in register r.
__device__ __forceinline__ f32x4 mfma16x16x32_bf16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The upper halves of two floats: bf16 by truncation, which never overflows.
__device__ __forceinline__ uint32_t high_halves(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
// Two floats rounded to bf16 (the empty asm keeps the compiler from converting
// each again where a half is used).
__device__ __forceinline__ uint32_t round_halves(float a, float b) {
    const bf16x2 h = {(__bf16)a, (__bf16)b};
    uint32_t u = __builtin_bit_cast(uint32_t, h);
    asm("" : "+v"(u));
    return u;
}
// x = p0 + p1 + p2 exactly (of values above 2^-110): p0 truncated, so that the
// largest floats stay finite, the others rounded.  An infinity's p1 is NaN.
__device__ __forceinline__ void split3(float a, float b, uint32_t &p0, uint32_t &p1, uint32_t &p2) {
    p0 = high_halves(a, b);
    const float ra = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u);
    const float rb = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
    p1 = round_halves(ra, rb);
    p2 = round_halves(ra - __uint_as_float(p1 << 16), rb - __uint_as_float(p1 & 0xffff0000u));
}
__device__ __forceinline__ void split3(f32x4 a, f32x4 b, bf16x8 (&p)[3]) {
    u32x4 u[3];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        uint32_t w0, w1, w2;
        split3(a[2 * i], a[2 * i + 1], w0, w1, w2);
        u[0][i] = w0;
        u[1][i] = w1;
        u[2][i] = w2;
        split3(b[2 * i], b[2 * i + 1], w0, w1, w2);
        u[0][2 + i] = w0;
        u[1][2 + i] = w1;
        u[2][2 + i] = w2;
    }
#pragma unroll
    for (int i = 0; i < 3; i++) p[i] = __builtin_bit_cast(bf16x8, u[i]);
}

__device__ __forceinline__ void split3(f32x4 a, bf16x4 (&p)[3]) {
    uint32_t u[3][2];
#pragma unroll
    for (int i = 0; i < 2; i++) split3(a[2 * i], a[2 * i + 1], u[0][i], u[1][i], u[2][i]);
#pragma unroll
    for (int i = 0; i < 3; i++) p[i] = __builtin_bit_cast(bf16x4, u32x2{u[i][0], u[i][1]});
}

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

// Four bf16 of column li of a 4 x 16 tile in LDS, whose row r is in the lanes 4 r
// .. 4 r + 3 of each 16-lane group (lane i gives the address of row i / 4, columns
// 4 (i % 4) .. + 3, and receives column i).
__device__ __forceinline__ bf16x4 read_tr(const char *p) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                          (__attribute__((address_space(3))) s16x4 *)p));
}
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

__device__ __forceinline__ bool finite8(f32x4 a, f32x4 b) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        m = max(m, __float_as_uint(a[e]) & 0x7fffffffu);
        m = max(m, __float_as_uint(b[e]) & 0x7fffffffu);
    }
    return m < 0x7f800000u;
}

// ---- the partition ----------------------------------------------------------------

// Keys [lo, hi) that a query at position pos of a request of len tokens sees: of those that
// its row of the table holds, however long the request is.
struct Seen {
    int lo, hi;
};
__device__ __forceinline__ Seen keys_seen(const CacheAttn &a, int len, int pos) {
    long long hi = len;
    if (a.block) hi = pos < 0 ? 0 : min(hi, ((long long)((unsigned)pos / a.block) + 1) * a.block);
    const long long lo = a.window ? max(0ll, hi - a.window) : 0;
    return {min((int)lo, a.row_keys), min((int)hi, a.row_keys)};
}

struct Tile {
    int r, start, len, pos;  // request, its first new token, its tokens, the first new one's position
    int row, rows;           // query rows (token of the request * group + head of the group)
    Seen any, all;           // keys that some row sees, that every row sees
    int step0, cost;         // first key step; their number, 1 where there is none, and kTileCost
};

// What a tile costs besides its key steps, in steps: queries fetched, first loads
// waited for, output written.  Without it a share of many short tiles takes twice as
// long as one of a long tile.
constexpr int kTileCost = 2;

__device__ __forceinline__ int start_of(const CacheAttn &a, int r) { return min(max(a.starts[r], 0), a.tokens); }
// The highest of the starts up to r, which is where request r begins: a row is one request's,
// whatever the starts, and the tiles are no more than a batch of so many tokens and requests has.
__device__ int highest_start(const CacheAttn &a, int r) {
    int h = 0;
#pragma unroll 1
    for (int i = 0; i <= r; i++) h = max(h, start_of(a, i));
    return h;
}
// In first_tile: the request's own start is not that one.  (Tiles stay below 2^26 + 2^12.)
constexpr int kFell = 1 << 30;

template <int BM, int STEP>
__device__ __forceinline__ Tile tile_of(const CacheAttn &a, const int *first_tile, int ti) {
    int lo = 0, hi = a.requests;  // first_tile[lo] <= ti < first_tile[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((first_tile[mid] & ~kFell) <= ti) lo = mid;
        else hi = mid;
    }
    Tile t;
    t.r = lo;
    const int first = first_tile[lo];
    t.start = start_of(a, lo);
    if (__builtin_expect(first & kFell, 0)) t.start = highest_start(a, lo);
    const int n = start_of(a, lo + 1) - t.start;
    t.len = max(a.lens[lo], 0);
    t.pos = t.len - n;
    t.row = (ti - (first & ~kFell)) * BM;
    t.rows = min(BM, n * a.group - t.row);
    const Seen s0 = keys_seen(a, t.len, t.pos + t.row / a.group);
    const Seen s1 = keys_seen(a, t.len, t.pos + (t.row + t.rows - 1) / a.group);
    t.any = {s0.lo, s1.hi};
    t.all = {s1.lo, s0.hi};
    t.step0 = t.any.lo / STEP;
    t.cost = max(1, (t.any.hi + STEP - 1) / STEP - t.step0) + kTileCost;
    return t;
}

// The same in scalar registers (all lanes have formed the same).
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ Tile uniform(const Tile &t) {
    return {uniform(t.r),   uniform(t.start), uniform(t.len),
            uniform(t.pos), uniform(t.row),   uniform(t.rows),
            {uniform(t.any.lo), uniform(t.any.hi)}, {uniform(t.all.lo), uniform(t.all.hi)},
            uniform(t.step0), uniform(t.cost)};
}

// What a workgroup knows of the partition: steps of all tiles of one head of the
// cache (units), the share of a workgroup, and where a given step lies.
struct Partition {
    int tiles;
    long long units, total, share;
    long long end, cost;  // of the tile of this thread's number: steps up to its end, and its own
    Tile mine;            // and the tile itself (TILE)
};
struct Place {
    int head, tile;
    long long into;  // steps of the tile before it
};

template <int BM, int STEP, int THREADS, bool TILE>
__device__ __forceinline__ Partition partition(const CacheAttn &a, int *first_tile, long long *tmp, int shares) {
    const int tid = threadIdx.x;
    Partition p;
    long long all = 0, base = 0;
    long long falls = 0;  // so far
    for (int r0 = 0; r0 < a.requests; r0 += THREADS) {
        const int r = r0 + tid;
        const bool there = r < a.requests;
        const int own = there ? start_of(a, r) : 0;
        int start = own, next = there ? start_of(a, r + 1) : 0;
        const long long fell = next < start;
        auto tiles_of = [&] { return ((long long)max(next - start, 0) * a.group + BM - 1) / BM; };
        long long tiles = tiles_of();
        // Falls are counted above the tiles.
        long long end = base + scan_all<THREADS>(tiles + (fell << 48), tmp, &all);
        falls += all >> 48;
        if (__builtin_expect(falls != 0, 0)) {
            start = there ? highest_start(a, r) : 0;
            tiles = tiles_of();
            end = base + scan_all<THREADS>(tiles, tmp, &all);
        }
        base += all;
        if (there) first_tile[r] = (int)(end - tiles) | (start != own ? kFell : 0);
    }
    if (tid == 0) first_tile[a.requests] = (int)base;
    __syncthreads();
    p.tiles = first_tile[a.requests];
    if constexpr (TILE) {
        p.mine = tid < p.tiles ? tile_of<BM, STEP>(a, first_tile, tid) : Tile{};
        p.cost = p.mine.cost;
    } else {
        p.cost = tid < p.tiles ? tile_of<BM, STEP>(a, first_tile, tid).cost : 0;
    }
    p.end = scan_all<THREADS>(p.cost, tmp, &p.units);
    for (int t0 = THREADS; t0 < p.tiles; t0 += THREADS) {
        const int ti = t0 + tid;
        scan_all<THREADS>(ti < p.tiles ? tile_of<BM, STEP>(a, first_tile, ti).cost : 0, tmp, &all);
        p.units += all;
    }
    p.total = p.units * a.cache.kv_heads;
    p.share = max(1ll, (p.total + shares - 1) / shares);
    return p;
}

// Steps of the first THREADS tiles.
template <int THREADS>
__device__ __forceinline__ long long first_units(const Partition &p, long long *tmp) {
    if (threadIdx.x == THREADS - 1) tmp[0] = p.end;
    __syncthreads();
    const long long n = tmp[0];
    __syncthreads();
    return n;
}

// The tile itself is left in `found_tile`, if that is asked for (TILE).
template <int BM, int STEP, int THREADS, bool TILE>
__device__ __forceinline__ Place find(const CacheAttn &a, const Partition &p, const int *first_tile, long long *tmp,
                                      long long unit, Tile *found_tile) {
    __shared__ long long found[2];
    Place at;
    at.head = (int)(unit / p.units);
    const long long x = unit - at.head * p.units;
    long long cost = p.cost, end = p.end, all = 0;
    for (int t0 = 0;;) {
        if (end - cost <= x && x < end) {
            found[0] = t0 + (int)threadIdx.x;
            found[1] = end - cost;
            if constexpr (TILE) *found_tile = t0 ? tile_of<BM, STEP>(a, first_tile, (int)found[0]) : p.mine;
        }
        t0 += THREADS;
        if (t0 >= p.tiles) break;
        const int ti = t0 + (int)threadIdx.x;
        const long long before = t0 == THREADS ? first_units<THREADS>(p, tmp) : all;
        cost = ti < p.tiles ? tile_of<BM, STEP>(a, first_tile, ti).cost : 0;
        long long some = 0;
        end = before + scan_all<THREADS>(cost, tmp, &some);
        all = before + some;
    }
    __syncthreads();
    at.tile = (int)found[0];
    at.into = x - found[1];
    __syncthreads();
    return at;
}

// The page of a key of a tile that sees some (of the nearest such key: no branch),
// and the key's slot, in the page of zeros behind the last where its page is not
// there.  Apart, so that a loop can load the page a step before it looks at it:
// looking waits for every load issued before.
__device__ __forceinline__ int page_of(const CacheAttn &a, const Tile &t, int key) {
    const int near = min(max(key, t.any.lo), t.any.hi - 1);
    return a.table[(size_t)t.r * a.max_pages + (near >> a.cache.page_shift)];
}
__device__ __forceinline__ int slot_of(const CacheAttn &a, int key, int page) {
    const int pages = a.cache.slots >> a.cache.page_shift;
    if ((unsigned)page >= (unsigned)pages) page = pages;
    return (page << a.cache.page_shift) + (key & ((1 << a.cache.page_shift) - 1));
}

// ---- one wave's arithmetic ---------------------------------------------------------

// QT tiles of 16 queries: their fragments (three parts), running maxima and sums,
// and O^T: o[df][u][r] = O[query 16 u + li][16 df + 4 lh + r].
template <int D, int QT>
struct Queries {
    static constexpr int C = D / 32, DF = D / 16;
    bf16x8 q[QT][C][3];
    f32x4 o[DF][QT];
    float m[QT], l[QT];
    Seen seen[QT];

    // Rows first .. first + 16 QT - 1 of the tile (rows past its end: zeros).
    __device__ __forceinline__ void load(const CacheAttn &a, const Tile &t, int g, int first, int li, int lh) {
#pragma unroll
        for (int u = 0; u < QT; u++) {
            const int in = first + 16 * u + li;
            const bool there = in < t.rows;
            const int row = t.row + (there ? in : 0), token = row / a.group, head = g * a.group + row % a.group;
            const float *src = a.q + ((size_t)(t.start + token) * a.heads + head) * a.head_dim;
#pragma unroll
            for (int c = 0; c < C; c++) {
                f32x4 x[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int d = 32 * c + 8 * lh + 4 * e;
                    x[e] = there && d < a.head_dim ? *reinterpret_cast<const f32x4 *>(src + d)
                                                   : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
                split3(x[0], x[1], q[u][c]);
            }
            seen[u] = there ? keys_seen(a, t.len, t.pos + token) : Seen{0, INT32_MAX};
            m[u] = -INFINITY;
            l[u] = 0.0f;
#pragma unroll
            for (int df = 0; df < DF; df++) o[df][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    // Scores of 32 keys from key on: the unseen ones out.  present: bit 16 t + i.
    __device__ __forceinline__ void mask(f32x4 (&s)[2][QT], int key, uint32_t present, int lh) const {
        asm volatile("" : "+s"(key));  // keeps what follows out of the steps that need none
#pragma unroll
        for (int u = 0; u < QT; u++) {
            // Bits [lo, hi) - key of 32, this lane's four of each tile lowest.
            const int lo = min(max(seen[u].lo - key, 0), 32), hi = min(max(seen[u].hi - key, 0), 32);
            const uint32_t bits =
                (present & (uint32_t)((1ull << hi) - 1) & ~(uint32_t)((1ull << lo) - 1)) >> (4 * lh);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (!(bits & (1u << (16 * t + r)))) s[t][u][r] = -INFINITY;
        }
    }

    // Brings the maxima up to those of H times 32 keys' scores.  They are only raised
    // where a score passes one by kMaxSlack, so most steps need no correction.
    // (Before any key was seen the maximum is -inf: any score passes it.)
    template <int H>
    __device__ __forceinline__ void raise(const f32x4 (&s)[H][2][QT], float scale) {
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
            mx[u] = v * scale;
            over |= mx[u] > m[u] + kMaxSlack;
        }
        if (__any(over)) {
#pragma unroll
            for (int u = 0; u < QT; u++) {
                const float mn = fmaxf(m[u], max_groups(mx[u]));
                const float corr = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[u] - mn);
                m[u] = mn;
                l[u] *= corr;
#pragma unroll
                for (int df = 0; df < DF; df++) o[df][u] *= corr;
            }
        }
    }

    // The scores of 32 keys become their weights, which are summed.
    __device__ __forceinline__ void weights(f32x4 (&s)[2][QT], float scale) {
#pragma unroll
        for (int u = 0; u < QT; u++) {
            const float off = m[u] == -INFINITY ? 0.0f : -m[u];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    s[t][u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][u][r], scale, off));
            l[u] += ((s[0][u][0] + s[0][u][1]) + (s[0][u][2] + s[0][u][3])) +
                    ((s[1][u][0] + s[1][u][1]) + (s[1][u][2] + s[1][u][3]));
        }
    }

    // O^T += V^T . P^T for 32 keys, of dims 16 d0 .. 16 (d0 + n) - 1; v: this lane's
    // address in the first plane.
    template <int NP, int D0, int N>
    __device__ __forceinline__ void add(const char *v, int plane, int vx, int vg, const bf16x8 (&p)[QT][3]) {
        // Two tiles of dims at a time, the small products first: 2 QT sums that do
        // not wait for each other.
#pragma unroll
        for (int d0 = D0; d0 < D0 + N; d0 += 2) {
            bf16x8 f[2][NP];
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    const char *at = v + i * plane + (((2 * (d0 + k) + vg) ^ vx) << 4);
                    const bf16x4 x = read_tr(at), y = read_tr(at + 16 * D * 2);
                    f[k][i] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                }
#pragma unroll
            for (int sum = 2; sum >= 0; sum--)
#pragma unroll
                for (int i = NP - 1; i >= 0; i--)
                    if (sum - i >= 0)
#pragma unroll
                        for (int k = 0; k < 2; k++)
#pragma unroll
                            for (int u = 0; u < QT; u++)
                                o[d0 + k][u] = mfma16x16x32_bf16(f[k][i], p[u][sum - i], o[d0 + k][u]);
        }
    }
};

// Swizzles of the planes in LDS ([key][D] bf16, in granules of 16 bytes).  K: a
// fragment read takes one granule of 16 rows.  V: a transposing read takes a pair of
// granules of 16 rows.
template <int D>
__device__ __forceinline__ int k_swizzle(int row) {
    return D == 64 ? (row >> 1) & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int v_swizzle(int row) {
    return D == 64 ? (row & 6) : 2 * (row & 7);
}

__device__ __forceinline__ float half_value(uint16_t h) { return (float)__builtin_bit_cast(_Float16, h); }

// Loads that pass by the caches: those of the few rows, whose tiles mostly read a row of the
// cache once (64 requests of 4 rows against 4096 keys each, 8 heads of 128 in bf16, 164 us,
// through the caches 184).  The second tile of 17 to 32 rows reads it again: of 64 requests no
// slower (342 and 381), of 16 up to 1.2 times (69 and 57).
template <bool NT, class T>
__device__ __forceinline__ T ld(const T *p) {
    if constexpr (NT) return __builtin_nontemporal_load(p);
    else return *p;
}

// Eight dims of a cache row as it is stored, of lane sg of the D / 8 that share the
// row, and their way to the planes.  Every load covers whole lines, so that none is
// asked for twice.  A load is at a base, wherever it can one that the wave shares (its
// rows in one page), plus 32 bits of a lane's own: the 64-bit products of a row's
// address are scalar then.
template <int KIND, int D>
struct Octet;
template <int D>
struct Octet<kCacheF32, D> {
    f32x4 a, b;  // dims 4 sg .. + 3, and D / 2 further
    static constexpr int kRow = 4 * D, kLane = 16;  // bytes
    template <bool NT>
    __device__ __forceinline__ void load(const char *base, uint32_t at) {
        a = ld<NT>(reinterpret_cast<const f32x4 *>(base + at));
        b = ld<NT>(reinterpret_cast<const f32x4 *>(base + at + 2 * D));
    }
    // To the row at `at` of the first plane.
    template <bool SCALED>
    __device__ __forceinline__ void stage(char *at, int plane, int sg, int swizzle, float) const {
        bf16x4 p[3];
        char *x = at + (((sg >> 1) ^ swizzle) << 4) + (sg & 1) * 8;
        split3(a, p);
#pragma unroll
        for (int i = 0; i < 3; i++) *reinterpret_cast<bf16x4 *>(x + i * plane) = p[i];
        x = at + (((D / 16 + (sg >> 1)) ^ swizzle) << 4) + (sg & 1) * 8;
        split3(b, p);
#pragma unroll
        for (int i = 0; i < 3; i++) *reinterpret_cast<bf16x4 *>(x + i * plane) = p[i];
    }
};
template <int D>
struct Octet<kCacheBf16, D> {
    bf16x8 x;  // dims 8 sg .. + 7
    static constexpr int kRow = 2 * D, kLane = 16;
    template <bool NT>
    __device__ __forceinline__ void load(const char *base, uint32_t at) {
        x = ld<NT>(reinterpret_cast<const bf16x8 *>(base + at));
    }
    template <bool SCALED>
    __device__ __forceinline__ void stage(char *at, int, int sg, int swizzle, float) const {
        *reinterpret_cast<bf16x8 *>(at + ((sg ^ swizzle) << 4)) = x;
    }
};
template <int D>
struct Octet<kCacheQ8, D> {
    u32x2 x;  // dims 8 sg .. + 7
    static constexpr int kRow = D, kLane = 8;
    template <bool NT>
    __device__ __forceinline__ void load(const char *base, uint32_t at) {
        x = ld<NT>(reinterpret_cast<const u32x2 *>(base + at));
    }
    // As integers, or times the scale d (18 bits: three parts).
    template <bool SCALED>
    __device__ __forceinline__ void stage(char *at, int plane, int sg, int swizzle, float d) const {
        f32x4 a, b;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            a[e] = (float)(int8_t)(x[0] >> (8 * e));
            b[e] = (float)(int8_t)(x[1] >> (8 * e));
        }
        at += (sg ^ swizzle) << 4;
        if constexpr (SCALED) {
            bf16x8 p[3];
            split3(a * d, b * d, p);
#pragma unroll
            for (int i = 0; i < 3; i++) *reinterpret_cast<bf16x8 *>(at + i * plane) = p[i];
        } else {
            *reinterpret_cast<u32x4 *>(at) = u32x4{high_halves(a[0], a[1]), high_halves(a[2], a[3]),
                                                   high_halves(b[0], b[1]), high_halves(b[2], b[3])};
        }
    }
};

// Values that are not finite become zeros; whether there were any.
template <int D>
__device__ __forceinline__ bool drop(Octet<kCacheF32, D> &x, uint16_t) {
    if (finite8(x.a, x.b)) return false;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (!(fabsf(x.a[e]) < INFINITY)) x.a[e] = 0.0f;
        if (!(fabsf(x.b[e]) < INFINITY)) x.b[e] = 0.0f;
    }
    return true;
}
template <int D>
__device__ __forceinline__ bool drop(Octet<kCacheBf16, D> &x, uint16_t) {
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (!(fabsf((float)x.x[e]) < INFINITY)) {
            x.x[e] = (__bf16)0.0f;
            bad = true;
        }
    return bad;
}
// (Of a block whose scale is not.)
template <int D>
__device__ __forceinline__ bool drop(Octet<kCacheQ8, D> &, uint16_t &d) {
    if ((d & 0x7c00) != 0x7c00) return false;
    d = 0;
    return true;
}

template <int KIND>
constexpr int kPartsOfK = KIND == kCacheF32 ? 3 : 1;
template <int KIND>
constexpr int kPartsOfV = KIND == kCacheBf16 ? 1 : 3;

// A value that is not finite in a step where some query does not see it was
// staged as zero: the dims of the queries that do see it become NaN here.  32 keys
// from key on; rare, so one by one.
template <int KIND, int D, int QT>
__device__ void add_not_finite(const CacheAttn &a, const Tile &t, int g, Queries<D, QT> &w, int key, int lh) {
    for (int i = 0; i < 32; i++) {
        const int slot = slot_of(a, key + i, page_of(a, t, key + i));
        if (slot >= a.cache.slots) continue;
        const size_t row = cache_row(a.cache, slot, g);
#pragma unroll
        for (int df = 0; df < D / 16; df++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const size_t at = row * D + 16 * df + 4 * lh + r;
                float v;
                if constexpr (KIND == kCacheF32) v = static_cast<const float *>(a.cache.v)[at];
                else if constexpr (KIND == kCacheBf16) v = (float)static_cast<const __bf16 *>(a.cache.v)[at];
                else v = half_value(a.cache.vd[at / 32]);
                if (fabsf(v) < INFINITY) continue;
#pragma unroll
                for (int u = 0; u < QT; u++)
                    if (key + i >= w.seen[u].lo && key + i < w.seen[u].hi) w.o[df][u][r] = NAN;
            }
    }
}

// The parts.  Where the last workgroup of a tile joins them (HERE) they are read and
// written past the L2 of an XCD (sc1), as the workgroups of a tile may be on several;
// a launch of its own sees them anyway.
template <bool HERE>
struct Parts {
    __amdgpu_buffer_rsrc_t base;
    __device__ __forceinline__ explicit Parts(const CacheAttn &a)
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
__device__ __forceinline__ uint32_t weights_at(const CacheAttn &a, uint32_t x, int in) {
    return 2u * a.shares * BM * D * 4 + (x * BM + in) * 8;
}

// Of a tile that is joined by a launch of its own, left by the workgroup of its first
// share behind the parts: a record for each share.
struct Joint {
    int start, row, rows;  // of the tile
    int head, last, part;  // its last share (-1: no tile goes on from this share), its first part
    int unused[2];
};
template <int BM, int D>
__device__ __forceinline__ Joint *joint_of(const CacheAttn &a, int w) {
    return reinterpret_cast<Joint *>(reinterpret_cast<char *>(a.parts) + weights_at<BM, D>(a, 2 * a.shares, 0)) + w;
}

// Row `in` of a tile, four dims from d on: the result, or a workgroup's part of it.
template <int BM, int D, bool HERE>
struct Output {
    const CacheAttn &a;
    const Tile &t;
    int g;
    int part;  // -1: the whole
    __device__ __forceinline__ void put(int in, int d, f32x4 v, float m, float l) const {
        if (in >= t.rows) return;
        if (part < 0) {
            if (d >= a.head_dim) return;
            const int row = t.row + in, token = row / a.group, head = g * a.group + row % a.group;
            const float inv = 1.0f / l;
            f32x4 y;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = l == 0.0f ? 0.0f : v[e] * inv;
            *reinterpret_cast<f32x4 *>(a.out + ((size_t)(t.start + token) * a.heads + head) * a.head_dim + d) = y;
        } else {
            const Parts<HERE> parts(a);
            parts.put(sums_at<BM, D>(part, in) + 4 * d, v);
            if (d == 0) parts.put(weights_at<BM, D>(a, part, in), m, l);
        }
    }
};

// Shares in the order of the steps, those of one XCD (workgroups go round-robin over
// the eight) next to each other: tiles of one head and request share K and V in its
// L2.
__device__ __forceinline__ int my_share(const CacheAttn &a) {
    return (blockIdx.x & 7) * (a.shares >> 3) + (blockIdx.x >> 3);
}

// A row's four dims of a part, or of several: O on the maximum m, and the sum of
// weights.
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

// The parts of shares w0 .. w1 (of w0 the one at part0) become the tile's output: rows
// from .. to - 1.  Of the workgroup's groups of D / 4 lanes (a group holds a row) as many
// share a row as the rows leave: a single query's parts are summed by all of them.
template <int BM, int D, int THREADS, bool HERE>
__device__ void join_parts(const CacheAttn &a, const Tile &t, int g, int w0, int w1, int part0, int from, int to,
                           char *smem) {
    Sums *some = reinterpret_cast<Sums *>(smem);
    const Output<BM, D, HERE> out{a, t, g, -1};
    const Parts<HERE> parts(a);
    constexpr int LANES = D / 4, GROUPS = THREADS / LANES;
    int rows = 1;  // at once
    while (rows < GROUPS && rows < to - from) rows *= 2;
    const int sharers = GROUPS / rows;
    const int group = threadIdx.x / LANES, d = 4 * (threadIdx.x % LANES);
    for (int in = from + group % rows; in < from + (to - from + rows - 1) / rows * rows; in += rows) {
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
        if (group < rows && in < to) out.put(in, d, sum.y, sum.m, sum.l);
    }
}

// Walks this workgroup's steps tile by tile: f(tile, head, first step, steps, part),
// no steps where a tile sees no key.  Without room for parts (a.parts null) every
// workgroup takes whole tiles.
//
// HERE: of the workgroups that hold a part of a tile the one that is done last joins
// them, in the order of the shares.  They count in the counter of the tile's first share
// (of which it is the last tile, so no other counts there), zero before and after.
template <int BM, int STEP, int THREADS, int D, bool HERE, class F>
__device__ __forceinline__ void walk(const CacheAttn &a, int *first_tile, char *smem, F f) {
    __shared__ long long tmp[THREADS / 64];
    __shared__ int is_last;
    const Partition p = partition<BM, STEP, THREADS, HERE>(a, first_tile, tmp, a.shares);
    const int w = my_share(a);
    const bool share = a.parts != nullptr;
    // Steps of this workgroup, or the numbers of its tiles.
    long long at = share ? w * p.share : w;
    const long long end = share ? min(at + p.share, p.total) : (long long)p.tiles * a.cache.kv_heads;
    int goes_on = -1;  // the last share of a tile that begins here and ends in a later one
    const auto leave = [&](const Joint &j) {
        if (!HERE && share && threadIdx.x == 0) *joint_of<BM, D>(a, w) = j;
    };
    if (at >= end) return leave(Joint{0, 0, 0, 0, -1});
    Place place = {0, 0, 0};
    __shared__ Tile found_tile;
    if (share) place = find<BM, STEP, THREADS, HERE>(a, p, first_tile, tmp, at, &found_tile);
    for (bool first = true; at < end; first = false) {
        if (!share) {
            place.head = (int)(at / p.tiles);
            place.tile = (int)(at - (long long)place.head * p.tiles);
        }
        // Few rows: the first tile as it was found (one token against 3461 keys 14.4 us,
        // formed again 14.6; many rows have no registers for it).
        const Tile t = uniform(HERE && share && first ? found_tile : tile_of<BM, STEP>(a, first_tile, place.tile));
        const int into = uniform((int)place.into), g = uniform(place.head);
        const int steps = share ? uniform((int)min(end - at, (long long)t.cost - into)) : t.cost;
        const bool whole = into == 0 && steps == t.cost;
        const int from = max(into - kTileCost, 0), to = max(into + steps - kTileCost, 0);
        f(t, g, t.step0 + from, t.any.lo < t.any.hi ? to - from : 0, whole ? -1 : 2 * w + (first ? 0 : 1));
        if (!HERE && !whole && into == 0) {
            goes_on = uniform((int)((at + t.cost - 1) / p.share));
            leave(Joint{t.start, t.row, t.rows, g, goes_on, 2 * w + (first ? 0 : 1)});
        }
        if (HERE && !whole) {
            const long long begin = at - into;
            const int w0 = uniform((int)(begin / p.share)), w1 = uniform((int)((begin + t.cost - 1) / p.share));
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
                join_parts<BM, D, THREADS, true>(a, t, g, w0, w1, 2 * w0 + (begin > w0 * p.share ? 1 : 0), 0,
                                                   t.rows, smem);
                __syncthreads();
            }
        }
        at += share ? steps : a.shares;
        place.into = 0;
        if (++place.tile == p.tiles) {
            place.tile = 0;
            place.head++;
        }
    }
    if (goes_on < 0) leave(Joint{0, 0, 0, 0, -1});
}

// ---- few rows -------------------------------------------------------------------

// A wave holds the rows of K or of V of one step in flight, never both: 64 KB to a CU
// at a row of 256 bytes.  Twice that lowers what the memory delivers (reading
// scattered pages of 16 KB and nothing else: 64 KB in flight a CU 6.8 TB/s, 128 KB
// 6.3, 256 KB 5.4), and the registers are the same for both.  (Shorter rows have less in flight,
// and reach less: 65536 keys in sixteen requests, 12 heads of 64 in bf16 42 us, 4.8 TB/s, 8 of
// 128 in Q8_0 52, 2.7, where the conversion of its bytes counts too.)  A Q8_0 value stays the
// integer it is; its scale joins its weight, once for each block of 32 dims (few
// weights, where the values of a step are many).
//
// Bound by the reads of K and V: a token each of 64 requests of 130 to 16384 keys, 32 / 8
// heads of 128 in bf16 (846 MB), takes 144 us, 5.9 TB/s; requests of one length
// 6.3 to 6.5 (reading alone: 6.4, past the caches 7.2).  Small calls are a chain of
// latencies (lengths, table, K, V, parts, counter, parts): one token against 3461 keys
// of 12 heads of 64 in floats 14.4 us.

template <int KIND>
constexpr int kFewParts = KIND == kCacheF32 ? 3 : 1;
template <int KIND, int D>
constexpr int few_wave_bytes() {
    // The planes of 32 keys, K's and then V's, and the scales of both, or the wave's O
    // at the end.
    constexpr int panel = kFewParts<KIND> * 32 * D * 2 + (KIND == kCacheQ8 ? 2 * 32 * (D / 32) * 4 : 0);
    constexpr int o = 16 * D * 4 + 128;
    return panel > o ? panel : o;
}
template <int KIND, int D>
constexpr int few_workgroups() {  // a CU
    return 4 * few_wave_bytes<KIND, D>() > 80 * 1024 ? 1 : 2;
}

// (Of wide floats LDS holds one workgroup a CU, which so may use every register: 64
// tokens against 3000 keys of 8 heads of 128 242 us, with half of them 267.)
template <int KIND, int D>
__global__ __launch_bounds__(256, (few_workgroups<KIND, D>())) void few_rows_kernel(CacheAttn a) {
    constexpr int BM = 16, STEP = 128, C = D / 32, WAVE = few_wave_bytes<KIND, D>();
    constexpr int NP = kFewParts<KIND>, PLANE = 32 * D * 2;
    constexpr int LPR = D / 8, RPP = 64 / LPR, PASSES = 32 / RPP;  // lanes a row, rows a pass
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int *first_tile = reinterpret_cast<int *>(smem + 4 * WAVE);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lh = lane >> 4;
    char *mine = smem + wave * WAVE;
    float *scales = reinterpret_cast<float *>(mine + NP * PLANE);  // [k, v][C][32]
    const int srow = lane / LPR, sg = lane % LPR;  // row of a pass and granule that this lane moves

    walk<BM, STEP, 256, D, true>(a, first_tile, smem, [&](const Tile &t, int g, int step0, int steps, int part) {
        Octet<KIND, D> x[PASSES];
        uint16_t d[C] = {};  // scales of key `lane & 31`
        auto load = [&](const void *base, const uint16_t *scale, int slot) {
            using O = Octet<KIND, D>;
            if (a.cache.page_shift >= 4) {  // the halves of a step are in one page each
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const char *rows = static_cast<const char *>(base) +
                                       cache_row(a.cache, __builtin_amdgcn_readlane(slot, 16 * h), g) * O::kRow;
#pragma unroll
                    for (int i = 0; i < PASSES / 2; i++)
                        x[h * (PASSES / 2) + i].template load<true>(rows, (i * RPP + srow) * O::kRow + sg * O::kLane);
                }
            } else {
#pragma unroll
                for (int i = 0; i < PASSES; i++)
                    x[i].template load<true>(static_cast<const char *>(base) +
                                                 cache_row(a.cache, __shfl(slot, i * RPP + srow, 64), g) * O::kRow,
                                             sg * O::kLane);
            }
            if constexpr (KIND == kCacheQ8) {
                const size_t row = cache_row(a.cache, slot, g);
#pragma unroll
                for (int c = 0; c < C; c++) d[c] = scale[row * C + c];
            }
        };
        // Of key `lane & 31` of a step.
        auto key_of = [&](int i) { return (step0 + i) * STEP + 32 * wave + (lane & 31); };
        int slot = 0, next_page = 0;
        if (steps) {
            const int page = page_of(a, t, key_of(0));
            next_page = page_of(a, t, key_of(1));
            slot = slot_of(a, key_of(0), page);
            load(a.cache.k, a.cache.kd, slot);
        }
        Queries<D, 1> w;  // (read behind the first keys)
        w.load(a, t, g, 0, li, lh);
        for (int i = 0; i < steps; i++) {
            const int key = (step0 + i) * STEP + 32 * wave;
            const uint32_t present = (uint32_t)__ballot(slot < a.cache.slots);
            const bool partial = key < t.all.lo || key + 32 > t.all.hi || present != 0xffffffffu;
            auto put_scales = [&](float *to) {
                if (KIND == kCacheQ8 && lane < 32) {
#pragma unroll
                    for (int c = 0; c < C; c++) to[32 * c + lane] = half_value(d[c]);
                }
            };
            put_scales(scales);
#pragma unroll
            for (int j = 0; j < PASSES; j++) {
                const int row = j * RPP + srow;
                x[j].template stage<false>(mine + row * (D * 2), PLANE, sg, k_swizzle<D>(row), 0.0f);
            }
            load(a.cache.v, a.cache.vd, slot);
            const int next = slot_of(a, key_of(i + 1), next_page);
            next_page = page_of(a, t, key_of(i + 2));
            wave_fence();
            f32x4 sx[1][2][1];
            f32x4(&s)[2][1] = sx[0];
            s[0][0] = s[1][0] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < C; c++) {
                bf16x8 f[2][NP];
                f32x4 y[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int row = 16 * j + li;
#pragma unroll
                    for (int e = 0; e < NP; e++)
                        f[j][e] = *reinterpret_cast<const bf16x8 *>(mine + e * PLANE + row * (D * 2) +
                                                                    (((4 * c + lh) ^ k_swizzle<D>(row)) << 4));
                    y[j] = KIND == kCacheQ8 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : s[j][0];
                }
#pragma unroll
                for (int sum = 2; sum >= 0; sum--)
#pragma unroll
                    for (int e = NP - 1; e >= 0; e--)
                        if (sum - e >= 0)
#pragma unroll
                            for (int j = 0; j < 2; j++) y[j] = mfma16x16x32_bf16(f[j][e], w.q[0][c][sum - e], y[j]);
#pragma unroll
                for (int j = 0; j < 2; j++)
                    if constexpr (KIND == kCacheQ8) {
                        const f32x4 z = *reinterpret_cast<const f32x4 *>(scales + 32 * c + 16 * j + 4 * lh);
#pragma unroll
                        for (int r = 0; r < 4; r++) s[j][0][r] = __builtin_fmaf(z[r], y[j][r], s[j][0][r]);
                    } else {
                        s[j][0] = y[j];
                    }
            }
            wave_fence();
            if (partial) w.mask(s, key, present, lh);
            w.raise(sx, a.scale_log2);
            w.weights(s, a.scale_log2);
            bool dropped = false;
            if (KIND == kCacheQ8 && partial) {
#pragma unroll
                for (int c = 0; c < C; c++) dropped |= drop(x[0], d[c]);
            }
            put_scales(scales + 32 * C);
#pragma unroll
            for (int j = 0; j < PASSES; j++) {
                uint16_t none = 0;
                if (KIND != kCacheQ8 && partial) dropped |= drop(x[j], none);
                const int row = j * RPP + srow;
                x[j].template stage<false>(mine + row * (D * 2), PLANE, sg, v_swizzle<D>(row), 0.0f);
            }
            slot = next;
            load(a.cache.k, a.cache.kd, slot);
            wave_fence();
            const int vrow = 4 * lh + (li >> 2);
            const char *v = mine + vrow * (D * 2) + (li & 1) * 8;
            const int vx = v_swizzle<D>(vrow), vg = (li & 3) >> 1;
            bf16x8 p[1][3];
            if constexpr (KIND == kCacheQ8) {
                auto block = [&](auto cc) {
                    constexpr int c = decltype(cc)::value;
                    const f32x4 *z = reinterpret_cast<const f32x4 *>(scales + 32 * (C + c) + 4 * lh);
                    split3(s[0][0] * z[0], s[1][0] * z[4], p[0]);
                    w.template add<1, 2 * c, 2>(v, PLANE, vx, vg, p);
                };
                block(std::integral_constant<int, 0>{});
                block(std::integral_constant<int, 1>{});
                if constexpr (C == 4) {
                    block(std::integral_constant<int, 2>{});
                    block(std::integral_constant<int, 3>{});
                }
            } else {
                split3(s[0][0], s[1][0], p[0]);
                w.template add<NP, 0, D / 16>(v, PLANE, vx, vg, p);
            }
            wave_fence();
            if (__any(dropped)) add_not_finite<KIND>(a, t, g, w, key, lh);
        }
        // The four waves' sums, each on its own maximum, joined by all threads.
        float *o = reinterpret_cast<float *>(mine);
#pragma unroll
        for (int df = 0; df < D / 16; df++) *reinterpret_cast<f32x4 *>(o + li * D + 16 * df + 4 * lh) = w.o[df][0];
        const float l = sum_groups(w.l[0]);
        if (lh == 0) {
            o[16 * D + 2 * li] = w.m[0];
            o[16 * D + 2 * li + 1] = l;
        }
        __syncthreads();
        const Output<BM, D, true> out{a, t, g, part};
        const int row = tid >> 4;
        float m = -INFINITY, sum = 0.0f, f[4];
#pragma unroll
        for (int v = 0; v < 4; v++) m = fmaxf(m, reinterpret_cast<float *>(smem + v * WAVE)[16 * D + 2 * row]);
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const float *x = reinterpret_cast<float *>(smem + v * WAVE) + 16 * D + 2 * row;
            f[v] = x[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x[0] - m);
            sum += x[1] * f[v];
        }
#pragma unroll
        for (int d = 4 * (tid & 15); d < D; d += 64) {
            f32x4 y{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int v = 0; v < 4; v++)
                y += *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(smem + v * WAVE) + row * D + d) * f[v];
            out.put(row, d, y, m, sum);
        }
        __syncthreads();
    });
}

// ---- many rows --------------------------------------------------------------------

// Bound by the matrix instructions and what does not hide under them (an 8-cycle issue
// of each, the softmax and the splits on the VALU).  12 heads of 64, 3457 tokens against
// 20742 keys in bf16 (three products of 220 GFLOP): 610 us, 1.08 PFLOP/s, where a large
// library product in bf16 reaches 1.31; 865 against 6920 floats (six of 18): 115 us,
// 0.96; 6 ragged causal chunks in Q8_0 with a window, 32 / 8 heads of 128 (three and six
// of 65 in all): 360 us, 0.81.

// Keys of a step.  (Wide floats, of six planes: 128 query rows of 8 heads against 65536 keys
// 214 us, with 64 keys 230; 2000 tokens of 32 / 8 heads against 20000 3230 and 3180.)
template <int KIND, int D>
constexpr int many_step() {
    return KIND == kCacheF32 && D == 128 ? 32 : 64;
}
template <int D>
constexpr int kManyThreads = D == 64 ? 256 : 512;
template <int KIND, int D>
constexpr int many_bytes() {
    constexpr int step = many_step<KIND, D>();
    return (kPartsOfK<KIND> + kPartsOfV<KIND>)*step * D * 2 + (KIND == kCacheQ8 ? step * (D / 32) * 4 : 0) + 2 * step +
           64;
}

template <int KIND, int D>
__global__ __launch_bounds__(kManyThreads<D>, kManyThreads<D> == 256 ? 2 : 1) void many_rows_kernel(CacheAttn a) {
    constexpr int THREADS = kManyThreads<D>, QT = 512 / THREADS, BM = 128, STEP = many_step<KIND, D>(), C = D / 32;
    constexpr int NPK = kPartsOfK<KIND>, NPV = kPartsOfV<KIND>, PLANE = STEP * D * 2;
    constexpr int LPR = D / 8, RPP = THREADS / LPR, PASSES = STEP / RPP;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char *kp = smem, *vp = smem + NPK * PLANE;
    float *k_scale = reinterpret_cast<float *>(smem + (NPK + NPV) * PLANE);  // [C][STEP]
    uint8_t *there = reinterpret_cast<uint8_t *>(k_scale) + (KIND == kCacheQ8 ? STEP * C * 4 : 0);  // [2][STEP]
    int *flags = reinterpret_cast<int *>(there + 2 * STEP);  // [2] a key is absent, [2] a value was dropped
    int *first_tile = reinterpret_cast<int *>(smem + many_bytes<KIND, D>());
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lh = lane >> 4;
    const int srow = tid / LPR, sg = tid % LPR;  // staged row of a pass, and granule

    walk<BM, STEP, THREADS, D, false>(a, first_tile, smem, [&](const Tile &t, int g, int step0, int steps, int part) {
        const int first = 16 * QT * wave;
        const bool works = first < t.rows;
        Octet<KIND, D> kr[PASSES], vr[PASSES];
        uint16_t kd[PASSES] = {}, vd[PASSES] = {};
        int slot[PASSES], page[PASSES];
        auto look_up = [&](int step) {
#pragma unroll
            for (int i = 0; i < PASSES; i++) page[i] = page_of(a, t, step * STEP + i * RPP + srow);
        };
        auto load = [&](int step) {
            using O = Octet<KIND, D>;
            const char *k = static_cast<const char *>(a.cache.k), *v = static_cast<const char *>(a.cache.v);
#pragma unroll
            for (int i = 0; i < PASSES; i++) {
                slot[i] = slot_of(a, step * STEP + i * RPP + srow, page[i]);
                // A wave's rows of a pass (four or eight) are in one page, or each has its own.
                size_t row;
                uint32_t at = sg * O::kLane;
                if (a.cache.page_shift >= 3) {
                    row = cache_row(a.cache, uniform(slot[i]), g);
                    at += (lane / LPR) * O::kRow;
                    kr[i].template load<false>(k + row * O::kRow, at);
                    vr[i].template load<false>(v + row * O::kRow, at);
                } else {
                    row = cache_row(a.cache, slot[i], g);
                    kr[i].template load<false>(k + row * O::kRow, at);
                    vr[i].template load<false>(v + row * O::kRow, at);
                }
                if constexpr (KIND == kCacheQ8) {
                    row = cache_row(a.cache, slot[i], g) * C + sg / 4;
                    kd[i] = a.cache.kd[row];
                    vd[i] = a.cache.vd[row];
                }
            }
        };
        if (steps) {
            look_up(step0);
            load(step0);
            look_up(step0 + 1);
        }
        if (tid < 4) flags[tid] = 0;
        Queries<D, QT> w;
        w.load(a, t, g, first, li, lh);
        for (int i = 0; i < steps; i++) {
            const int key = (step0 + i) * STEP;
            const bool edge = key < t.all.lo || key + STEP > t.all.hi;
            __syncthreads();  // the panels' last readers are done
            bool absent = false, dropped = false;
#pragma unroll
            for (int j = 0; j < PASSES; j++) {
                const int row = j * RPP + srow;
                absent |= slot[j] >= a.cache.slots;
                if (sg == 0) there[(i & 1) * STEP + row] = slot[j] < a.cache.slots;
                if (edge) dropped |= drop(vr[j], vd[j]);
                kr[j].template stage<false>(kp + row * (D * 2), PLANE, sg, k_swizzle<D>(row), 0.0f);
                if (KIND == kCacheQ8 && sg % 4 == 0) k_scale[(sg / 4) * STEP + row] = half_value(kd[j]);
                vr[j].template stage<true>(vp + row * (D * 2), PLANE, sg, v_swizzle<D>(row), half_value(vd[j]));
            }
            if (absent) flags[i & 1] = 1;
            if (dropped) flags[2 + (i & 1)] = 1;
            if (i + 1 < steps) {
                load(step0 + i + 1);
                look_up(step0 + i + 2);
            }
            __syncthreads();
            if (tid == 0) flags[(i + 1) & 1] = flags[2 + ((i + 1) & 1)] = 0;
            if (!works) continue;
            const bool partial = edge || flags[i & 1];
            const bool fix = flags[2 + (i & 1)];
            constexpr int H = STEP / 32;
            f32x4 s[H][2][QT];
#pragma unroll
            for (int h = 0; h < H; h++) {
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int u = 0; u < QT; u++) s[h][j][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < C; c++) {
                    bf16x8 f[2][NPK];
                    f32x4 x[2][QT];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int row = 32 * h + 16 * j + li;
#pragma unroll
                        for (int e = 0; e < NPK; e++)
                            f[j][e] = *reinterpret_cast<const bf16x8 *>(kp + e * PLANE + row * (D * 2) +
                                                                        (((4 * c + lh) ^ k_swizzle<D>(row)) << 4));
#pragma unroll
                        for (int u = 0; u < QT; u++)
                            x[j][u] = KIND == kCacheQ8 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : s[h][j][u];
                    }
#pragma unroll
                    for (int sum = 2; sum >= 0; sum--)
#pragma unroll
                        for (int e = NPK - 1; e >= 0; e--)
                            if (sum - e >= 0)
#pragma unroll
                                for (int j = 0; j < 2; j++)
#pragma unroll
                                    for (int u = 0; u < QT; u++)
                                        x[j][u] = mfma16x16x32_bf16(f[j][e], w.q[u][c][sum - e], x[j][u]);
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        if constexpr (KIND == kCacheQ8) {
                            const f32x4 d =
                                *reinterpret_cast<const f32x4 *>(k_scale + c * STEP + 32 * h + 16 * j + 4 * lh);
#pragma unroll
                            for (int u = 0; u < QT; u++)
#pragma unroll
                                for (int r = 0; r < 4; r++)
                                    s[h][j][u][r] = __builtin_fmaf(d[r], x[j][u][r], s[h][j][u][r]);
                        } else {
#pragma unroll
                            for (int u = 0; u < QT; u++) s[h][j][u] = x[j][u];
                        }
                }
            }
            if (partial)
#pragma unroll
                for (int h = 0; h < H; h++) {
                    const uint32_t present = (uint32_t)__ballot(there[(i & 1) * STEP + 32 * h + (lane & 31)] != 0);
                    w.mask(s[h], key + 32 * h, present, lh);
                }
            w.raise(s, a.scale_log2);
            const int vrow = 4 * lh + (li >> 2);
#pragma unroll
            for (int h = 0; h < H; h++) {
                bf16x8 p[QT][3];
                w.weights(s[h], a.scale_log2);
#pragma unroll
                for (int u = 0; u < QT; u++) split3(s[h][0][u], s[h][1][u], p[u]);
                w.template add<NPV, 0, D / 16>(vp + (32 * h + vrow) * (D * 2) + (li & 1) * 8, PLANE, v_swizzle<D>(vrow),
                                    (li & 3) >> 1, p);
            }
            if (fix)
                for (int h = 0; h < H; h++) add_not_finite<KIND>(a, t, g, w, key + 32 * h, lh);
        }
        const Output<BM, D, false> out{a, t, g, part};
#pragma unroll
        for (int u = 0; u < QT; u++) {
            const float l = sum_groups(w.l[u]);
#pragma unroll
            for (int df = 0; df < D / 16; df++)
                out.put(first + 16 * u + li, 16 * df + 4 * lh, w.o[df][u], w.m[u], l);
        }
        __syncthreads();
    });
}

// Joins the parts of many_rows_kernel, whose tiles would keep the last workgroup of
// each busy for long (a frame against eight 115 us this way, 138 the other; the few
// rows of the other kernel are joined there: one token 15.2 us against 18.2).  A
// workgroup takes so few rows that each has two of its groups of lanes: the parts of a
// row are a chain of loads (128 tokens against 4096 keys of 12 heads of 64 in floats 33.0
// us, with twice the rows 36.7, with half 30.5, but three chunks of 900 57.2, 55.6, 61.0).
template <int D>
constexpr int kJoinRows = 512 / D;
template <int BM, int D>
__global__ __launch_bounds__(256) void join_kernel(CacheAttn a) {
    __shared__ __attribute__((aligned(16))) char smem[256 * sizeof(Sums)];
    const Joint j = *joint_of<BM, D>(a, blockIdx.x);
    const int from = blockIdx.y * kJoinRows<D>;
    if (j.last < 0 || from >= j.rows) return;
    Tile t{};
    t.start = uniform(j.start);
    t.row = uniform(j.row);
    t.rows = uniform(j.rows);
    join_parts<BM, D, 256, false>(a, t, uniform(j.head), blockIdx.x, uniform(j.last), uniform(j.part), from,
                                  min(from + kJoinRows<D>, t.rows), smem);
}

template <int KIND, int D>
hipError_t run_kind(hipStream_t s, const CacheAttn &a, bool few) {
    const size_t lds = few ? 4 * few_wave_bytes<KIND, D>() : many_bytes<KIND, D>();
    const size_t index = ((size_t)a.requests + 1) * sizeof(int);
    static std::atomic<uint64_t> done_few{0}, done_many{0};
    constexpr size_t most = (kMaxRequests + 1) * sizeof(int);
    hipError_t e = few ? ensure_dynamic_lds(few_rows_kernel<KIND, D>, 4 * few_wave_bytes<KIND, D>() + most, done_few)
                       : ensure_dynamic_lds(many_rows_kernel<KIND, D>, many_bytes<KIND, D>() + most, done_many);
    if (e != hipSuccess) return e;
    if (few) few_rows_kernel<KIND, D><<<a.shares, 256, lds + index, s>>>(a);
    else many_rows_kernel<KIND, D><<<a.shares, kManyThreads<D>, lds + index, s>>>(a);
    e = hipGetLastError();
    if (e != hipSuccess || few || !a.parts) return e;
    join_kernel<128, D><<<dim3(a.shares, 128 / kJoinRows<D>), 256, 0, s>>>(a);
    return hipGetLastError();
}

constexpr int kShares = 512;

// Whether requests of these query rows (new tokens times the heads that share a head
// of the cache) go to tiles of 16, by their average.  More rows read K and V once
// for each 16; tiles of 128 do the arithmetic of 128 whatever they hold.  Measured in
// us, tiles of 16 / of 128, for 16, 32, 64 and 128 rows against 65536 keys of one request
// and 4096 of sixteen (f32 and bf16 heads: 12 of 64; wide: 8 of 128 for 32):
//   f32        78/117 133/118 220/143 472/169    74/116 133/119 214/141 367/169
//   f32 wide  102/155 169/158 314/162 602/215    91/144 145/147 283/154 572/215
//   bf16       49/71   71/73  103/89  226/96     42/71   69/73  108/89  179/96
//   bf16 wide  76/88  102/90  170/91  315/116    58/79   63/80   92/82  198/110
//   Q8_0       47/117  67/119 114/135 215/142    41/116  67/117 114/133 209/139
//   Q8_0 wide  68/161  84/164 135/165 253/194    48/152  72/154 118/156 233/185
// Fewer keys, whose number the host does not know, favour the tiles of 16 more: 64 rows
// against 4096 of one request f32 24/33, bf16 18/29, Q8_0 19/33.  So floats keep 32 rows, where
// the table has the tiles of 128 ahead: against 300, 1000 and 4096 keys of one request f32 14/17
// 15/20 21/26, wide 18/18 20/21 30/30; of sixteen 26/27 48/43 136/114, wide 24/28 50/51 159/147.
// The average is the call's: a chunk beside single tokens sends all to one form.  A chunk of 2000
// with 63 tokens, 4096 keys each, 32 / 8 heads of 128: bf16 621 us in one call, 448 in two, Q8_0
// 1113 and 611; a chunk of 449: 316 and 271, 339 and 285.
bool few_rows(const CacheView &c, size_t rows, size_t requests) {
    return rows <= (c.kind == kCacheQ8 ? 64 : 32) * requests;
}

// As many workgroups as run at once: two a CU, one of eight waves (Q8_0 chunks of 32 /
// 8 heads of 128: 368 us, with two 388) or of the LDS of wide floats.
int shares_of(const CacheView &c, bool few) {
    return c.width == 128 && (!few || c.kind == kCacheF32) ? kShares / 2 : kShares;
}

}  // namespace

static_assert(kShares <= kAttnCounters, "a counter for each share");

size_t cache_attn_floats(const CacheView &cache, size_t tokens, size_t group, size_t requests) {
    const bool few = few_rows(cache, tokens * group, requests);
    const size_t shares = shares_of(cache, few);
    return 2 * shares * (few ? 16 : 128) * (cache.width + 2) + (few ? 0 : shares * sizeof(Joint) / sizeof(float));
}

hipError_t launch_cache_attn(hipStream_t s, CacheAttn a) {
    const bool few = few_rows(a.cache, (size_t)a.tokens * a.group, (size_t)a.requests);
    const bool wide = a.cache.width == 128;
    a.shares = shares_of(a.cache, few);
    // What a row of the table holds, short of where a step past it no longer counts in 31 bits.
    a.row_keys = (int)std::min(a.max_pages << a.cache.page_shift, (long long)INT32_MAX - 4095);
    switch (a.cache.kind) {
        case kCacheF32: return wide ? run_kind<kCacheF32, 128>(s, a, few) : run_kind<kCacheF32, 64>(s, a, few);
        case kCacheBf16: return wide ? run_kind<kCacheBf16, 128>(s, a, few) : run_kind<kCacheBf16, 64>(s, a, few);
        default: return wide ? run_kind<kCacheQ8, 128>(s, a, few) : run_kind<kCacheQ8, 64>(s, a, few);
    }
}

}  // namespace vh
