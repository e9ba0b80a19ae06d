// Rows in 8-bit floating point (e4m3) with a power-of-two scale for each 128 values,
// and products with them (kernels.h Fp8Rows).
//
// Quantising: a block's exponent e is the least with all of its finite values within
// 448 * 2^e (448 is the largest e4m3), a code is x * 2^-e rounded to nearest even: the
// scaling is exact, so a value is rounded once.  A block is 4 + 1 bytes a value of
// traffic, bound by HBM.
//
// Products go through f16: every e4m3 is a half, and products of two are exact in the
// f32 sums of v_mfma_f32_16x16x32_f16.  The fp8 matrix instructions would take half
// the time, but keep only some 14 bits below the largest product of a group of k
// (measured on N(0, 1): 1.5e-5 of the result's norm at any K, the same for
// the scaled and the plain form), which is no 32-bit sum.  The conversion
// (v_cvt_scalef32_pk_f16_fp8) takes a power-of-two scale: a block's exponent relative to
// the largest of its row, so that one f32 sum runs over all of K and the rows' exponents
// join behind it.  That is exact while a row's exponents are within 15 of each other (blocks
// of zeros aside).  Rows that are wider say so (fp8_row), and a wave of a tile that meets one forms
// its 16 rows' sums again, each block's on its own exponents, as the products of few rows do
// it: what is small in one side's row may stand against what is large in the other's.
//
// Storage, "panels": 16 rows x 128 values are 2048 bytes, [half 2][lane 64][16]: lane
// (row li, lh) of half h holds values 32 lh + 16 h .. + 15 of its row, so that a
// fragment is one 16-byte read of consecutive lanes everywhere: memory to LDS, LDS to
// registers, or memory to registers.  (Any order of k does for a product, as long as
// both sides have it.)
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "common.h"
#include "kernels.h"
#include "split_gemm.h"

namespace vh {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr size_t kMaxGrid = 65536;  // of the kernels that walk their tiles
constexpr size_t kMaxThreads = (size_t)1 << 32, kMaxGridY = 65535;  // of a launch

// The exponent of a block whose largest finite magnitude has these bits: 448 = 1.75 * 2^8.
__device__ __forceinline__ int block_exponent(uint32_t amax) {
    const int e = (int)(amax >> 23) - 135 + ((amax & 0x7fffff) > 0x600000 ? 1 : 0);
    return max(e, -127);
}
__device__ __forceinline__ float pow2(int e) {  // -126 <= e <= 127
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Where dword c (values 4 c .. + 3) of row r is in a panel in LDS, and 16 bytes of lane `lane` of
// half h: as in memory, but for the row, which is swizzled so that the dwords of two rows
// of 32 lanes go to different banks.
__device__ __forceinline__ int panel_at(int r, int c) {
    const int h = (c >> 2) & 1, lh = c >> 3;
    return h * 1024 + (lh * 16 + (r ^ (4 * lh + 2 * h))) * 16 + (c & 3) * 4;
}
__device__ __forceinline__ int panel_lane(int lane, int h) {
    return h * 1024 + (lane ^ (4 * (lane >> 4) + 2 * h)) * 16;
}

// Largest magnitude's bits, of the finite values alone.
__device__ __forceinline__ uint32_t finite_max(uint32_t mx, float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    return max(mx, b < 0x7f800000u ? b : 0u);
}
__device__ __forceinline__ int e4m3_of(f32x4 v) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
}
// For rows that may hold what is not finite.
__device__ __forceinline__ f32x4 scaled(f32x4 v, float inv) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = fabsf(v[i]) < INFINITY ? v[i] * inv : NAN;
    return v;
}

// Four values of a row of k floats from column d on (zeros past its end).
template <bool VEC>
__device__ __forceinline__ f32x4 row4(const float *row, size_t d, size_t k) {
    if constexpr (VEC) {
        if (d < k) return *reinterpret_cast<const f32x4 *>(row + d);
        return f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = d + i < k ? row[d + i] : 0.0f;
    return v;
}

// 16 rows' floats of a block, 32 lanes a row: of the nearest there are, so that no load is in a
// branch (where every one would be waited for); clear_panel takes out what was not asked
// for.  VEC: whole float4 at 32 bits of a lane's own, below 2^24 values a row.
constexpr size_t kVecK = (size_t)1 << 24;
template <bool VEC, bool NT>
__device__ __forceinline__ void load_panel(const float *x, const Fp8Rows &w, size_t tile, size_t b, int lane,
                                           f32x4 (&v)[8]) {
    asm volatile("" : "+v"(lane));
    const int side = lane >> 5, c = lane & 31;
    const int last = (int)min((size_t)16, w.rows - tile * 16) - 1;
    if constexpr (VEC) {
        const char *base = reinterpret_cast<const char *>(x + tile * 16 * w.k);
        const uint32_t at = (uint32_t)min(b * 128 + 4 * c, w.k - 4) * 4, row_bytes = (uint32_t)w.k * 4;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const f32x4 *p = reinterpret_cast<const f32x4 *>(base + (at + min(2 * i + side, last) * row_bytes));
            v[i] = NT ? __builtin_nontemporal_load(p) : *p;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float *row = x + (tile * 16 + min(2 * i + side, last)) * w.k;
#pragma unroll
            for (int j = 0; j < 4; j++) v[i][j] = row[min(b * 128 + 4 * c + j, w.k - 1)];
        }
    }
}
__device__ __forceinline__ void clear_panel(const Fp8Rows &w, size_t tile, size_t b, int lane, f32x4 (&v)[8]) {
    if (tile * 16 + 16 <= w.rows && b * 128 + 128 <= w.k) return;
    const int side = lane >> 5, c = lane & 31;
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (tile * 16 + 2 * i + side >= w.rows || b * 128 + 4 * c + j >= w.k) v[i][j] = 0.0f;
}
// Largest of the 32 lanes of a row, in each of them.
__device__ __forceinline__ uint32_t row_umax(uint32_t v) {
    v = dpp_umax<0x140>(dpp_umax<0x141>(dpp_umax<0x4e>(dpp_umax<0xb1>(v))));
    return max(v, (uint32_t)__shfl_xor((int)v, 16, kWave));
}
// Their codes; `to`: 2048 bytes of the wave's own.  Lanes 0 .. 7 of either half get the
// exponents of rows 2 lane + half, kEmpty where all values are zeros.
constexpr int kEmpty = -128;
__device__ __forceinline__ int quantize_panel(f32x4 (&v)[8], const Fp8Rows &out, size_t tile, size_t b, int lane,
                                              char *to) {
    // Opaque: what follows from the lane (addresses, masks) is formed for each panel anew, not kept
    // over the loop in 90 registers.
    asm volatile("" : "+v"(lane));
    const int c = lane & 31, side = lane >> 5;
    clear_panel(out, tile, b, lane, v);
    uint32_t mx[8], most = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        mx[i] = row_umax(absmax4(0, v[i]));
        most = max(most, mx[i]);
    }
    if (__any(most >= 0x7f800000u)) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                m = finite_max(m, v[i][j]);
                v[i][j] = fabsf(v[i][j]) < INFINITY ? v[i][j] : NAN;
            }
            mx[i] = row_umax(m);
        }
    }
    int mine = kEmpty;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int e = block_exponent(mx[i]);
        *reinterpret_cast<int *>(to + panel_at(2 * i + side, c)) = e4m3_of(v[i] * pow2(-e));
        if (c == i) mine = mx[i] ? e : kEmpty;
    }
    wave_sync();
    char *at = reinterpret_cast<char *>(out.codes) + (tile * fp8_blocks(out.k) + b) * 2048 + lane * 16;
#pragma unroll
    for (int h = 0; h < 2; h++)
        *reinterpret_cast<u32x4 *>(at + h * 1024) = *reinterpret_cast<const u32x4 *>(to + panel_lane(lane, h));
    wave_sync();
    if (c < 8) out.exps[b * fp8_rows16(out.rows) + tile * 16 + 2 * c + side] = (uint8_t)(max(mine, -127) + 127);
    return mine;
}

// A workgroup takes 16 rows, its waves their blocks in turn.  Rows past the end become
// zeros.  Bound by HBM where there are many rows (13828 x 4096 58.7 us, 4.8 TB/s); the next
// block's floats asked for ahead, or fewer waves a workgroup, are no faster.
constexpr int kQuantThreads = 512, kQuantBlocks = 256;  // whose exponents stay in LDS
template <bool VEC, bool NT>
__global__ __launch_bounds__(kQuantThreads) void quantize_fp8_kernel(const float *x, Fp8Rows out) {
    constexpr int W = kQuantThreads / 64;
    __shared__ __attribute__((aligned(16))) char stage[W][2048];
    __shared__ int wave_max[W][16], wave_min[W][16];
    __shared__ uint8_t codes[kQuantBlocks * 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 31, row = 2 * c + (lane >> 5);
    const size_t kb = fp8_blocks(out.k), rows16 = fp8_rows16(out.rows);
    for (size_t tile = blockIdx.x; tile < rows16 / 16; tile += gridDim.x) {
        int most = -127, least = 127;
        for (size_t b = wave; b < kb; b += W) {
            f32x4 v[8];
            load_panel<VEC, NT>(x, out, tile, b, lane, v);
            const int e = quantize_panel(v, out, tile, b, lane, stage[wave]);
            if (c < 8 && b < kQuantBlocks) codes[b * 16 + row] = (uint8_t)(max(e, -127) + 127);
            most = max(most, e);
            if (e != kEmpty) least = min(least, e);
        }
        if (c < 8) {
            wave_max[wave][row] = most;
            wave_min[wave][row] = least;
        }
        __syncthreads();
        // Thread t writes row t % 16 of the blocks t / 16, ...
        most = wave_max[0][tid & 15];
        least = wave_min[0][tid & 15];
#pragma unroll
        for (int w = 1; w < W; w++) {
            most = max(most, wave_max[w][tid & 15]);
            least = min(least, wave_min[w][tid & 15]);
        }
        if (tid < 16) out.row_e[tile * 16 + tid] = fp8_row(most, least);
        for (size_t i = tid; i < kb * 16; i += kQuantThreads) {
            const size_t at = (i >> 4) * rows16 + tile * 16 + (i & 15);
            out.rel[at] = fp8_relative(i < kQuantBlocks * 16 ? codes[i] : out.exps[at], most);
        }
        __syncthreads();
    }
}

// Where there are few rows: codes and exponents alone, a wave a panel; then what follows from
// the exponents, until when `rel` says which blocks are all zeros.
template <bool VEC>
__global__ __launch_bounds__(64) void quantize_panels_kernel(const float *x, Fp8Rows out) {
    __shared__ __attribute__((aligned(16))) char stage[2048];
    f32x4 v[8];
    load_panel<VEC, false>(x, out, blockIdx.y, blockIdx.x, threadIdx.x, v);
    const int e = quantize_panel(v, out, blockIdx.y, blockIdx.x, threadIdx.x, stage);
    const int c = threadIdx.x & 31, row = 2 * c + (threadIdx.x >> 5);
    if (c < 8) out.rel[blockIdx.x * fp8_rows16(out.rows) + blockIdx.y * 16 + row] = e == kEmpty;
}
__global__ __launch_bounds__(256) void relative_fp8_kernel(Fp8Rows out) {
    __shared__ int some[16][16], low[16][16];
    const int tid = threadIdx.x, r = tid & 15, part = tid >> 4;
    const size_t kb = fp8_blocks(out.k), rows16 = fp8_rows16(out.rows), row = (size_t)blockIdx.x * 16 + r;
    int most = 0, least = 254;
    for (size_t b = part; b < kb; b += 16) {
        const int e = out.exps[b * rows16 + row];
        most = max(most, e);
        if (!out.rel[b * rows16 + row]) least = min(least, e);
    }
    some[part][r] = most;
    low[part][r] = least;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; i++) {
        most = max(most, some[i][r]);
        least = min(least, low[i][r]);
    }
    if (part == 0) out.row_e[row] = fp8_row(most - 127, least - 127);
    for (size_t b = part; b < kb; b += 16) out.rel[b * rows16 + row] = fp8_relative(out.exps[b * rows16 + row], most - 127);
}

// The values that the codes stand for, a wave a panel; through LDS, so that rows are written in 512
// bytes at once.  Bound by HBM (13828 x 4096 44 us, 6.4 TB/s); 865 x 768 4.1 us, a launch and two latencies.
template <bool VEC, bool NT>
__global__ __launch_bounds__(256) void dequantize_fp8_kernel(Fp8Rows in, float *out) {
    __shared__ __attribute__((aligned(16))) char stage[4][2048];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 31, side = lane >> 5;
    const size_t kb = fp8_blocks(in.k), rows16 = fp8_rows16(in.rows), tiles = rows16 / 16 * kb;
    for (size_t i0 = (size_t)blockIdx.x * 4; i0 < tiles; i0 += (size_t)gridDim.x * 4) {
        const size_t i = i0 + wave;
        if (i >= tiles) break;
        const size_t tile = i / kb, b = i - tile * kb;
        const char *at = reinterpret_cast<const char *>(in.codes) + i * 2048 + lane * 16;
        char *to = stage[wave];
#pragma unroll
        for (int h = 0; h < 2; h++)
            *reinterpret_cast<u32x4 *>(to + panel_lane(lane, h)) = *reinterpret_cast<const u32x4 *>(at + h * 1024);
        wave_sync();
#pragma unroll
        for (int r0 = 0; r0 < 8; r0++) {
            const int r = 2 * r0 + side;
            const size_t row = tile * 16 + r, d = b * 128 + 4 * c;
            const int word = *reinterpret_cast<const int *>(to + panel_at(r, c));
            const int e = (int)in.exps[b * rows16 + row] - 127;
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(word, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
            const f32x4 v{ldexpf(lo[0], e), ldexpf(lo[1], e), ldexpf(hi[0], e), ldexpf(hi[1], e)};
            if (row >= in.rows || d >= in.k) continue;
            float *y = out + row * in.k + d;
            if constexpr (VEC && NT) {
                __builtin_nontemporal_store(v, reinterpret_cast<f32x4 *>(y));
            } else if constexpr (VEC) {
                *reinterpret_cast<f32x4 *>(y) = v;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (d + j < in.k) y[j] = v[j];
            }
        }
        wave_sync();
    }
}

// ---- products ------------------------------------------------------------------------

// 8 codes as halves, times the power of two `scale`.
__device__ __forceinline__ f16x8 halves(uint32_t w0, uint32_t w1, float scale) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, scale, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, scale, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, scale, false);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, scale, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Four consecutive outputs of row m, columns n .. n + 3, from their sums.
template <Epi EPI>
__device__ __forceinline__ void put4(const Fp8Gemm &g, size_t m, size_t n, f32x4 v) {
    if (m >= g.m || n >= g.n) return;
    float *c = g.c + m * g.n + n;
    const int count = (int)min((size_t)4, g.n - n);
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const size_t at = n + min(r, count - 1);
        if (g.bias) v[r] += g.bias[at];
        if (EPI == Epi::Gelu) v[r] = gelu_fast_form(v[r]);
        else if (g.gamma) v[r] *= g.gamma[at];
    }
    if ((g.n & 3) == 0) {
        if (EPI == Epi::Residual) v += *reinterpret_cast<const f32x4 *>(c);
        stream_store(reinterpret_cast<f32x4 *>(c), v);
    } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (r < count) c[r] = EPI == Epi::Residual ? c[r] + v[r] : v[r];
    }
}

// What joins a block's sum of 16 columns of B (panel nt) to the others: exponents of the columns 4 lh .. + 3,
// or a checkpoint's scale as a significand in [1, 2) and an exponent (far below every sum for a zero), so
// that no intermediate is larger than the product: with the scale multiplied in behind the exponents of rows
// whose other scales are far above it, a finite product passed the floats on its way.
struct Scale {
    float significand;
    int e[4];
};
template <bool BLOCKS>
__device__ __forceinline__ Scale block_scale(const Fp8Gemm &g, size_t nt, size_t b, int lh) {
    Scale s{1.0f, {}};
    if constexpr (BLOCKS) {
        const float v = g.b_scales[nt / 8 * fp8_blocks(g.b.k) + b];
        s.significand = 2.0f * __builtin_amdgcn_frexp_mantf(v);
        const int e = v == 0.0f ? -1000 : __builtin_amdgcn_frexp_expf(v) - 1;
#pragma unroll
        for (int r = 0; r < 4; r++) s.e[r] = e;
    } else {
        const uint32_t e = *reinterpret_cast<const uint32_t *>(g.b.exps + b * fp8_rows16(g.b.rows) + nt * 16 + 4 * lh);
#pragma unroll
        for (int r = 0; r < 4; r++) s.e[r] = (int)((e >> (8 * r)) & 255) - 127;
    }
    return s;
}
__device__ __forceinline__ void join_block(f32x4 &acc, f32x4 part, int ea, const Scale &s) {
#pragma unroll
    for (int r = 0; r < 4; r++) acc[r] = __builtin_fmaf(s.significand, __builtin_ldexpf(part[r], ea + s.e[r]), acc[r]);
}

// The sums of 16 rows (panel mt of A) by 16 TN columns (panels nt .. of B; past the end the last), a block after the
// other on its own exponents, from memory: of rows too wide for the sums of a tile.  The loads of a block's
// panels are in flight together (865 x 768 by 3072 with a wide row in every 16 20.9 us, without 12.7; 13828 x 4096 by
// 8192 2.35 ms and 0.85).
template <int TN, bool BLOCKS>
__device__ __forceinline__ void wide_sums(const Fp8Gemm &g, size_t mt, size_t nt, int lane, f32x4 (&acc)[TN]) {
    const size_t kb = fp8_blocks(g.a.k), a16 = fp8_rows16(g.a.rows), last = fp8_rows16(g.b.rows) / 16 - 1;
    mt = min(mt, a16 / 16 - 1);
#pragma unroll
    for (int j = 0; j < TN; j++) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (size_t b = 0; b < kb; b++) {
        u32x4 x[2], y[TN][2];
        Scale s[TN];
        const int ea = (int)g.a.exps[b * a16 + mt * 16 + (lane & 15)] - 127;
#pragma unroll
        for (int h = 0; h < 2; h++)
            x[h] = *reinterpret_cast<const u32x4 *>(g.a.codes + (mt * kb + b) * 2048 + h * 1024 + lane * 16);
#pragma unroll
        for (int j = 0; j < TN; j++) {
            const size_t panel = min(nt + j, last);
            s[j] = block_scale<BLOCKS>(g, panel, b, lane >> 4);
#pragma unroll
            for (int h = 0; h < 2; h++)
                y[j][h] = *reinterpret_cast<const u32x4 *>(g.b.codes + (panel * kb + b) * 2048 + h * 1024 + lane * 16);
        }
#pragma unroll
        for (int j = 0; j < TN; j++) {
            f32x4 part{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    part = mfma16x16x32_f16(halves(y[j][h][2 * e], y[j][h][2 * e + 1], 1.0f),
                                            halves(x[h][2 * e], x[h][2 * e + 1], 1.0f), part);
            join_block(acc[j], part, ea, s[j]);
        }
    }
}

// The lane, from no register: what it gives is not kept over a loop.  (Tiles of 256 have none to spare:
// the reload of one that was spilled waits for the copies before it: 13824 x 4096 by 8192 796 us,
// so 735.)
__device__ __forceinline__ int fresh_lane() {
    int lane;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
    return lane;
}

// C = A . B^T, a workgroup of WM x WN waves a tile of BM x BN.  Two stages of 128 k in
// LDS; D^T = B . A^T, so that a lane holds four consecutive columns of its row.
// BLOCKS: B has float scales for 128 x 128 values (b_rel) on top of its rows' exponents.
//
// What bounds it: tiles of 256 (waves of 128 x 64, 1.7 other vector instructions a matrix
// instruction) the matrix cores at the clock that they leave, 13824 x 4096 by 8192 721 us, 1286
// TFLOP/s at 2.15 GHz in a row of a hundred (the first ones after a pause take 750 to 910 us, at 2.06 down
// to 1.7 GHz), where a library's product of 8192^3 halves has 1139; tiles of 128 (waves of 64 x 32, 3.5,
// with BLOCKS 4.5) the issue of instructions, 4001 x 2200 by 5001 107 us, BLOCKS 114; tiles of 64
// (waves of 32 x 32, 5) the same and the start of a tile, 865 x 768 by 3072 11.7 us.  Waves of 64 x
// 64 for the middle ones, in tiles of 256 x 128, 133 and 136 us, in tiles of 128 of four waves, 114.5
// and 115: fewer waves hide less.  Three stages in LDS are no faster.
constexpr int kStages = 2;
template <int BM, int BN>
constexpr int kStageBytes = (BM + BN) * 128 + (BM + BN) * 2;  // codes, relative exponents
template <int BM, int BN, int WM, int WN, Epi EPI, bool BLOCKS>
__global__ __launch_bounds__(WM *WN * 64, 2) void fp8_gemm_kernel(Fp8Gemm g) {
    constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
    constexpr int CODES = (BM + BN) * 128, STAGE = kStageBytes<BM, BN>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr bool kSpare = TM * TN < 32;  // registers
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM;

    // Workgroups go round-robin over the 8 XCDs: each takes a run of tiles, eight
    // rows of tiles deep, so that its L2 holds what they share.
    const int per = (g.tiles + 7) / 8, item = (blockIdx.x % 8) * per + blockIdx.x / 8;
    if (item >= g.tiles || (int)(blockIdx.x / 8) >= per) return;
    constexpr int DEEP = 8;
    const int group = item / (DEEP * g.n_tiles), m_first = group * DEEP, deep = min(DEEP, g.m_tiles - m_first);
    const int in = item - group * DEEP * g.n_tiles;
    const int mt = m_first + in % deep, nt = in / deep;

    const size_t kb = fp8_blocks(g.a.k), a16 = fp8_rows16(g.a.rows), b16 = fp8_rows16(g.b.rows);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)smem;
    // Units of 1 KB: halves of panels, A's then B's; then the blocks' relative exponents.
    auto copy = [&](size_t b, int buf, int lane) {
#pragma unroll
        for (int i = 0; i < (BM + BN) / 8 / NW; i++) {
            const int u = wave + i * NW;
            const bool is_a = u < BM / 8;
            const size_t t = is_a ? min((size_t)mt * (BM / 16) + u / 2, a16 / 16 - 1)
                                  : min((size_t)nt * (BN / 16) + (u - BM / 8) / 2, b16 / 16 - 1);
            const char *from = reinterpret_cast<const char *>(is_a ? g.a.codes : g.b.codes) + (t * kb + b) * 2048 + (u & 1) * 1024;
            copy16_to_lds(from, lane * 16, __builtin_amdgcn_readfirstlane(lds0 + buf * STAGE + u * 1024));
        }
        // Eight rows a lane (past the end: the last eight); half of the waves A's, half B's, so that
        // every wave has as many copies.
        const bool is_a = wave < NW / 2;
        const int rows = (is_a ? BM : BN) / (NW / 2), first = wave % (NW / 2) * rows;
        if (lane < rows / 8) {
            const size_t r16 = is_a ? a16 : b16;
            const uint32_t row = (uint32_t)(is_a ? mt * BM : nt * BN) + first + lane * 8;
            const uint32_t at = min(row, (uint32_t)r16 - 8) * 2;
            copy16_to_lds((is_a ? g.a.rel : g.b.rel) + b * r16, at,
                          __builtin_amdgcn_readfirstlane(lds0 + buf * STAGE + CODES + ((is_a ? 0 : BM) + first) * 2));
        }
    };
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    static_assert((BM + BN) / 8 % NW == 0 && BM / (NW / 2) % 8 == 0 && BN / (NW / 2) % 8 == 0 && NW % 2 == 0);
    copy(0, 0, tid & 63);
    for (size_t b = 0; b < kb; b++) {
        const int buf = (int)(b % kStages);
        split_wait<0>();  // this stage landed
        __builtin_amdgcn_s_barrier();
        const int lane = kSpare ? tid & 63 : fresh_lane(), li = lane & 15;
        if (b + 1 < kb) copy(b + 1, buf ^ 1, lane);
        const char *as = smem + buf * STAGE + wm * TM * 2048 + lane * 16;
        const char *bs = smem + buf * STAGE + BM * 128 + wn * TN * 2048 + lane * 16;
        const uint16_t *rs = reinterpret_cast<const uint16_t *>(smem + buf * STAGE + CODES);
        float ra[TM], rb[TN];
#pragma unroll
        for (int i = 0; i < TM; i++) ra[i] = __uint_as_float((uint32_t)rs[(wm * TM + i) * 16 + li] << 16);
#pragma unroll
        for (int j = 0; j < TN; j++)
            rb[j] = BLOCKS ? 1.0f : __uint_as_float((uint32_t)rs[BM + (wn * TN + j) * 16 + li] << 16);
        if constexpr (BLOCKS) {
            // A block's sum from zero, a row of tiles at a time, then onto the others by its scale.
            const size_t n_block = min(((size_t)nt * BN + wn * TN * 16) / 128, (b16 - 1) / 128);
            const float s = g.b_rel[n_block * kb + b];
            f16x8 fb[TN][4];
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const u32x4 y = *reinterpret_cast<const u32x4 *>(bs + j * 2048 + h * 1024);
                    fb[j][2 * h] = halves(y[0], y[1], 1.0f);
                    fb[j][2 * h + 1] = halves(y[2], y[3], 1.0f);
                }
#pragma unroll
            for (int i = 0; i < TM; i++) {
                f16x8 fa[4];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const u32x4 x = *reinterpret_cast<const u32x4 *>(as + i * 2048 + h * 1024);
                    fa[2 * h] = halves(x[0], x[1], ra[i]);
                    fa[2 * h + 1] = halves(x[2], x[3], ra[i]);
                }
                f32x4 part[TN];
#pragma unroll
                for (int j = 0; j < TN; j++) part[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int j = 0; j < TN; j++) part[j] = mfma16x16x32_f16(fb[j][e], fa[e], part[j]);
#pragma unroll
                for (int j = 0; j < TN; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[i][j][r] = __builtin_fmaf(part[j][r], s, acc[i][j][r]);
            }
            continue;
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            u32x4 x[TM], y[TN];
#pragma unroll
            for (int j = 0; j < TN; j++) y[j] = *reinterpret_cast<const u32x4 *>(bs + j * 2048 + h * 1024);
#pragma unroll
            for (int i = 0; i < TM; i++) x[i] = *reinterpret_cast<const u32x4 *>(as + i * 2048 + h * 1024);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                f16x8 fb[TN];
#pragma unroll
                for (int j = 0; j < TN; j++) fb[j] = halves(y[j][2 * e], y[j][2 * e + 1], rb[j]);
#pragma unroll
                for (int i = 0; i < TM; i++) {
                    const f16x8 fa = halves(x[i][2 * e], x[i][2 * e + 1], ra[i]);
#pragma unroll
                    for (int j = 0; j < TN; j++) acc[i][j] = mfma16x16x32_f16(fb[j], fa, acc[i][j]);
                }
            }
        }
    }
    // 16 rows at a time through LDS of the wave's own, so that a row is written in one piece,
    // whatever its alignment (1239 x 50 x 7838, no multiple of four, from floats: 63 us without, 25 with).
    constexpr int W = TN * 16, PITCH = W + 4;
    static_assert(NW * 16 * PITCH * 4 <= kStages * STAGE, "room for every wave's rows");
    __syncthreads();
    float *rows = reinterpret_cast<float *>(smem) + wave * 16 * PITCH;
    const int lane = kSpare ? tid & 63 : fresh_lane(), li = lane & 15, lh = lane >> 4;
    const size_t n0 = (size_t)nt * BN + wn * W;
    const bool whole = (g.n & 3) == 0;
    const int lanes = whole ? W / 4 : W, row0 = lane / lanes, step = 64 / lanes;
    const size_t n = n0 + (lane % lanes) * (whole ? 4 : 1);
    f32x4 bias{0.0f, 0.0f, 0.0f, 0.0f}, gamma{1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const size_t at = min(n + (whole ? r : 0), g.n - 1);
        if (g.bias) bias[r] = g.bias[at];
        if (g.gamma) gamma[r] = g.gamma[at];
    }
    auto finish = [&](float v, int r) {
        v += bias[r];
        return EPI == Epi::Gelu ? gelu_fast_form(v) : v * gamma[r];
    };
    // The rows' exponents join the sums, those of wide rows are formed again.
    int row_a[TM], row_b[TN][4], wide_a = 0, wide_b = 0;
#pragma unroll
    for (int i = 0; i < TM; i++) wide_a |= row_a[i] = g.a.row_e[min((size_t)mt * BM + (wm * TM + i) * 16 + li, a16 - 1)];
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) wide_b |= row_b[j][r] = g.b.row_e[min(n0 + 16 * j + 4 * lh + r, b16 - 1)];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                acc[i][j][r] = ldexpf(acc[i][j][r], fp8_row_exponent(row_a[i]) + fp8_row_exponent(row_b[j][r]));
    if (__any((wide_a | wide_b) & 1)) {
#pragma unroll
        for (int i = 0; i < TM; i++)
            if (__any((row_a[i] | wide_b) & 1))
                wide_sums<TN, BLOCKS>(g, (size_t)mt * (BM / 16) + wm * TM + i, n0 / 16, lane, acc[i]);
    }
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const size_t m0 = (size_t)mt * BM + (wm * TM + i) * 16;
#pragma unroll
        for (int j = 0; j < TN; j++) *reinterpret_cast<f32x4 *>(rows + li * PITCH + 16 * j + 4 * lh) = acc[i][j];
        wave_sync();
        if (n < g.n) {
            for (int r0 = row0; r0 < 16 && m0 + r0 < g.m; r0 += step) {
                float *c = g.c + (m0 + r0) * g.n + n;
                if (whole) {
                    f32x4 v = *reinterpret_cast<const f32x4 *>(rows + r0 * PITCH + 4 * (lane % lanes));
#pragma unroll
                    for (int r = 0; r < 4; r++) v[r] = finish(v[r], r);
                    if (EPI == Epi::Residual) v += *reinterpret_cast<const f32x4 *>(c);
                    stream_store(reinterpret_cast<f32x4 *>(c), v);
                } else {
                    const float v = finish(rows[r0 * PITCH + lane % lanes], 0);
                    *c = EPI == Epi::Residual ? *c + v : v;
                }
            }
        }
        wave_sync();
    }
}

// Few rows: 16 MT rows by 16 columns a workgroup, whose waves share K between them, memory
// to registers; B is read once, past the caches.  A block's sum joins the others on its own
// exponents.  FUSED (MT = 1): A are floats, which every workgroup quantises itself.  Bound by a
// launch and the latency of a block: one row of 768 by 2304 4.3 us.
constexpr int kFewWaves = 8;
template <int MT, bool FUSED, bool BLOCKS, Epi EPI>
__global__ __launch_bounds__(kFewWaves * 64) void fp8_few_kernel(Fp8Gemm g, const float *x) {
    __shared__ f32x4 sums[kFewWaves][MT][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, lh = lane >> 4;
    const size_t kb = fp8_blocks(g.b.k), nt = blockIdx.x, mt = (size_t)blockIdx.y * MT;
    const size_t a16 = fp8_rows16(g.m);
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (size_t b = wave; b < kb; b += kFewWaves) {
        const char *from = reinterpret_cast<const char *>(g.b.codes) + (nt * kb + b) * 2048 + lane * 16;
        u32x4 y[2];
#pragma unroll
        for (int h = 0; h < 2; h++) y[h] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(from + h * 1024));
        const Scale s = block_scale<BLOCKS>(g, nt, b, lh);
#pragma unroll
        for (int i = 0; i < MT; i++) {
            u32x4 a[2];
            int ea;
            if constexpr (FUSED) {
                f32x4 v[8];
                uint32_t mx = 0;
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    const size_t d = b * 128 + 32 * lh + 4 * c;
                    v[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    if ((size_t)li < g.m) v[c] = g.b.k % 4 == 0 ? row4<true>(x + li * g.b.k, d, g.b.k) : row4<false>(x + li * g.b.k, d, g.b.k);
#pragma unroll
                    for (int j = 0; j < 4; j++) mx = finite_max(mx, v[c][j]);
                }
                mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16, kWave));
                mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, kWave));
                ea = block_exponent(mx);
                const float inv = pow2(-ea);
#pragma unroll
                for (int c = 0; c < 8; c++) a[c / 4][c % 4] = (uint32_t)e4m3_of(scaled(v[c], inv));
            } else {
                const size_t t = min(mt + i, a16 / 16 - 1);
                const char *at = reinterpret_cast<const char *>(g.a.codes) + (t * kb + b) * 2048 + lane * 16;
#pragma unroll
                for (int h = 0; h < 2; h++) a[h] = *reinterpret_cast<const u32x4 *>(at + h * 1024);
                ea = (int)g.a.exps[b * a16 + t * 16 + li] - 127;
            }
            f32x4 part{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    part = mfma16x16x32_f16(halves(y[h][2 * e], y[h][2 * e + 1], 1.0f),
                                            halves(a[h][2 * e], a[h][2 * e + 1], 1.0f), part);
            join_block(acc[i], part, ea, s);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; i++) sums[wave][i][lane] = acc[i];
    __syncthreads();
    for (int i = wave; i < MT; i += kFewWaves) {
        f32x4 v = sums[0][i][lane];
#pragma unroll
        for (int w = 1; w < kFewWaves; w++) v += sums[w][i][lane];
        put4<EPI>(g, (mt + i) * 16 + li, nt * 16 + 4 * lh, v);
    }
}

template <int BM, int BN, int WM, int WN, Epi EPI, bool BLOCKS>
hipError_t launch_tile(hipStream_t s, Fp8Gemm g) {
    constexpr size_t bytes = kStages * kStageBytes<BM, BN>;
    static std::atomic<uint64_t> done{0};
    hipError_t e = ensure_dynamic_lds(fp8_gemm_kernel<BM, BN, WM, WN, EPI, BLOCKS>, bytes, done);
    if (e != hipSuccess) return e;
    const size_t mt = (g.m + BM - 1) / BM, nt = (g.n + BN - 1) / BN;
    if (mt * nt >= kMaxThreads / (WM * WN * 64)) return hipErrorInvalidConfiguration;
    g.m_tiles = (int)mt;
    g.n_tiles = (int)nt;
    g.tiles = (int)(mt * nt);
    fp8_gemm_kernel<BM, BN, WM, WN, EPI, BLOCKS><<<(g.tiles + 7) / 8 * 8, WM * WN * 64, bytes, s>>>(g);
    return hipGetLastError();
}

template <Epi EPI, bool BLOCKS>
hipError_t launch_epi(hipStream_t s, const Fp8Gemm &g, Fp8Plan plan, const float *x) {
    if (plan == Fp8Plan::Fused || plan == Fp8Plan::Few) {
        const dim3 grid((unsigned)((g.n + 15) / 16), (unsigned)((g.m + 63) / 64));
        constexpr int threads = kFewWaves * 64;
        if (plan == Fp8Plan::Fused) fp8_few_kernel<1, true, BLOCKS, EPI><<<grid, threads, 0, s>>>(g, x);
        else if (g.m <= 16) fp8_few_kernel<1, false, BLOCKS, EPI><<<grid, threads, 0, s>>>(g, nullptr);
        else if (g.m <= 32) fp8_few_kernel<2, false, BLOCKS, EPI><<<grid, threads, 0, s>>>(g, nullptr);
        else fp8_few_kernel<4, false, BLOCKS, EPI><<<grid, threads, 0, s>>>(g, nullptr);
        return hipGetLastError();
    }
    if (plan == Fp8Plan::Tile64) return launch_tile<64, 64, 2, 2, EPI, BLOCKS>(s, g);
    if (plan == Fp8Plan::Tile128) return launch_tile<128, 128, 2, 4, EPI, BLOCKS>(s, g);
    return launch_tile<256, 256, 2, 4, EPI, BLOCKS>(s, g);
}

template <bool BLOCKS>
hipError_t launch_blocks(hipStream_t s, const Fp8Gemm &g, Epi epi, Fp8Plan plan, const float *x) {
    if (epi == Epi::Gelu) return launch_epi<Epi::Gelu, BLOCKS>(s, g, plan, x);
    if (epi == Epi::Residual) return launch_epi<Epi::Residual, BLOCKS>(s, g, plan, x);
    return launch_epi<Epi::Store, BLOCKS>(s, g, plan, x);
}

}  // namespace

// Whether the floats pass by the caches (4001 x 2200 from memory 10.3 us, through the caches 12.3;
// 13828 x 4096 58.7 and 62.1; 865 x 768 4.4 and 4.05).
constexpr size_t kFp8StreamBytes = (size_t)32 << 20;

hipError_t launch_quantize_fp8(hipStream_t s, const float *x, const Fp8Rows &out, bool products_of_few) {
    const size_t tiles = fp8_rows16(out.rows) / 16, kb = fp8_blocks(out.k);
    const bool vec = out.k % 4 == 0 && out.k <= kVecK;
    // Few rows: a wave a panel (100 x 6000 in 7.8 us, two launches, against 14.2 of one workgroup for
    // 16 rows; 865 x 768 7.0 against 4.9).
    if (products_of_few || (tiles <= 64 && kb > 16)) {
        const dim3 grid((unsigned)kb, (unsigned)tiles);
        if (vec) quantize_panels_kernel<true><<<grid, 64, 0, s>>>(x, out);
        else quantize_panels_kernel<false><<<grid, 64, 0, s>>>(x, out);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess || products_of_few) return e;
        relative_fp8_kernel<<<(unsigned)tiles, 256, 0, s>>>(out);
        return hipGetLastError();
    }
    const unsigned grid = (unsigned)std::min(tiles, kMaxGrid);
    if (!vec) quantize_fp8_kernel<false, false><<<grid, kQuantThreads, 0, s>>>(x, out);
    else if (out.rows * out.k * 4 >= kFp8StreamBytes) quantize_fp8_kernel<true, true><<<grid, kQuantThreads, 0, s>>>(x, out);
    else quantize_fp8_kernel<true, false><<<grid, kQuantThreads, 0, s>>>(x, out);
    return hipGetLastError();
}

hipError_t launch_dequantize_fp8(hipStream_t s, const Fp8Rows &in, float *out) {
    const size_t tiles = fp8_rows16(in.rows) / 16 * fp8_blocks(in.k);
    const unsigned grid = (unsigned)std::min((tiles + 3) / 4, kMaxGrid);
    // Past the caches (13828 x 4096 57 us, so 44; 55312 x 1100, whose rows are no whole lines, quantised
    // and read back, in other memory each time, 143 and 134).
    if (in.k % 4 == 0 && in.rows * in.k * 4 >= kFp8StreamBytes) dequantize_fp8_kernel<true, true><<<grid, 256, 0, s>>>(in, out);
    else if (in.k % 4 == 0) dequantize_fp8_kernel<true, false><<<grid, 256, 0, s>>>(in, out);
    else dequantize_fp8_kernel<false, false><<<grid, 256, 0, s>>>(in, out);
    return hipGetLastError();
}

// By a model of the launch, in us, fitted to 24 shapes measured with each form: the few rows'
// form takes a wave's blocks one after the other (1.0) or what all workgroups have to read and
// multiply, and as long again for each round of 1024 of them; tiles of 64 and 128 one tile on its
// own, or rounds of as many as are resident (1024 and 512); tiles of 256 whole rounds of 256.
Fp8Plan fp8_plan(size_t m, size_t n, size_t k, bool floats) {
    const auto tiles = [&](size_t b) { return (double)((m + b - 1) / b) * (double)((n + b - 1) / b); };
    const double kb = (double)fp8_blocks(k), groups = (double)((n + 15) / 16) * (double)((m + 63) / 64);
    const double each = m <= 16 ? 4.2e-4 : m <= 32 ? 5.6e-4 : 8.4e-4;
    // Where a launch has the workgroups; there is no output large enough for tiles of 256 not to.
    const auto fits = [&](size_t b, size_t threads) { return tiles(b) < (double)(kMaxThreads / threads); };
    const bool few = (n + 15) / 16 < kMaxThreads / (kFewWaves * 64) && (m + 15) / 16 <= kMaxGridY;
    double best = !few ? INFINITY : 2.6 + std::max(std::ceil(kb / kFewWaves), groups * kb * each) + 5 * std::max(0.0, groups / 1024 - 1);
    // Fused while a wave quantises one block (one row of 768 for 2304 outputs 4.0 us, in two launches
    // 5.8; 16 rows 5.8 and 7.3; of 3072 for 768 8.0 and 6.6).
    Fp8Plan plan = floats && m <= 16 && kb <= kFewWaves && groups <= 1024 ? Fp8Plan::Fused : Fp8Plan::Few;
    const auto offer = [&](Fp8Plan p, double us) {
        if (us < best) {
            best = us;
            plan = p;
        }
    };
    if (fits(64, 256)) offer(Fp8Plan::Tile64, std::max(4.2 + 0.57 * kb, tiles(64) / 1024 * (5 + 1.05 * kb)));
    if (fits(128, 512)) offer(Fp8Plan::Tile128, std::max(7 + 1.0 * kb, tiles(128) / 512 * (8 + 1.85 * kb)));
    offer(Fp8Plan::Tile256, std::ceil(tiles(256) / 256) * (16 + 3.0 * kb));
    static const char *asked = getenv("VESTRA_HIP_FP8_TILE");
    if (asked) {
        const int a = atoi(asked);
        if (a == 15 && floats && m <= 16) return Fp8Plan::Fused;
        if (a == 16) return Fp8Plan::Few;
        if (a == 64) return Fp8Plan::Tile64;
        if (a == 128) return Fp8Plan::Tile128;
        if (a == 256) return Fp8Plan::Tile256;
    }
    return plan;
}

hipError_t launch_gemm_fp8(hipStream_t s, const Fp8Gemm &g, Epi epi, Fp8Plan plan, const float *x) {
    return g.b_scales ? launch_blocks<true>(s, g, epi, plan, x) : launch_blocks<false>(s, g, epi, plan, x);
}

}  // namespace vh
