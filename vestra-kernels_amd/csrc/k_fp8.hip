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
// join behind it.  A value is then off by at most 2^-25 of 2^E, E the row's largest
// exponent (448 * 2^E the largest value it can hold): nothing while a row's
// exponents are within 15 of each other, and 2^-33 of the largest value at the worst.
//
// Storage, "panels": 16 rows x 128 values are 2048 bytes, [half 2][lane 64][16]: lane
// (row li, lh) of half h holds values 32 lh + 16 h .. + 15 of its row, so that a
// fragment is one 16-byte read of consecutive lanes everywhere: memory to LDS, LDS to
// registers, or memory to registers.  (Any order of k does for a product, as long as
// both sides have it.)
#include <algorithm>

#include "common.h"
#include "kernels.h"
#include "split_gemm.h"

namespace vh {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kQuantThreads = 512;
constexpr size_t kMaxGrid = 65536;  // of the kernels that walk their tiles

// The exponent of a block whose largest finite magnitude has these bits: 448 = 1.75 * 2^8.
__device__ __forceinline__ int block_exponent(uint32_t amax) {
    const int e = (int)(amax >> 23) - 135 + ((amax & 0x7fffff) > 0x600000 ? 1 : 0);
    return max(e, -127);
}
__device__ __forceinline__ float pow2(int e) {  // -126 <= e <= 127
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Where dword c (values 4 c .. + 3) of row r is in a panel.
__device__ __forceinline__ int panel_at(int r, int c) { return ((c >> 2) & 1) * 1024 + ((c >> 3) * 16 + r) * 16 + (c & 3) * 4; }

// Largest finite magnitude's bits.
__device__ __forceinline__ uint32_t finite_max(uint32_t mx, float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    return max(mx, b < 0x7f800000u ? b : 0u);
}
__device__ __forceinline__ int e4m3_of(f32x4 v, float inv) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = fabsf(v[i]) < INFINITY ? v[i] * inv : NAN;
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
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

// A workgroup takes 16 rows, its waves their blocks in turn; 32 lanes a row's block.
// Rows past the end become zeros.
template <bool VEC>
__global__ __launch_bounds__(kQuantThreads) void quantize_fp8_kernel(const float *x, Fp8Rows out) {
    __shared__ __attribute__((aligned(16))) char stage[kQuantThreads / 64][2048];
    __shared__ int row_max[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 31, side = lane >> 5;
    const size_t kb = fp8_blocks(out.k), rows16 = fp8_rows16(out.rows);
    for (size_t tile = blockIdx.x; tile < rows16 / 16; tile += gridDim.x) {
        if (threadIdx.x < 16) row_max[threadIdx.x] = -127;
        __syncthreads();
        for (size_t b = wave; b < kb; b += kQuantThreads / 64) {
            f32x4 v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const size_t row = tile * 16 + 2 * i + side;
                v[i] = row < out.rows ? row4<VEC>(x + row * out.k, b * 128 + 4 * c, out.k)
                                      : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            char *to = stage[wave];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                uint32_t mx = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) mx = finite_max(mx, v[i][j]);
                mx = dpp_umax<0x140>(dpp_umax<0x141>(dpp_umax<0x4e>(dpp_umax<0xb1>(mx))));
                mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16, kWave));
                const int e = block_exponent(mx), r = 2 * i + side;
                *reinterpret_cast<int *>(to + panel_at(r, c)) = e4m3_of(v[i], pow2(-e));
                if (c == 0) {
                    out.exps[b * rows16 + tile * 16 + r] = (uint8_t)(e + 127);
                    atomicMax(&row_max[r], e);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            char *at = reinterpret_cast<char *>(out.codes) + (tile * kb + b) * 2048 + lane * 16;
#pragma unroll
            for (int h = 0; h < 2; h++)
                *reinterpret_cast<u32x4 *>(at + h * 1024) = *reinterpret_cast<const u32x4 *>(to + h * 1024 + lane * 16);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        __syncthreads();
        if (threadIdx.x < 16) out.row_e[tile * 16 + threadIdx.x] = row_max[threadIdx.x];
        for (size_t i = threadIdx.x; i < kb * 16; i += kQuantThreads) {
            const size_t at = (i >> 4) * rows16 + tile * 16 + (i & 15);
            out.rel[at] = fp8_relative(out.exps[at], row_max[i & 15]);
        }
        __syncthreads();
    }
}

// The values that the codes stand for.
template <bool VEC>
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
            *reinterpret_cast<u32x4 *>(to + h * 1024 + lane * 16) = *reinterpret_cast<const u32x4 *>(at + h * 1024);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
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
            if constexpr (VEC) {
                *reinterpret_cast<f32x4 *>(y) = v;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (d + j < in.k) y[j] = v[j];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
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

// C = A . B^T, a workgroup of WM x WN waves a tile of BM x BN.  Two stages of 128 k in
// LDS; D^T = B . A^T, so that a lane holds four consecutive columns of its row.
// BLOCKS: B has float scales for 128 x 128 values (b_scales) instead of its exponents.
template <int BM, int BN, int WM, int WN, Epi EPI, bool BLOCKS>
__global__ __launch_bounds__(WM *WN * 64, 2) void fp8_gemm_kernel(Fp8Gemm g) {
    constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
    constexpr int CODES = (BM + BN) * 128, STAGE = CODES + (BM + BN) * 2;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lh = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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
    auto copy = [&](size_t b, int buf) {
#pragma unroll
        for (int u = wave; u < (BM + BN) / 8; u += NW) {
            const bool is_a = u < BM / 8;
            const size_t t = is_a ? min((size_t)mt * (BM / 16) + u / 2, a16 / 16 - 1)
                                  : min((size_t)nt * (BN / 16) + (u - BM / 8) / 2, b16 / 16 - 1);
            const char *from = reinterpret_cast<const char *>(is_a ? g.a.codes : g.b.codes) + (t * kb + b) * 2048 + (u & 1) * 1024;
            copy16_to_lds(from, lane * 16, __builtin_amdgcn_readfirstlane(lds0 + buf * STAGE + u * 1024));
        }
        for (int u = wave; u < (BM + BN + 511) / 512; u += NW) {
            // Eight rows a lane (past the end: the last eight).
            const int r = u * 512 + lane * 8;
            if (r < BM + BN) {
                const bool is_a = r < BM;
                const size_t row = is_a ? min((size_t)mt * BM + r, a16 - 8) : min((size_t)nt * BN + r - BM, b16 - 8);
                const uint16_t *from = is_a ? g.a.rel + b * a16 + row : g.b.rel + b * b16 + row;
                *reinterpret_cast<u32x4 *>(smem + buf * STAGE + CODES + r * 2) = *reinterpret_cast<const u32x4 *>(from);
            }
        }
    };
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    copy(0, 0);
    for (size_t b = 0; b < kb; b++) {
        const int buf = b & 1;
        split_wait<0>();
        __syncthreads();
        if (b + 1 < kb) copy(b + 1, buf ^ 1);
        const char *as = smem + buf * STAGE + wm * TM * 2048 + lane * 16;
        const char *bs = smem + buf * STAGE + BM * 128 + wn * TN * 2048 + lane * 16;
        const uint16_t *rs = reinterpret_cast<const uint16_t *>(smem + buf * STAGE + CODES);
        float ra[TM], rb[TN];
#pragma unroll
        for (int i = 0; i < TM; i++) ra[i] = __uint_as_float((uint32_t)rs[(wm * TM + i) * 16 + li] << 16);
#pragma unroll
        for (int j = 0; j < TN; j++)
            rb[j] = BLOCKS ? 1.0f : __uint_as_float((uint32_t)rs[BM + (wn * TN + j) * 16 + li] << 16);
        f32x4 part[TM][TN];
        if constexpr (BLOCKS) {
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++) part[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        auto &sum = [&]() -> f32x4(&)[TM][TN] {
            if constexpr (BLOCKS) return part;
            else return acc;
        }();
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
                    for (int j = 0; j < TN; j++) sum[i][j] = mfma16x16x32_f16(fb[j], fa, sum[i][j]);
                }
            }
        }
        if constexpr (BLOCKS) {
            const size_t n_block = min(((size_t)nt * BN + wn * TN * 16) / 128, (b16 - 1) / 128);
            const float s = g.b_scales[n_block * kb + b];
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[i][j][r] = __builtin_fmaf(part[i][j][r], s, acc[i][j][r]);
        }
    }
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const size_t m = (size_t)mt * BM + (wm * TM + i) * 16 + li;
        const int ea = g.a.row_e[min(m, a16 - 1)];
#pragma unroll
        for (int j = 0; j < TN; j++) {
            const size_t n = (size_t)nt * BN + (wn * TN + j) * 16 + 4 * lh;
            f32x4 v = acc[i][j];
#pragma unroll
            for (int r = 0; r < 4; r++)
                v[r] = ldexpf(v[r], ea + (BLOCKS ? 0 : g.b.row_e[min(n + r, b16 - 1)]));
            put4<EPI>(g, m, n, v);
        }
    }
}

template <int BM, int BN, int WM, int WN, Epi EPI, bool BLOCKS>
hipError_t launch_tile(hipStream_t s, Fp8Gemm g) {
    constexpr size_t bytes = 2 * ((BM + BN) * 128 + (BM + BN) * 2);
    static std::atomic<uint64_t> done{0};
    hipError_t e = ensure_dynamic_lds(fp8_gemm_kernel<BM, BN, WM, WN, EPI, BLOCKS>, bytes, done);
    if (e != hipSuccess) return e;
    const size_t mt = (g.m + BM - 1) / BM, nt = (g.n + BN - 1) / BN;
    if (mt * nt > (size_t)1 << 22) return hipErrorInvalidConfiguration;
    g.m_tiles = (int)mt;
    g.n_tiles = (int)nt;
    g.tiles = (int)(mt * nt);
    fp8_gemm_kernel<BM, BN, WM, WN, EPI, BLOCKS><<<(g.tiles + 7) / 8 * 8, WM * WN * 64, bytes, s>>>(g);
    return hipGetLastError();
}

template <Epi EPI, bool BLOCKS>
hipError_t launch_epi(hipStream_t s, const Fp8Gemm &g) {
    return launch_tile<128, 128, 2, 2, EPI, BLOCKS>(s, g);
}

}  // namespace

hipError_t launch_quantize_fp8(hipStream_t s, const float *x, const Fp8Rows &out) {
    const unsigned grid = (unsigned)std::min(fp8_rows16(out.rows) / 16, kMaxGrid);
    if (out.k % 4 == 0) quantize_fp8_kernel<true><<<grid, kQuantThreads, 0, s>>>(x, out);
    else quantize_fp8_kernel<false><<<grid, kQuantThreads, 0, s>>>(x, out);
    return hipGetLastError();
}

hipError_t launch_dequantize_fp8(hipStream_t s, const Fp8Rows &in, float *out) {
    const size_t tiles = fp8_rows16(in.rows) / 16 * fp8_blocks(in.k);
    const unsigned grid = (unsigned)std::min((tiles + 3) / 4, kMaxGrid);
    if (in.k % 4 == 0) dequantize_fp8_kernel<true><<<grid, 256, 0, s>>>(in, out);
    else dequantize_fp8_kernel<false><<<grid, 256, 0, s>>>(in, out);
    return hipGetLastError();
}

hipError_t launch_gemm_fp8(hipStream_t s, const Fp8Gemm &g, Epi epi) {
    if (g.b_scales) {
        if (epi == Epi::Gelu) return launch_epi<Epi::Gelu, true>(s, g);
        if (epi == Epi::Residual) return launch_epi<Epi::Residual, true>(s, g);
        return launch_epi<Epi::Store, true>(s, g);
    }
    if (epi == Epi::Gelu) return launch_epi<Epi::Gelu, false>(s, g);
    if (epi == Epi::Residual) return launch_epi<Epi::Residual, false>(s, g);
    return launch_epi<Epi::Store, false>(s, g);
}

}  // namespace vh
