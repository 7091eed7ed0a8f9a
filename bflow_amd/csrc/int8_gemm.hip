// Rows of 8-bit integers against rows of 8-bit integers, with a scale for each row of either side, and the quantisation in front of it
// (gfx950 only).
//
//   out[i][j] = alpha * sa[i] * sb[j] * sum_k a[i][k] b[j][k]        sums exact in 32-bit integers (|k| < 2^17)
//   q[k] = nearest whole number to 127 x[k] / max|x| (halves to even, exactly), scale = max|x| / 127
//
// The integer matrix rate is twice the fp16 rate; at a feature dimension of 256 the correlation volume leaves the matrix cores' bound for the
// memory's.
#include "common.h"
#include "tile_nt.h"

namespace {
using namespace bflow;
using namespace bflow::nt;

enum { F32 = 0, F16 = 1, BF16 = 2 };
template <int DT> struct OutT { typedef float T; };
template <> struct OutT<F16> { typedef _Float16 T; };
template <> struct OutT<BF16> { typedef __bf16 T; };

struct GemmArgs {
    const signed char *a, *b;
    const float *sa, *sb;
    void* out;
    long long a0, a1, b0, b1, sa0, sa1, sb0, sb1, o0, o1;   // strides of the two batch dimensions (elements)
    int lda, ldb;
    long long ldo;
    int M, N, K, n1;        // n1: size of the inner batch dimension
    float alpha;
    int tiles_m, tiles_n;
};

// bytes k .. k + 15 of a fragment: those at or behind K become zero
__device__ __forceinline__ i32x4 cut(i32x4 v, int k, int K) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const int left = K - k - 4 * d;
        v[d] &= left >= 4 ? -1 : left <= 0 ? 0 : (1 << (8 * left)) - 1;
    }
    return v;
}

// BM x BN tile; wave (wm, wn) keeps WM x WN of it.
template <int BM, int BN, int WM, int WN>
struct ByteTile {
    static constexpr int ACROSS = BN / WN, WAVES = (BM / WM) * ACROSS, THREADS = 64 * WAVES, MT = WM / 32, NT = WN / 32;
    static constexpr int STAGE = (BM + BN) * CHUNK, LDS = 2 * STAGE, PIECES = (BM + BN) / 8;
    static_assert(PIECES % WAVES == 0, "whole pieces for every wave");
    i32x16 acc[MT][NT];

    __device__ __forceinline__ void issue(rsrc_t a, int lda, int va, rsrc_t b, int ldb, int vb, int chunk, char* stage, int wave) {
#pragma unroll
        for (int i = 0; i < PIECES / WAVES; ++i) {
            const int p = wave + i * WAVES;
            if (p < BM / 8) dma_piece(a, stage + p * 1024, va, p * 8 * lda + chunk * CHUNK);
            else dma_piece(b, stage + p * 1024, vb, (p - BM / 8) * 8 * ldb + chunk * CHUNK);
        }
    }
    template <bool CUT> __device__ __forceinline__ void multiply(const char* as, const char* bs, int lane, int k, int K) {
#pragma unroll
        for (int sub = 0; sub < 4; ++sub) {
            i32x4 av[MT], bv[NT];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                av[i] = frag(as + i * 32 * CHUNK, lane, sub);
                if (CUT) av[i] = cut(av[i], k + sub * 32 + (lane >> 5) * 16, K);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) bv[j] = frag(bs + j * 32 * CHUNK, lane, sub);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av[i], bv[j], acc[i][j], 0, 0, 0);
        }
    }
    __device__ __forceinline__ void run(rsrc_t a, int lda, rsrc_t b, int ldb, int K, char* lds) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wm = wave / ACROSS, wn = wave % ACROSS;
        const int va = lane_offset(lane, lda), vb = lane_offset(lane, ldb), chunks = (K + CHUNK - 1) / CHUNK;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int k = 0; k < 16; ++k) acc[i][j][k] = 0;
        issue(a, lda, va, b, ldb, vb, 0, lds, wave);
        wait_chunk();
        __builtin_amdgcn_s_barrier();
        for (int c = 0; c < chunks; ++c) {
            if (c + 1 < chunks) issue(a, lda, va, b, ldb, vb, c + 1, lds + ((c + 1) & 1) * STAGE, wave);
            const char* as = lds + (c & 1) * STAGE + wm * WM * CHUNK;
            const char* bs = lds + (c & 1) * STAGE + (BM + wn * WN) * CHUNK;
            if ((c + 1) * CHUNK <= K) multiply<false>(as, bs, lane, 0, 0);
            else multiply<true>(as, bs, lane, c * CHUNK, K);
            wait_chunk();
            __builtin_amdgcn_s_barrier();
        }
    }
};

template <class Tile, int BM, int BN, int DT>
__global__ __launch_bounds__(Tile::THREADS) void i8_gemm_kernel(GemmArgs g) {
    typedef typename OutT<DT>::T T;
    __shared__ __attribute__((aligned(1024))) char lds[Tile::LDS];
    const int z = blockIdx.y, z0 = z / g.n1, z1 = z - z0 * g.n1;
    const int tm = blockIdx.x % g.tiles_m, tn = blockIdx.x / g.tiles_m;
    const int m0 = tm * BM, n0 = tn * BN;
    const int row_bytes = (g.K + 15) & ~15;
    const signed char* a = g.a + z0 * g.a0 + z1 * g.a1 + (long long)m0 * g.lda;
    const signed char* b = g.b + z0 * g.b0 + z1 * g.b1 + (long long)n0 * g.ldb;
    Tile t;
    t.run(rows_rsrc(a, min(g.M - m0, BM), g.lda, row_bytes), g.lda, rows_rsrc(b, min(g.N - n0, BN), g.ldb, row_bytes), g.ldb, g.K, lds);
    const float *sa = g.sa + z0 * g.sa0 + z1 * g.sa1, *sb = g.sb + z0 * g.sb0 + z1 * g.sb1;
    T* out = (T*)g.out + z0 * g.o0 + z1 * g.o1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int mw = m0 + wave / Tile::ACROSS * Tile::MT * 32 + (lane >> 5) * 4, nw = n0 + wave % Tile::ACROSS * Tile::NT * 32 + (lane & 31);
#pragma unroll
    for (int i = 0; i < Tile::MT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = mw + i * 32 + q * 8 + e;
                if (row >= g.M) continue;
                const float s = sa[row] * g.alpha;
#pragma unroll
                for (int j = 0; j < Tile::NT; ++j) {
                    const int col = nw + j * 32;
                    if (col < g.N) out[(long long)row * g.ldo + col] = (T)((float)t.acc[i][j][q * 4 + e] * s * sb[col]);
                }
            }
}

typedef ByteTile<64, 64, 32, 32> Small;

// ---------------------------------------------------------------------------------------------------------------------- quantisation
// |x| as an integer that orders like it, NaN above all
__device__ __forceinline__ unsigned magnitude(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }

struct Quant {
    float most, inv;
    __device__ __forceinline__ explicit Quant(unsigned bits) : most(__builtin_bit_cast(float, bits)), inv(127.f / most) {}
    __device__ __forceinline__ float scale() const { return most / 127.f; }
    // rows without a finite maximum, and empty ones, hold zeros: their scale (infinite, NaN, 0) says the rest
    __device__ __forceinline__ bool none() const { return !(most > 0.f && most < __builtin_inff()); }
    // x * inv is off by less than 127 * 2^-22 = 3.1e-5; nearer to a half than that, 64 bits decide (a quotient of 24-bit numbers is never
    // nearer to a half than 2^-25 of itself without being one).  A maximum so small that inv overflows ends there too: the test fails on NaN.
    __device__ __forceinline__ int operator()(float x) const {
        const float t = x * inv, r = __builtin_rintf(t);
        if (fabsf(fabsf(t - r) - 0.5f) > 4e-5f) return (int)r;
        return (int)__builtin_rint((double)x * 127.0 / (double)most);
    }
};

template <int DT> __device__ __forceinline__ float load1(const void* p, long long i) {
    if constexpr (DT == F32) return ((const float*)p)[i];
    else if constexpr (DT == F16) return (float)((const _Float16*)p)[i];
    else return __builtin_bit_cast(float, (unsigned)((const unsigned short*)p)[i] << 16);
}
__device__ __forceinline__ unsigned wave_most(unsigned v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
    return v;
}

// One wave for a row: x (rows, K), ld elements apart -> q (rows, ldq), zeros behind K.
template <int DT>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const void* x, long long ld, long long rows, int K, signed char* q, int ldq, float* scale) {
    const int lane = threadIdx.x & 63;
    for (long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (long long)gridDim.x * 4) {
        unsigned most = 0;
        for (int k = lane; k < K; k += 64) most = max(most, magnitude(load1<DT>(x, row * ld + k)));
        const Quant f(wave_most(most));
        const bool none = f.none();
        if (lane == 0) scale[row] = f.scale();
        for (int k = lane * 4; k < ldq; k += 256) {
            unsigned w = 0;
            for (int e = 0; e < 4; ++e)
                if (k + e < K && !none) w |= (unsigned)(f(load1<DT>(x, row * ld + k + e)) & 255) << (8 * e);
            *reinterpret_cast<unsigned*>(q + row * ldq + k) = w;
        }
    }
}

// 64 pixels of a workgroup, all D channels.  Row r of q is pixel r, or in the 4 x 8 tile order of the look-up (tiled); rows without a pixel
// are zero with scale 0.  PACKED: x is the fp16-pair operand (hi, lo planes of 32 channels by `np` pixels), else (B, D, h, w) in 32 bits.
template <bool PACKED>
__global__ __launch_bounds__(256) void quantize_pixels_kernel(const float* x, const _Float16* hi, const _Float16* lo, int D, int h, int w, int np, int rows, int tiled,
                                                              signed char* q, float* scale) {
    __shared__ unsigned most[4][64];
    const int b = blockIdx.y, p = threadIdx.x & 63, c = threadIdx.x >> 6, r = blockIdx.x * 64 + p;
    int pix = -1;
    if (r < rows) {
        if (tiled) {
            const int across = (w + 7) / 8, tile = r >> 5, y = tile / across * 4 + ((r & 31) >> 3), xx = tile % across * 8 + (r & 7);
            if (y < h && xx < w) pix = y * w + xx;
        } else pix = r;
    }
    auto value = [&](int d) {
        if constexpr (PACKED) {
            const long long i = (((long long)b * (D / 32) + d / 32) * np + pix) * 32 + d % 32;
            return fmaf((float)lo[i], SPLIT_LO_INV, (float)hi[i]);
        } else return x[((long long)b * D + d) * h * w + pix];
    };
    const int per = (D / 4 + 3) / 4 * 4, first = c * per, last = min(D, first + per);     // this thread's channels, in fours
    unsigned m = 0;
    if (pix >= 0)
        for (int d = first; d < last; ++d) m = max(m, magnitude(value(d)));
    most[c][p] = m;
    __syncthreads();
    const Quant f(max(max(most[0][p], most[1][p]), max(most[2][p], most[3][p])));
    const bool none = f.none();
    if (r >= rows) return;
    if (c == 0) scale[(long long)b * rows + r] = f.scale();
    for (int d = first; d < last; d += 4) {
        unsigned v = 0;
        if (!none)
            for (int e = 0; e < 4; ++e) v |= (unsigned)(f(value(d + e)) & 255) << (8 * e);
        *reinterpret_cast<unsigned*>(q + ((long long)b * rows + r) * D + d) = v;
    }
}
}  // namespace

extern "C" int bflow_i8_gemm(const bflow_i8_gemm_t* d, bflow_stream_t stream) {
    BFLOW_REQUIRE(d, BFLOW_E_ARG, "i8_gemm: null descriptor");
    BFLOW_REQUIRE(d->a && d->b && d->scale_a && d->scale_b && d->out, BFLOW_E_ARG, "i8_gemm: null pointer");
    BFLOW_REQUIRE(d->M >= 1 && d->N >= 1 && d->K >= 1 && d->batch0 >= 1 && d->batch1 >= 1, BFLOW_E_ARG, "i8_gemm: sizes %d x %d x %d, batch %d x %d", d->M, d->N, d->K,
                  d->batch0, d->batch1);
    BFLOW_REQUIRE(d->K <= BFLOW_I8_MAX_K, BFLOW_E_LIMIT, "i8_gemm: K = %d > %d (32-bit sums)", d->K, BFLOW_I8_MAX_K);
    BFLOW_REQUIRE(d->dtype >= F32 && d->dtype <= BF16, BFLOW_E_ARG, "i8_gemm: dtype %d", d->dtype);
    const int row = (d->K + 15) & ~15;
    BFLOW_REQUIRE(d->lda >= row && d->ldb >= row && d->lda <= BFLOW_I8_MAX_LD && d->ldb <= BFLOW_I8_MAX_LD && d->ldo >= d->N, BFLOW_E_ARG,
                  "i8_gemm: leading dimensions %d, %d, %lld for K = %d, N = %d", d->lda, d->ldb, d->ldo, d->K, d->N);
    BFLOW_REQUIRE(((uintptr_t)d->a | (uintptr_t)d->b | (unsigned)d->lda | (unsigned)d->ldb | (unsigned long long)d->a_stride0 | (unsigned long long)d->a_stride1 |
                   (unsigned long long)d->b_stride0 | (unsigned long long)d->b_stride1) % 16 == 0, BFLOW_E_ARG, "i8_gemm: operands and their strides are multiples of 16 bytes");
    const long long batch = (long long)d->batch0 * d->batch1;
    BFLOW_REQUIRE(batch <= 65535, BFLOW_E_LIMIT, "i8_gemm: %lld matrices > 65535", batch);
    GemmArgs g = {(const signed char*)d->a, (const signed char*)d->b, d->scale_a, d->scale_b, d->out, d->a_stride0, d->a_stride1, d->b_stride0, d->b_stride1,
                  d->sa_stride0, d->sa_stride1, d->sb_stride0, d->sb_stride1, d->out_stride0, d->out_stride1, d->lda, d->ldb, d->ldo, d->M, d->N, d->K, d->batch1, d->alpha,
                  ceil_div(d->M, 64), ceil_div(d->N, 64)};
    BFLOW_REQUIRE((long long)g.tiles_m * g.tiles_n < (1LL << 31), BFLOW_E_LIMIT, "i8_gemm: too many tiles");
    const auto kernel = d->dtype == F32 ? i8_gemm_kernel<Small, 64, 64, F32> : d->dtype == F16 ? i8_gemm_kernel<Small, 64, 64, F16> : i8_gemm_kernel<Small, 64, 64, BF16>;
    hipLaunchKernelGGL(kernel, dim3(g.tiles_m * g.tiles_n, (unsigned)batch), dim3(256), 0, (hipStream_t)stream, g);
    return launch_status("i8_gemm");
}

extern "C" int bflow_i8_quantize_rows(const void* x, int dtype, long long ld, long long rows, int K, signed char* q, int ldq, float* scale, bflow_stream_t stream) {
    BFLOW_REQUIRE(x && q && scale, BFLOW_E_ARG, "i8_quantize_rows: null pointer");
    BFLOW_REQUIRE(rows >= 1 && K >= 1 && ld >= 0 && ldq >= K && ldq % 16 == 0 && (uintptr_t)q % 16 == 0, BFLOW_E_ARG, "i8_quantize_rows: %lld rows of %d, strides %lld, %d", rows, K, ld,
                  ldq);
    BFLOW_REQUIRE(dtype >= F32 && dtype <= BF16, BFLOW_E_ARG, "i8_quantize_rows: dtype %d", dtype);
    const auto kernel = dtype == F32 ? quantize_rows_kernel<F32> : dtype == F16 ? quantize_rows_kernel<F16> : quantize_rows_kernel<BF16>;
    const long long wgs = (rows + 3) / 4;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(wgs < 65536 ? wgs : 65536)), dim3(256), 0, (hipStream_t)stream, x, ld, rows, K, q, ldq, scale);
    return launch_status("i8_quantize_rows");
}

extern "C" int bflow_i8_quantize_pixels(const float* x, const void* x_hi, const void* x_lo, int np, int B, int D, int h, int w, int tiled, signed char* q, float* scale,
                                        bflow_stream_t stream) {
    BFLOW_REQUIRE(q && scale && (x || (x_hi && x_lo)) && !(x && x_hi), BFLOW_E_ARG, "i8_quantize_pixels: null pointer, or both forms of x");
    BFLOW_REQUIRE(B >= 1 && B <= 65535 && D >= 16 && D % 16 == 0 && h >= 1 && w >= 1 && (long long)h * w < (1LL << 28), BFLOW_E_ARG,
                  "i8_quantize_pixels: B = %d, D = %d (a multiple of 16), %d x %d pixels", B, D, h, w);
    BFLOW_REQUIRE(x || (D % 32 == 0 && np >= h * w), BFLOW_E_ARG, "i8_quantize_pixels: packed operand of %d rows for %d pixels, D = %d (a multiple of 32)", np, h * w, D);
    BFLOW_REQUIRE((uintptr_t)q % 16 == 0, BFLOW_E_ARG, "i8_quantize_pixels: q is not aligned to 16 bytes");
    const int rows = tiled ? (h + 3) / 4 * ((w + 7) / 8) * 32 : h * w;
    const dim3 grid((rows + 63) / 64, B);
    if (x) hipLaunchKernelGGL(quantize_pixels_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, x, nullptr, nullptr, D, h, w, 0, rows, tiled, q, scale);
    else hipLaunchKernelGGL(quantize_pixels_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, nullptr, (const _Float16*)x_hi, (const _Float16*)x_lo, D, h, w, np, rows, tiled, q, scale);
    return launch_status("i8_quantize_pixels");
}
