// Orthogonalisation of a list of matrices by quintic Newton-Schulz steps, and the Muon step around it (gfx950 only).
//
//   X0 = X / (|X|_F + eps);   steps times:   A = X X^T,   B = b A + c A^2,   X <- a X + B X          (X r x s, r <= s; tall matrices transposed)
//
// A list is worked off TOGETHER: every launch below covers one phase of all its matrices (up to 64; the table travels in the kernel
// arguments), because the filters of a network are many and small and a step is a chain of 3 products.
//
// Number format: X, A and B are carried as fp16 pairs (value = hi + lo * 2^-11, common.h) and multiplied in three matrix passes
// (hi*hi, hi*lo, lo*hi) with 32-bit sums: the accuracy of 32-bit arithmetic at a third of the fp16 rate, 3 times the rate of the 32-bit
// matrix instructions.  All sums of squares are taken in 64 bits.  Powers of two keep the pairs in the range where hi is a normal number:
// X is stored times sx ~ sqrt(r s) (entries of root mean square 1 at the start), A times 2^12, B times 2^10.  The host refuses coefficients
// whose iterates leave [0, 2], so |X| <= 2, |A| <= 4, |B| < 64 and nothing saturates.  Where |X|_F is below eps, X0 is small as a whole and
// would sink under the pairs' smallest numbers: X carries a further 2^g (A and B 2^2g), g = floor(log2((|X| + eps) / |X|)) at the start and
// less by the steps' largest gain from step to step, so that 2^g |X| <= 1 holds (g is 0 for any gradient that is not vanishing).  a X is added from X itself and not folded into B:
// with it in B, the rounding of B's diagonal costs twice the error on matrices with weak directions.
//
// Layouts (workspace): an operand row is a row of 128-byte chunks of 32 columns, [32 hi | 32 lo] (tile_nt.h), rows and columns padded to 64
// with zeros.  X is held twice, by rows (X, for the Gram product) and by columns (Xt, the right operand of B X): both products then read
// both operands along the contraction.
#include <cmath>
#include "common.h"
#include "tile_nt.h"

namespace {
using namespace bflow;
using namespace bflow::nt;

constexpr int MOST = BFLOW_NS_MAX_MATRICES;
constexpr float SA = 4096.f, SB = 1024.f;
constexpr int NORM_MIN = 16384, NORM_PARTS = 1024;   // elements of one partial sum of squares at least; partials of a matrix at most

struct Work {          // one matrix inside the products
    long long off;     // bytes from the workspace
    int r, s;          // rows <= columns
    int tile0;         // first workgroup of this launch
    int split;         // Gram: k chunks of one workgroup
};
struct Entry {         // one matrix where it enters
    const void* src;   // the matrix, or the gradient (step)
    float* momentum;   // step only
    long long ld, off;
    int r, s;
    int tile0, per;    // first workgroup; elements of one partial (norm)
    int tall;
};
struct Exit {          // one matrix where it leaves
    void* dst;         // the result, or the weights (step)
    long long ld, off;
    int r, s;
    int tile0, tall;
    float size;        // step: 0.2 sqrt(max(m, n))
};
struct Works { Work m[MOST]; int count; };
struct Entries { Entry m[MOST]; int count; };
struct Exits { Exit m[MOST]; int count; };
static_assert(sizeof(Entries) <= 4096 && sizeof(Exits) <= 4096 && sizeof(Works) <= 4096, "the tables are kernel arguments");

__host__ __device__ inline int up64(int x) { return (x + 63) & ~63; }
__host__ __device__ inline long long mat_bytes(int r, int s) { return 4LL * up64(r) * up64(s); }
// regions of a matrix, from its `off`: norm partials, g of the start, X, Xt (two, alternating), A, B
__host__ __device__ inline long long g_at(long long off) { return off + NORM_PARTS * 8; }
__host__ __device__ inline long long x_at(long long off) { return g_at(off) + 256; }
__host__ __device__ inline long long xt_at(long long off, int r, int s, int which) { return x_at(off) + (1 + which) * mat_bytes(r, s); }
__host__ __device__ inline long long a_at(long long off, int r, int s) { return x_at(off) + 3 * mat_bytes(r, s); }
__host__ __device__ inline long long b_at(long long off, int r, int s) { return a_at(off, r, s) + mat_bytes(r, r); }
__host__ inline long long end_at(long long off, int r, int s) { return b_at(off, r, s) + mat_bytes(r, r); }

// sx: the power of two next to sqrt(r s), at most 2^14 (|X| <= 2 then stays below the largest fp16)
__host__ __device__ inline int x_exponent(int r, int s) {
    const double e = 0.5 * log2((double)r * (double)s);
    const int k = (int)(e + 0.5);
    return k > 14 ? 14 : k;
}

template <class T>
__device__ __forceinline__ int find(const T* m, int count, int wg) {
    int at = 0;
    for (int step = MOST / 2; step > 0; step >>= 1)
        if (at + step < count && m[at + step].tile0 <= wg) at += step;
    return at;
}

enum { F32 = 0, F16 = 1, BF16 = 2 };
template <int DT> __device__ __forceinline__ float load1(const void* p, long long i) {
    if constexpr (DT == F32) return ((const float*)p)[i];
    else if constexpr (DT == F16) return (float)((const _Float16*)p)[i];
    else return __builtin_bit_cast(float, (unsigned)((const unsigned short*)p)[i] << 16);
}
template <int DT> __device__ __forceinline__ void store1(void* p, long long i, float v) {
    if constexpr (DT == F32) ((float*)p)[i] = v;
    else if constexpr (DT == F16) ((_Float16*)p)[i] = (_Float16)v;
    else ((__bf16*)p)[i] = (__bf16)v;      // round to nearest even
}

// position of (row, col) in an operand of `cols` padded columns, in halves; the lo half is 32 further
__device__ __forceinline__ long long at(int row, int col, int cols) { return (long long)row * (2 * cols) + (col >> 5) * 64 + (col & 31); }
__device__ __forceinline__ float pair_value(_Float16 h, _Float16 l) { return fmaf((float)l, SPLIT_LO_INV, (float)h); }
__device__ __forceinline__ void put1(_Float16* m, long long i, float v) {
    _Float16 h, l;
    split1(v, h, l);
    m[i] = h;
    m[i + 32] = l;
}
__device__ __forceinline__ void put4(_Float16* m, long long i, const float v[4]) {
    half4 h, l;
#pragma unroll
    for (int k = 0; k < 4; ++k) { _Float16 a, b; split1(v[k], a, b); h[k] = a; l[k] = b; }
    *reinterpret_cast<half4*>(m + i) = h;
    *reinterpret_cast<half4*>(m + i + 32) = l;
}
__device__ __forceinline__ void get4(const _Float16* m, long long i, float v[4]) {
    const half4 h = *reinterpret_cast<const half4*>(m + i), l = *reinterpret_cast<const half4*>(m + i + 32);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = pair_value(h[k], l[k]);
}

// ------------------------------------------------------------------------------------------------------------------------------ entry
// Element e of the source in its own order (row-major over the m x n of the user).
template <int DT, bool STEP>
__device__ __forceinline__ float entering(const Entry& m, int i, int j, float mu, bool nesterov, bool update) {
    const float g = load1<DT>(m.src, (long long)i * m.ld + j);
    if constexpr (!STEP) return g;
    const long long e = (long long)i * (m.tall ? m.r : m.s) + j;          // momentum is dense
    float v = m.momentum[e];
    if (update) { v = fmaf(mu, v, g); m.momentum[e] = v; }
    return nesterov ? fmaf(mu, v, g) : v;
}

// Sum of squares of one stretch of a matrix, in 64 bits; the step's momentum is brought up to date on the way.
template <int DT, bool STEP>
__global__ __launch_bounds__(256) void ns_norm_kernel(Entries t, char* ws, float mu, int nesterov) {
    __shared__ double part[4];
    const int k = find(t.m, t.count, blockIdx.x);
    const Entry m = t.m[k];
    const int cols = m.tall ? m.r : m.s;
    const long long n = (long long)m.r * m.s, first = (long long)(blockIdx.x - m.tile0) * m.per;
    const long long last = first + m.per < n ? first + m.per : n;
    double sum = 0;
    for (long long e = first + threadIdx.x; e < last; e += 256) {
        const int i = (int)(e / cols), j = (int)(e - (long long)i * cols);
        const float u = entering<DT, STEP>(m, i, j, mu, nesterov, true);
        sum += (double)u * (double)u;
    }
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) ((double*)(ws + m.off))[blockIdx.x - m.tile0] = part[0] + part[1] + part[2] + part[3];
}

// X and Xt of a 64 x 64 tile, scaled to sx / (|X| + eps), zeros in the padding.
template <int DT, bool STEP>
__global__ __launch_bounds__(256) void ns_pack_kernel(Entries t, char* ws, float mu, int nesterov, float eps) {
    __shared__ double part[4];
    __shared__ float tile[64][65];
    const int k = find(t.m, t.count, blockIdx.x);
    const Entry m = t.m[k];
    const int R = up64(m.r), S = up64(m.s), across = S / 64;
    const int w = blockIdx.x - m.tile0, r0 = (w / across) * 64, s0 = (w - (w / across) * across) * 64;
    const long long n = (long long)m.r * m.s;
    const int parts = (int)((n + m.per - 1) / m.per);
    double sum = 0;
    for (int i = threadIdx.x; i < parts; i += 256) sum += ((const double*)(ws + m.off))[i];
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = part[0] + part[1] + part[2] + part[3];
    const double norm = sqrt(sum);
    // (NaN and infinite norms: the comparison is false, g = 0)
    const int g = norm > 0. && norm < (double)eps ? (int)log2((norm + (double)eps) / norm) : 0;
    if (w == 0 && threadIdx.x == 0) *(int*)(ws + g_at(m.off)) = g;
    const double scale = ldexp(1.0, x_exponent(m.r, m.s) + g) / (norm + (double)eps);
    const int fast = threadIdx.x & 63, slow = threadIdx.x >> 6;
    const int i0 = m.tall ? s0 : r0, j0 = m.tall ? r0 : s0;               // of the user's matrix
    const int rows = m.tall ? m.s : m.r, cols = m.tall ? m.r : m.s;
    for (int i = slow; i < 64; i += 4) {
        float v = 0.f;
        if (i0 + i < rows && j0 + fast < cols) v = (float)((double)entering<DT, STEP>(m, i0 + i, j0 + fast, mu, nesterov, false) * scale);
        tile[i][fast] = v;
    }
    __syncthreads();
    _Float16* x = (_Float16*)(ws + x_at(m.off));
    _Float16* xt = (_Float16*)(ws + xt_at(m.off, m.r, m.s, 0));
    for (int i = slow; i < 64; i += 4) {
        const float across_v = tile[i][fast], down_v = tile[fast][i];     // (i, fast) and (fast, i) of the user's tile
        put1(x, at(r0 + i, s0 + fast, S), m.tall ? down_v : across_v);
        put1(xt, at(s0 + i, r0 + fast, R), m.tall ? across_v : down_v);
    }
}

// g of a step: what the start had, less `drop` for the growth since
__device__ __forceinline__ int g_of(const char* ws, long long off, int drop) { return max(*(const int*)(ws + g_at(off)) - drop, 0); }

// --------------------------------------------------------------------------------------------------------------------------- products
// BM x BN tile of A B^T on pairs; wave (wm, wn) keeps WM x WN of it.
template <int BM, int BN, int WM, int WN>
struct PairTile {
    static constexpr int ACROSS = BN / WN, WAVES = (BM / WM) * ACROSS, THREADS = 64 * WAVES, MT = WM / 32, NT = WN / 32;
    static constexpr int STAGE = (BM + BN) * CHUNK, LDS = 2 * STAGE, PIECES = (BM + BN) / 8;
    static_assert(PIECES % WAVES == 0, "whole pieces for every wave");
    f32x16 hh[MT][NT], xx[MT][NT];

    __device__ __forceinline__ void issue(rsrc_t a, int lda, int va, rsrc_t b, int ldb, int vb, int chunk, char* stage, int wave) {
#pragma unroll
        for (int i = 0; i < PIECES / WAVES; ++i) {
            const int p = wave + i * WAVES;
            if (p < BM / 8) dma_piece(a, stage + p * 1024, va, p * 8 * lda + chunk * CHUNK);
            else dma_piece(b, stage + p * 1024, vb, (p - BM / 8) * 8 * ldb + chunk * CHUNK);
        }
    }

    __device__ __forceinline__ void run(rsrc_t a, int lda, rsrc_t b, int ldb, int chunk0, int chunks, char* lds) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wm = wave / ACROSS, wn = wave % ACROSS;
        const int va = lane_offset(lane, lda), vb = lane_offset(lane, ldb);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int k = 0; k < 16; ++k) { hh[i][j][k] = 0.f; xx[i][j][k] = 0.f; }
        issue(a, lda, va, b, ldb, vb, chunk0, lds, wave);
        wait_chunk();
        __builtin_amdgcn_s_barrier();
        for (int c = 0; c < chunks; ++c) {
            if (c + 1 < chunks) issue(a, lda, va, b, ldb, vb, chunk0 + c + 1, lds + ((c + 1) & 1) * STAGE, wave);
            const char* as = lds + (c & 1) * STAGE + wm * WM * CHUNK;
            const char* bs = lds + (c & 1) * STAGE + (BM + wn * WN) * CHUNK;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                half8 ah[MT], al[MT], bh[NT], bl[NT];
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    ah[i] = __builtin_bit_cast(half8, frag(as + i * 32 * CHUNK, lane, sub));
                    al[i] = __builtin_bit_cast(half8, frag(as + i * 32 * CHUNK, lane, 2 + sub));
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    bh[j] = __builtin_bit_cast(half8, frag(bs + j * 32 * CHUNK, lane, sub));
                    bl[j] = __builtin_bit_cast(half8, frag(bs + j * 32 * CHUNK, lane, 2 + sub));
                }
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        hh[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bh[j], hh[i][j], 0, 0, 0);
                        xx[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bl[j], xx[i][j], 0, 0, 0);
                        xx[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[i], bh[j], xx[i][j], 0, 0, 0);
                    }
            }
            wait_chunk();
            __builtin_amdgcn_s_barrier();
        }
    }

    // f(row, col, v[4]): 4 consecutive rows of column `col` of the tile; the 32 lanes of a half wave hold 32 neighbouring columns
    template <class F> __device__ __forceinline__ void each4(F f) const {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wm = wave / ACROSS, wn = wave % ACROSS;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = fmaf(xx[i][j][q * 4 + k], SPLIT_LO_INV, hh[i][j][q * 4 + k]);
                    f(wm * WM + i * 32 + q * 8 + (lane >> 5) * 4, wn * WN + j * 32 + (lane & 31), v);
                }
    }
};

typedef PairTile<64, 64, 32, 32> Small;

// tile t of the lower triangle (diagonal included), row by row
__device__ __forceinline__ void lower(int t, int& i, int& j) {
    i = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    j = t - i * (i + 1) / 2;
}

// One stretch of the contraction of one 64 x 64 tile of X X^T, lower triangle; partials in the order of the registers.
__global__ __launch_bounds__(256) void ns_gram_kernel(Works t, const char* ws, float* parts) {
    __shared__ __attribute__((aligned(1024))) char lds[Small::LDS];
    const int k = find(t.m, t.count, blockIdx.x);
    const Work m = t.m[k];
    const int R = up64(m.r), S = up64(m.s), chunks = S / 32, splits = (chunks + m.split - 1) / m.split;
    const int w = blockIdx.x - m.tile0, tile = w / splits, part = w - tile * splits;
    int ti, tj;
    lower(tile, ti, tj);
    const char* x = ws + x_at(m.off);
    const int ld = S * 4;
    Small p;
    p.run(rows_rsrc(x + (long long)ti * 64 * ld, R - ti * 64, ld, ld), ld, rows_rsrc(x + (long long)tj * 64 * ld, R - tj * 64, ld, ld), ld, part * m.split,
          min(m.split, chunks - part * m.split), lds);
    float* out = parts + (long long)blockIdx.x * 4096 + threadIdx.x * 4;
    int q = 0;
    p.each4([&](int, int, const float v[4]) { *reinterpret_cast<float4*>(out + (q++) * 1024) = make_float4(v[0], v[1], v[2], v[3]); });
}

// A = the sum of the partials, as pairs, both triangles.  t.tile0: as in the Gram launch.
__global__ __launch_bounds__(256) void ns_gram_sum_kernel(Works t, Works sums, char* ws, const float* parts) {
    const int k = find(sums.m, sums.count, blockIdx.x);
    const Work m = t.m[k];
    const int R = up64(m.r), chunks = up64(m.s) / 32, splits = (chunks + m.split - 1) / m.split;
    const int tile = blockIdx.x - sums.m[k].tile0;
    int ti, tj;
    lower(tile, ti, tj);
    const float* in = parts + ((long long)m.tile0 + (long long)tile * splits) * 4096 + threadIdx.x * 4;
    const float scale = ldexpf(SA, -2 * x_exponent(m.r, m.s));
    _Float16* a = (_Float16*)(ws + a_at(m.off, m.r, m.s));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = 0; p < splits; ++p) {
            const float4 v = *reinterpret_cast<const float4*>(in + (long long)p * 4096 + q * 1024);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        const float v[4] = {s.x * scale, s.y * scale, s.z * scale, s.w * scale};
        const int row = ti * 64 + (wave >> 1) * 32 + q * 8 + (lane >> 5) * 4, col = tj * 64 + (wave & 1) * 32 + (lane & 31);
#pragma unroll
        for (int e = 0; e < 4; ++e) put1(a, at(row + e, col, R), v[e]);
        if (ti != tj) put4(a, at(col, row, R), v);
    }
}

// B = b A + c A^2, lower tiles computed, both triangles written.
__global__ __launch_bounds__(256) void ns_poly_kernel(Works t, char* ws, float b, float c, int drop) {
    __shared__ __attribute__((aligned(1024))) char lds[Small::LDS];
    const int k = find(t.m, t.count, blockIdx.x);
    const Work m = t.m[k];
    const int R = up64(m.r), ld = R * 4;
    int ti, tj;
    lower(blockIdx.x - m.tile0, ti, tj);
    const char* a = ws + a_at(m.off, m.r, m.s);
    Small p;
    p.run(rows_rsrc(a + (long long)ti * 64 * ld, R - ti * 64, ld, ld), ld, rows_rsrc(a + (long long)tj * 64 * ld, R - tj * 64, ld, ld), ld, 0, R / 32, lds);
    _Float16* out = (_Float16*)(ws + b_at(m.off, m.r, m.s));
    const float fb = b * (SB / SA), fc = ldexpf(c * (SB / (SA * SA)), -2 * g_of(ws, m.off, drop));
    p.each4([&](int r, int cc, const float d[4]) {
        const int row = ti * 64 + r, col = tj * 64 + cc;
        float av[4], v[4];
        get4((const _Float16*)a, at(col, row, R), av);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = fmaf(fb, av[e], fc * d[e]); put1(out, at(row + e, col, R), v[e]); }
        if (ti != tj) put4(out, at(col, row, R), v);
    });
}

// X <- a X + B X.  Both orders of the new X.
__global__ __launch_bounds__(256) void ns_apply_kernel(Works t, char* ws, int from, float a, int drop, int drop_next) {
    __shared__ __attribute__((aligned(1024))) char lds[Small::LDS];
    const int k = find(t.m, t.count, blockIdx.x);
    const Work m = t.m[k];
    const int R = up64(m.r), S = up64(m.s), ld = R * 4, down = R / 64;
    const int w = blockIdx.x - m.tile0, r0 = (w % down) * 64, s0 = (w / down) * 64;
    const char* b = ws + b_at(m.off, m.r, m.s);
    const char* xt = ws + xt_at(m.off, m.r, m.s, from);
    Small p;
    p.run(rows_rsrc(b + (long long)r0 * ld, R - r0, ld, ld), ld, rows_rsrc(xt + (long long)s0 * ld, S - s0, ld, ld), ld, 0, R / 32, lds);
    _Float16* x = (_Float16*)(ws + x_at(m.off));
    _Float16* to = (_Float16*)(ws + xt_at(m.off, m.r, m.s, 1 - from));
    const int g = g_of(ws, m.off, drop), down_g = g_of(ws, m.off, drop_next) - g;
    const float fx = ldexpf(a, down_g), fd = ldexpf(1.f / SB, down_g - 2 * g);
    p.each4([&](int r, int c, const float d[4]) {
        const int row = r0 + r, col = s0 + c;
        float xv[4], v[4];
        get4((const _Float16*)xt, at(col, row, R), xv);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = fmaf(fx, xv[e], d[e] * fd); put1(x, at(row + e, col, S), v[e]); }
        put4(to, at(col, row, R), v);
    });
}

// The last X <- a X + B X: to the user's matrix, or into the weights.
template <int DT, bool STEP>
__global__ __launch_bounds__(256) void ns_leave_kernel(Exits t, const char* ws, int from, float a, int drop, float lr, const float* lr_device, float decay) {
    __shared__ __attribute__((aligned(1024))) char lds[Small::LDS];
    const int k = find(t.m, t.count, blockIdx.x);
    const Exit m = t.m[k];
    const int R = up64(m.r), S = up64(m.s), ld = R * 4, down = R / 64;
    const int w = blockIdx.x - m.tile0, r0 = (w % down) * 64, s0 = (w / down) * 64;
    const char* b = ws + b_at(m.off, m.r, m.s);
    const char* xt = ws + xt_at(m.off, m.r, m.s, from);
    Small p;
    p.run(rows_rsrc(b + (long long)r0 * ld, R - r0, ld, ld), ld, rows_rsrc(xt + (long long)s0 * ld, S - s0, ld, ld), ld, 0, R / 32, lds);
    const int g = g_of(ws, m.off, drop), unit = -x_exponent(m.r, m.s) - g;
    const float fd = ldexpf(1.f / SB, -2 * g);
    if constexpr (STEP) lr = lr_device ? *lr_device : lr;
    const float keep = 1.f - lr * decay, rate = lr * m.size;
    p.each4([&](int r, int c, const float d[4]) {
        const int row = r0 + r, col = s0 + c;
        float xv[4];
        get4((const _Float16*)xt, at(col, row, R), xv);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (row + e >= m.r || col >= m.s) continue;
            const float v = ldexpf(fmaf(a, xv[e], d[e] * fd), unit);
            const long long i = m.tall ? (long long)col * m.ld + row + e : (long long)(row + e) * m.ld + col;
            if constexpr (STEP) ((float*)m.dst)[i] = fmaf(-rate, v, ((const float*)m.dst)[i] * keep);
            else store1<DT>(m.dst, i, v);
        }
    });
}

// ------------------------------------------------------------------------------------------------------------------------------ host
constexpr int GRAM_WGS = 1024, GRAM_MIN = 8;   // workgroups of the Gram launch aimed at; k chunks of one of them at least

struct Plan {
    Works gram, sum, poly, apply;
    Entries norm, pack;
    Exits leave;
    long long tiles_gram, tiles_sum, tiles_poly, tiles_apply, tiles_norm, tiles_pack, parts_at, bytes;
};

// The launches of one group of matrices; returns false where a count passes what a grid or an int holds.
bool lay_out(const bflow_ns_matrix_t* m, int count, Plan& p) {
    long long off = 0, work = 0;
    p.tiles_gram = p.tiles_sum = p.tiles_poly = p.tiles_apply = p.tiles_norm = p.tiles_pack = 0;
    for (int i = 0; i < count; ++i) {
        const int r = m[i].rows < m[i].cols ? m[i].rows : m[i].cols, s = m[i].rows < m[i].cols ? m[i].cols : m[i].rows;
        const long long T = up64(r) / 64;
        work += T * (T + 1) / 2 * (up64(s) / 32);
    }
    for (int i = 0; i < count; ++i) {
        const int tall = m[i].rows > m[i].cols;
        const int r = tall ? m[i].cols : m[i].rows, s = tall ? m[i].rows : m[i].cols;
        const long long T = up64(r) / 64, U = up64(s) / 64, n = (long long)r * s, chunks = 2 * U;
        long long split = (work + GRAM_WGS - 1) / GRAM_WGS;
        split = split < GRAM_MIN ? GRAM_MIN : split;
        split = split > chunks ? chunks : split;
        long long per = (n + NORM_PARTS - 1) / NORM_PARTS;
        per = per < NORM_MIN ? NORM_MIN : per;
        p.gram.m[i] = {off, r, s, (int)p.tiles_gram, (int)split};
        p.sum.m[i] = {off, r, s, (int)p.tiles_sum, 0};
        p.poly.m[i] = {off, r, s, (int)p.tiles_poly, 0};
        p.apply.m[i] = {off, r, s, (int)p.tiles_apply, 0};
        p.norm.m[i] = {m[i].src, m[i].momentum, m[i].src_ld, off, r, s, (int)p.tiles_norm, (int)per, tall};
        p.pack.m[i] = p.norm.m[i];
        p.pack.m[i].tile0 = (int)p.tiles_pack;
        p.leave.m[i] = {m[i].dst, m[i].dst_ld, off, r, s, (int)p.tiles_apply, tall, 0.2f * sqrtf((float)s)};
        p.tiles_gram += T * (T + 1) / 2 * ((chunks + split - 1) / split);
        p.tiles_sum += T * (T + 1) / 2;
        p.tiles_poly += T * (T + 1) / 2;
        p.tiles_apply += T * U;
        p.tiles_norm += (n + per - 1) / per;
        p.tiles_pack += T * U;
        off = (end_at(off, r, s) + 255) & ~255LL;
    }
    p.gram.count = p.sum.count = p.poly.count = p.apply.count = p.norm.count = p.pack.count = p.leave.count = count;
    p.parts_at = off;
    p.bytes = off + p.tiles_gram * 4096 * 4;
    return p.tiles_gram < (1LL << 30) && p.tiles_apply < (1LL << 30);
}

const char* bad(const bflow_ns_matrix_t* m, int count) {
    if (!m || count < 0) return "null table or negative count";
    for (int i = 0; i < count; ++i) {
        if (m[i].rows < 1 || m[i].cols < 1 || m[i].rows > BFLOW_NS_MAX_SIDE || m[i].cols > BFLOW_NS_MAX_SIDE) return "a side outside 1 .. BFLOW_NS_MAX_SIDE";
        if ((long long)m[i].rows * m[i].cols > (1LL << 30)) return "more than 2^30 elements";
    }
    return nullptr;
}

// Largest |x| that the steps make of any x in [0, 1] (the coefficients have to keep the iterates inside the pairs' range), and the largest
// gain |x'| / |x| of one step there.
double reach(int steps, double a, double b, double c, double* gain) {
    double most = 0;
    *gain = 1;
    for (int i = 0; i <= 4096; ++i) {
        double x = i / 4096.0;
        for (int k = 0; k < steps; ++k) {
            const double f = a + x * x * (b + c * x * x);
            x *= f;
            if (!(std::fabs(x) <= most)) most = std::fabs(x);
            if (!(most < 1e6)) return 1e6;
            if (std::fabs(f) > *gain) *gain = std::fabs(f);
        }
    }
    return most;
}

template <int DT, bool STEP>
int launch_all(const Plan& p, int steps, float a, float b, float c, float eps, double gain, char* ws, float mu, int nesterov, float lr, const float* lr_device, float decay,
               hipStream_t st) {
    float* parts = (float*)(ws + p.parts_at);
    hipLaunchKernelGGL((ns_norm_kernel<DT, STEP>), dim3(p.tiles_norm), dim3(256), 0, st, p.norm, ws, mu, nesterov);
    hipLaunchKernelGGL((ns_pack_kernel<DT, STEP>), dim3(p.tiles_pack), dim3(256), 0, st, p.pack, ws, mu, nesterov, eps);
    const double bits = log2(gain);
    for (int k = 0; k < steps; ++k) {
        const int drop = (int)std::ceil(k * bits), next = (int)std::ceil((k + 1) * bits);
        hipLaunchKernelGGL(ns_gram_kernel, dim3(p.tiles_gram), dim3(256), 0, st, p.gram, ws, parts);
        hipLaunchKernelGGL(ns_gram_sum_kernel, dim3(p.tiles_sum), dim3(256), 0, st, p.gram, p.sum, ws, parts);
        hipLaunchKernelGGL(ns_poly_kernel, dim3(p.tiles_poly), dim3(256), 0, st, p.poly, ws, b, c, drop);
        if (k + 1 < steps) hipLaunchKernelGGL(ns_apply_kernel, dim3(p.tiles_apply), dim3(256), 0, st, p.apply, ws, k & 1, a, drop, next);
        else hipLaunchKernelGGL((ns_leave_kernel<DT, STEP>), dim3(p.tiles_apply), dim3(256), 0, st, p.leave, ws, k & 1, a, drop, lr, lr_device, decay);
    }
    return launch_status("newton_schulz");
}

int check(const bflow_ns_matrix_t* m, int count, int steps, float a, float b, float c, float eps, const void* ws, long long ws_bytes, bool step, double* gain) {
    const char* why = bad(m, count);
    BFLOW_REQUIRE(!why, BFLOW_E_ARG, "newton_schulz: %s", why);
    BFLOW_REQUIRE(steps >= 1 && steps <= 32, BFLOW_E_ARG, "newton_schulz: %d steps (1 .. 32)", steps);
    BFLOW_REQUIRE(eps > 0.f && eps < 1.f, BFLOW_E_ARG, "newton_schulz: eps %g outside (0, 1)", (double)eps);
    const double most = reach(steps, a, b, c, gain);
    BFLOW_REQUIRE(most <= 1.9 && std::fabs(b) * 4 + std::fabs(c) * 16 < 63, BFLOW_E_ARG,
                  "newton_schulz: coefficients (%g, %g, %g) take a singular value in [0, 1] to %g: the iterates must stay below 1.9", (double)a, (double)b,
                  (double)c, most);
    BFLOW_REQUIRE(!count || (ws && ((uintptr_t)ws & 255) == 0), BFLOW_E_ARG, "newton_schulz: workspace null or not aligned to 256 bytes");
    const long long need = bflow_ns_workspace_bytes(m, count);
    BFLOW_REQUIRE(need >= 0 && ws_bytes >= need, BFLOW_E_ARG, "newton_schulz: workspace of %lld bytes, %lld needed", ws_bytes, need);
    for (int i = 0; i < count; ++i)
        BFLOW_REQUIRE(m[i].src && m[i].dst && m[i].src_ld >= m[i].cols && m[i].dst_ld >= m[i].cols && (!step || m[i].momentum), BFLOW_E_ARG,
                      "newton_schulz: matrix %d: null pointer or a row shorter than its columns", i);
    return 0;
}
}  // namespace

extern "C" long long bflow_ns_workspace_bytes(const bflow_ns_matrix_t* m, int count) {
    if (const char* why = bad(m, count)) {
        set_error("newton_schulz: %s", why);
        return BFLOW_E_ARG;
    }
    long long most = 0;
    for (int i = 0; i < count; i += MOST) {
        static thread_local Plan p;
        if (!lay_out(m + i, count - i < MOST ? count - i : MOST, p)) {
            set_error("newton_schulz: too many tiles");
            return BFLOW_E_LIMIT;
        }
        most = p.bytes > most ? p.bytes : most;
    }
    return most;
}

extern "C" int bflow_ns_orthogonalize(const bflow_ns_matrix_t* m, int count, int dtype, int steps, float a, float b, float c, float eps, void* ws, long long ws_bytes,
                                      bflow_stream_t stream) {
    BFLOW_REQUIRE(dtype >= F32 && dtype <= BF16, BFLOW_E_ARG, "ns_orthogonalize: dtype %d", dtype);
    double gain;
    if (const int rc = check(m, count, steps, a, b, c, eps, ws, ws_bytes, false, &gain)) return rc;
    for (int i = 0; i < count; i += MOST) {
        static thread_local Plan p;
        lay_out(m + i, count - i < MOST ? count - i : MOST, p);
        const auto go = dtype == F32 ? launch_all<F32, false> : dtype == F16 ? launch_all<F16, false> : launch_all<BF16, false>;
        if (const int rc = go(p, steps, a, b, c, eps, gain, (char*)ws, 0.f, 0, 0.f, nullptr, 0.f, (hipStream_t)stream)) return rc;
    }
    return 0;
}

extern "C" int bflow_muon_step(const bflow_ns_matrix_t* m, int count, int steps, float a, float b, float c, float eps, float momentum, int nesterov, float lr,
                               const float* lr_device, float weight_decay, void* ws, long long ws_bytes, bflow_stream_t stream) {
    double gain;
    if (const int rc = check(m, count, steps, a, b, c, eps, ws, ws_bytes, true, &gain)) return rc;
    for (int i = 0; i < count; i += MOST) {
        static thread_local Plan p;
        lay_out(m + i, count - i < MOST ? count - i : MOST, p);
        if (const int rc = launch_all<F32, true>(p, steps, a, b, c, eps, gain, (char*)ws, momentum, nesterov, lr, lr_device, weight_decay, (hipStream_t)stream)) return rc;
    }
    return 0;
}
