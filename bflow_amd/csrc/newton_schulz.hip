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
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>
#include "common.h"
#include "tile_nt.h"

namespace {
using namespace bflow;
using namespace bflow::nt;

constexpr int MOST = BFLOW_NS_MAX_MATRICES;
constexpr float SA = 4096.f, SB = 1024.f;
constexpr int NORM_MIN = 4096, NORM_PARTS = 1024;   // elements of one partial sum of squares at least; partials of a matrix at most
constexpr int LARGE_BLOCKS = 512;                   // 64 x 64 blocks of the Gram matrices from which the large tiles are taken

struct Work {          // one matrix inside the products
    long long off;     // bytes from the workspace
    int r, s;          // rows <= columns
    int tile0;         // first workgroup of this launch
    int ex;            // log2 sx
};
struct Entry {         // one matrix where it enters
    const void* src;   // the matrix, or the gradient (step)
    float* momentum;   // step only
    long long ld, off;
    int r, s;
    int tile0, per;    // first workgroup; elements of one partial (norm)
    int tall, ex;
};
struct Exit {          // one matrix where it leaves
    void* dst;         // the result, or the weights (step)
    long long ld, off;
    int r, s;
    int tile0, tall;
    float size;        // step: 0.2 sqrt(max(m, n))
    int ex;
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
inline int x_exponent(int r, int s) {
    const double e = 0.5 * log2((double)r * (double)s);
    const int k = (int)(e + 0.5);
    return k > 14 ? 14 : k;
}

// The matrix that a workgroup works on: each lane looks at one matrix' first workgroup.
template <class T>
__device__ __forceinline__ int find(const T* m, int count, int wg) {
    const int lane = threadIdx.x & 63;
    const bool before = lane < count && m[lane < count ? lane : 0].tile0 <= wg;
    return __builtin_amdgcn_readfirstlane(__builtin_popcountll(__ballot(before)) - 1);
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

// p (1 - lr decay) - rate x, the decay beside the update: 1 - lr decay in 32 bits is 1 where lr decay is below 2^-25, as it is in training (1e-4 each).
// (An infinite weight stays what it is: its decay is that of the largest number.)
__device__ __forceinline__ float stepped(float p, float x, float rate, float shrink) {
    return p - fmaf(shrink, __builtin_amdgcn_fmed3f(p, -FLT_MAX, FLT_MAX), rate * x);
}

// position of (row, col) in an operand of `cols` padded columns, in halves; the lo half is 32 further
__device__ __forceinline__ long long at(int row, int col, int cols) { return (long long)row * (2 * cols) + (col >> 5) * 64 + (col & 31); }
__device__ __forceinline__ float pair_value(_Float16 h, _Float16 l) { return fmaf((float)l, SPLIT_LO_INV, (float)h); }
// A number as a pair: split1 (common.h) without its clamp, as nothing here leaves the range.  NaN stays NaN in both halves.
__device__ __forceinline__ void pair_of(float x, _Float16& h, _Float16& l) {
    h = fabsf(x) < 6.103515625e-05f ? (_Float16)0.f : (_Float16)x;
    l = (_Float16)((x - (float)h) * SPLIT_LO_SCALE);
}
__device__ __forceinline__ void put8(_Float16* m, long long i, half8 h, half8 l) {
    *reinterpret_cast<half8*>(m + i) = h;
    *reinterpret_cast<half8*>(m + i + 32) = l;
}
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

// A BM x BN tile of 32-bit numbers in LDS, to be written by columns of four rows, read by rows of eight and by columns of eight: the groups of four
// columns are permuted by the row's eighth, so that none of the three meets itself in a bank more than twice.
template <int BN> struct Turn {
    __device__ static __forceinline__ int at(int row, int col) { return row * BN + ((((col >> 2) ^ ((row >> 3) & 7)) << 2) | (col & 3)); }
    __device__ static __forceinline__ void row8(const float* t, int row, int col, float v[8]) {      // col a multiple of 8
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float4 x = *reinterpret_cast<const float4*>(t + at(row, col + 4 * h));
            v[4 * h] = x.x; v[4 * h + 1] = x.y; v[4 * h + 2] = x.z; v[4 * h + 3] = x.w;
        }
    }
    __device__ static __forceinline__ void put_row8(float* t, int row, int col, const float v[8]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) *reinterpret_cast<float4*>(t + at(row, col + 4 * h)) = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
    }
    // pairs in the place of the numbers: split once, read by columns without arithmetic
    __device__ static __forceinline__ void put_pairs(float* t, int row, int col, half8 h, half8 l) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = __builtin_bit_cast(float, half2_t{h[k], l[k]});
        put_row8(t, row, col, v);
    }
    __device__ static __forceinline__ void pairs8(const float* t, int row, int col, half8& h, half8& l) {
        float v[8];
        row8(t, row, col, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const half2_t p = __builtin_bit_cast(half2_t, v[k]);
            h[k] = p[0];
            l[k] = p[1];
        }
    }
    __device__ static __forceinline__ void col8(const float* t, int row, int col, half8& h, half8& l) {      // row a multiple of 8
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const half2_t p = __builtin_bit_cast(half2_t, t[at(row + k, col)]);
            h[k] = p[0];
            l[k] = p[1];
        }
    }
};

// ------------------------------------------------------------------------------------------------------------------------------ entry
// What enters the iteration at an element of the user's matrix, the step's momentum being up to date.
template <int DT, bool STEP>
__device__ __forceinline__ float entering(const Entry& m, long long from, long long dense, float mu, bool nesterov) {
    const float g = load1<DT>(m.src, from);
    if constexpr (!STEP) return g;
    const float v = m.momentum[dense];
    return nesterov ? fmaf(mu, v, g) : v;
}

// Sum of squares of one stretch of a matrix, in 64 bits; the step's momentum is brought up to date on the way.  Bound by memory: 12.6 million numbers of
// a step (gradient read, momentum read and written, 151 MB) 27 us, 5.6 TB/s.
template <int DT, bool STEP>
__global__ __launch_bounds__(256) void ns_norm_kernel(Entries t, char* ws, float mu, int nesterov) {
    __shared__ double part[4];
    const int k = find(t.m, t.count, blockIdx.x);
    const Entry m = t.m[k];
    const unsigned cols = m.tall ? m.r : m.s;
    const bool dense = m.ld == cols;
    const unsigned n = (unsigned)m.r * (unsigned)m.s, first = (blockIdx.x - m.tile0) * (unsigned)m.per, last = min(first + (unsigned)m.per, n);   // n <= 2^30
    double sum = 0;
    constexpr int TOGETHER = 8;                         // loads in front of the stores, which would hold them back
    for (unsigned e0 = first + threadIdx.x; e0 < last; e0 += 256 * TOGETHER) {
        float g[TOGETHER], v[TOGETHER];
#pragma unroll
        for (int u = 0; u < TOGETHER; ++u) {
            const unsigned e = min(e0 + 256 * u, last - 1);
            g[u] = load1<DT>(m.src, dense ? (long long)e : (long long)(e / cols) * m.ld + e % cols);
            if constexpr (STEP) v[u] = m.momentum[e];
        }
#pragma unroll
        for (int u = 0; u < TOGETHER; ++u) {
            if (e0 + 256 * u >= last) break;
            float x = g[u];
            if constexpr (STEP) {
                const float now = fmaf(mu, v[u], x);
                m.momentum[e0 + 256 * u] = now;
                x = nesterov ? fmaf(mu, now, x) : now;
            }
            sum += (double)x * (double)x;
        }
    }
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) ((double*)(ws + m.off))[blockIdx.x - m.tile0] = part[0] + part[1] + part[2] + part[3];
}

// X and (`both`) Xt of a 64 x 64 tile, scaled to sx / (|X| + eps), zeros in the padding.  Bound by memory: the same 12.6 million numbers (8 bytes in, 8
// out each) 43 us, 4.7 TB/s; a list of small ones by its latency (a network's filters, 5.3 million numbers: 20 us).
template <int DT, bool STEP>
__global__ __launch_bounds__(256) void ns_pack_kernel(Entries t, char* ws, float mu, int nesterov, double eps, int both) {
    __shared__ double part[4];
    __shared__ __attribute__((aligned(16))) float tile[64 * 64];
    const int k = find(t.m, t.count, blockIdx.x);
    const Entry m = t.m[k];
    const int R = up64(m.r), S = up64(m.s), across = S / 64;
    const int w = blockIdx.x - m.tile0, r0 = (w / across) * 64, s0 = (w - (w / across) * across) * 64;
    const int fast = threadIdx.x & 63, slow = threadIdx.x >> 6;
    const int i0 = m.tall ? s0 : r0, j0 = m.tall ? r0 : s0;               // of the user's matrix
    const int rows = m.tall ? m.s : m.r, cols = m.tall ? m.r : m.s;
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int i = i0 + slow + 4 * e, j = j0 + fast;
        v[e] = i < rows && j < cols ? entering<DT, STEP>(m, (long long)i * m.ld + j, (long long)i * cols + j, mu, nesterov) : 0.f;
    }
    const int parts = (int)(((long long)m.r * m.s + m.per - 1) / m.per);
    double sum = 0;
    for (int i = threadIdx.x; i < parts; i += 256) sum += ((const double*)(ws + m.off))[i];
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = part[0] + part[1] + part[2] + part[3];
    const double norm = sqrt(sum);
    // (NaN and infinite norms: the comparison is false, g = 0)
    const int g = norm > 0. && norm < eps ? (int)log2((norm + eps) / norm) : 0;
    if (w == 0 && threadIdx.x == 0) *(int*)(ws + g_at(m.off)) = g;
    const double scale = ldexp(1.0, m.ex + g) / (norm + eps);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        _Float16 h, l;
        pair_of((float)((double)v[e] * scale), h, l);
        tile[Turn<64>::at(slow + 4 * e, fast)] = __builtin_bit_cast(float, half2_t{h, l});
    }
    __syncthreads();
    // rows of the user's tile are rows of X, or (tall) of Xt
    _Float16* x = (_Float16*)(ws + x_at(m.off));
    _Float16* xt = (_Float16*)(ws + xt_at(m.off, m.r, m.s, 0));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int it = threadIdx.x + i * 256, line = it >> 3, eight = (it & 7) * 8;
        half8 ah, al, dh, dl;
        Turn<64>::pairs8(tile, line, eight, ah, al);
        Turn<64>::col8(tile, eight, line, dh, dl);
        if (both || !m.tall) put8(m.tall ? xt : x, m.tall ? at(s0 + line, r0 + eight, R) : at(r0 + line, s0 + eight, S), ah, al);
        if (both || m.tall) put8(m.tall ? x : xt, m.tall ? at(r0 + line, s0 + eight, S) : at(s0 + line, r0 + eight, R), dh, dl);
    }
}

// Tile t of a lower triangle, diagonal included, row by row: (0, 0), (1, 0), (1, 1), (2, 0), ...
__device__ __forceinline__ void lower32(int t, int& i, int& j) {
    i = 0;
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    j = t - i * (i + 1) / 2;
}

// g of a step: what the start had, less `drop` for the growth since
__device__ __forceinline__ int g_of(const char* ws, long long off, int drop) { return max(*(const int*)(ws + g_at(off)) - drop, 0); }

// --------------------------------------------------------------------------------------------------------------------------- products
// BM x BN tile of A B^T.  A group of waves has WM x WN of it each; KG groups share the contraction (a stage holds a chunk for each) and are summed
// in LDS, in a fixed order.  Three matrix passes over the 32 columns of a chunk.
// At 4096 x 4096 (three passes counted): X 1.10 PFLOP/s of fp16, A and B 1.00, matrix cores busy 65 and 55 % of the cycles at a clock that power holds down.
// A library product of plain fp16 reaches 1.49 here.
template <int BM_, int BN_, int WM, int WN, int KG_, int STAGES>
struct Product {
    static constexpr int BM = BM_, BN = BN_, KG = KG_;
    static constexpr int ACROSS = BN / WN, WAVES = (BM / WM) * ACROSS, THREADS = 64 * WAVES * KG, MT = WM / 32, NT = WN / 32;
    static constexpr int COLUMNS = 32;                   // of a chunk
    static constexpr int CHUNK_BYTES = (BM + BN) * CHUNK, STAGE = KG * CHUNK_BYTES, TILE = BM * BN * 4;
    static constexpr int LDS = STAGES * STAGE > KG * TILE ? STAGES * STAGE : KG * TILE;
    static_assert(BM / 8 % WAVES == 0 && BN / 8 % WAVES == 0 && WAVES % 2 == 0, "whole pieces of either operand for every wave, all odd or all even");
    typedef Turn<BN> T;

    // rounds of a contraction over `columns`, a multiple of 64: each group of waves takes a chunk in each
    __host__ __device__ static inline int rounds_of(int columns) { return (columns / COLUMNS + KG - 1) / KG; }

    // Leaves KG tiles in LDS (Turn order); the workgroup is synchronised.  a, b: descriptors of the tile's rows, `columns` (a multiple of 64) long;
    // rounds first .. last of them.
    __device__ static __forceinline__ void run(rsrc_t a, int lda, rsrc_t b, int ldb, int columns, char* lds) { run(a, lda, b, ldb, columns, lds, 0, rounds_of(columns)); }
    __device__ static __forceinline__ void run(rsrc_t a, int lda, rsrc_t b, int ldb, int columns, char* lds, int first, int last) {
        const int chunks = min(columns / COLUMNS, last * KG);
        const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = w / WAVES, wave = w % WAVES;
        const int wm = wave / ACROSS, wn = wave % ACROSS;
        const int va = lane_offset(lane, lda, wave), vb = lane_offset(lane, ldb, wave);
        f32x16 hh[MT][NT], xx[MT][NT];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int k = 0; k < 16; ++k) { hh[i][j][k] = 0.f; xx[i][j][k] = 0.f; }
        const int rounds = last - first;
        auto issue = [&](int round) {
            char* stage = lds + (round % STAGES) * STAGE + group * CHUNK_BYTES;
            const int c = (first + round) * KG + group;
            const bool there = c < chunks;                           // behind the last chunk: zeros
            const int at = there ? c * COLUMNS * 4 : 0;
#pragma unroll
            for (int i = 0; i < BM / 8 / WAVES; ++i)
                dma_piece(a, stage + (wave + i * WAVES) * 1024, there ? va + (wave + i * WAVES) * 8 * lda : OUTSIDE, at);
#pragma unroll
            for (int i = 0; i < BN / 8 / WAVES; ++i)
                dma_piece(b, stage + BM * CHUNK + (wave + i * WAVES) * 1024, there ? vb + (wave + i * WAVES) * 8 * ldb : OUTSIDE, at);
        };
        constexpr int PIECES = (BM + BN) / 8 / WAVES;
#pragma unroll
        for (int r = 0; r < STAGES - 1; ++r) issue(r);
        for (int r = 0; r < rounds; ++r) {
            // this wave's part of round r has landed (STAGES - 2 rounds may be in flight behind it), its reads of round r - 1 have returned; behind the
            // barrier that holds for every wave, and the stage of round r - 1 may be filled again
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * PIECES) : "memory");
            __builtin_amdgcn_s_barrier();
            issue(r + STAGES - 1);
            const char* as = lds + (r % STAGES) * STAGE + group * CHUNK_BYTES + wm * WM * CHUNK;
            const char* bs = lds + (r % STAGES) * STAGE + group * CHUNK_BYTES + (BM + wn * WN) * CHUNK;
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
        }
        wait_chunk();                          // also the pieces behind the last round: the tiles take their place
        __builtin_amdgcn_s_barrier();
        float* t = (float*)(lds + group * TILE);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    t[T::at(wm * WM + i * 32 + (k >> 2) * 8 + (lane >> 5) * 4 + (k & 3), wn * WN + j * 32 + (lane & 31))] = fmaf(xx[i][j][k], SPLIT_LO_INV, hh[i][j][k]);
        __syncthreads();
    }

    __device__ static __forceinline__ void sum8(const char* lds, int row, int col, float v[8]) {
        T::row8((const float*)lds, row, col, v);
#pragma unroll
        for (int g = 1; g < KG; ++g) {
            float u[8];
            T::row8((const float*)(lds + g * TILE), row, col, u);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] += u[k];
        }
    }
    static constexpr int EIGHTS = BM * BN / 8, ITEMS = (EIGHTS + THREADS - 1) / THREADS;     // pieces of eight; of a thread
    // Piece n of a thread: eight columns of a row.  False where the thread has none.
    __device__ static __forceinline__ bool row_piece(int n, int& row, int& col) {
        const int i = threadIdx.x + n * THREADS;
        row = i / (BN / 8);
        col = i % (BN / 8) * 8;
        return EIGHTS % THREADS == 0 || i < EIGHTS;
    }
    // f(n, row, col, v): every piece of the tile once, made into what the tile holds; g(row, col, h, l): the same as pairs, to be written
    template <class F, class G> __device__ static __forceinline__ void rows(char* lds, F f, G g) {
#pragma unroll
        for (int n = 0; n < ITEMS; ++n) {
            int row, col;
            if (!row_piece(n, row, col)) continue;
            float v[8];
            sum8(lds, row, col, v);
            f(n, row, col, v);
            half8 h, l;
#pragma unroll
            for (int k = 0; k < 8; ++k) { _Float16 a, b; pair_of(v[k], a, b); h[k] = a; l[k] = b; }
            g(row, col, h, l);
            T::put_pairs((float*)lds, row, col, h, l);
        }
    }
    // the same for a tile that stays in 32 bits
    template <class F> __device__ static __forceinline__ void values(char* lds, F f) {
#pragma unroll
        for (int n = 0; n < ITEMS; ++n) {
            int row, col;
            if (!row_piece(n, row, col)) continue;
            float v[8];
            sum8(lds, row, col, v);
            f(n, row, col, v);
            T::put_row8((float*)lds, row, col, v);
        }
    }
    // g(row, col, h, l): eight rows of a column of the pairs that `rows` left
    template <class G> __device__ static __forceinline__ void columns(const char* lds, G g) {
#pragma unroll
        for (int n = 0; n < ITEMS; ++n) {
            const int i = threadIdx.x + n * THREADS, col = i / (BM / 8), row = i % (BM / 8) * 8;
            if (EIGHTS % THREADS != 0 && i >= EIGHTS) continue;
            half8 h, l;
            T::col8((const float*)lds, row, col, h, l);
            g(row, col, h, l);
        }
    }
    // The pairs at a thread's pieces of an operand of `cols` padded columns, read ahead of the product: one after another between the stores they
    // would cost a memory latency each.
    struct Ahead {
        half8 h[ITEMS], l[ITEMS];
        __device__ __forceinline__ void load(const _Float16* m, int row0, int col0, int rows, int cols) {
#pragma unroll
            for (int n = 0; n < ITEMS; ++n) {
                int row, col;
                row_piece(n, row, col);
                const long long i = at(min(row0 + row, rows - 1), min(col0 + col, cols - 8), cols);
                h[n] = *reinterpret_cast<const half8*>(m + i);
                l[n] = *reinterpret_cast<const half8*>(m + i + 32);
            }
        }
        __device__ __forceinline__ float operator()(int n, int e) const { return pair_value(h[n][e], l[n][e]); }
    };
};

template <class P> __host__ __device__ inline int lower_tiles(int R) { const int down = (R + P::BM - 1) / P::BM; return down * (down + 1) / 2; }
// Tile t of a lower triangle, bands of BAND rows of tiles, each walked column by column; an XCD (workgroups go round them) takes an eighth of that walk, so
// that what it works on at one time shares rows: 4096 x 4096 4147 -> 4082 us, 8 of 1024 x 1024 870 -> 852 (whole calls, fp32).
constexpr int BAND = 8;
template <class P> __device__ __forceinline__ void lower(int t, int R, int& r0, int& c0) {
    static_assert(P::BM == P::BN, "square tiles");
    const int down = (R + P::BM - 1) / P::BM, total = lower_tiles<P>(R);
    const int x = t & 7, at = x * (total >> 3) + min(x, total & 7) + (t >> 3);
    int band = 0;
    while ((band + BAND) * (band + BAND + 1) / 2 <= at) band += BAND;        // rows in front of the band
    const int in = at - band * (band + 1) / 2, high = min(BAND, down - band);
    int i, j;
    if (in < band * high) {
        j = in / high;
        i = band + in - j * high;
    } else {
        lower32(in - band * high, i, j);
        i += band;
        j += band;
    }
    r0 = i * P::BM;
    c0 = j * P::BN;
}
// Tile t of a rectangle, in the same order: 24 of 640 x 640 903 -> 835 us, 2944 x 2944 2012 -> 1990; powers of two lose or gain up to 1 % (8 of 1024 x
// 1024 868 -> 872, 4096 x 4096 4217 -> 4242 in fp32, 4250 -> 4212 in bf16: there any order shares).
template <class P> __device__ __forceinline__ void panel(int t, int R, int S, int& r0, int& s0) {
    const int down = (R + P::BM - 1) / P::BM, across = (S + P::BN - 1) / P::BN, total = down * across;
    const int x = t & 7, at = x * (total >> 3) + min(x, total & 7) + (t >> 3);
    const int band = at / (BAND * across), in = at - band * BAND * across, high = min(BAND, down - band * BAND), j = in / high;
    r0 = (band * BAND + in - j * high) * P::BM;
    s0 = j * P::BN;
}
// What of a symmetric matrix a tile writes: 64 x 64 blocks on the diagonal once, those below it to both sides, those above not at all (another tile's
// mirror; the two differ in the last bit, and one writer keeps the result the same from run to run).
__device__ __forceinline__ bool mine(int row, int col) { return row >> 6 >= col >> 6; }
__device__ __forceinline__ bool mirrored(int row, int col) { return row >> 6 > col >> 6; }

// The tail of a launch: a tile of the large set takes a CU alone, so 528 of them (4096 rows) are two rounds of 256 and one of 16.  Tiles from `whole` on
// are cut along the contraction into `parts` workgroups each, which leave 32-bit sums in `room`, and ns_join_kernel adds them in their order.  Whole
// tiles keep their common walk along the contraction; dealing all of it out evenly lost that, and with it the L2 (189 -> 232 us).
struct Tail { int whole, parts, first; float* room; };      // first: the last workgroup is dispatched first
// This workgroup's tile, and its part of n rounds; false: a whole tile.
__device__ __forceinline__ bool cut_tile(const Tail& l, int wg, int& tile, int& part) {
    part = 0;
    tile = wg;
    if (wg < l.whole) return false;
    tile = l.whole + (wg - l.whole) / l.parts;
    part = (wg - l.whole) % l.parts;
    return true;
}
template <class P> __device__ __forceinline__ void leave_part(const Tail& l, int wg, const char* lds) {
    float* to = l.room + (long long)(wg - l.whole) * P::BM * P::BN;
#pragma unroll
    for (int i = 0; i < P::ITEMS; ++i) {
        int row, col;
        if (!P::row_piece(i, row, col)) continue;
        float v[8];
        P::sum8(lds, row, col, v);
#pragma unroll
        for (int h = 0; h < 2; ++h) *reinterpret_cast<float4*>(to + row * P::BN + col + 4 * h) = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
    }
}

// A = X X^T as pairs, both triangles.
template <class P> __device__ __forceinline__ void gram_out(const Work& m, char* ws, int r0, int c0, char* lds) {
    const int R = up64(m.r);
    const float scale = ldexpf(SA, -2 * m.ex);
    _Float16* a = (_Float16*)(ws + a_at(m.off, m.r, m.s));
    P::rows(lds, [&](int, int, int, float v[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= scale;
    }, [&](int row, int col, half8 h, half8 l) {
        if (r0 + row < R && c0 + col < R && mine(r0 + row, c0 + col)) put8(a, at(r0 + row, c0 + col, R), h, l);
    });
    if (r0 + P::BM <= c0 + 64) return;                  // nothing of the tile lies below the diagonal blocks
    __syncthreads();
    P::columns(lds, [&](int row, int col, half8 h, half8 l) {
        if (r0 + row < R && c0 + col < R && mirrored(r0 + row, c0 + col)) put8(a, at(c0 + col, r0 + row, R), h, l);
    });
}
template <class P>
__global__ __launch_bounds__(P::THREADS, 2) void ns_gram_kernel(Works t, Tail l, char* ws) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    int tile, part, r0, c0;
    const int wg = l.first ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    const bool cut = cut_tile(l, wg, tile, part);
    const int k = find(t.m, t.count, tile);
    const Work m = t.m[k];
    const int R = up64(m.r), S = up64(m.s), ld = S * 4, n = P::rounds_of(S);
    lower<P>(tile - m.tile0, R, r0, c0);
    const char* x = ws + x_at(m.off);
    P::run(rows_rsrc(x + (long long)r0 * ld, min(P::BM, R - r0), ld, ld), ld, rows_rsrc(x + (long long)c0 * ld, min(P::BN, R - c0), ld, ld), ld, S, lds,
           cut ? (int)((long long)n * part / l.parts) : 0, cut ? (int)((long long)n * (part + 1) / l.parts) : n);
    if (cut) leave_part<P>(l, wg, lds);
    else gram_out<P>(m, ws, r0, c0, lds);
}

// B = b A + c A^2, both triangles.
template <class P> __device__ __forceinline__ void poly_out(const Work& m, char* ws, int r0, int c0, char* lds, const typename P::Ahead& av, float b, float c, int drop) {
    const int R = up64(m.r);
    _Float16* out = (_Float16*)(ws + b_at(m.off, m.r, m.s));
    const float fb = b * (SB / SA), fc = ldexpf(c * (SB / (SA * SA)), -2 * g_of(ws, m.off, drop));
    P::rows(lds, [&](int n, int, int, float v[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(fb, av(n, e), fc * v[e]);
    }, [&](int row, int col, half8 h, half8 l) {
        if (r0 + row < R && c0 + col < R && mine(r0 + row, c0 + col)) put8(out, at(r0 + row, c0 + col, R), h, l);
    });
    if (r0 + P::BM <= c0 + 64) return;
    __syncthreads();
    P::columns(lds, [&](int row, int col, half8 h, half8 l) {
        if (r0 + row < R && c0 + col < R && mirrored(r0 + row, c0 + col)) put8(out, at(c0 + col, r0 + row, R), h, l);
    });
}
template <class P>
__global__ __launch_bounds__(P::THREADS, 2) void ns_poly_kernel(Works t, Tail l, char* ws, float b, float c, int drop) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    int tile, part, r0, c0;
    const int wg = l.first ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    const bool cut = cut_tile(l, wg, tile, part);
    const int k = find(t.m, t.count, tile);
    const Work m = t.m[k];
    const int R = up64(m.r), ld = R * 4, n = P::rounds_of(R);
    lower<P>(tile - m.tile0, R, r0, c0);
    const char* a = ws + a_at(m.off, m.r, m.s);
    typename P::Ahead av;
    av.load((const _Float16*)a, r0, c0, R, R);
    P::run(rows_rsrc(a + (long long)r0 * ld, min(P::BM, R - r0), ld, ld), ld, rows_rsrc(a + (long long)c0 * ld, min(P::BN, R - c0), ld, ld), ld, R, lds,
           cut ? (int)((long long)n * part / l.parts) : 0, cut ? (int)((long long)n * (part + 1) / l.parts) : n);
    if (cut) leave_part<P>(l, wg, lds);
    else poly_out<P>(m, ws, r0, c0, lds, av, b, c, drop);
}

// The tail's tiles, 64 x 64 of one a workgroup: the parts added, then what the product does with a tile.
enum { GRAM = 0, POLY = 1 };
template <class P, int WHAT>
__global__ __launch_bounds__(256) void ns_join_kernel(Works t, Tail l, char* ws, float b, float c, int drop) {
    typedef Product<64, 64, 32, 32, 1, 2> J;
    static_assert(J::THREADS == 256, "as launched");
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    constexpr int DOWN = P::BM / 64, ACROSS = P::BN / 64;
    const int in = blockIdx.x % (DOWN * ACROSS), rank = blockIdx.x / (DOWN * ACROSS), tile = l.whole + rank, dr = in / ACROSS * 64, dc = in % ACROSS * 64;
    const int k = find(t.m, t.count, tile);
    const Work m = t.m[k];
    const int R = up64(m.r);
    int r0, c0;
    lower<P>(tile - m.tile0, R, r0, c0);
    if (r0 + dr >= R || c0 + dc > r0 + dr) return;      // outside, or above the diagonal
    typename J::Ahead av;
    if (WHAT == POLY) av.load((const _Float16*)(ws + a_at(m.off, m.r, m.s)), r0 + dr, c0 + dc, R, R);
    const float* from = l.room + (long long)rank * l.parts * P::BM * P::BN + dr * P::BN + dc;
    float v[J::ITEMS][8];
#pragma unroll
    for (int i = 0; i < J::ITEMS; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
#pragma unroll 4
    for (int n = 0; n < l.parts; ++n)
#pragma unroll
        for (int i = 0; i < J::ITEMS; ++i) {
            int row, col;
            J::row_piece(i, row, col);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 y = *reinterpret_cast<const float4*>(from + (long long)n * P::BM * P::BN + row * P::BN + col + 4 * h);
                v[i][4 * h] += y.x; v[i][4 * h + 1] += y.y; v[i][4 * h + 2] += y.z; v[i][4 * h + 3] += y.w;
            }
        }
#pragma unroll
    for (int i = 0; i < J::ITEMS; ++i) {
        int row, col;
        J::row_piece(i, row, col);
        J::T::put_row8((float*)lds, row, col, v[i]);
    }
    __syncthreads();
    if (WHAT == GRAM) gram_out<J>(m, ws, r0 + dr, c0 + dc, lds);
    else poly_out<J>(m, ws, r0 + dr, c0 + dc, lds, av, b, c, drop);
}

// X <- a X + B X, by rows (in place: a tile reads and writes its own part alone) and by columns (from one Xt to the other).
template <class P>
__global__ __launch_bounds__(P::THREADS, 2) void ns_apply_kernel(Works t, char* ws, int from, float a, int drop, int drop_next) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int k = find(t.m, t.count, blockIdx.x);
    const Work m = t.m[k];
    const int R = up64(m.r), S = up64(m.s), ld = R * 4;
    int r0, s0;
    panel<P>(blockIdx.x - m.tile0, R, S, r0, s0);
    const char* b = ws + b_at(m.off, m.r, m.s);
    const char* xt = ws + xt_at(m.off, m.r, m.s, from);
    _Float16* x = (_Float16*)(ws + x_at(m.off));
    typename P::Ahead xv;
    xv.load(x, r0, s0, R, S);
    P::run(rows_rsrc(b + (long long)r0 * ld, min(P::BM, R - r0), ld, ld), ld, rows_rsrc(xt + (long long)s0 * ld, min(P::BN, S - s0), ld, ld), ld, R, lds);
    _Float16* to = (_Float16*)(ws + xt_at(m.off, m.r, m.s, 1 - from));
    const int g = g_of(ws, m.off, drop), down_g = g_of(ws, m.off, drop_next) - g;
    const float fx = ldexpf(a, down_g), fd = ldexpf(1.f / SB, down_g - 2 * g);
    P::rows(lds, [&](int n, int, int, float v[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(fx, xv(n, e), v[e] * fd);
    }, [&](int row, int col, half8 h, half8 l) {
        if (r0 + row < R && s0 + col < S) put8(x, at(r0 + row, s0 + col, S), h, l);
    });
    __syncthreads();
    P::columns(lds, [&](int row, int col, half8 h, half8 l) {
        if (r0 + row < R && s0 + col < S) put8(to, at(s0 + col, r0 + row, R), h, l);
    });
}

// The last X <- a X + B X: to the user's matrix, or into the weights.
template <class P, int DT, bool STEP>
__global__ __launch_bounds__(P::THREADS, 2) void ns_leave_kernel(Exits t, const char* ws, int from, float a, int drop, float lr, const float* lr_device, float decay) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int k = find(t.m, t.count, blockIdx.x);
    const Exit m = t.m[k];
    const int R = up64(m.r), S = up64(m.s), ld = R * 4;
    int r0, s0;
    panel<P>(blockIdx.x - m.tile0, R, S, r0, s0);
    const char* b = ws + b_at(m.off, m.r, m.s);
    const char* xt = ws + xt_at(m.off, m.r, m.s, from);
    typename P::Ahead xv;
    xv.load((const _Float16*)(ws + x_at(m.off)), r0, s0, R, S);
    P::run(rows_rsrc(b + (long long)r0 * ld, min(P::BM, R - r0), ld, ld), ld, rows_rsrc(xt + (long long)s0 * ld, min(P::BN, S - s0), ld, ld), ld, R, lds);
    const int g = g_of(ws, m.off, drop), unit = -m.ex - g;
    const float fd = ldexpf(1.f / SB, -2 * g);
    if constexpr (STEP) lr = lr_device ? *lr_device : lr;
    const float shrink = lr * decay, rate = lr * m.size;
    P::values(lds, [&](int n, int, int, float v[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = ldexpf(fmaf(a, xv(n, e), v[e] * fd), unit);
    });
    __syncthreads();
    // element by element along the user's rows (any address, whole lines), the weights of sixteen of them read together
    constexpr int N = P::BM * P::BN / P::THREADS, AT_ONCE = 16;
    static_assert(N % AT_ONCE == 0, "whole batches");
    if constexpr (DT == F32) {
        // four of a row at a time where they stand at multiples of 16 bytes: a step of 4 of 1024 x 1024 and 2 of 1024 x 4096
        // 132 -> 110 us (the same in the panels below: 1 of 236 us, left out)
        if (!m.tall && ((uintptr_t)m.dst | (unsigned long long)m.ld * 4) % 16 == 0 && m.s % 4 == 0) {
            constexpr int FOURS = N / 4 < 8 ? N / 4 : 8;
            static_assert(N / 4 % FOURS == 0, "whole batches");
#pragma unroll 1
            for (int n0 = 0; n0 < N / 4; n0 += FOURS) {
                float4 v[FOURS], p[FOURS];
                float* at[FOURS];
#pragma unroll
                for (int n = 0; n < FOURS; ++n) {
                    const int i = threadIdx.x + (n0 + n) * P::THREADS, row = i / (P::BN / 4), col = i % (P::BN / 4) * 4;
                    at[n] = r0 + row < m.r && s0 + col < m.s ? (float*)m.dst + (long long)(r0 + row) * m.ld + s0 + col : nullptr;
                    v[n] = *reinterpret_cast<const float4*>((const float*)lds + P::T::at(row, col));
                    if constexpr (STEP) p[n] = at[n] ? *reinterpret_cast<const float4*>(at[n]) : float4{0.f, 0.f, 0.f, 0.f};
                }
#pragma unroll
                for (int n = 0; n < FOURS; ++n) {
                    if (!at[n]) continue;
                    if constexpr (STEP) v[n] = make_float4(stepped(p[n].x, v[n].x, rate, shrink), stepped(p[n].y, v[n].y, rate, shrink), stepped(p[n].z, v[n].z, rate, shrink), stepped(p[n].w, v[n].w, rate, shrink));
                    *reinterpret_cast<float4*>(at[n]) = v[n];
                }
            }
            return;
        }
    }
#pragma unroll 1
    for (int n0 = 0; n0 < N; n0 += AT_ONCE) {
        long long at[AT_ONCE];
        float v[AT_ONCE], p[AT_ONCE];
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
            const int i = threadIdx.x + (n0 + n) * P::THREADS;
            const int row = m.tall ? i % P::BM : i / P::BN, col = m.tall ? i / P::BM : i % P::BN;
            const bool in = r0 + row < m.r && s0 + col < m.s;
            at[n] = !in ? -1 : m.tall ? (long long)(s0 + col) * m.ld + r0 + row : (long long)(r0 + row) * m.ld + s0 + col;
            v[n] = ((const float*)lds)[P::T::at(row, col)];
            if constexpr (STEP) p[n] = in ? ((const float*)m.dst)[at[n]] : 0.f;
        }
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n)
            if (at[n] >= 0) {
                if constexpr (STEP) ((float*)m.dst)[at[n]] = stepped(p[n], v[n], rate, shrink);
                else store1<DT>(m.dst, at[n], v[n]);
            }
    }
}

// ----------------------------------------------------------------------------------------------------------------------------- panels
// Matrices of at most 256 rows (the filters of a network): what bounds the products above is memory, X by rows and by columns to and fro.  Here a
// workgroup takes PANELS of X, all R rows by 64 columns, held by rows alone.  Once a panel is in LDS it is multiplied by B, updated in place,
// written back, and multiplied by its own transpose, all from LDS; X crosses the chip once each way a step.  The Gram parts of a matrix' workgroups
// are added, in order, where B is made of them.  A step is two launches instead of three.
//   apply   D[s][r'] = sum_r X[r][s] B[r'][r]: the left operand needs eight rows of one column in a lane, which the transposing LDS read gives;
//           four neighbouring columns of a row leave a lane together, so a panel is updated by 8-byte reads and writes.
//   Gram    lower 32 x 32 tiles dealt over the waves; a panel's product is added to sums that stay in registers (16 a tile) from panel to panel.
// B stays in LDS up to 128 rows and is streamed by chunks of 32 columns above (three or four in flight).
// The filters of a network (64 x 245 to 256 x 1152, 47 of them, 5.3 million numbers): 26 us for update and Gram, 7 + 6 for B; matrix cores busy 21 % of the
// cycles.  What bounds it is one panel of 256 rows, a workgroup's chain of 8 chunks, update, Gram (14 us), of which there is hardly one for each CU.
constexpr int PANEL_ROWS = 256, PANEL_THREADS = 512;

struct PanelWork {     // one matrix
    long long off;
    short r, ex;       // rows; log2 sx
    int s;
    int wg0, square0, sum0;  // first workgroup of the panel launches, of those that make B, of those that add the parts
    int per;           // panels of a workgroup
};
struct PanelWorks { PanelWork m[MOST]; int count; };
struct PanelExit {     // where a matrix leaves
    void* dst;
    long long ld;
    float size;
    int tall;
};
struct PanelExits { PanelExit m[MOST]; };
static_assert(sizeof(PanelWorks) + sizeof(PanelExits) <= 4096, "the tables are kernel arguments");
// regions: norm partials, g, X, B, A, the Gram parts (32 bits, lower tiles)
__host__ __device__ inline long long pb_at(long long off, int r, int s) { return x_at(off) + mat_bytes(r, s); }
__host__ __device__ inline long long pa_at(long long off, int r, int s) { return pb_at(off, r, s) + mat_bytes(r, r); }
__host__ __device__ inline long long parts_at(long long off, int r, int s) { return pa_at(off, r, s) + mat_bytes(r, r); }
__host__ __device__ inline int panels_of(int s) { return up64(s) / 64; }
__host__ __device__ inline long long part_size(int R) { return (long long)(R / 32) * (R / 32 + 1) / 2 * 1024; }      // lower 32 x 32 tiles, in numbers

template <class F> __device__ __forceinline__ int find_by(int count, int wg, F first) {
    const int lane = threadIdx.x & 63;
    const bool before = lane < count && first(lane < count ? lane : 0) <= wg;
    return __builtin_amdgcn_readfirstlane(__builtin_popcountll(__ballot(before)) - 1);
}

typedef short short4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4_t* tr_t;
__device__ __forceinline__ half4 tr_read(const char* p) {
    return __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_t)p));
}
__device__ __forceinline__ half8 join(half4 a, half4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

enum { FIRST = 0, MIDDLE = 1, LAST = 2 };     // Gram alone; update and Gram; update alone, to the user

template <int RT> struct PanelSize {
    static constexpr int R = 64 * RT, IMAGE = 2 * R * CHUNK, STAGE = R * CHUNK;
    static constexpr bool RESIDENT = RT <= 2;
    static constexpr int STAGES = RESIDENT ? 2 * RT : RT == 3 ? 4 : 3;
    static constexpr int IMAGES = RESIDENT ? 2 : 1;        // room for the next panel beside the current one
    static constexpr int LDS = IMAGES * IMAGE + STAGES * STAGE;
};

struct Numbers {       // of a step
    int drop, drop_next;
    float a, lr;
    const float* lr_device;
    float decay;
};

template <int RT, int MODE, int DT, bool STEP>
__device__ __forceinline__ void panel_body(const PanelWork& m, const PanelExit& o, char* ws, int slice, const Numbers& nu, char* lds) {
    typedef PanelSize<RT> P;
    constexpr int R = P::R, STAGES = P::STAGES, AT = (RT + 1) / 2, GRAM = RT * (2 * RT + 1), GT = (GRAM + 7) / 8;
    const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int S = up64(m.s), ldx = S * 4, ldb = R * 4, panels = S / 64;
    char* x = ws + x_at(m.off);
    char* stages = lds + P::IMAGES * P::IMAGE;
    const rsrc_t rx = rows_rsrc(x, R, ldx, ldx), rb = rows_rsrc(ws + pb_at(m.off, m.r, m.s), R, ldb, ldb);
    const int vx = lane_offset(lane, ldx, w), vb = lane_offset(lane, ldb, w);
    const int g = MODE == FIRST ? 0 : g_of(ws, m.off, nu.drop), down_g = MODE == MIDDLE ? g_of(ws, m.off, nu.drop_next) - g : 0;
    const float fx = ldexpf(nu.a, down_g), fd = ldexpf(1.f / SB, down_g - 2 * g);
    const int unit = MODE == LAST ? -m.ex - g : 0;

    auto load_panel = [&](int p, char* image) {   // 2 chunks x R rows, 8 rows a piece
#pragma unroll
        for (int i = 0; i < 2 * RT; ++i) {
            const int q = w + i * 8, j = q / (8 * RT), piece = q - j * 8 * RT;
            dma_piece(rx, image + j * R * CHUNK + piece * 1024, vx + piece * 8 * ldx, (p * 2 + j) * CHUNK);
        }
    };
    auto load_b = [&](int c, int stage) {         // chunk c of B, all its rows; behind the last one zeros
        const bool there = c < 2 * RT;
#pragma unroll
        for (int i = 0; i < RT; ++i)
            dma_piece(rb, stages + stage * P::STAGE + (w + i * 8) * 1024, there ? vb + (w + i * 8) * 8 * ldb : OUTSIDE, there ? c * CHUNK : 0);
    };

    // apply: column block sb, row tiles t0, t0 + 4
    const int sb = w & 1, t0 = w >> 1;
    // transposing read u (rows + 4 u), half l (hi, lo): lane 16 k + i fetches row i / 4, four columns at 16 (k & 1) + 4 (i % 4), eight rows further for k >= 2
    int tr[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int l = 0; l < 2; ++l) {
            const int row = h * 8 + u * 4 + ((lane & 15) >> 2), seg = ((lane & 16) >> 3) + ((lane & 3) >> 1) + 4 * l;
            tr[u][l] = sb * R * CHUNK + row * CHUNK + ((seg ^ swizzle(row)) << 4) + (lane & 1) * 8;
        }
    f32x16 sums[GT];
    if (MODE != LAST)
#pragma unroll
        for (int t = 0; t < GT; ++t)
#pragma unroll
            for (int k = 0; k < 16; ++k) sums[t][k] = 0.f;

    const int first = slice * m.per, last = min(first + m.per, panels);
    if (P::RESIDENT) {
        load_panel(first, lds);
        if (MODE != FIRST)
#pragma unroll
            for (int c = 0; c < 2 * RT; ++c) load_b(c, c);
    }
    for (int p = first; p < last; ++p) {
        char* image = lds + (P::RESIDENT ? (p - first) & 1 : 0) * P::IMAGE;
        if (P::RESIDENT) {
            // this panel has landed: loads and stores leave vmcnt in order, and behind its pieces stand the 2 RT stores of the panel before it at most
            if (MODE == MIDDLE && p > first) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * RT) : "memory");
            else wait_chunk();
            __builtin_amdgcn_s_barrier();         // for every wave; and the other image is free
            if (p + 1 < last) load_panel(p + 1, lds + ((p + 1 - first) & 1) * P::IMAGE);
        } else {
            load_panel(p, image);
            if (MODE == FIRST) {
                wait_chunk();
                __builtin_amdgcn_s_barrier();
            } else {
#pragma unroll
                for (int c = 0; c < STAGES - 1; ++c) load_b(c, c);
            }
        }
        if (MODE != FIRST) {
            f32x16 hh[AT], xx[AT];
#pragma unroll
            for (int n = 0; n < AT; ++n)
#pragma unroll
                for (int k = 0; k < 16; ++k) { hh[n][k] = 0.f; xx[n][k] = 0.f; }
            int stage = 0;
#pragma unroll 1
            for (int c = 0; c < 2 * RT; ++c) {
                if (!P::RESIDENT) {               // chunk c (and, before it, the panel) has landed; the stage of chunk c - 1 is free
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * RT) : "memory");
                    __builtin_amdgcn_s_barrier();
                    load_b(c + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
                }
                const char* bs = stages + stage * P::STAGE;
                stage = stage == STAGES - 1 ? 0 : stage + 1;
#pragma unroll
                for (int sub = 0; sub < 2; ++sub) {
                    const char* at = image + (c * 32 + sub * 16) * CHUNK;
                    const half8 xh = join(tr_read(at + tr[0][0]), tr_read(at + tr[1][0])), xl = join(tr_read(at + tr[0][1]), tr_read(at + tr[1][1]));
#pragma unroll
                    for (int n = 0; n < AT; ++n)
                        if (t0 + 4 * n < 2 * RT) {
                            const char* rows = bs + (t0 + 4 * n) * 32 * CHUNK;
                            const half8 bh = __builtin_bit_cast(half8, frag(rows, lane, sub)), bl = __builtin_bit_cast(half8, frag(rows, lane, 2 + sub));
                            hh[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xh, bh, hh[n], 0, 0, 0);
                            xx[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xh, bl, xx[n], 0, 0, 0);
                            xx[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xl, bh, xx[n], 0, 0, 0);
                        }
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();         // every wave has read the old panel
#pragma unroll
            for (int n = 0; n < AT; ++n)
                if (t0 + 4 * n < 2 * RT) {
                    const int row = (t0 + 4 * n) * 32 + l31;
                    char* mine = image + sb * R * CHUNK + row * CHUNK + h * 8;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        char *ph = mine + ((q ^ swizzle(row)) << 4), *pl = mine + (((q + 4) ^ swizzle(row)) << 4);
                        half4 xh = *reinterpret_cast<const half4*>(ph), xl = *reinterpret_cast<const half4*>(pl);
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float d = fmaf(xx[n][q * 4 + e], SPLIT_LO_INV, hh[n][q * 4 + e]);
                            v[e] = fmaf(fx, pair_value(xh[e], xl[e]), d * fd);
                        }
                        if (MODE == LAST) {       // the result itself, in the place of the pairs
                            *reinterpret_cast<float2*>(ph) = make_float2(ldexpf(v[0], unit), ldexpf(v[1], unit));
                            *reinterpret_cast<float2*>(pl) = make_float2(ldexpf(v[2], unit), ldexpf(v[3], unit));
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) { _Float16 a, b; pair_of(v[e], a, b); xh[e] = a; xl[e] = b; }
                            *reinterpret_cast<half4*>(ph) = xh;
                            *reinterpret_cast<half4*>(pl) = xl;
                        }
                    }
                }
            __syncthreads();
        }
        if (MODE == MIDDLE) {                     // back to memory: 256 bytes of a row together
#pragma unroll
            for (int n = 0; n < 2 * RT; ++n) {
                const int i = threadIdx.x + n * PANEL_THREADS, seg = i & 7, j = (i >> 3) & 1, row = i >> 4;
                *reinterpret_cast<i32x4*>(x + (long long)row * ldx + (p * 2 + j) * CHUNK + seg * 16) =
                    *reinterpret_cast<const i32x4*>(image + j * R * CHUNK + row * CHUNK + ((seg ^ swizzle(row)) << 4));
            }
        }
        if (MODE == LAST) {
            const float lr = STEP ? (nu.lr_device ? *nu.lr_device : nu.lr) : 0.f, shrink = lr * nu.decay, rate = lr * o.size;
            // element by element along the user's rows, eight of a thread together
            constexpr int AT_ONCE = 8;
#pragma unroll 1
            for (int n0 = 0; n0 < 8 * RT; n0 += AT_ONCE) {
                long long to[AT_ONCE];
                float v[AT_ONCE], old[AT_ONCE];
#pragma unroll
                for (int n = 0; n < AT_ONCE; ++n) {
                    const int i = threadIdx.x + (n0 + n) * PANEL_THREADS, row = o.tall ? i % R : i >> 6, col = o.tall ? i / R : i & 63, s = p * 64 + col;
                    const bool in = row < m.r && s < m.s;
                    to[n] = !in ? -1 : o.tall ? (long long)s * o.ld + row : (long long)row * o.ld + s;
                    const int seg = ((col & 31) >> 3) + ((col & 2) << 1);
                    v[n] = *reinterpret_cast<const float*>(image + (col >> 5) * R * CHUNK + row * CHUNK + ((seg ^ swizzle(row)) << 4) + ((col >> 2) & 1) * 8 + (col & 1) * 4);
                    if constexpr (STEP) old[n] = in ? ((const float*)o.dst)[to[n]] : 0.f;
                }
#pragma unroll
                for (int n = 0; n < AT_ONCE; ++n)
                    if (to[n] >= 0) {
                        if constexpr (STEP) ((float*)o.dst)[to[n]] = stepped(old[n], v[n], rate, shrink);
                        else store1<DT>(o.dst, to[n], v[n]);
                    }
            }
        }
        if (MODE != LAST) {
#pragma unroll
            for (int t = 0; t < GT; ++t) {
                const int tile = w + t * 8;
                if (tile >= GRAM) continue;
                int i, j;
                lower32(tile, i, j);
                f32x16 gh, gx;
#pragma unroll
                for (int k = 0; k < 16; ++k) { gh[k] = 0.f; gx[k] = 0.f; }
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int sub = 0; sub < 2; ++sub) {
                        const char *ai = image + c * R * CHUNK + i * 32 * CHUNK, *aj = image + c * R * CHUNK + j * 32 * CHUNK;
                        const half8 ih = __builtin_bit_cast(half8, frag(ai, lane, sub)), il = __builtin_bit_cast(half8, frag(ai, lane, 2 + sub));
                        const half8 jh = __builtin_bit_cast(half8, frag(aj, lane, sub)), jl = __builtin_bit_cast(half8, frag(aj, lane, 2 + sub));
                        gh = __builtin_amdgcn_mfma_f32_32x32x16_f16(ih, jh, gh, 0, 0, 0);
                        gx = __builtin_amdgcn_mfma_f32_32x32x16_f16(ih, jl, gx, 0, 0, 0);
                        gx = __builtin_amdgcn_mfma_f32_32x32x16_f16(il, jh, gx, 0, 0, 0);
                    }
#pragma unroll
                for (int k = 0; k < 16; ++k) sums[t][k] += fmaf(gx[k], SPLIT_LO_INV, gh[k]);
            }
        }
        if (!P::RESIDENT) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();         // every wave is done with the panel and the stages
        }
    }
    if (MODE != LAST) {                           // the lower tiles, each in the order of the registers: whole lines
        float* part = (float*)(ws + parts_at(m.off, m.r, m.s)) + (long long)slice * part_size(R) + lane * 4;
#pragma unroll
        for (int t = 0; t < GT; ++t) {
            const int tile = w + t * 8;
            if (tile >= GRAM) continue;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<float4*>(part + tile * 1024 + q * 256) = make_float4(sums[t][q * 4], sums[t][q * 4 + 1], sums[t][q * 4 + 2], sums[t][q * 4 + 3]);
        }
    }
}

template <int MODE, int DT, bool STEP>
__device__ __forceinline__ void panel_switch(const PanelWork& m, const PanelExit& o, char* ws, const Numbers& nu, char* lds) {
    const int slice = blockIdx.x - m.wg0;
    switch (up64(m.r) / 64) {
        case 1: panel_body<1, MODE, DT, STEP>(m, o, ws, slice, nu, lds); break;
        case 2: panel_body<2, MODE, DT, STEP>(m, o, ws, slice, nu, lds); break;
        case 3: panel_body<3, MODE, DT, STEP>(m, o, ws, slice, nu, lds); break;
        default: panel_body<4, MODE, DT, STEP>(m, o, ws, slice, nu, lds); break;
    }
}
__global__ __launch_bounds__(PANEL_THREADS, 2) void ns_panel_first_kernel(PanelWorks t, char* ws) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    panel_switch<FIRST, F32, false>(t.m[find_by(t.count, blockIdx.x, [&](int i) { return t.m[i].wg0; })], PanelExit{}, ws, Numbers{}, lds);
}
__global__ __launch_bounds__(PANEL_THREADS, 2) void ns_panel_middle_kernel(PanelWorks t, char* ws, Numbers nu) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    panel_switch<MIDDLE, F32, false>(t.m[find_by(t.count, blockIdx.x, [&](int i) { return t.m[i].wg0; })], PanelExit{}, ws, nu, lds);
}
template <int DT, bool STEP>
__global__ __launch_bounds__(PANEL_THREADS, 2) void ns_panel_last_kernel(PanelWorks t, PanelExits leave, char* ws, Numbers nu) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int k = find_by(t.count, blockIdx.x, [&](int i) { return t.m[i].wg0; });
    panel_switch<LAST, DT, STEP>(t.m[k], leave.m[k], ws, nu, lds);
}

// Four numbers of A, rows 8 q + 4 h .. + 3 of column `lane % 32` of a tile: the sum of the Gram parts, as pairs.  TOGETHER: eight parts at once on their
// way, the last again where there are fewer -- for few workgroups, that wait for every load (64 x 576: 8.1 -> 6.3 us; a launch of many tiles: 5.6 -> 6.4).
template <bool TOGETHER> __device__ __forceinline__ void summed(const float* f, long long one, int slices, float scale, half4& hi, half4& lo) {
    float4 s = *reinterpret_cast<const float4*>(f);
    auto add = [&](float4 v) { s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w; };
    if constexpr (TOGETHER) {
        for (int n = 1; n < slices; n += 8) {
            float4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = *reinterpret_cast<const float4*>(f + min(n + u, slices - 1) * one);
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (n + u < slices) add(v[u]);
        }
    } else {
#pragma unroll 8
        for (int n = 1; n < slices; ++n) add(*reinterpret_cast<const float4*>(f + n * one));
    }
    const float v[4] = {s.x * scale, s.y * scale, s.z * scale, s.w * scale};
#pragma unroll
    for (int e = 0; e < 4; ++e) { _Float16 a, l; pair_of(v[e], a, l); hi[e] = a; lo[e] = l; }
}
__device__ __forceinline__ int slices_of(const PanelWork& m) { return (panels_of(m.s) + m.per - 1) / m.per; }

// A = the sum of the Gram parts, on its own launch: where there are many parts, adding them where B is made would have every tile's workgroup read
// half of them or more.  A workgroup adds one 32 x 32 tile and writes it to both sides.
__global__ __launch_bounds__(256) void ns_panel_sum_kernel(PanelWorks t, char* ws) {
    __shared__ half2_t tile[32][33];
    const PanelWork m = t.m[find_by(t.count, blockIdx.x, [&](int i) { return t.m[i].sum0; })];
    const int R = up64(m.r), n = blockIdx.x - m.sum0, lane = threadIdx.x & 63, q = threadIdx.x >> 6, col = lane & 31, row = q * 8 + (lane >> 5) * 4;
    int i, j;
    lower32(n, i, j);
    half4 hi, lo;
    summed<false>((const float*)(ws + parts_at(m.off, m.r, m.s)) + n * 1024 + threadIdx.x * 4, part_size(R), slices_of(m), ldexpf(SA, -2 * m.ex), hi, lo);
    _Float16* a = (_Float16*)(ws + pa_at(m.off, m.r, m.s));
    if (i != j) {                                 // column by column: the tile on the other side of the diagonal
        *reinterpret_cast<half4*>(a + at(j * 32 + col, i * 32 + row, R)) = hi;
        *reinterpret_cast<half4*>(a + at(j * 32 + col, i * 32 + row, R) + 32) = lo;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[row + e][col] = half2_t{hi[e], lo[e]};
    __syncthreads();
    const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) { hi[e] = tile[r][c + e][0]; lo[e] = tile[r][c + e][1]; }
    *reinterpret_cast<half4*>(a + at(i * 32 + r, j * 32 + c, R)) = hi;
    *reinterpret_cast<half4*>(a + at(i * 32 + r, j * 32 + c, R) + 32) = lo;
}

// B = b A + c A^2 of matrices of at most 256 rows: a 64 x 64 tile of the lower triangle a workgroup; the two blocks of 64 rows of A that it needs stand
// whole in LDS.  SUMMED: A is in memory; otherwise the parts are added on the way.
typedef Product<64, 64, 32, 32, 2, 2> PanelSquare;     // (its way of writing a tile; two groups of waves share the contraction)
constexpr int panel_square_lds(int R) { return 2 * (R / 32) * 64 * CHUNK + PanelSquare::KG * PanelSquare::TILE; }

template <bool SUMMED>
__global__ __launch_bounds__(PANEL_THREADS, 2) void ns_panel_square_kernel(PanelWorks t, char* ws, float b, float c, int drop) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const PanelWork m = t.m[find_by(t.count, blockIdx.x, [&](int i) { return t.m[i].square0; })];
    const int R = up64(m.r), chunks = R / 32;
    int ti, tj;
    lower32(blockIdx.x - m.square0, ti, tj);
    char *tiles = lds, *image = lds + PanelSquare::KG * PanelSquare::TILE;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int blk = 0; blk < (ti == tj ? 1 : 2); ++blk) {
        const int row0 = (blk ? tj : ti) * 64;
        char* to = image + blk * chunks * 64 * CHUNK;
        if constexpr (SUMMED) {
            const int ld = R * 4;
            const rsrc_t ra = rows_rsrc(ws + pa_at(m.off, m.r, m.s) + (long long)row0 * ld, 64, ld, ld);
            const int va = lane_offset(lane, ld, w) + w * 8 * ld;
            for (int cc = 0; cc < chunks; ++cc) dma_piece(ra, to + cc * 64 * CHUNK + w * 1024, va, cc * CHUNK);
        } else {
            const float* parts = (const float*)(ws + parts_at(m.off, m.r, m.s));
            const float scale = ldexpf(SA, -2 * m.ex);
            const int slices = slices_of(m), col = lane & 31, row = (w & 3) * 8 + (lane >> 5) * 4;
            for (int n = w >> 2; n < 2 * chunks; n += 2) {       // 32 x 32 tiles of the block, four waves each
                const int half = n & 1, i = row0 / 32 + half, j = n >> 1, up = max(i, j), left = min(i, j);
                half4 hi, lo;
                summed<true>(parts + (up * (up + 1) / 2 + left) * 1024 + (w & 3) * 256 + lane * 4, part_size(R), slices, scale, hi, lo);
                char* at = to + (j * 64 + half * 32) * CHUNK;
                if (i >= j) {                                    // four rows of a column
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        char* r = at + (row + e) * CHUNK + (col & 7) * 2;
                        *reinterpret_cast<_Float16*>(r + (((col >> 3) ^ swizzle(row + e)) << 4)) = hi[e];
                        *reinterpret_cast<_Float16*>(r + ((((col >> 3) + 4) ^ swizzle(row + e)) << 4)) = lo[e];
                    }
                } else {                                         // from the other side of the diagonal: four columns of a row
                    char* r = at + col * CHUNK + (row & 4) * 2;
                    *reinterpret_cast<half4*>(r + (((row >> 3) ^ swizzle(col)) << 4)) = hi;
                    *reinterpret_cast<half4*>(r + ((((row >> 3) + 4) ^ swizzle(col)) << 4)) = lo;
                }
            }
        }
    }
    if constexpr (SUMMED) wait_chunk();
    __syncthreads();
    const char *rows_i = image, *rows_j = image + (ti == tj ? 0 : chunks * 64 * CHUNK);
    const int group = w >> 2, wm = (w >> 1) & 1, wn = w & 1;
    f32x16 hh, xx;
#pragma unroll
    for (int e = 0; e < 16; ++e) { hh[e] = 0.f; xx[e] = 0.f; }
    for (int cc = group; cc < chunks; cc += 2)
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const char *ai = rows_i + (cc * 64 + wm * 32) * CHUNK, *aj = rows_j + (cc * 64 + wn * 32) * CHUNK;
            const half8 ih = __builtin_bit_cast(half8, frag(ai, lane, sub)), il = __builtin_bit_cast(half8, frag(ai, lane, 2 + sub));
            const half8 jh = __builtin_bit_cast(half8, frag(aj, lane, sub)), jl = __builtin_bit_cast(half8, frag(aj, lane, 2 + sub));
            hh = __builtin_amdgcn_mfma_f32_32x32x16_f16(ih, jh, hh, 0, 0, 0);
            xx = __builtin_amdgcn_mfma_f32_32x32x16_f16(ih, jl, xx, 0, 0, 0);
            xx = __builtin_amdgcn_mfma_f32_32x32x16_f16(il, jh, xx, 0, 0, 0);
        }
    float* mine_t = (float*)(tiles + group * PanelSquare::TILE);
#pragma unroll
    for (int e = 0; e < 16; ++e)
        mine_t[PanelSquare::T::at(wm * 32 + (e >> 2) * 8 + (lane >> 5) * 4 + (e & 3), wn * 32 + (lane & 31))] = fmaf(xx[e], SPLIT_LO_INV, hh[e]);
    __syncthreads();
    _Float16* out = (_Float16*)(ws + pb_at(m.off, m.r, m.s));
    const float fb = b * (SB / SA), fc = ldexpf(c * (SB / (SA * SA)), -2 * g_of(ws, m.off, drop));
    PanelSquare::rows(tiles, [&](int, int row, int col, float v[8]) {
        const char* at = rows_i + ((tj * 2 + (col >> 5)) * 64 + row) * CHUNK;
        const int seg = (col & 31) >> 3;
        const half8 ah = *reinterpret_cast<const half8*>(at + ((seg ^ swizzle(row)) << 4)), al = *reinterpret_cast<const half8*>(at + (((seg + 4) ^ swizzle(row)) << 4));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(fb, pair_value(ah[e], al[e]), fc * v[e]);
    }, [&](int row, int col, half8 h, half8 l) { put8(out, at(ti * 64 + row, tj * 64 + col, R), h, l); });
    if (ti == tj) return;
    __syncthreads();
    PanelSquare::columns(tiles, [&](int row, int col, half8 h, half8 l) { put8(out, at(tj * 64 + col, ti * 64 + row, R), h, l); });
}

// ------------------------------------------------------------------------------------------------------------------------------ tiny
// Matrices of at most 32 rows (heads, first layers, everything small in a list): one workgroup does all of it in one launch, in 64 bits.
// All steps are polynomials of the starting Gram matrix S and commute with it: each multiplies by P = a + b S + c S^2 from the left and turns S into
// P S P, so that the last X is the product of the P times the first X.  X is read twice, for S and for the end; the steps run on r x r matrices in
// LDS.  In 32 bits that form loses what matters (an error of S in a weak direction grows with it, to 1e-4 in five steps); in 64 it costs little at
// this size, products of 32-bit numbers are exact in it, and the result is off by its last rounding alone -- where the pairs above would do a little
// worse than 32 bits (X is held to 2^-23, and few terms average).
// v_mfma_f64_16x16x4: lane l holds row l % 16, k = l / 16 of the left operand, column l % 16 of the right one, and rows l / 16 + 4 e of the result.
constexpr int TINY_ROWS = 32, TINY_THREADS = 512, TINY_LD = 33;
// Numbers of a matrix: one workgroup reads them twice, in front of the panels of the list's other matrices (2 x 2: 10 us, 16 x 512 and 32 x 256: 13 and 17
// us, 32 x 640 31 us -- the panels take 13 us a step and any number of matrices).  More of them with 8 rows and less, where pairs would be worse than
// 32 bits (2 x 1152: by a quarter) and a thread a column is quick (4 x 2304: 13 us, in the step 17; 8 x 8000 40, 2 x 60000 85).
constexpr int TINY_FEW = 8;
constexpr long long TINY_NUMBERS = 1 << 13, TINY_NUMBERS_FEW = 1 << 17;
typedef double f64x4 __attribute__((ext_vector_type(4)));
struct TinyTable { bflow_ns_matrix_t m[MOST]; };
struct TinyNumbers {
    double a, b, c, eps;
    int steps, nesterov;
    float mu, lr, decay;
    const float* lr_device;
};

// tile (ti, tj) of X Y, R x R matrices in LDS
template <int R> __device__ __forceinline__ f64x4 tiny_product(const double* x, const double* y, int ti, int tj, int lane) {
    const double* xr = x + (ti * 16 + (lane & 15)) * TINY_LD + (lane >> 4);
    const double* yc = y + (lane >> 4) * TINY_LD + tj * 16 + (lane & 15);
    f64x4 d = {0., 0., 0., 0.}, d2 = {0., 0., 0., 0.};
#pragma unroll
    for (int k = 0; k < R; k += 8) {                    // two chains: the instruction's latency is its length
        d = __builtin_amdgcn_mfma_f64_16x16x4f64(xr[k], yc[k * TINY_LD], d, 0, 0, 0);
        d2 = __builtin_amdgcn_mfma_f64_16x16x4f64(xr[k + 4], yc[(k + 4) * TINY_LD], d2, 0, 0, 0);
    }
    return d + d2;
}

// NV > 0: at most NV rows (4 or 8), whose 16-row tiles would be mostly padding: S and the end by ordinary 64-bit arithmetic, a column a thread.
template <int NT, int NV, int DT, bool STEP>
__device__ __forceinline__ void tiny_body(const bflow_ns_matrix_t& m, const TinyNumbers& nu, double* S, double* room) {
    constexpr int WAVES = TINY_THREADS / 64, SQUARE = TINY_ROWS * TINY_LD, R = NT * 16, AHEAD = 4 / NT;
    double *P = room, *T = room + SQUARE, *Q = room + 2 * SQUARE;
    const bool tall = m.rows > m.cols;
    const int r = tall ? m.cols : m.rows, s = tall ? m.rows : m.cols;
    const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (i, j) of the r x s matrix, zero outside.  No branch around the loads, those outside read the last element inside; and they stand in front of all
    // stores of their batch, so that the whole batch is in flight together.
    struct Raw { float x, v; };
    auto read = [&](int i, int j) -> Raw {
        const int ic = min(i, r - 1), jc = min(j, s - 1), row = tall ? jc : ic, col = tall ? ic : jc;
        const float x = load1<DT>(m.src, (long long)row * m.src_ld + col);
        if constexpr (!STEP) return {x, 0.f};
        else return {x, m.momentum[(long long)row * m.cols + col]};
    };
    auto number = [&](Raw n, int i, int j, bool update) -> float {
        const bool inside = i < r && j < s;
        if constexpr (!STEP) return inside ? n.x : 0.f;
        if (update) {
            n.v = fmaf(nu.mu, n.v, n.x);
            if (inside) m.momentum[tall ? (long long)j * m.cols + i : (long long)i * m.cols + j] = n.v;
        }
        return !inside ? 0.f : nu.nesterov ? fmaf(nu.mu, n.v, n.x) : n.v;
    };
    if constexpr (NV > 0) {
        constexpr int PAIRS = NV * (NV + 1) / 2, TOGETHER = NV == 4 ? 4 : 2;
        double acc[PAIRS];
#pragma unroll
        for (int n = 0; n < PAIRS; ++n) acc[n] = 0;
        for (int j = threadIdx.x; j < s; j += TOGETHER * TINY_THREADS) {
            Raw raw[TOGETHER][NV];
            float x[TOGETHER][NV];
#pragma unroll
            for (int u = 0; u < TOGETHER; ++u)
#pragma unroll
                for (int i = 0; i < NV; ++i) raw[u][i] = read(i, j + u * TINY_THREADS);
#pragma unroll
            for (int u = 0; u < TOGETHER; ++u)
#pragma unroll
                for (int i = 0; i < NV; ++i) x[u][i] = number(raw[u][i], i, j + u * TINY_THREADS, true);
#pragma unroll
            for (int u = 0; u < TOGETHER; ++u)
#pragma unroll
                for (int i = 0, n = 0; i < NV; ++i)
#pragma unroll
                    for (int k = 0; k <= i; ++k, ++n) acc[n] = fma((double)x[u][i], (double)x[u][k], acc[n]);
        }
#pragma unroll
        for (int n = 0; n < PAIRS; ++n) {
            const double v = wave_sum(acc[n]);
            if (lane == 0) room[w * PAIRS + n] = v;
        }
        for (int i = threadIdx.x; i < R * R; i += TINY_THREADS) S[(i / R) * TINY_LD + i % R] = 0;
        __syncthreads();
        if (threadIdx.x < PAIRS) {
            int i = 0, n = threadIdx.x;
            while (n > i) n -= ++i;                     // (0, 0), (1, 0), (1, 1), ...
            double sum = 0;
#pragma unroll
            for (int k = 0; k < WAVES; ++k) sum += room[k * PAIRS + threadIdx.x];
            S[i * TINY_LD + n] = sum;
            S[n * TINY_LD + i] = sum;
        }
    } else {
        // S = X X^T, before the norm is known; AHEAD blocks of 16 columns are read together
        f64x4 acc[3] = {{0., 0., 0., 0.}, {0., 0., 0., 0.}, {0., 0., 0., 0.}};
        for (int c0 = w * 16; c0 < s; c0 += AHEAD * WAVES * 16) {
            Raw raw[AHEAD][NT][4];
            float x[AHEAD][NT][4];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) raw[u][n][e] = read(n * 16 + l15, c0 + u * WAVES * 16 + g * 4 + e);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[u][n][e] = number(raw[u][n][e], n * 16 + l15, c0 + u * WAVES * 16 + g * 4 + e, true);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double x0 = x[u][0][e], x1 = x[u][NT - 1][e];
                    acc[0] = __builtin_amdgcn_mfma_f64_16x16x4f64(x0, x0, acc[0], 0, 0, 0);
                    if (NT == 2) {
                        acc[1] = __builtin_amdgcn_mfma_f64_16x16x4f64(x1, x0, acc[1], 0, 0, 0);
                        acc[2] = __builtin_amdgcn_mfma_f64_16x16x4f64(x1, x1, acc[2], 0, 0, 0);
                    }
                }
        }
#pragma unroll
        for (int n = 0; n < 2 * NT - 1; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) room[(w * 3 + n) * 256 + (g + 4 * e) * 16 + l15] = acc[n][e];
        __syncthreads();
        for (int i = threadIdx.x; i < (2 * NT - 1) * 256; i += TINY_THREADS) {
            double sum = 0;
#pragma unroll
            for (int k = 0; k < WAVES; ++k) sum += room[k * 768 + i];
            const int n = i >> 8, row = ((i >> 4) & 15) + (n > 0 ? 16 : 0), col = (i & 15) + (n == 2 ? 16 : 0);
            S[row * TINY_LD + col] = sum;
            if (n == 1) S[col * TINY_LD + row] = sum;
        }
    }
    __syncthreads();
    double trace = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) trace += S[i * TINY_LD + i];
    const double scale = 1. / (sqrt(trace) + nu.eps);
    __syncthreads();
    for (int i = threadIdx.x; i < R * R; i += TINY_THREADS) {
        double& v = S[(i / R) * TINY_LD + i % R];
        v = v * scale * scale;                          // (the square of 1 / eps may be infinite)
    }
    __syncthreads();
    // four waves make P Q, four P S and then P S P
    const int tile = w & 3, ti = tile >> (NT - 1), tj = tile & (NT - 1);
    const bool on = tile < NT * NT, left = w < 4;
    const int at = (ti * 16 + g) * TINY_LD + tj * 16 + l15;     // of number e: 4 e rows further
    for (int k = 0; k < nu.steps; ++k) {
        if (left && on) {
            const f64x4 d = tiny_product<R>(S, S, ti, tj, lane);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                P[at + 4 * e * TINY_LD] = (ti == tj && g + 4 * e == l15 ? nu.a : 0.) + nu.b * S[at + 4 * e * TINY_LD] + nu.c * d[e];
        }
        __syncthreads();
        f64x4 d = {0., 0., 0., 0.};
        if (on && !(left && k == 0)) d = tiny_product<R>(P, left ? Q : S, ti, tj, lane);
        if (!left && on)
#pragma unroll
            for (int e = 0; e < 4; ++e) T[at + 4 * e * TINY_LD] = d[e];
        __syncthreads();
        if (left && on)
#pragma unroll
            for (int e = 0; e < 4; ++e) Q[at + 4 * e * TINY_LD] = k == 0 ? P[at + 4 * e * TINY_LD] : d[e];
        if (!left && on) {
            d = tiny_product<R>(T, P, ti, tj, lane);
#pragma unroll
            for (int e = 0; e < 4; ++e) S[at + 4 * e * TINY_LD] = d[e];      // (S was last read in front of the barrier)
        }
        __syncthreads();
    }
    // the last X
    const float lr = STEP ? (nu.lr_device ? *nu.lr_device : nu.lr) : 0.f, shrink = lr * nu.decay, rate = lr * 0.2f * sqrtf((float)s);
    if constexpr (NV > 0) {
        constexpr int TOGETHER = NV == 4 ? 4 : 2;
        for (int j0 = threadIdx.x; j0 < s; j0 += TOGETHER * TINY_THREADS) {
            Raw raw[TOGETHER][NV];
            float old[TOGETHER][NV];
            auto place = [&](int i, int j) { return tall ? (long long)j * m.dst_ld + i : (long long)i * m.dst_ld + j; };
#pragma unroll
            for (int u = 0; u < TOGETHER; ++u)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int j = j0 + u * TINY_THREADS;
                    raw[u][i] = read(i, j);
                    if constexpr (STEP) old[u][i] = ((const float*)m.dst)[place(min(i, r - 1), min(j, s - 1))];
                }
#pragma unroll
            for (int u = 0; u < TOGETHER; ++u) {
                const int j = j0 + u * TINY_THREADS;
                double x[NV];
#pragma unroll
                for (int i = 0; i < NV; ++i) x[i] = number(raw[u][i], i, j, false);
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    double d = 0;
#pragma unroll
                    for (int k = 0; k < NV; ++k) d = fma(Q[i * TINY_LD + k], x[k], d);
                    if (i >= r || j >= s) continue;
                    const float v = (float)(d * scale);
                    if constexpr (STEP) ((float*)m.dst)[place(i, j)] = stepped(old[u][i], v, rate, shrink);
                    else store1<DT>(m.dst, place(i, j), v);
                }
            }
        }
    } else {
        double q[NT][R / 4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < R / 4; ++k) q[n][k] = Q[(n * 16 + l15) * TINY_LD + 4 * k + g] * scale;
        for (int c0 = w * 16; c0 < s; c0 += AHEAD * WAVES * 16) {
            float x[AHEAD][R / 4];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int k = 0; k < R / 4; ++k) x[u][k] = number(read(4 * k + g, c0 + u * WAVES * 16 + l15), 4 * k + g, c0 + u * WAVES * 16 + l15, false);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int j = c0 + u * WAVES * 16 + l15;
                f64x4 d[NT];
                float old[NT][4];
                long long to[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    d[n] = f64x4{0., 0., 0., 0.};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = n * 16 + g + 4 * e;
                        to[n][e] = i >= r || j >= s ? -1 : tall ? (long long)j * m.dst_ld + i : (long long)i * m.dst_ld + j;
                        if constexpr (STEP) old[n][e] = ((const float*)m.dst)[max(to[n][e], 0LL)];
                    }
                }
#pragma unroll
                for (int k = 0; k < R / 4; ++k)
#pragma unroll
                    for (int n = 0; n < NT; ++n) d[n] = __builtin_amdgcn_mfma_f64_16x16x4f64(q[n][k], (double)x[u][k], d[n], 0, 0, 0);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (to[n][e] >= 0) {
                            const float v = (float)d[n][e];
                            if constexpr (STEP) ((float*)m.dst)[to[n][e]] = stepped(old[n][e], v, rate, shrink);
                            else store1<DT>(m.dst, to[n][e], v);
                        }
            }
        }
    }
}

template <int DT, bool STEP>
__global__ __launch_bounds__(TINY_THREADS) void ns_tiny_kernel(TinyTable t, TinyNumbers nu) {
    __shared__ double S[TINY_ROWS * TINY_LD];
    __shared__ double room[TINY_THREADS / 64 * 3 * 256];      // the waves' parts of S; then P, T and Q
    static_assert(3 * TINY_ROWS * TINY_LD <= TINY_THREADS / 64 * 3 * 256, "three matrices fit the parts");
    const bflow_ns_matrix_t m = t.m[blockIdx.x];
    const int r = min(m.rows, m.cols);
    if (r <= 4) tiny_body<1, 4, DT, STEP>(m, nu, S, room);
    else if (r <= 8) tiny_body<1, 8, DT, STEP>(m, nu, S, room);
    else if (r <= 16) tiny_body<1, 0, DT, STEP>(m, nu, S, room);
    else tiny_body<2, 0, DT, STEP>(m, nu, S, room);
}

// ------------------------------------------------------------------------------------------------------------------------------ host
// Two sets of tiles.  Small: the filters of a network; few tiles, so four groups of waves share a contraction.  Large: many.
struct SmallSet {
    typedef Product<64, 64, 32, 32, 4, 2> Square;      // A and B
    typedef Product<64, 128, 32, 32, 1, 3> Panel;      // X
};
struct LargeSet {
    typedef Product<128, 128, 64, 64, 2, 2> Square;    // (a CU alone)
    typedef Product<128, 128, 64, 64, 1, 2> Panel;
};

// Tiles of a square product that are not cut; parts of those behind them (0: none); whether they are dispatched from the last one on.
struct Cut { int whole, parts, first; };

struct Plan {
    Works square, panel;
    Entries norm, pack;
    Exits leave;
    long long tiles_square, tiles_panel, tiles_sum, tiles_norm, tiles_pack, bytes;
    bool large;
    Cut gram, poly;
    long long room;        // where the parts of cut tiles stand
    bool panels;           // every matrix of at most PANEL_ROWS rows: `works` instead of `square` and `panel`
    PanelWorks works;
    int lds_panel, lds_square;
};

template <class Set> void lay_out_products(Plan& p) {
    for (int i = 0; i < p.square.count; ++i) {
        const int r = p.square.m[i].r, s = p.square.m[i].s, R = up64(r), S = up64(s);
        p.square.m[i].tile0 = (int)p.tiles_square;
        p.panel.m[i] = p.square.m[i];
        p.panel.m[i].tile0 = p.leave.m[i].tile0 = (int)p.tiles_panel;
        p.tiles_square += lower_tiles<typename Set::Square>(R);
        p.tiles_panel += (long long)((R + Set::Panel::BM - 1) / Set::Panel::BM) * ((S + Set::Panel::BN - 1) / Set::Panel::BN);
    }
}

// Loads of the CUs as pieces of work are dealt out in order, each to the least loaded: CUs of one load stand together.
constexpr int CUS = 256;
struct Loads {
    struct { double load; long long cus; } at[2 * MOST + 8];
    int count = 1;
    double most = 0;
    Loads() { at[0] = {0, CUS}; }
    void deal(double length, long long pieces) {
        while (pieces > 0) {
            const double load = at[0].load + length;
            const long long n = pieces < at[0].cus ? pieces : at[0].cus;
            pieces -= n;
            if (n == at[0].cus) {
                for (int i = 1; i < count; ++i) at[i - 1] = at[i];
                --count;
            } else {
                at[0].cus -= n;
            }
            int i = count;
            while (i > 0 && at[i - 1].load > load) --i;
            if (i > 0 && at[i - 1].load == load) {
                at[i - 1].cus += n;
            } else {
                for (int j = count; j > i; --j) at[j] = at[j - 1];
                at[i] = {load, n};
                ++count;
            }
            most = std::max(most, load);
        }
    }
};

// Which tiles of a product of the large set are cut, by the time that the dealing gives, in rounds (1.3 us): a whole tile
// takes 3 more and a part 2, the join 4, and writing and reading a part a 40th.  Either the
// last tiles that would leave most CUs idle, as many parts as there are CUs for them, or all tiles of the list's longest matrices (they stand last) in two
// to four parts; a part has eight rounds or so (CUT_COLUMNS) at least.  Calls without and with it: 2944 x 2944 in fp32 2255 / 1985 us,
// 4096 x 4096 4495 / 4075, 8 of 1024 x 1024 892 / 856, a step of 4 of 1024 x 1024 and 2 of 1024 x 4096 1073 / 1004; 2048 x 2048 whole 790,
// in three parts 829.  (256 columns at least: 24 of 640 x 640 893 / 937; 1024: 2944 x 2944 2079.)
constexpr int CUT_COLUMNS = 512;
constexpr long long CUT_PIECES = 1024;
template <int WHAT> Cut plan_cut(const Works& w) {
    typedef LargeSet::Square Q;
    const auto columns = [&](int i) { return up64(WHAT == GRAM ? w.m[i].s : w.m[i].r); };
    const auto tiles = [&](int i) { return (long long)lower_tiles<Q>(up64(w.m[i].r)); };
    long long total = 0;
    for (int i = 0; i < w.count; ++i) total += tiles(i);
    const auto time = [&](long long whole, int parts) {      // the last matrix' tiles start first
        Loads loads;
        long long left = total - whole, skip = left;
        for (int i = w.count - 1; i >= 0 && left > 0; --i) {
            const long long n = std::min(left, tiles(i));
            loads.deal((double)Q::rounds_of(columns(i)) / parts + 2, n * parts);
            left -= n;
        }
        for (int i = w.count - 1; i >= 0; --i) {
            const long long n = std::min(skip, tiles(i));
            skip -= n;
            loads.deal(Q::rounds_of(columns(i)) + 3, tiles(i) - n);
        }
        return loads.most + (whole < total ? 4 + (double)(total - whole) * parts / 40 : 0);
    };
    const auto most_parts = [&](long long whole) {           // by the shortest of the cut tiles, to the nearest 128 columns upwards
        int shortest = 1 << 30;
        long long seen = total;
        for (int i = w.count - 1; i >= 0 && seen > whole; --i) {
            shortest = std::min(shortest, columns(i));
            seen -= tiles(i);
        }
        return (shortest + 64) / CUT_COLUMNS;
    };
    // Lengths that differ start with the longest, which stand last.  The last tiles of many alike come last: in front they would end the common walk of the
    // others (4096 x 4096 4.08 -> 4.12 ms).
    const int differ = columns(0) != columns(w.count - 1);
    Cut best = {(int)total, 0, differ};
    double least = time(total, 1);
    const auto consider = [&](long long whole, int parts, int first) {
        if (parts < 2 || whole >= total || (total - whole) * parts > CUT_PIECES || parts > most_parts(whole)) return;
        const double t = time(whole, parts);
        if (t < least) { least = t; best = {(int)whole, parts, first}; }
    };
    const long long last = total % CUS;
    if (total > CUS && last) consider(total - last, (int)std::min<long long>(CUS / last, most_parts(total - last)), 0);
    long long whole = total;
    int borders = 0;
    for (int i = w.count - 1; i >= 0 && borders < 4; --i) {
        whole -= tiles(i);
        if (i > 0 && columns(i - 1) == columns(i)) continue;
        ++borders;
        for (int parts = 2; parts <= 4; ++parts) consider(whole, parts, 1);
    }
    return best;
}

// Panels of a workgroup.  A panel takes COST microseconds by its rows; the workgroups of a list (one for each CU at most, where that can be) should take
// the same time, the least that does it.
constexpr int PANEL_WGS = 256;
constexpr double PANEL_COST[5] = {0, 2, 3.5, 7, 14};
constexpr double PART_COST = 0.35;     // of adding a part where B is made, for each 64 rows; a launch that adds them costs 4 us
void lay_out_panels(Plan& p) {
    const int count = p.works.count;
    auto per_of = [&](int i, double time) {
        const double n = time / PANEL_COST[up64(p.works.m[i].r) / 64];
        const int panels = panels_of(p.works.m[i].s);
        return n < 1 ? 1 : n > panels ? panels : (int)n;
    };
    double time = 2;
    for (;; time *= 1.1) {
        long long wgs = 0;
        bool one = true;                 // a matrix in one piece each: no fewer workgroups to be had
        for (int i = 0; i < count; ++i) {
            const int panels = panels_of(p.works.m[i].s), per = per_of(i, time);
            wgs += (panels + per - 1) / per;
            one = one && per == panels;
        }
        if (wgs <= PANEL_WGS || one) break;
    }
    long long wgs = 0, squares = 0, sums = 0, off = 0;
    double adding = 0;
    p.lds_panel = p.lds_square = 0;
    for (int i = 0; i < count; ++i) {
        PanelWork& m = p.works.m[i];
        const int R = up64(m.r), panels = panels_of(m.s), lds = R == 64 ? PanelSize<1>::LDS : R == 128 ? PanelSize<2>::LDS : R == 192 ? PanelSize<3>::LDS : PanelSize<4>::LDS;
        m.per = per_of(i, time);
        const long long slices = (panels + m.per - 1) / m.per;
        m.off = p.norm.m[i].off = p.pack.m[i].off = p.leave.m[i].off = off;
        m.wg0 = (int)wgs;
        m.square0 = (int)squares;
        m.sum0 = (int)sums;
        wgs += slices;
        squares += (long long)(R / 64) * (R / 64 + 1) / 2;
        sums += part_size(R) / 1024;
        adding = std::max(adding, PART_COST * slices * R / 64);
        off = (parts_at(off, m.r, m.s) + slices * part_size(R) * 4 + 255) & ~255LL;
        p.lds_panel = lds > p.lds_panel ? lds : p.lds_panel;
        p.lds_square = panel_square_lds(R) > p.lds_square ? panel_square_lds(R) : p.lds_square;
    }
    p.tiles_panel = wgs;
    p.tiles_square = squares;
    p.tiles_sum = adding > 4 ? sums : 0;
    p.bytes = off;
}

// The launches of one group of matrices; returns false where a count passes what a grid holds.
bool lay_out(const bflow_ns_matrix_t* given, int count, Plan& p) {
    long long off = 0, blocks = 0;
    bflow_ns_matrix_t m[MOST];
    std::copy(given, given + count, m);
    const auto shorter = [](const bflow_ns_matrix_t& a, const bflow_ns_matrix_t& b) { return std::max(a.rows, a.cols) < std::max(b.rows, b.cols); };
    for (int i = 1; i < count; ++i)                     // the longest contractions last
        for (int j = i; j > 0 && shorter(m[j], m[j - 1]); --j) std::swap(m[j], m[j - 1]);
    p.tiles_square = p.tiles_panel = p.tiles_norm = p.tiles_pack = 0;
    p.square.count = p.panel.count = p.norm.count = p.pack.count = p.leave.count = count;
    for (int i = 0; i < count; ++i) {
        const int tall = m[i].rows > m[i].cols;
        const int r = tall ? m[i].cols : m[i].rows, s = tall ? m[i].rows : m[i].cols;
        const long long T = up64(r) / 64, U = up64(s) / 64, n = (long long)r * s;
        long long per = (n + NORM_PARTS - 1) / NORM_PARTS;
        per = per < NORM_MIN ? NORM_MIN : per;
        p.square.m[i] = {off, r, s, 0, x_exponent(r, s)};
        p.norm.m[i] = {m[i].src, m[i].momentum, m[i].src_ld, off, r, s, (int)p.tiles_norm, (int)per, tall, x_exponent(r, s)};
        p.pack.m[i] = p.norm.m[i];
        p.pack.m[i].tile0 = (int)p.tiles_pack;
        p.leave.m[i] = {m[i].dst, m[i].dst_ld, off, r, s, 0, tall, 0.2f * sqrtf((float)s), x_exponent(r, s)};
        blocks += T * (T + 1) / 2;
        p.tiles_norm += (n + per - 1) / per;
        p.tiles_pack += T * U;
        off = (end_at(off, r, s) + 255) & ~255LL;
    }
    p.panels = true;
    p.works.count = count;
    for (int i = 0; i < count; ++i) {
        p.panels = p.panels && p.square.m[i].r <= PANEL_ROWS;
        if (p.panels) p.works.m[i] = {0, (short)p.square.m[i].r, (short)p.square.m[i].ex, p.square.m[i].s, 0, 0, 0, 1};
    }
    if (p.panels) {
        lay_out_panels(p);
        return p.tiles_pack < (1LL << 30);
    }
    // One 1024 x 1024 (136 blocks): 261 us in small tiles, 452 in large ones; 8 of 512 x 512 (288): 304 / 329; 2048 x 2048 (528): 958 / 800;
    // 12 of 640 x 640 (660): 615 / 504; 8192 x 8192: 47.5 / 33.3 ms.
    p.large = blocks >= LARGE_BLOCKS;
    if (p.large) lay_out_products<LargeSet>(p);
    else lay_out_products<SmallSet>(p);
    p.gram = p.poly = {(int)p.tiles_square, 0, 0};
    p.room = off;
    if (p.large) {
        p.gram = plan_cut<GRAM>(p.square);
        p.poly = plan_cut<POLY>(p.square);
        const long long most = std::max((p.tiles_square - p.gram.whole) * p.gram.parts, (p.tiles_square - p.poly.whole) * p.poly.parts);
        off += most * LargeSet::Square::TILE;
    }
    p.bytes = off;
    return p.tiles_pack < (1LL << 30);
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
    static thread_local struct { int steps; double a, b, c, most, gain; } last = {0, 0, 0, 0, 0, 0};     // 20000 polynomials: once for a user's coefficients
    if (last.steps == steps && last.a == a && last.b == b && last.c == c) {
        *gain = last.gain;
        return last.most;
    }
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
    last = {steps, a, b, c, most, *gain};
    return most;
}

template <class K> int allow_lds(K kernel, int bytes) {
    if (bytes <= 65536) return 0;
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    BFLOW_REQUIRE(e == hipSuccess, (int)e, "newton_schulz: %s", hipGetErrorString(e));
    return 0;
}

template <class Set, int DT, bool STEP>
int launch_products(const Plan& p, int steps, float a, float b, float c, double gain, char* ws, float lr, const float* lr_device, float decay, hipStream_t st) {
    typedef typename Set::Square Q;
    typedef typename Set::Panel P;
    const auto gram = ns_gram_kernel<Q>;
    const auto poly = ns_poly_kernel<Q>;
    const auto apply = ns_apply_kernel<P>;
    const auto leave = ns_leave_kernel<P, DT, STEP>;
    for (const int rc : {allow_lds(gram, Q::LDS), allow_lds(poly, Q::LDS), allow_lds(apply, P::LDS), allow_lds(leave, P::LDS)})
        if (rc) return rc;
    const auto tail = [&](Cut c) { return Tail{c.whole, c.parts, c.first, (float*)(ws + p.room)}; };
    const auto cut = [&](Cut c) { return (int)p.tiles_square - c.whole; };
    const auto grid = [&](Cut c) { return dim3(c.whole + cut(c) * c.parts); };
    const auto joins = [&](Cut c) { return dim3(cut(c) * (Q::BM / 64) * (Q::BN / 64)); };
    const double bits = log2(gain);
    for (int k = 0; k < steps; ++k) {
        const int drop = (int)std::ceil(k * bits), next = (int)std::ceil((k + 1) * bits);
        hipLaunchKernelGGL(gram, grid(p.gram), dim3(Q::THREADS), Q::LDS, st, p.square, tail(p.gram), ws);
        if constexpr (std::is_same_v<Set, LargeSet>)
            if (cut(p.gram)) hipLaunchKernelGGL((ns_join_kernel<Q, GRAM>), joins(p.gram), dim3(256), 64 * 64 * 4, st, p.square, tail(p.gram), ws, b, c, drop);
        hipLaunchKernelGGL(poly, grid(p.poly), dim3(Q::THREADS), Q::LDS, st, p.square, tail(p.poly), ws, b, c, drop);
        if constexpr (std::is_same_v<Set, LargeSet>)
            if (cut(p.poly)) hipLaunchKernelGGL((ns_join_kernel<Q, POLY>), joins(p.poly), dim3(256), 64 * 64 * 4, st, p.square, tail(p.poly), ws, b, c, drop);
        if (k + 1 < steps) hipLaunchKernelGGL(apply, dim3(p.tiles_panel), dim3(P::THREADS), P::LDS, st, p.panel, ws, k & 1, a, drop, next);
        else hipLaunchKernelGGL(leave, dim3(p.tiles_panel), dim3(P::THREADS), P::LDS, st, p.leave, ws, k & 1, a, drop, lr, lr_device, decay);
    }
    return launch_status("newton_schulz");
}

template <int DT, bool STEP>
int launch_panels(const Plan& p, int steps, float a, float b, float c, double gain, char* ws, float lr, const float* lr_device, float decay, hipStream_t st) {
    const auto last = ns_panel_last_kernel<DT, STEP>;
    for (const int rc : {allow_lds(ns_panel_first_kernel, p.lds_panel), allow_lds(ns_panel_middle_kernel, p.lds_panel), allow_lds(last, p.lds_panel), allow_lds(ns_panel_square_kernel<true>, p.lds_square),
                         allow_lds(ns_panel_square_kernel<false>, p.lds_square)})
        if (rc) return rc;
    const double bits = log2(gain);
    PanelExits exits;
    for (int i = 0; i < p.works.count; ++i) exits.m[i] = {p.leave.m[i].dst, p.leave.m[i].ld, p.leave.m[i].size, p.leave.m[i].tall};
    const dim3 grid(p.tiles_panel), block(PANEL_THREADS);
    hipLaunchKernelGGL(ns_panel_first_kernel, grid, block, p.lds_panel, st, p.works, ws);
    for (int k = 0; k < steps; ++k) {
        const Numbers nu = {(int)std::ceil(k * bits), (int)std::ceil((k + 1) * bits), a, lr, lr_device, decay};
        if (p.tiles_sum) hipLaunchKernelGGL(ns_panel_sum_kernel, dim3(p.tiles_sum), dim3(256), 0, st, p.works, ws);
        const auto square = p.tiles_sum ? ns_panel_square_kernel<true> : ns_panel_square_kernel<false>;
        hipLaunchKernelGGL(square, dim3(p.tiles_square), block, p.lds_square, st, p.works, ws, b, c, nu.drop);
        if (k + 1 < steps) hipLaunchKernelGGL(ns_panel_middle_kernel, grid, block, p.lds_panel, st, p.works, ws, nu);
        else hipLaunchKernelGGL(last, grid, block, p.lds_panel, st, p.works, exits, ws, nu);
    }
    return launch_status("newton_schulz");
}

template <int DT, bool STEP>
int launch_all(const Plan& p, int steps, float a, float b, float c, double eps, double gain, char* ws, float mu, int nesterov, float lr, const float* lr_device, float decay,
               hipStream_t st) {
    hipLaunchKernelGGL((ns_norm_kernel<DT, STEP>), dim3(p.tiles_norm), dim3(256), 0, st, p.norm, ws, mu, nesterov);
    hipLaunchKernelGGL((ns_pack_kernel<DT, STEP>), dim3(p.tiles_pack), dim3(256), 0, st, p.pack, ws, mu, nesterov, eps, (int)!p.panels);
    if (p.panels) return launch_panels<DT, STEP>(p, steps, a, b, c, gain, ws, lr, lr_device, decay, st);
    return (p.large ? launch_products<LargeSet, DT, STEP> : launch_products<SmallSet, DT, STEP>)(p, steps, a, b, c, gain, ws, lr, lr_device, decay, st);
}

int check(const bflow_ns_matrix_t* m, int count, int steps, double a, double b, double c, double eps, const void* ws, long long ws_bytes, bool step, double* gain) {
    const char* why = bad(m, count);
    BFLOW_REQUIRE(!why, BFLOW_E_ARG, "newton_schulz: %s", why);
    BFLOW_REQUIRE(steps >= 1 && steps <= 32, BFLOW_E_ARG, "newton_schulz: %d steps (1 .. 32)", steps);
    BFLOW_REQUIRE(eps >= 1e-300 && eps < 1, BFLOW_E_ARG, "newton_schulz: eps %g outside [1e-300, 1)", eps);
    const double most = reach(steps, a, b, c, gain);
    BFLOW_REQUIRE(most <= 1.9 && std::fabs(b) * 4 + std::fabs(c) * 16 < 63, BFLOW_E_ARG,
                  "newton_schulz: coefficients (%g, %g, %g) take a singular value in [0, 1] to %g: the iterates must stay below 1.9", a, b, c, most);
    const long long need = bflow_ns_workspace_bytes(m, count);
    BFLOW_REQUIRE(need <= 0 || (ws && ((uintptr_t)ws & 255) == 0), BFLOW_E_ARG, "newton_schulz: workspace null or not aligned to 256 bytes");
    BFLOW_REQUIRE(need >= 0 && ws_bytes >= need, BFLOW_E_ARG, "newton_schulz: workspace of %lld bytes, %lld needed", ws_bytes, need);
    for (int i = 0; i < count; ++i)
        BFLOW_REQUIRE(m[i].src && m[i].dst && m[i].src_ld >= m[i].cols && m[i].dst_ld >= m[i].cols && (!step || m[i].momentum), BFLOW_E_ARG,
                      "newton_schulz: matrix %d: null pointer or a row shorter than its columns", i);
    return 0;
}
bool tiny(const bflow_ns_matrix_t& m) {
    const int r = m.rows < m.cols ? m.rows : m.cols;
    return r <= TINY_ROWS && (long long)m.rows * m.cols <= (r <= TINY_FEW ? TINY_NUMBERS_FEW : TINY_NUMBERS);
}

// f(group, n) for the matrices of a list that are tiny, or those that are not, MOST at a time.  f returns a status.
template <class F> long long for_groups(const bflow_ns_matrix_t* m, int count, bool want_tiny, F f) {
    bflow_ns_matrix_t group[MOST];
    int n = 0;
    for (int i = 0; i < count; ++i) {
        if (tiny(m[i]) == want_tiny) group[n++] = m[i];
        if (n == MOST || (i + 1 == count && n)) {
            if (const long long rc = f(group, n)) return rc;
            n = 0;
        }
    }
    return 0;
}

template <int DT, bool STEP>
int launch_list(const bflow_ns_matrix_t* m, int count, int steps, double a, double b, double c, double eps, double gain, char* ws, float mu, int nesterov, float lr,
                const float* lr_device, float decay, hipStream_t st) {
    long long rc = for_groups(m, count, true, [&](const bflow_ns_matrix_t* group, int n) -> long long {
        TinyTable t = {};
        for (int i = 0; i < n; ++i) t.m[i] = group[i];
        hipLaunchKernelGGL((ns_tiny_kernel<DT, STEP>), dim3(n), dim3(TINY_THREADS), 0, st, t, TinyNumbers{a, b, c, eps, steps, nesterov, mu, lr, decay, lr_device});
        return launch_status("newton_schulz");
    });
    if (rc) return (int)rc;
    return (int)for_groups(m, count, false, [&](const bflow_ns_matrix_t* group, int n) -> long long {
        static thread_local Plan p;
        lay_out(group, n, p);
        return launch_all<DT, STEP>(p, steps, (float)a, (float)b, (float)c, eps, gain, ws, mu, nesterov, lr, lr_device, decay, st);
    });
}
}  // namespace

extern "C" long long bflow_ns_workspace_bytes(const bflow_ns_matrix_t* m, int count) {
    if (const char* why = bad(m, count)) {
        set_error("newton_schulz: %s", why);
        return BFLOW_E_ARG;
    }
    long long most = 0;
    const long long rc = for_groups(m, count, false, [&](const bflow_ns_matrix_t* group, int n) -> long long {
        static thread_local Plan p;
        if (!lay_out(group, n, p)) {
            set_error("newton_schulz: too many tiles");
            return BFLOW_E_LIMIT;
        }
        most = p.bytes > most ? p.bytes : most;
        return 0;
    });
    return rc ? rc : most;
}

extern "C" int bflow_ns_orthogonalize(const bflow_ns_matrix_t* m, int count, int dtype, int steps, double a, double b, double c, double eps, void* ws,
                                      long long ws_bytes, bflow_stream_t stream) {
    BFLOW_REQUIRE(dtype >= F32 && dtype <= BF16, BFLOW_E_ARG, "ns_orthogonalize: dtype %d", dtype);
    double gain;
    if (const int rc = check(m, count, steps, a, b, c, eps, ws, ws_bytes, false, &gain)) return rc;
    const auto go = dtype == F32 ? launch_list<F32, false> : dtype == F16 ? launch_list<F16, false> : launch_list<BF16, false>;
    return go(m, count, steps, a, b, c, eps, gain, (char*)ws, 0.f, 0, 0.f, nullptr, 0.f, (hipStream_t)stream);
}

extern "C" int bflow_muon_step(const bflow_ns_matrix_t* m, int count, int steps, double a, double b, double c, double eps, float momentum, int nesterov,
                               float lr, const float* lr_device, float weight_decay, void* ws, long long ws_bytes, bflow_stream_t stream) {
    double gain;
    if (const int rc = check(m, count, steps, a, b, c, eps, ws, ws_bytes, true, &gain)) return rc;
    return launch_list<F32, true>(m, count, steps, a, b, c, eps, gain, (char*)ws, momentum, nesterov, lr, lr_device, weight_decay, (hipStream_t)stream);
}
