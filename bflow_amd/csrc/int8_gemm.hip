// Rows of 8-bit integers against rows of 8-bit integers, with a scale for each row of either side, and the quantisation in front of it
// (gfx950 only).
//
//   out[i][j] = (alpha * sa[i]) * sb[j] * sum_k a[i][k] b[j][k]      sums exact in 32-bit integers (k < 2^17), then 32-bit floating point
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
    int wide;               // the output's rows start at multiples of 16 bytes
};

// sum (alpha scale_a) scale_b, rounded to 32 bits before it is rounded to 16: left to itself the compiler joins the last product and the rounding to fp16
// into one instruction in some kernels, and a row's bits would depend on which one takes it.
template <class T> __device__ __forceinline__ T scaled(int sum, float sa, float sb) {
    float v = (float)sum * sa * sb;
    if constexpr (sizeof(T) == 2) asm("" : "+v"(v));
    return (T)v;
}

// bytes k .. k + 15 of a fragment: those at or behind K become zero
__device__ __forceinline__ i32x4 cut(i32x4 v, int k, int K) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const int left = K - k - 4 * d;
        v[d] &= left >= 4 ? -1 : left <= 0 ? 0 : (1 << (8 * left)) - 1;
    }
    return v;
}

// BM x BN tile; wave (wm, wn) keeps WM x WN of it.  8192^3 in 256 x 256 tiles, many calls in a row: 475 us, 2.32 POP/s (the library's 8-bit product, to 32-bit
// integers without scales, in turn with it: 452); single calls on a rested card 516 (483).  Matrix cores busy 60 % of the cycles at a clock that power
// holds down.
template <int BM, int BN, int WM, int WN>
struct ByteTile {
    static constexpr int M = BM, N = BN, ACROSS = BN / WN, WAVES = (BM / WM) * ACROSS, THREADS = 64 * WAVES, MT = WM / 32, NT = WN / 32;
    static constexpr int STAGE = (BM + BN) * CHUNK, LDS = 2 * STAGE;
    static_assert(BM / 8 % WAVES == 0 && BN / 8 % WAVES == 0 && WAVES % 2 == 0, "whole pieces of either operand for every wave, all odd or all even");
    // B is the instruction's first operand: lane l then holds row l % 32 of a 32 x 32 block, four neighbouring columns in neighbouring registers
    i32x16 acc[MT][NT];

    static constexpr int PA = BM / 8 / WAVES, PB = BN / 8 / WAVES;
    __device__ __forceinline__ void issue(rsrc_t a, const int (&va)[PA], rsrc_t b, const int (&vb)[PB], int chunk, char* stage, int wave) {
#pragma unroll
        for (int i = 0; i < PA; ++i) dma_piece(a, stage + (wave + i * WAVES) * 1024, va[i], chunk * CHUNK);
#pragma unroll
        for (int i = 0; i < PB; ++i) dma_piece(b, stage + BM * CHUNK + (wave + i * WAVES) * 1024, vb[i], chunk * CHUNK);
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
                for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bv[j], av[i], acc[i][j], 0, 0, 0);
        }
    }
    __device__ __forceinline__ void run(rsrc_t a, int lda, rsrc_t b, int ldb, int K, char* lds) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wm = wave / ACROSS, wn = wave % ACROSS;
        const int chunks = (K + CHUNK - 1) / CHUNK;
        int va[PA], vb[PB];
#pragma unroll
        for (int i = 0; i < PA; ++i) va[i] = lane_offset(lane, lda, wave) + (wave + i * WAVES) * 8 * lda;
#pragma unroll
        for (int i = 0; i < PB; ++i) vb[i] = lane_offset(lane, ldb, wave) + (wave + i * WAVES) * 8 * ldb;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int k = 0; k < 16; ++k) acc[i][j][k] = 0;
        issue(a, va, b, vb, 0, lds, wave);
        wait_chunk();
        __builtin_amdgcn_s_barrier();
        const char *as = lds + wm * WM * CHUNK, *bs = lds + (BM + wn * WN) * CHUNK;
        const int whole = K / CHUNK;
        for (int c = 0; c < whole; ++c) {
            if (c + 1 < chunks) issue(a, va, b, vb, c + 1, lds + ((c + 1) & 1) * STAGE, wave);
            multiply<false>(as + (c & 1) * STAGE, bs + (c & 1) * STAGE, lane, 0, 0);
            wait_chunk();
            __builtin_amdgcn_s_barrier();
        }
        if (whole < chunks) {
            multiply<true>(as + (whole & 1) * STAGE, bs + (whole & 1) * STAGE, lane, whole * CHUNK, K);
            wait_chunk();
            __builtin_amdgcn_s_barrier();
        }
    }
};

// Workgroup -> tile.  Workgroups go round the 8 XCDs, each with an L2 of its own: XCD x takes the x-th eighth of the tiles in an order that walks
// bands of GROUP tile rows column by column, so that the tiles an XCD works on at one time share their rows of A and B.
constexpr int GROUP = 8;
__device__ __forceinline__ void place(int id, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int total = tiles_m * tiles_n, q = total >> 3, r = total & 7, x = id & 7;
    const int at = x * q + min(x, r) + (id >> 3);
    const int band = at / (GROUP * tiles_n), in = at - band * GROUP * tiles_n, high = min(GROUP, tiles_m - band * GROUP);
    tn = in / high;
    tm = band * GROUP + in - tn * high;
}

template <class Tile, int DT>
__global__ __launch_bounds__(Tile::THREADS, 2) void i8_gemm_kernel(GemmArgs g) {
    typedef typename OutT<DT>::T T;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int z = blockIdx.y, z0 = z / g.n1, z1 = z - z0 * g.n1;
    int tm, tn;
    place(blockIdx.x, g.tiles_m, g.tiles_n, tm, tn);
    const int m0 = tm * Tile::M, n0 = tn * Tile::N;
    const int row_bytes = (g.K + 15) & ~15;
    const signed char* a = g.a + z0 * g.a0 + z1 * g.a1 + (long long)m0 * g.lda;
    const signed char* b = g.b + z0 * g.b0 + z1 * g.b1 + (long long)n0 * g.ldb;
    Tile t;
    t.run(rows_rsrc(a, min(g.M - m0, Tile::M), g.lda, row_bytes), g.lda, rows_rsrc(b, min(g.N - n0, Tile::N), g.ldb, row_bytes), g.ldb, g.K, lds);
    const float *sa = g.sa + z0 * g.sa0 + z1 * g.sa1, *sb = g.sb + z0 * g.sb0 + z1 * g.sb1;
    T* out = (T*)g.out + z0 * g.o0 + z1 * g.o1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // The stages are free (every wave is past its last barrier).  A wave turns its tile in a part of LDS of its own, 32 rows at a time: four
    // columns of a row leave a lane at once, and 16 bytes of a row a lane go to memory, 64 lanes on whole lines.  (Straight from the registers a
    // 16-bit store instruction covers 128 bytes instead of 1024: 8192 x 4800 x 4800 x 256 took three times as long.)
    constexpr int ROW = Tile::NT * 32 * (int)sizeof(T) + 16, VEC = 16 / (int)sizeof(T), LANES = Tile::NT * 32 / VEC;   // bytes of a row, elements of a lane, lanes of a row
    static_assert(Tile::WAVES * 32 * ROW + Tile::N * 4 <= Tile::LDS, "the turning space and the scales of b fit the stages");
    char* turn = lds + wave * 32 * ROW;
    float* scale_b = (float*)(lds + Tile::WAVES * 32 * ROW);
    for (int i = threadIdx.x; i < Tile::N; i += Tile::THREADS) scale_b[i] = n0 + i < g.N ? sb[n0 + i] : 0.f;
    __syncthreads();
    const int mw = m0 + wave / Tile::ACROSS * Tile::MT * 32, nw = n0 + wave % Tile::ACROSS * Tile::NT * 32;
    const int col = nw + (lane % LANES) * VEC;
    const bool wide = g.wide && col + VEC <= g.N;
#pragma unroll
    for (int i = 0; i < Tile::MT; ++i) {
        const int mine = mw + i * 32 + (lane & 31);
        const float s = mine < g.M ? sa[mine] * g.alpha : 0.f;
#pragma unroll
        for (int j = 0; j < Tile::NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                typedef T T4 __attribute__((ext_vector_type(4)));
                const f32x4 c = *reinterpret_cast<const f32x4*>(scale_b + nw - n0 + j * 32 + q * 8 + (lane >> 5) * 4);
                T4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = scaled<T>(t.acc[i][j][q * 4 + e], s, c[e]);
                *reinterpret_cast<T4*>(turn + (lane & 31) * ROW + (j * 32 + q * 8 + (lane >> 5) * 4) * (int)sizeof(T)) = v;
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the wave's own writes; no other wave touches this part
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += 64 / LANES) {
            const int r = r0 + lane / LANES, row = mw + i * 32 + r;
            const char* from = turn + r * ROW + (lane % LANES) * 16;
            if (row < g.M) {
                T* o = out + (long long)row * g.ldo + col;
                if (wide) *reinterpret_cast<i32x4*>(o) = *reinterpret_cast<const i32x4*>(from);
                else
                    for (int e = 0; e < VEC && col + e < g.N; ++e) o[e] = reinterpret_cast<const T*>(from)[e];
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

typedef ByteTile<64, 64, 32, 32> Small;
typedef ByteTile<128, 128, 64, 64> Middle;
typedef ByteTile<256, 256, 128, 64> Large;

// Short rows (K <= 256) and many of them on both sides -- the correlation volume: what is written dwarfs what is read and computed, so the stores
// have to run all the time.  A workgroup keeps 256 rows of b (the output's columns) in registers, 64 in a wave, and lets rows of a stream past:
// chunks of 32 rows in a ring of SLOTS, filled by LDS-DMA SLOTS - 1 chunks ahead; a chunk's results are turned in LDS and stored 16 bytes a lane.
// Three workgroups share a CU, so that one's stores run beside another's products (two with a deeper ring: +8 % time).
// vmcnt counts loads and stores and retires them in order: a wave issues PW pieces and NS stores a chunk, always (what lies outside is dropped by
// the bounds check), so "chunk c has landed" is a fixed count that leaves the stores of SLOTS - 1 chunks in flight.
// 4 x 4800 x 4800 x 256 to fp16: 51 us, 184 MB written, 3.6 TB/s (a fill: 6.8, a copy 5.1).
constexpr int STREAM_WGS = 2048;       // workgroups aimed at
constexpr int STREAM_ROWS = 512;       // rows of a that a workgroup takes at most (their scales wait in LDS)
struct StreamArgs {
    GemmArgs g;
    int panels, ranges, rows;          // column panels, row ranges, rows of a range (a multiple of 32)
};

template <int KC, int DT>
__global__ __launch_bounds__(256, 3) void i8_stream_kernel(StreamArgs s) {
    typedef typename OutT<DT>::T T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    const GemmArgs& g = s.g;
    constexpr int SLOTS = 3, SLOT = 32 * KC * CHUNK, PW = KC, NT = 2;
    constexpr int TURN = 128 / (int)sizeof(T), TURNS = 64 / TURN;            // columns turned at a time: 128 bytes of a row
    constexpr int ROW = 128 + 16, VEC = 16 / (int)sizeof(T), NS = 4 * TURNS; // 8 lanes a row, 8 rows a store
    __shared__ __attribute__((aligned(1024))) char ring[SLOTS * SLOT];
    __shared__ __attribute__((aligned(16))) char turns[4 * 32 * ROW];
    __shared__ __attribute__((aligned(16))) float scale_a[STREAM_ROWS], scale_b[256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int z = blockIdx.y, z0 = z / g.n1, z1 = z - z0 * g.n1;
    const int range = blockIdx.x / s.panels, n0 = (blockIdx.x - range * s.panels) * 256, m0 = range * s.rows;
    const int rows = min(s.rows, g.M - m0), chunks = (rows + 31) / 32;
    const int row_bytes = (g.K + 15) & ~15;
    const float *sa = g.sa + z0 * g.sa0 + z1 * g.sa1 + m0, *sb = g.sb + z0 * g.sb0 + z1 * g.sb1 + n0;
    for (int i = threadIdx.x; i < s.rows; i += 256) scale_a[i] = i < rows ? sa[i] * g.alpha : 0.f;
    scale_b[threadIdx.x] = n0 + (int)threadIdx.x < g.N ? sb[threadIdx.x] : 0.f;
    // the wave's columns, whole
    const int nw = n0 + wave * 64;
    const rsrc_t rb = rows_rsrc(g.b + z0 * g.b0 + z1 * g.b1 + (long long)nw * g.ldb, min(g.N - nw, 64), g.ldb, row_bytes);
    i32x4 bv[NT][KC * 4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int u = 0; u < KC * 4; ++u) {
            const int k = u * 32 + (lane >> 5) * 16;
            bv[j][u] = cut(__builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rb, (j * 32 + (lane & 31)) * g.ldb + k, 0, 0)), k, g.K);
        }
    const rsrc_t ra = rows_rsrc(g.a + z0 * g.a0 + z1 * g.a1 + (long long)m0 * g.lda, rows, g.lda, row_bytes);
    const rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc((void*)((T*)g.out + z0 * g.o0 + z1 * g.o1 + (long long)m0 * g.ldo), 0, 0x7fffffff, 0x00020000);
    const int va = lane_offset(lane, g.lda, wave);
    // a chunk lies as KC columns of 32 rows x 128 bytes; a wave moves eight rows of each
    auto issue = [&](int c, int slot) {
#pragma unroll
        for (int i = 0; i < PW; ++i)
            dma_piece(ra, ring + slot * SLOT + i * 32 * CHUNK + wave * 1024, va + (c * 32 + wave * 8) * g.lda, i * CHUNK);
    };
    __syncthreads();                    // the scales
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int c = 0; c < SLOTS - 1; ++c) issue(c, c);
    char* turn = turns + wave * 32 * ROW;
    int slot = 0;
    for (int c = 0; c < chunks; ++c) {
        if (c < SLOTS - 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((SLOTS - 2) * PW) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((SLOTS - 2) * PW + (SLOTS - 1) * NS) : "memory");
        __builtin_amdgcn_s_barrier();
        issue(c + SLOTS - 1, slot == 0 ? SLOTS - 1 : slot - 1);     // (behind the last chunk: rows outside, zeros into a slot that nobody reads)
        const char* as = ring + slot * SLOT;
        slot = slot == SLOTS - 1 ? 0 : slot + 1;
        i32x16 acc[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[j][k] = 0;
#pragma unroll
        for (int u = 0; u < KC * 4; ++u) {
            const i32x4 av = frag(as + u / 4 * 32 * CHUNK, lane, u & 3);
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bv[j][u], av, acc[j], 0, 0, 0);
        }
        const float sr = scale_a[c * 32 + (lane & 31)];
#pragma unroll
        for (int t = 0; t < TURNS; ++t) {
#pragma unroll
            for (int j = t * NT / TURNS; j < (t + 1) * NT / TURNS; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int at = j * 32 + q * 8 + (lane >> 5) * 4;
                    const f32x4 sc = *reinterpret_cast<const f32x4*>(scale_b + wave * 64 + at);
                    T4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = scaled<T>(acc[j][q * 4 + e], sr, sc[e]);
                    *reinterpret_cast<T4*>(turn + (lane & 31) * ROW + (at - t * TURN) * (int)sizeof(T)) = v;
                }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // the wave's own writes; no other wave touches this part
            const int col = nw + t * TURN + (lane & 7) * VEC;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + (lane >> 3), row = c * 32 + r;
                const i32x4 v = *reinterpret_cast<const i32x4*>(turn + r * ROW + (lane & 7) * 16);
                const unsigned off = row < rows && col < g.N ? (unsigned)(((long long)row * g.ldo + col) * (int)sizeof(T)) : 0x80000000u;
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), ro, off, 0, 2);   // nt: what is written is not read here
            }
            if (t + 1 < TURNS) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // no piece lands in LDS that is no longer this workgroup's
}

// Few rows on one side (R <= 16 * RT), the other side's rows (many) read once: 16 of them for a workgroup, straight from memory into the
// fragments, the contraction split over its four waves and joined in LDS.  `many` is b (the output's columns) or a, by the strides given.
// One row at N = K = 4096: 6.5 us, 2.6 TB/s; few workgroups, each waiting for memory once or twice, and the launch itself.
struct SkinnyArgs {
    const signed char *few, *many;
    const float *sf, *sm;
    void* out;
    long long f0, f1, m0, m1, sf0, sf1, sm0, sm1, o0, o1;
    int ldf, ldm;
    long long of, om;      // strides of the output along the few and the many rows
    int F, M, K, n1;
    float alpha;
    int few_is_a;          // alpha scale_a goes first, as in the other kernels: a row has the same bits however many stand beside it
};
constexpr int SKINNY_AHEAD = 8;    // steps of 64 k in flight

template <int RT, int DT>
__global__ __launch_bounds__(256) void i8_skinny_kernel(SkinnyArgs g) {
    typedef typename OutT<DT>::T T;
    __shared__ i32x4 part[4][RT][64];
    const int z = blockIdx.y, z0 = z / g.n1, z1 = z - z0 * g.n1;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r0 = blockIdx.x * 16;
    const int row_bytes = (g.K + 15) & ~15;
    const rsrc_t many = rows_rsrc(g.many + z0 * g.m0 + z1 * g.m1 + (long long)r0 * g.ldm, min(16, g.M - r0), g.ldm, row_bytes);
    const rsrc_t few = rows_rsrc(g.few + z0 * g.f0 + z1 * g.f1, g.F, g.ldf, row_bytes);
    const int steps = (g.K + 63) / 64, per = (steps + 3) / 4, first = wave * per, last = min(steps, first + per);
    const int k_lane = (lane >> 4) * 16, vm = (lane & 15) * g.ldm + k_lane, vf = (lane & 15) * g.ldf + k_lane;
    i32x4 acc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t] = i32x4{0, 0, 0, 0};
    for (int s = first; s < last; s += SKINNY_AHEAD) {
        i32x4 mv[SKINNY_AHEAD], fv[RT][SKINNY_AHEAD];
#pragma unroll
        for (int u = 0; u < SKINNY_AHEAD; ++u) {
            const int k = min(s + u, last - 1) * 64;        // (behind the last step: read again, not counted)
            mv[u] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(many, vm, k, 0));
#pragma unroll
            for (int t = 0; t < RT; ++t) fv[t][u] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(few, vf + t * 16 * g.ldf, k, 0));
        }
#pragma unroll
        for (int u = 0; u < SKINNY_AHEAD; ++u) {
            const i32x4 m = s + u < last ? cut(mv[u], (s + u) * 64 + k_lane, g.K) : i32x4{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fv[t][u], m, acc[t], 0, 0, 0);
        }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    // lane: column (of the many) lane % 16, rows (of the few) 4 * (lane / 16) .. + 3
    const int col = r0 + (lane & 15);
    if (wave < RT && col < g.M) {
        const i32x4 v = part[0][wave][lane] + part[1][wave][lane] + part[2][wave][lane] + part[3][wave][lane];
        const float sm = g.sm[z0 * g.sm0 + z1 * g.sm1 + col];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = wave * 16 + (lane >> 4) * 4 + e;
            if (row < g.F) {
                const float sf = g.sf[z0 * g.sf0 + z1 * g.sf1 + row];
                ((T*)g.out)[z0 * g.o0 + z1 * g.o1 + row * g.of + col * g.om] = scaled<T>(v[e], (g.few_is_a ? sf : sm) * g.alpha, g.few_is_a ? sm : sf);
            }
        }
    }
}

// A launch has fewer than 2^32 threads along x.
bool fits(long long wgs, int threads) { return wgs * threads < (1LL << 32); }

template <class Tile>
int launch_tiles(GemmArgs g, int dtype, unsigned batch, hipStream_t st) {
    g.tiles_m = ceil_div(g.M, Tile::M);
    g.tiles_n = ceil_div(g.N, Tile::N);
    BFLOW_REQUIRE(fits((long long)g.tiles_m * g.tiles_n, Tile::THREADS), BFLOW_E_LIMIT, "i8_gemm: too many tiles for %d x %d", g.M, g.N);
    const auto kernel = dtype == F32 ? i8_gemm_kernel<Tile, F32> : dtype == F16 ? i8_gemm_kernel<Tile, F16> : i8_gemm_kernel<Tile, BF16>;
    if (Tile::LDS > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, Tile::LDS);
        BFLOW_REQUIRE(e == hipSuccess, (int)e, "i8_gemm: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL(kernel, dim3(g.tiles_m * g.tiles_n, batch), dim3(Tile::THREADS), Tile::LDS, st, g);
    return launch_status("i8_gemm");
}
int launch_stream(const GemmArgs& g, int dtype, unsigned batch, hipStream_t st) {
    StreamArgs s = {g, ceil_div(g.N, 256), 0, 0};
    const long long panels = (long long)s.panels * batch, chunks = ceil_div(g.M, 32);
    long long ranges = (STREAM_WGS + panels - 1) / panels, per = (chunks + ranges - 1) / ranges;
    per = per > STREAM_ROWS / 32 ? STREAM_ROWS / 32 : per;
    s.rows = (int)per * 32;
    s.ranges = ceil_div(g.M, s.rows);
    BFLOW_REQUIRE(fits((long long)s.panels * s.ranges, 256), BFLOW_E_LIMIT, "i8_gemm: too many panels for %d x %d", g.M, g.N);
    const bool one = g.K <= CHUNK;
    const auto kernel = one ? (dtype == F32 ? i8_stream_kernel<1, F32> : dtype == F16 ? i8_stream_kernel<1, F16> : i8_stream_kernel<1, BF16>)
                            : (dtype == F32 ? i8_stream_kernel<2, F32> : dtype == F16 ? i8_stream_kernel<2, F16> : i8_stream_kernel<2, BF16>);
    hipLaunchKernelGGL(kernel, dim3(s.panels * s.ranges, batch), dim3(256), 0, st, s);
    return launch_status("i8_gemm");
}
template <int RT>
int launch_skinny(const SkinnyArgs& g, int dtype, unsigned batch, hipStream_t st) {
    BFLOW_REQUIRE(fits((g.M + 15LL) / 16, 256), BFLOW_E_LIMIT, "i8_gemm: %d rows beside %d, fewer than 2^28 are taken", g.M, g.F);
    const auto kernel = dtype == F32 ? i8_skinny_kernel<RT, F32> : dtype == F16 ? i8_skinny_kernel<RT, F16> : i8_skinny_kernel<RT, BF16>;
    hipLaunchKernelGGL(kernel, dim3((g.M + 15) / 16, batch), dim3(256), 0, st, g);
    return launch_status("i8_gemm");
}

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

// One wave for a row: x (rows, K), ld elements apart -> q (rows, ldq), zeros behind K; the row is read twice, an element a lane, so that few or long rows
// wait for one load after another.  bf16: 1 x 4096 16 us, 64 x 4096 19, 8192 x 8192 87 (the second reading from the caches: 2.3 TB/s); 4800 x 567 in fp32 7.4.
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

// Row r of a plane -> its pixel, -1 outside the map: in order, or in the 4 x 8 tile order of the look-up.
__device__ __forceinline__ int pixel_of(int r, int rows, int tiled, int h, int w) {
    if (r >= rows) return -1;
    if (!tiled) return r;
    const int across = (w + 7) / 8, tile = r >> 5, ty = tile / across, y = ty * 4 + ((r & 31) >> 3), x = (tile - ty * across) * 8 + (r & 7);
    return y < h && x < w ? y * w + x : -1;
}

// Maps (B, D, h, w) in 32 bits.  A workgroup takes 64 rows of the result, a lane a row, a wave a sixteenth of the channels (of 256 of them at a
// time): all loads of a thread are in flight at once and are kept, the whole numbers are turned in LDS and leave as whole rows.  10 us for
// 4 x 256 x 60 x 80 (19.7 MB in, 4.9 out); four waves walking the channels twice took 43.
// Both operands of a volume share a launch (the second one's maps behind the first one's): 11 + 6 us -> 12 for 1 and 4 maps of 256 x 60 x 80.
constexpr int SEG = 256;
struct Maps { bflow_i8_maps_t v[2]; int rows[2]; };
// the operand of a map of the launch, and which of its maps
__device__ __forceinline__ int operand_of(const Maps& m, int& b) {
    b = blockIdx.y;
    if (b < m.v[0].B) return 0;
    b -= m.v[0].B;
    return 1;
}
__global__ __launch_bounds__(1024) void quantize_pixels_kernel(Maps m, int D, int h, int w) {
    __shared__ unsigned most[16][64];
    __shared__ __attribute__((aligned(16))) signed char turn[64][SEG + 16];
    int b;
    const int item = operand_of(m, b), rows = m.rows[item], p = threadIdx.x & 63, c = threadIdx.x >> 6, r0 = blockIdx.x * 64;
    if (r0 >= rows) return;                         // (the other operand has more)
    const int pix = pixel_of(r0 + p, rows, m.v[item].tiled, h, w);
    const float* from = m.v[item].x + (long long)b * D * h * w + pix;
    signed char* q = m.v[item].q;
    float* scale = m.v[item].scale;
    const long long plane = (long long)h * w;
    float v[16];
    auto load = [&](int d0) {                       // this thread's channels of the segment: d0 + c * per ..
        const int n = min(SEG, D - d0), per = n / 16;
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = e < per && pix >= 0 ? from[(d0 + c * per + e) * plane] : 0.f;
    };
    unsigned top = 0;
    for (int d0 = 0; d0 < D; d0 += SEG) {
        load(d0);
#pragma unroll
        for (int e = 0; e < 16; ++e) top = max(top, magnitude(v[e]));
    }
    most[c][p] = top;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 16; ++e) top = max(top, most[e][p]);
    const Quant f(top);
    const bool none = f.none();
    if (c == 0 && r0 + p < rows) scale[(long long)b * rows + r0 + p] = f.scale();
    for (int d0 = 0; d0 < D; d0 += SEG) {
        if (D > SEG) load(d0);
        const int n = min(SEG, D - d0), per = n / 16;
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (e < per) turn[p][c * per + e] = none ? 0 : (signed char)f(v[e]);
        __syncthreads();
        for (int i = threadIdx.x; i < 64 * per; i += 1024) {
            const int r = i / per, k = (i - r * per) * 16;
            if (r0 + r < rows) *reinterpret_cast<i32x4*>(q + ((long long)b * rows + r0 + r) * D + d0 + k) = *reinterpret_cast<const i32x4*>(&turn[r][k]);
        }
        __syncthreads();
    }
}

// The conv engine's operand: hi and lo planes, 32 channels of a pixel together.  Four lanes a row, eight channels each of a block of 32.  1 and 4 maps of
// 256 x 60 x 80, both operands of a volume: 13 us (24.6 MB in, 6.1 out, 2.3 TB/s).
__global__ __launch_bounds__(256) void quantize_packed_kernel(Maps mm, int KB, int h, int w) {
    int b;
    const int item = operand_of(mm, b), rows = mm.rows[item], np = mm.v[item].np;
    const _Float16 *hi = (const _Float16*)mm.v[item].x_hi, *lo = (const _Float16*)mm.v[item].x_lo;
    signed char* q = mm.v[item].q;
    float* scale = mm.v[item].scale;
    const int lane = threadIdx.x & 63, r = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 16 + (lane >> 2), pix = pixel_of(r, rows, mm.v[item].tiled, h, w);
    const long long at = ((long long)b * KB * np + max(pix, 0)) * 32 + (lane & 3) * 8, step = (long long)np * 32;
    constexpr int KEEP = 8;                         // blocks of 32 channels kept in registers; further ones are read twice
    half8 vh[KEEP], vl[KEEP];
    unsigned m = 0;
    auto worst = [&](half8 a, half8 l) {
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, magnitude(fmaf((float)l[e], SPLIT_LO_INV, (float)a[e])));
    };
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
        if (k < KB) {
            vh[k] = *reinterpret_cast<const half8*>(hi + at + k * step);
            vl[k] = *reinterpret_cast<const half8*>(lo + at + k * step);
        }
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
        if (k < KB) worst(vh[k], vl[k]);
    for (int k = KEEP; k < KB; ++k) worst(*reinterpret_cast<const half8*>(hi + at + k * step), *reinterpret_cast<const half8*>(lo + at + k * step));
    m = max(m, (unsigned)__shfl_xor((int)m, 1, 64));
    m = max(m, (unsigned)__shfl_xor((int)m, 2, 64));
    if (pix < 0) m = 0;
    const Quant f(m);
    const bool none = f.none();
    if (r >= rows) return;
    if ((lane & 3) == 0) scale[(long long)b * rows + r] = f.scale();
    signed char* to = q + ((long long)b * rows + r) * KB * 32 + (lane & 3) * 8;
    auto put = [&](int k, half8 a, half8 l) {
        unsigned u[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (!none) u[e >> 2] |= (unsigned)(f(fmaf((float)l[e], SPLIT_LO_INV, (float)a[e])) & 255) << (8 * (e & 3));
        *reinterpret_cast<uint2*>(to + k * 32) = make_uint2(u[0], u[1]);
    };
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
        if (k < KB) put(k, vh[k], vl[k]);
    for (int k = KEEP; k < KB; ++k) put(k, *reinterpret_cast<const half8*>(hi + at + k * step), *reinterpret_cast<const half8*>(lo + at + k * step));
}
}  // namespace

extern "C" int bflow_i8_gemm(const bflow_i8_gemm_t* d, bflow_stream_t stream) {
    BFLOW_REQUIRE(d, BFLOW_E_ARG, "i8_gemm: null descriptor");
    BFLOW_REQUIRE(d->a && d->b && d->scale_a && d->scale_b && d->out, BFLOW_E_ARG, "i8_gemm: null pointer");
    BFLOW_REQUIRE(d->M >= 1 && d->N >= 1 && d->K >= 1 && d->batch0 >= 1 && d->batch1 >= 1, BFLOW_E_ARG, "i8_gemm: sizes %d x %d x %d, batch %d x %d", d->M, d->N, d->K,
                  d->batch0, d->batch1);
    BFLOW_REQUIRE(d->K <= BFLOW_I8_MAX_K, BFLOW_E_LIMIT, "i8_gemm: K = %d > %d (32-bit sums)", d->K, BFLOW_I8_MAX_K);
    BFLOW_REQUIRE(d->M <= BFLOW_I8_MAX_SIZE && d->N <= BFLOW_I8_MAX_SIZE, BFLOW_E_LIMIT, "i8_gemm: %d x %d, a side above %d", d->M, d->N, BFLOW_I8_MAX_SIZE);
    BFLOW_REQUIRE(d->dtype >= F32 && d->dtype <= BF16, BFLOW_E_ARG, "i8_gemm: dtype %d", d->dtype);
    const int row = (d->K + 15) & ~15;
    BFLOW_REQUIRE(d->lda >= row && d->ldb >= row && d->lda <= BFLOW_I8_MAX_LD && d->ldb <= BFLOW_I8_MAX_LD && d->ldo >= d->N, BFLOW_E_ARG,
                  "i8_gemm: leading dimensions %d, %d, %lld for K = %d, N = %d", d->lda, d->ldb, d->ldo, d->K, d->N);
    BFLOW_REQUIRE(((uintptr_t)d->a | (uintptr_t)d->b | (unsigned)d->lda | (unsigned)d->ldb | (unsigned long long)d->a_stride0 | (unsigned long long)d->a_stride1 |
                   (unsigned long long)d->b_stride0 | (unsigned long long)d->b_stride1) % 16 == 0, BFLOW_E_ARG, "i8_gemm: operands and their strides are multiples of 16 bytes");
    const long long batch = (long long)d->batch0 * d->batch1;
    BFLOW_REQUIRE(batch <= 65535, BFLOW_E_LIMIT, "i8_gemm: %lld matrices > 65535", batch);
    const int size = d->dtype == F32 ? 4 : 2;
    const GemmArgs g = {(const signed char*)d->a, (const signed char*)d->b, d->scale_a, d->scale_b, d->out, d->a_stride0, d->a_stride1, d->b_stride0, d->b_stride1,
                        d->sa_stride0, d->sa_stride1, d->sb_stride0, d->sb_stride1, d->out_stride0, d->out_stride1, d->lda, d->ldb, d->ldo, d->M, d->N, d->K, d->batch1,
                        d->alpha, 0, 0, ((uintptr_t)d->out | (unsigned long long)size * (unsigned long long)(d->ldo | d->out_stride0 | d->out_stride1)) % 16 == 0};
    const hipStream_t st = (hipStream_t)stream;
    // Few rows on one side: 6.4 us against 11.9 for one row at N = K = 4096, 10.0 against 12.1 for 32, 11.9 either way for 48.
    if (d->M <= 32 || d->N <= 32) {
        const SkinnyArgs s = d->M <= d->N ? SkinnyArgs{g.a, g.b, g.sa, g.sb, g.out, g.a0, g.a1, g.b0, g.b1, g.sa0, g.sa1, g.sb0, g.sb1, g.o0, g.o1, g.lda, g.ldb, g.ldo, 1, g.M, g.N, g.K, g.n1, g.alpha, 1}
                                          : SkinnyArgs{g.b, g.a, g.sb, g.sa, g.out, g.b0, g.b1, g.a0, g.a1, g.sb0, g.sb1, g.sa0, g.sa1, g.o0, g.o1, g.ldb, g.lda, 1, g.ldo, g.N, g.M, g.K, g.n1, g.alpha, 0};
        return s.F <= 16 ? launch_skinny<1>(s, d->dtype, (unsigned)batch, st) : launch_skinny<2>(s, d->dtype, (unsigned)batch, st);
    }
    // Short rows, whole 16-byte stores: 55 us against 64 (256 x 256 tiles) for 4 x 4800 x 4800 x 256 in fp16, 81 against 88 in fp32, 709 against 1233
    // for 6 x 16384 x 16384 x 256; with less than a panel on either side it has nothing to stream.
    if (d->K <= 256 && d->M >= 256 && d->N >= 256 && g.wide && d->N % (16 / size) == 0 && d->lda <= 1 << 20 && (long long)STREAM_ROWS * d->ldo * size < (1LL << 31))
        return launch_stream(g, d->dtype, (unsigned)batch, st);
    // Tiles by the rounds that they take on 256 CUs, priced by what a round took at K = 4096: 256 tiles of 256 x 256 79 us, 512 of 128 x 128 (two on a
    // CU) 44, 1024 of 64 x 64 (four) 28.  Captured calls in a row, tiles of 256 / 128 / 64: 8192^3 470 / 534 / 802 us; 4096^3 67 / 75 / 105; 2048^3 31 / 15 /
    // 16; 1024^3 18 / 9.3 / 5.8.
    auto price = [&](int side, long long room, int us) { return ((long long)ceil_div(d->M, side) * ceil_div(d->N, side) * batch + room - 1) / room * us; };
    const long long large = price(256, 256, 79), middle = price(128, 512, 44), small = price(64, 1024, 28);
    if (small <= middle && small <= large) return launch_tiles<Small>(g, d->dtype, (unsigned)batch, st);
    if (middle <= large) return launch_tiles<Middle>(g, d->dtype, (unsigned)batch, st);
    return launch_tiles<Large>(g, d->dtype, (unsigned)batch, st);
}

// Rows at any address -> rows at multiples of 16 bytes: dwords are read where they stand and shifted together.  No word is read that holds none of
// the row's bytes.
struct PadArgs { bflow_i8_pad_t v[2]; };
__global__ __launch_bounds__(256) void pad_rows_kernel(PadArgs p) {
    const bflow_i8_pad_t d = p.v[blockIdx.y];
    const int across = d.ldd / 16;
    const long long n = d.rows * across;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const long long row = i / across;
        const int k = (int)(i - row * across) * 16;
        const uintptr_t from = (uintptr_t)d.src + row * d.ld + k;
        const int shift = (int)(from & 3), bytes = min(16, d.K - k) + shift;      // counted from the first word
        const unsigned* w = (const unsigned*)(from - shift);
        unsigned x[5];
#pragma unroll
        for (int e = 0; e < 5; ++e) x[e] = 4 * e < bytes ? w[e] : 0u;
        i32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (int)__builtin_amdgcn_alignbyte(x[e + 1], x[e], shift);
        *reinterpret_cast<i32x4*>((char*)d.dst + row * d.ldd + k) = cut(v, k, d.K);      // (the last word may hold bytes of what follows the row)
    }
}

extern "C" int bflow_i8_pad_rows(const bflow_i8_pad_t* items, int count, bflow_stream_t stream) {
    BFLOW_REQUIRE(items && count >= 1 && count <= 2, BFLOW_E_ARG, "i8_pad_rows: one or two operands");
    PadArgs p = {};
    long long most = 0;
    for (int i = 0; i < count; ++i) {
        const bflow_i8_pad_t& d = items[i];
        BFLOW_REQUIRE(d.src && d.dst && d.rows >= 1 && d.K >= 1 && d.ldd >= d.K && d.ldd % 16 == 0 && (uintptr_t)d.dst % 16 == 0, BFLOW_E_ARG,
                      "i8_pad_rows: %lld rows of %d, ldd %d", d.rows, d.K, d.ldd);
        p.v[i] = d;
        most = d.rows * (d.ldd / 16) > most ? d.rows * (d.ldd / 16) : most;
    }
    hipLaunchKernelGGL(pad_rows_kernel, dim3(stream_grid(most, 256), count), dim3(256), 0, (hipStream_t)stream, p);
    return launch_status("i8_pad_rows");
}

extern "C" int bflow_i8_quantize_rows(const void* x, int dtype, long long ld, long long rows, int K, signed char* q, int ldq, float* scale, bflow_stream_t stream) {
    BFLOW_REQUIRE(x && q && scale, BFLOW_E_ARG, "i8_quantize_rows: null pointer");
    BFLOW_REQUIRE(rows >= 1 && K >= 1 && ld >= 0 && ldq >= K && ldq % 16 == 0 && (uintptr_t)q % 16 == 0, BFLOW_E_ARG, "i8_quantize_rows: %lld rows of %d, strides %lld, %d", rows, K, ld,
                  ldq);
    BFLOW_REQUIRE(dtype >= F32 && dtype <= BF16, BFLOW_E_ARG, "i8_quantize_rows: dtype %d", dtype);
    BFLOW_REQUIRE(K <= BFLOW_I8_MAX_SIZE && ldq <= BFLOW_I8_MAX_SIZE, BFLOW_E_LIMIT, "i8_quantize_rows: rows of %d, %d apart, above %d", K, ldq, BFLOW_I8_MAX_SIZE);
    const auto kernel = dtype == F32 ? quantize_rows_kernel<F32> : dtype == F16 ? quantize_rows_kernel<F16> : quantize_rows_kernel<BF16>;
    const long long wgs = (rows + 3) / 4;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(wgs < 65536 ? wgs : 65536)), dim3(256), 0, (hipStream_t)stream, x, ld, rows, K, q, ldq, scale);
    return launch_status("i8_quantize_rows");
}

extern "C" int bflow_i8_quantize_maps(const bflow_i8_maps_t* items, int count, int D, int h, int w, bflow_stream_t stream) {
    BFLOW_REQUIRE(items && count >= 1 && count <= 2, BFLOW_E_ARG, "i8_quantize_pixels: one or two operands");
    BFLOW_REQUIRE(D >= 16 && D % 16 == 0 && h >= 1 && w >= 1 && (long long)h * w < (1LL << 28), BFLOW_E_ARG, "i8_quantize_pixels: D = %d (a multiple of 16), %d x %d pixels",
                  D, h, w);
    Maps m = {};
    long long maps = 0;
    int most = 0;
    const bool plain = items[0].x;
    for (int i = 0; i < count; ++i) {
        const bflow_i8_maps_t& v = items[i];
        BFLOW_REQUIRE(v.q && v.scale && (v.x || (v.x_hi && v.x_lo)) && !(v.x && v.x_hi), BFLOW_E_ARG, "i8_quantize_pixels: null pointer, or both forms of x");
        BFLOW_REQUIRE(plain == (v.x != nullptr), BFLOW_E_ARG, "i8_quantize_pixels: two operands of different form");
        BFLOW_REQUIRE(v.B >= 1 && v.B <= 65535, BFLOW_E_ARG, "i8_quantize_pixels: B = %d", v.B);
        BFLOW_REQUIRE(plain || (D % 32 == 0 && v.np >= h * w), BFLOW_E_ARG, "i8_quantize_pixels: packed operand of %d rows for %d pixels, D = %d (a multiple of 32)", v.np, h * w, D);
        BFLOW_REQUIRE((uintptr_t)v.q % 16 == 0, BFLOW_E_ARG, "i8_quantize_pixels: q is not aligned to 16 bytes");
        const long long places = v.tiled ? (long long)((h + 3) / 4) * ((w + 7) / 8) * 32 : (long long)h * w;
        BFLOW_REQUIRE(places <= 1 << 30, BFLOW_E_LIMIT, "i8_quantize_pixels: %lld places of %d x %d pixels", places, h, w);
        m.v[i] = v;
        m.rows[i] = (int)places;
        maps += v.B;
        most = m.rows[i] > most ? m.rows[i] : most;
    }
    BFLOW_REQUIRE(maps <= 65535, BFLOW_E_LIMIT, "i8_quantize_pixels: %lld maps > 65535", maps);
    BFLOW_REQUIRE(fits((most + 63) / 64, plain ? 1024 : 256), BFLOW_E_LIMIT, "i8_quantize_pixels: %d places of %d x %d pixels", most, h, w);
    const dim3 grid((most + 63) / 64, (unsigned)maps);
    if (plain) hipLaunchKernelGGL(quantize_pixels_kernel, grid, dim3(1024), 0, (hipStream_t)stream, m, D, h, w);
    else hipLaunchKernelGGL(quantize_packed_kernel, grid, dim3(256), 0, (hipStream_t)stream, m, D / 32, h, w);
    return launch_status("i8_quantize_pixels");
}

extern "C" int bflow_i8_quantize_pixels(const float* x, const void* x_hi, const void* x_lo, int np, int B, int D, int h, int w, int tiled, signed char* q, float* scale,
                                        bflow_stream_t stream) {
    const bflow_i8_maps_t one = {x, x_hi, x_lo, q, scale, np, B, tiled, 0};
    return bflow_i8_quantize_maps(&one, 1, D, h, w, stream);
}
