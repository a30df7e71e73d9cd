// Weight gradient of a projection whose input is held in 8 bits: dst[b] (k x n) = restored[b]^T * upstream[b] (m x n).
#include "rt_pack8.h"

#include <atomic>

namespace {

// ---- f32 -----------------------------------------------------------------------------------------------------------------------------
// A restored value has 7 significant bits and is a bf16 number exactly.  An f32 number v is the exact sum of three bf16 numbers: v cut to
// its upper 16 bits, what is left cut again, and the last 8 bits.  A product of two bf16 numbers is exact in f32, so three bf16 matrix
// products accumulated in f32 give the f32 product, at a sixteenth of the f32 matrix instructions' time each.  (Of an element below
// 2^-110 the last parts may fall below the normal range, where the matrix unit may take them as 0: at most 2^-126 of it.)
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16_a1 __attribute__((aligned(1)));

// Upper halves of two words, the first one's in the lower half of the result.
__device__ __forceinline__ uint32_t uppers(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ __forceinline__ uint32_t bits(float v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ float number(uint32_t b) { return __builtin_bit_cast(float, b); }

// The three parts of eight numbers, one below the other in the summed dim, as the matrix instructions take them.
struct Parts { u32x4 p[3]; };
__device__ __forceinline__ Parts parts_of(const uint32_t (&v)[8]) {
    Parts out;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t h[2], m[2], l[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            h[e] = v[2 * j + e];
            const float x = number(h[e]);
            // inf - inf: an infinity has no further parts (a NaN is one in all of them)
            const float r = __builtin_fabsf(x) == __builtin_inff() ? 0.0f : x - number(h[e] & 0xffff0000u);
            m[e] = bits(r);
            l[e] = bits(r - number(m[e] & 0xffff0000u));
        }
        out.p[0][j] = uppers(h[0], h[1]);
        out.p[1][j] = uppers(m[0], m[1]);
        out.p[2][j] = uppers(l[0], l[1]);
    }
    return out;
}

// Bound by the matrix instructions: 16384 x 4096 x 4096 takes 1358 us (1340 to 1390 from run to run), three bf16 products at 1215 TFLOP/s
// (the card's bf16 matmul of 8192^3 runs at 1154), 405 TFLOP/s of f32; short shares by what surrounds them: 65536 x 256 x 320 takes 54 us,
// of which 6 are the join, about 10 the first loads and the partial results, and 24 steps of 1.5 us the rest.
//
// dst tile of BI x BJ by WI x WJ waves, kStep rows of both operands staged in LDS at a time, two buffers.  LDS holds 16-byte pieces of
// eight rows of one column, [part][row group][column]: what a lane of the 32x32x16 matrix instruction takes is one piece, and neither
// the writes nor the reads of a wave meet in a bank.
constexpr int kStep = 32, kGroups = kStep / 8;
template <int BI, int BJ> struct Stage {
    u32x4 x[kGroups][BI];
    u32x4 y[3][kGroups][BJ];
};

// Which rows a block sums: split `s` of `splits` takes whole steps.
struct Share { uint64_t from, to; };
__device__ __forceinline__ Share share_of(uint64_t m, uint32_t splits, uint32_t s) {
    const uint64_t steps = (m + kStep - 1) / kStep, per = steps / splits, more = steps % splits;
    const uint64_t a = s * per + (s < more ? s : more), n = per + (s < more ? 1 : 0);
    const uint64_t to = (a + n) * kStep;
    return Share{a * kStep, to < m ? to : m};
}

struct Product {
    const int8_t* codes;
    const uint8_t* exps;
    const void* up;
    void* out;                        // dst, or the splits' partial results, each as large as dst
    uint64_t b, m, k, n;
    uint32_t ti, tj, splits;          // tiles of dst, shares of the rows
    uint64_t batch0;                  // first batch of the launch
};
// Tile of a block: batch-major, then the splits; within one (batch, split) the tiles in bands of eight along i, so that blocks that run
// at the same time on one XCD (every eighth block) share columns of both operands in its L2: XCD x takes the x-th eighth of the tiles.
struct Where { uint64_t batch; uint32_t split, i, j; };
__device__ __forceinline__ Where where(const Product& p) {
    const uint32_t tiles = p.ti * p.tj, total = gridDim.x;
    uint32_t t = blockIdx.x;
    const uint32_t xcd = t % 8, more = total % 8;
    t = xcd * (total / 8) + (xcd < more ? xcd : more) + t / 8;
    Where w;
    const uint32_t bs = t / tiles;
    t -= bs * tiles;
    w.batch = p.batch0 + bs / p.splits;
    w.split = bs % p.splits;
    const uint32_t band = t / (8 * p.tj), rows = p.ti - band * 8 < 8 ? p.ti - band * 8 : 8;
    t -= band * 8 * p.tj;
    w.i = band * 8 + t % rows;
    w.j = t / rows;
    return w;
}

// One step of the loop works on three steps of the rows at once: the matrix instructions take the one in the current buffer, the next one
// is turned into parts and written to the other buffer, and the one after that is on its way from memory into registers.  EVEN: k is
// even, so a lane's two codes lie in one group.  The matrix instructions come first, so that the loads have all of them to arrive behind
// (16384 x 4096 x 4096 1400 -> 1320 us); not so with odd k and its twice as many loads (16000 x 2001 x 2003 410 us, the other way round
// 430 us).
template <int BI, int BJ, int WI, int WJ, int DEPTH, bool EVEN>
__global__ __launch_bounds__(WI * WJ * 64) void pack8_matmul_f32_kernel(Product p) {
    constexpr int kThreads = WI * WJ * 64, FI = BI / WI / 32, FJ = BJ / WJ / 32;             // 32 x 32 pieces of a wave
    constexpr int kYEach = kGroups * BJ / kThreads;                                          // row groups of y a lane stages
    static_assert(kGroups * BI / 2 == kThreads && kYEach * kThreads == kGroups * BJ, "staging covers the tile once");
    extern __shared__ __align__(16) char lds[];
    Stage<BI, BJ>* stage = reinterpret_cast<Stage<BI, BJ>*>(lds);
    const Where at = where(p);
    const Share share = share_of(p.m, p.splits, at.split);
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wi = w / WJ, wj = w % WJ;
    const uint64_t i0 = (uint64_t)at.i * BI, j0 = (uint64_t)at.j * BJ;
    // staging: the lane's two columns of x and one row group; kYEach row groups of one column of y
    const int xc = tid % (BI / 2) * 2, xg = tid / (BI / 2);
    const int yc = tid % BJ, yg = tid / BJ * kYEach;
    // addresses: a wave-uniform start of each row and one 32-bit offset (k and n are below 2^25); columns behind the last one load it
    const uint32_t k = (uint32_t)p.k, n = (uint32_t)p.n;
    const uint32_t xcol = i0 + xc < k ? (uint32_t)i0 + xc : (EVEN ? k - 2 : k - 1), xnext = xcol + 1 < k ? 1u : 0u;
    const uint32_t ycol = j0 + yc < n ? (uint32_t)j0 + yc : n - 1;
    const uint64_t xrow = at.batch * p.m;
    const float* up = static_cast<const float*>(p.up) + at.batch * p.m * p.n;

    // EVEN: two codes in cx, their exponent byte in ex; else one each in [0] and [1].  Bits of y.
    struct Held { uint32_t cx[EVEN ? 1 : 2][8], ex[EVEN ? 1 : 2][8], yv[kYEach][8]; };
    Held held[DEPTH];
    auto load_row_of_x = [&](Held& d, int r, uint64_t from, uint32_t off) {       // from: a wave-uniform row; off: the lane's place from its start
        const uint64_t e = (xrow + from) * k;
        const int8_t* codes = p.codes + e;
        const uint8_t* exps = p.exps + e / kP8Group;
        const uint32_t rem = (uint32_t)e % kP8Group;
        if constexpr (EVEN) {
            d.cx[0][r] = *reinterpret_cast<const u16_a1*>(codes + off);
            d.ex[0][r] = exps[(rem + off) / kP8Group];
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                d.cx[q][r] = (uint8_t)codes[off + q * xnext];
                d.ex[q][r] = exps[(rem + off + q * xnext) / kP8Group];
            }
        }
    };
    const uint32_t xoff = (uint32_t)(xg * 8) * k + xcol, yoff = (uint32_t)(yg * 8) * n + ycol;
    auto load_whole = [&](Held& d, uint64_t m0) {
#pragma unroll
        for (int r = 0; r < 8; ++r) load_row_of_x(d, r, m0 + r, xoff);
#pragma unroll
        for (int g = 0; g < kYEach; ++g)
#pragma unroll
            for (int r = 0; r < 8; ++r) d.yv[g][r] = bits((up + (m0 + g * 8 + r) * n)[yoff]);
    };
    auto load = [&](Held& d, uint64_t m0) {
        if (m0 >= share.to) return;
        if (m0 + kStep <= share.to) {
            load_whole(d, m0);
        } else {                                                 // rows behind the last one load it
            const int rows = (int)(share.to - m0);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const int row = xg * 8 + r < rows ? xg * 8 + r : rows - 1;
                load_row_of_x(d, r, m0, (uint32_t)row * k + xcol);
            }
#pragma unroll
            for (int g = 0; g < kYEach; ++g)
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const int row = (yg + g) * 8 + r < rows ? (yg + g) * 8 + r : rows - 1;
                    d.yv[g][r] = bits((up + m0 * n)[(uint32_t)row * n + ycol]);
                }
        }
    };
    auto store = [&](Held& d, Stage<BI, BJ>& st) {
        u32x4 a, b;
#pragma unroll
        for (int r = 0; r < 8; r += 2) {
            uint32_t v[2][2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                constexpr int kSecond = EVEN ? 0 : 1, kShift = EVEN ? 8 : 0;
                v[q][0] = bits(p8_value<float>((int8_t)d.cx[0][r + q], d.ex[0][r + q]));
                v[q][1] = bits(p8_value<float>((int8_t)(d.cx[kSecond][r + q] >> kShift), d.ex[kSecond][r + q]));
            }
            a[r / 2] = uppers(v[0][0], v[1][0]);
            b[r / 2] = uppers(v[0][1], v[1][1]);
        }
        st.x[xg][xc] = a;
        st.x[xg][xc + 1] = b;
#pragma unroll
        for (int g = 0; g < kYEach; ++g) {
            const Parts q = parts_of(d.yv[g]);
#pragma unroll
            for (int s = 0; s < 3; ++s) st.y[s][yg + g][yc] = q.p[s];
        }
    };
    auto mask = [&](Held& d, uint64_t m0) {                               // rows behind the last one are zeros
        const int rows = share.to - m0 < (uint64_t)kStep ? (int)(share.to - m0) : kStep;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
#pragma unroll
            for (int q = 0; q < (EVEN ? 1 : 2); ++q)
                if (xg * 8 + r >= rows) d.cx[q][r] = d.ex[q][r] = 0u;
#pragma unroll
            for (int g = 0; g < kYEach; ++g)
                if ((yg + g) * 8 + r >= rows) d.yv[g][r] = 0u;
        }
    };

    f32x16 acc[FI][FJ];
#pragma unroll
    for (int a = 0; a < FI; ++a)
#pragma unroll
        for (int b = 0; b < FJ; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.0f;
    auto multiply = [&](const Stage<BI, BJ>& st) {
#pragma unroll
        for (int half = 0; half < kStep / 16; ++half) {
            const int g = half * 2 + (lane >> 5), c = lane & 31;
            bf16x8 xa[FI];
#pragma unroll
            for (int a = 0; a < FI; ++a) xa[a] = __builtin_bit_cast(bf16x8, st.x[g][(wi * FI + a) * 32 + c]);
#pragma unroll
            for (int s = 2; s >= 0; --s) {                       // the smallest parts first
                bf16x8 yb[FJ];
#pragma unroll
                for (int b = 0; b < FJ; ++b) yb[b] = __builtin_bit_cast(bf16x8, st.y[s][g][(wj * FJ + b) * 32 + c]);
#pragma unroll
                for (int a = 0; a < FI; ++a)
#pragma unroll
                    for (int b = 0; b < FJ; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xa[a], yb[b], acc[a][b], 0, 0, 0);
            }
        }
    };

    if (share.from < share.to) {
        const uint32_t steps = (uint32_t)((share.to - share.from + kStep - 1) / kStep);
        auto row_of = [&](uint32_t t) { return share.from + (uint64_t)t * kStep; };
        load(held[0], row_of(0));
        if (steps == 1) mask(held[0], row_of(0));
        store(held[0], stage[0]);
        // step t is held in set (t - 1) % DEPTH
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) load(held[d], row_of(1 + d));
        __syncthreads();
        uint32_t t = 0;
        for (; t + 2 * DEPTH + 1 < steps; t += DEPTH) {          // DEPTH steps a turn, so that the sets are named at compile time; whole ones
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                if constexpr (EVEN) multiply(stage[(t + d) & 1]);
                store(held[d], stage[(t + d + 1) & 1]);
                load_whole(held[d], row_of(t + d + 1 + DEPTH));
                if constexpr (!EVEN) multiply(stage[(t + d) & 1]);
                __syncthreads();
            }
        }
#pragma unroll
        for (int q = 0; q < 2 * DEPTH; ++q, ++t) {               // what is left: at most 2 DEPTH steps, the last one with rows missing
            if (t + 1 < steps) {
                if (t + 2 == steps) mask(held[q % DEPTH], row_of(t + 1));
                store(held[q % DEPTH], stage[(t + 1) & 1]);
                if (q < DEPTH) load(held[q % DEPTH], row_of(t + 1 + DEPTH));
                multiply(stage[t & 1]);
                __syncthreads();
            }
        }
        multiply(stage[(steps - 1) & 1]);
    }
    float* out = static_cast<float*>(p.out) + ((uint64_t)at.split * p.b + at.batch) * p.k * p.n;
#pragma unroll
    for (int a = 0; a < FI; ++a)
#pragma unroll
        for (int b = 0; b < FJ; ++b) {
            const uint64_t j = j0 + (wj * FJ + b) * 32 + (lane & 31);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint64_t i = i0 + (wi * FI + a) * 32 + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3);
                if (i < p.k && j < p.n) out[i * p.n + j] = acc[a][b][r];
            }
        }
}

// ---- f64 -----------------------------------------------------------------------------------------------------------------------------
typedef double f64x4 __attribute__((ext_vector_type(4)));
constexpr int kStep64 = 16;

// Bound by the f64 matrix instructions: 8192 x 2048 x 2048 takes 1127 us, 61 TFLOP/s (the card's f64 matmul reaches 73).
// SIDE x SIDE of dst by WI x WJ waves, the 16x16x4 matrix instruction, kStep64 rows staged at a time, ahead as in the f32 kernel.  The
// pitch of the staged rows, in words, is 32 more than a multiple of 64: the two rows that half a wave reads lie on the two halves of the
// banks.
template <int SIDE, int WI, int WJ>
__global__ __launch_bounds__(WI * WJ * 64) void pack8_matmul_f64_kernel(Product p) {
    constexpr int kPitch = SIDE + 16, FI = SIDE / WI / 16, FJ = SIDE / WJ / 16;
    static_assert(WI * WJ * 64 == SIDE * kStep64 / 4, "a lane stages four rows of one column");
    __shared__ double xs[2][kStep64][kPitch], ys[2][kStep64][kPitch];
    const Where at = where(p);
    const Share share = share_of(p.m, p.splits, at.split);
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, wi = w / WJ, wj = w % WJ;
    const uint64_t i0 = (uint64_t)at.i * SIDE, j0 = (uint64_t)at.j * SIDE;
    const int c = tid % SIDE, r0 = tid / SIDE * 4;
    const uint32_t k = (uint32_t)p.k, n = (uint32_t)p.n;
    const uint32_t xcol = i0 + c < k ? (uint32_t)i0 + c : k - 1, ycol = j0 + c < n ? (uint32_t)j0 + c : n - 1;
    const double* up = static_cast<const double*>(p.up) + at.batch * p.m * p.n;
    int32_t cx[4];
    uint32_t ex[4];
    double yv[4];
    const uint32_t xoff = (uint32_t)r0 * k + xcol, yoff = (uint32_t)r0 * n + ycol;
    auto load_row = [&](int r, uint64_t from, uint32_t xo, uint32_t yo) {        // from: a wave-uniform row; xo, yo: places from its start
        const uint64_t e = (at.batch * p.m + from) * k;
        cx[r] = (p.codes + e)[xo];
        ex[r] = (p.exps + e / kP8Group)[((uint32_t)e % kP8Group + xo) / kP8Group];
        yv[r] = (up + from * n)[yo];
    };
    auto load = [&](uint64_t m0) {
        if (m0 >= share.to) return;
        const int rows = share.to - m0 < (uint64_t)kStep64 ? (int)(share.to - m0) : kStep64;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t row = r0 + r < rows ? r0 + r : rows - 1;
            load_row(r, m0, row * k + xcol, row * n + ycol);
        }
    };
    auto store = [&](int b) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            xs[b][r0 + r][c] = p8_value<double>(cx[r], ex[r]);
            ys[b][r0 + r][c] = yv[r];
        }
    };
    auto mask = [&](uint64_t m0) {                               // rows behind the last one are zeros
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (m0 + r0 + r >= share.to) { cx[r] = 0; ex[r] = 0u; yv[r] = 0.0; }
    };
    f64x4 acc[FI][FJ];
#pragma unroll
    for (int a = 0; a < FI; ++a)
#pragma unroll
        for (int b = 0; b < FJ; ++b) acc[a][b] = f64x4{0.0, 0.0, 0.0, 0.0};
    auto multiply = [&](int cur) {
#pragma unroll
        for (int q = 0; q < kStep64 / 4; ++q) {
            const int row = q * 4 + (lane >> 4), cc = lane & 15;
            double xa[FI], yb[FJ];
#pragma unroll
            for (int a = 0; a < FI; ++a) xa[a] = xs[cur][row][(wi * FI + a) * 16 + cc];
#pragma unroll
            for (int b = 0; b < FJ; ++b) yb[b] = ys[cur][row][(wj * FJ + b) * 16 + cc];
#pragma unroll
            for (int a = 0; a < FI; ++a)
#pragma unroll
                for (int b = 0; b < FJ; ++b) acc[a][b] = __builtin_amdgcn_mfma_f64_16x16x4f64(xa[a], yb[b], acc[a][b], 0, 0, 0);
        }
    };
    if (share.from < share.to) {
        const uint32_t steps = (uint32_t)((share.to - share.from + kStep64 - 1) / kStep64);
        auto row_of = [&](uint32_t t) { return share.from + (uint64_t)t * kStep64; };
        load(row_of(0));
        if (steps == 1) mask(row_of(0));
        store(0);
        load(row_of(1));
        __syncthreads();
        uint32_t t = 0;
        for (; t + 3 < steps; ++t) {                             // whole steps
            store((t + 1) & 1);
#pragma unroll
            for (int r = 0; r < 4; ++r) load_row(r, row_of(t + 2) + r, xoff, yoff);
            multiply(t & 1);
            __syncthreads();
        }
#pragma unroll
        for (int q = 0; q < 2; ++q, ++t) {                       // what is left: at most two steps, the last one with rows missing
            if (t + 1 < steps) {
                if (t + 2 == steps) mask(row_of(t + 1));
                store((t + 1) & 1);
                if (q == 0) load(row_of(t + 2));
                multiply(t & 1);
                __syncthreads();
            }
        }
        multiply((steps - 1) & 1);
    }
    double* out = static_cast<double*>(p.out) + ((uint64_t)at.split * p.b + at.batch) * p.k * p.n;
#pragma unroll
    for (int a = 0; a < FI; ++a)
#pragma unroll
        for (int b = 0; b < FJ; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint64_t i = i0 + (wi * FI + a) * 16 + r * 4 + (lane >> 4), j = j0 + (wj * FJ + b) * 16 + (lane & 15);
                if (i < p.k && j < p.n) out[i * p.n + j] = acc[a][b][r];
            }
}

// ---- the splits' partial results, added in order -----------------------------------------------------------------------------------------
// The W waves of a block add a W-th of the splits each for 64 elements, eight loads in flight, then their sums are added in order.
// 85 splits of 256 x 320 f32: 6 us, 28 MB out of the caches and 1280 short blocks.
template <class T, int W> __global__ __launch_bounds__(W * 64) void pack8_matmul_join_kernel(const T* __restrict__ part, T* __restrict__ dst, uint64_t n, uint32_t splits) {
    __shared__ T sums[W][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t i = (uint64_t)blockIdx.x * 64 + lane, at = i < n ? i : n - 1;
    const uint32_t from = splits * w / W, to = splits * (w + 1) / W;
    T s = (T)0;
#pragma unroll 8
    for (uint32_t k = from; k < to; ++k) s += part[k * n + at];
    sums[w][lane] = s;
    __syncthreads();
    if (w == 0 && i < n) {
        T all = sums[0][lane];
#pragma unroll
        for (int v = 1; v < W; ++v) all += sums[v][lane];
        dst[i] = all;
    }
}

// Shares of the rows: enough blocks to fill the card, each share long enough to pay for its partial result.
uint32_t splits_for(rt_ctx* ctx, uint64_t tiles, uint64_t m, uint64_t least_rows, uint64_t blocks_per_cu) {
    const uint64_t want = (uint64_t)ctx->num_cus * blocks_per_cu, most = m / least_rows;
    uint64_t s = tiles >= want ? 1 : want / tiles;
    s = s < most ? s : most;
    return (uint32_t)(s < 1 ? 1 : s);
}

template <class T> int32_t join(rt_ctx* ctx, const void* part, void* dst, uint64_t n, uint32_t splits) {
    const dim3 grid((uint32_t)((n + 63) / 64));
    // many splits of a small result: more waves for each, where blocks are few (512 splits of 64 x 64 f32 26 -> 22 us with the product; 85 of
    // 256 x 320 would lose 2 us)
    if (splits >= 32 && grid.x <= (uint32_t)ctx->num_cus) hipLaunchKernelGGL((pack8_matmul_join_kernel<T, 16>), grid, dim3(1024), 0, ctx->stream, (const T*)part, (T*)dst, n, splits);
    else hipLaunchKernelGGL((pack8_matmul_join_kernel<T, 4>), grid, dim3(256), 0, ctx->stream, (const T*)part, (T*)dst, n, splits);
    RT_HIP(hipGetLastError());
    return RT_OK;
}

// `launch(part, blocks)` for all batches, by blocks of `threads`, over as many launches as that takes: the lanes of a grid are numbered in
// 32 bits.  More than one launch comes with one split only (few tiles are split).
constexpr uint64_t kMostLanes = 1ull << 31;
template <class Launch> int32_t batch_launches(Product p, uint32_t threads, Launch launch) {
    const uint64_t per = (uint64_t)p.ti * p.tj * p.splits, most = kMostLanes / threads / per;
    if (!most) return rt_fail(RT_E_INVALID, "pack8 matmul backward: the result is too large for one launch");
    for (; p.batch0 < p.b; p.batch0 += most) {
        launch(p, (uint32_t)((p.b - p.batch0 < most ? p.b - p.batch0 : most) * per));
        RT_HIP(hipGetLastError());
    }
    return RT_OK;
}

template <int BI, int BJ, int WI, int WJ, int DEPTH, bool EVEN> int32_t f32_launch(rt_ctx* ctx, const Product& p) {
    constexpr size_t bytes = 2 * sizeof(Stage<BI, BJ>);
    auto kernel = pack8_matmul_f32_kernel<BI, BJ, WI, WJ, DEPTH, EVEN>;
    static std::atomic<uint64_t> allowed{0};                     // more than 64 KiB of LDS has to be asked for, once a device
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (!(allowed.load() & bit) || ctx->device > 63) {
        RT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
        allowed.fetch_or(bit);
    }
    return batch_launches(p, WI * WJ * 64, [&](const Product& part, uint32_t blocks) {
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(WI * WJ * 64), bytes, ctx->stream, part);
    });
}

template <bool EVEN> int32_t f32_any(rt_ctx* ctx, const Product& p, int shape) {
    // steps that are on their way from memory: two, but for an odd k and its twice as many registers (65536 x 257 x 320 145 us with two,
    // 90 us with one; 65536 x 256 x 320 50.3 and 51.1 us)
    constexpr int kDepth = EVEN ? 2 : 1;
    if (shape == 0) return f32_launch<256, 256, 2, 4, 1, EVEN>(ctx, p);
    if (shape == 1) return f32_launch<256, 128, 4, 2, kDepth, EVEN>(ctx, p);
    return f32_launch<128, 128, 2, 2, kDepth, EVEN>(ctx, p);
}

int32_t run_product(rt_ctx* ctx, int dtype, Product p, void* dst) {
    struct Shape { uint64_t bi, bj, least_rows, per_cu; double rate; };
    // The tile's shape: the larger, the fewer conversions there are for each matrix instruction.  `rate` is what a shape reaches of the
    // first one's rate on a result it divides (16384 x 4096 x 4096, measured together: 1318, 1569 and 1765 us -- the smaller ones are better than that on
    // short shares, hence less weight); the shape with the least padded area at its rate is taken, of those that give every CU a block.
    static const Shape f32[3] = {{256, 256, 512, 1, 1.0}, {256, 128, 256, 1, 0.8}, {128, 128, 64, 2, 0.6}};
    static const Shape f64[2] = {{128, 128, 128, 2, 1.0}, {64, 64, 64, 4, 1.0}};
    auto tiles_of = [&](const Shape& s) { return p.b * ((p.k + s.bi - 1) / s.bi) * ((p.n + s.bj - 1) / s.bj); };
    int shape = dtype == RT_F64 && tiles_of(f64[0]) * (p.m / f64[0].least_rows) < (uint64_t)ctx->num_cus ? 1 : 0;
    Shape s = f64[shape & 1];
    if (dtype == RT_F32) {
        double best = 0;
        for (int c = 2; c >= 0; --c) {
            const uint64_t tiles = tiles_of(f32[c]), most = p.m / f32[c].least_rows, blocks = tiles * (most ? most : 1);
            if (c < 2 && blocks < (uint64_t)ctx->num_cus) continue;              // would not fill the card
            const double cost = (double)tiles * f32[c].bi * f32[c].bj / f32[c].rate;
            if (c == 2 || cost < best) { best = cost; shape = c; }
        }
        s = f32[shape];
    }
    const uint64_t tiles = tiles_of(s);
    p.ti = (uint32_t)((p.k + s.bi - 1) / s.bi);
    p.tj = (uint32_t)((p.n + s.bj - 1) / s.bj);
    const uint64_t n = p.b * p.k * p.n;
    p.splits = splits_for(ctx, tiles, p.m, s.least_rows, s.per_cu);
    p.out = dst;
    if (p.splits > 1) RT_TRY(rt_scratch(ctx, n * p.splits * rt_elem_size(dtype), &p.out));
    if (dtype == RT_F64) {
        RT_TRY(batch_launches(p, shape == 0 ? 512 : 256, [&](const Product& part, uint32_t blocks) {
            if (shape == 0) hipLaunchKernelGGL((pack8_matmul_f64_kernel<128, 4, 2>), dim3(blocks), dim3(512), 0, ctx->stream, part);
            else hipLaunchKernelGGL((pack8_matmul_f64_kernel<64, 2, 2>), dim3(blocks), dim3(256), 0, ctx->stream, part);
        }));
    } else {
        RT_TRY(p.k % 2 == 0 ? f32_any<true>(ctx, p, shape) : f32_any<false>(ctx, p, shape));
    }
    if (p.splits == 1) return RT_OK;
    return dtype == RT_F32 ? join<float>(ctx, p.out, dst, n, p.splits) : join<double>(ctx, p.out, dst, n, p.splits);
}

bool product(uint64_t a, uint64_t b, uint64_t c, uint64_t* out) {
    const uint64_t most = 1ull << 40;                           // elements: beyond any device memory
    *out = 0;
    if (!a || !b || !c) return true;
    if (a > most || b > most / a || c > most / (a * b)) return false;
    *out = a * b * c;
    return true;
}

}  // namespace

extern "C" int32_t rt_pack8_matmul_backward(rt_ctx* ctx, int32_t dtype, const void* codes, uint64_t codes_len, const void* exps, uint64_t exps_len,
                                            const void* upstream, uint64_t upstream_len, void* dst, uint64_t dst_len, uint64_t b, uint64_t m, uint64_t k,
                                            uint64_t n) {
    const char* what = "pack8 matmul backward";
    if (dtype != RT_F32 && dtype != RT_F64) return rt_fail(RT_E_DTYPE, "%s: f32 / f64 only", what);
    uint64_t nx, ny, nd;
    if (!product(b, m, k, &nx) || !product(b, m, n, &ny) || !product(b, k, n, &nd)) return rt_fail(RT_E_INVALID, "%s: sizes are too large", what);
    if (k >= (1ull << 25) || n >= (1ull << 25)) return rt_fail(RT_E_INVALID, "%s: k and n have to be below 2^25", what);
    const uint64_t groups = (nx + kP8Group - 1) / kP8Group;
    const int es = rt_elem_size(dtype);
    if (codes_len < nx || exps_len < groups) return rt_fail(RT_E_OUT_OF_BOUNDS, "%s: codes or exps are shorter than b * m * k elements need", what);
    if (upstream_len < ny) return rt_fail(RT_E_OUT_OF_BOUNDS, "%s: upstream is shorter than b * m * n", what);
    if (dst_len < nd) return rt_fail(RT_E_OUT_OF_BOUNDS, "%s: dst is shorter than b * k * n", what);
    if (!nd) return rt_ctx_enter(ctx);
    if (!dst || (nx && (!codes || !exps)) || (ny && !upstream)) return rt_fail(RT_E_INVALID, "%s: null buffer", what);
    if (reinterpret_cast<uintptr_t>(dst) % es || (ny && reinterpret_cast<uintptr_t>(upstream) % es))
        return rt_fail(RT_E_INVALID, "%s: an operand is not aligned to its elements", what);
    const ByteSpan ds = rt_run_span(dst, es, 0, nd);
    if ((ny && rt_spans_meet(ds, rt_run_span(upstream, es, 0, ny))) ||
        (nx && (rt_spans_meet(ds, rt_run_span(codes, 1, 0, nx)) || rt_spans_meet(ds, rt_run_span(exps, 1, 0, groups)))))
        return rt_fail(RT_E_INVALID, "%s: dst overlaps an input", what);
    RT_TRY(rt_ctx_enter(ctx));
    CtxGuard g(ctx);
    return run_product(ctx, dtype, Product{(const int8_t*)codes, (const uint8_t*)exps, upstream, nullptr, b, m, k, n, 0, 0, 1, 0}, dst);
}
