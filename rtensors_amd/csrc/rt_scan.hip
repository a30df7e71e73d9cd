// Gated linear recurrence along a dim and its backward pass (include/rt_hip.h has the formulas).
#include "rt_pack8.h"
#include "rt_unary_math.h"

#include <stddef.h>

#include <atomic>

namespace {

constexpr int kSBlock = 256;

// A load that is marked as touched once -- where the wave's stretch is a whole number of cache lines.  Rows that are no multiple of a line
// share lines between neighbouring columns' waves, and a line that is dropped after the first is fetched again: (1, 50000, 1111) f32
// forward 179 us with the mark, 158 us without; (1, 65536, 4096) 549 us with it, 558 us without.
template <bool ONCE, class T> __device__ __forceinline__ T once(const T* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(p);
    else return *p;
}

// The same for a store: the backward pass, with two outputs, gains from lines that wait in the L2 for their other half ((32, 1000, 1500)
// f32 284 -> 246 us, (1, 50000, 1111) from the 8-bit form 287 -> 279 us), the forward pass does not (158 -> 165 us), nor does f64, whose
// stretches are twice as long ((2, 8192, 1000) backward 166 -> 174 us).
template <bool ONCE, class T> __device__ __forceinline__ void put_once(T v, T* p) {
    if constexpr (ONCE) __builtin_nontemporal_store(v, p);
    else *p = v;
}

// x and h of the backward pass: whole values or the 8-bit form
template <class T> struct Whole {
    static constexpr bool kHeld = false;
    const T* p;
    // element i of the run that starts at `base` (wave-uniform; base + i does not leave the run, base alone may)
    template <bool ONCE = true> __device__ __forceinline__ T at(uint64_t base, uint32_t i) const { return once<ONCE>(p + base + i); }
};
template <class T> struct Held {
    static constexpr bool kHeld = true;
    const int8_t* codes;
    const uint8_t* exps;
    template <bool ONCE = true> __device__ __forceinline__ T at(uint64_t base, uint32_t i) const {
        const uint64_t e = base + i;
        return p8_value<T>(codes[e], exps[e / kP8Group]);
    }
};

template <class T> struct ScanArgs {
    const T *gate, *x, *state;
    const uint8_t* reset;
    T *h, *last;
    uint64_t outer, steps, inner;
    uint64_t col0;           // first column of a launch with one lane a column
};
template <class T, class S> struct BackArgs {
    const T* gate;
    S x, h;
    const T* state;
    const uint8_t* reset;
    const T *dh, *dlast;
    T *dgate, *dx, *dstate;
    uint64_t outer, steps, inner;
    uint64_t col0;
};

// One lane per column, the steps one after the other: for a token and a few steps more, where a launch is most of the time ((64, 1, 2048)
// f32 2.8 us in the kernel), and for so many columns that they fill the card ((2000, 8, 4096) f32 linear 149 us, 5.5 TB/s).
template <class T, int FORM>
__global__ __launch_bounds__(kSBlock) void scan_columns_kernel(ScanArgs<T> a) {
    const uint64_t col = a.col0 + (uint64_t)blockIdx.x * kSBlock + threadIdx.x;
    if (col >= a.outer * a.inner) return;
    const uint64_t o = col / a.inner, i = col - o * a.inner;
    T p = a.state ? a.state[col] : (T)0;
    bool none = !a.state;
    for (uint64_t t = 0; t < a.steps; ++t) {
        const uint64_t at = (o * a.steps + t) * a.inner + i;
        const bool cut = none || (a.reset && a.reset[o * a.steps + t]);
        const T g = a.gate[at], x = a.x[at];
        if constexpr (FORM == RT_SCAN_LINEAR) {
            p = cut ? x : g * p + x;
        } else {
            const RtGate<T> q = rt_gate_of(g);
            p = cut ? q.r * x : q.s * p + q.r * x;
        }
        a.h[at] = p;
        none = false;
    }
    if (a.last) a.last[col] = p;
}

template <class T, int FORM, class S>
__global__ __launch_bounds__(kSBlock) void scan_backward_columns_kernel(BackArgs<T, S> a) {
    const uint64_t col = a.col0 + (uint64_t)blockIdx.x * kSBlock + threadIdx.x;
    if (col >= a.outer * a.inner) return;
    const uint64_t o = col / a.inner, i = col - o * a.inner;
    T carry = a.dlast ? a.dlast[col] : (T)0;          // a[t + 1] * D[t + 1]
    for (uint64_t t = a.steps; t-- > 0;) {
        const uint64_t at = (o * a.steps + t) * a.inner + i;
        const bool cut = a.reset && a.reset[o * a.steps + t];
        const bool none = cut || (t == 0 && !a.state);
        const T d = a.dh[at] + carry;
        const T g = a.gate[at];
        const T p = none ? (T)0 : (t == 0 ? a.state[col] : a.h.at(at - a.inner, 0));
        if constexpr (FORM == RT_SCAN_LINEAR) {
            a.dgate[at] = none ? (T)0 : d * p;
            a.dx[at] = d;
            carry = cut ? (T)0 : g * d;
        } else {
            const RtGate<T> q = rt_gate_of(g);
            const T x = a.x.at(at, 0);
            a.dgate[at] = d * (p - x) * (q.s * q.r);
            a.dx[at] = q.r * d;
            carry = cut ? (T)0 : q.s * d;
        }
    }
    if (a.dstate) a.dstate[col] = carry;
}

// ---- tiles along the steps ---------------------------------------------------------------------------------------------------------
// A prefix scan in one pass with look-back to the tiles before ("Single-pass Parallel Prefix Scan with Decoupled Look-back", Merrill and
// Garland, 2016), of pairs.
// Two stretches of the recurrence join as (A1, H1), (A2, H2) -> (A1 A2, A2 H1 + H2): A is the product of a stretch's factors, H what
// it ends at from a state of zero.  A block takes a tile of the steps for 64 columns, holds it in registers, and needs one thing from
// the tiles before: the state it starts from.  So that the data are read once, the tiles of a column run in the same launch and hand
// states on through words in memory: a tile publishes (A, H) as soon as it has them, and its end state once it knows its start; a
// tile that starts looks at the kWindow tiles before it, takes the nearest end state that is there, and goes through the (A, H) from
// there on.  An end state is always A * start + H of its own tile, however many tiles it was found over, so the bits do not depend on
// which block ran when.
//
// Every wait ends: the tiles of a line of columns are numbered by the line's counter as blocks start, all tiles a block waits for have
// lower numbers, so they have started, and the lowest unfinished one waits for nobody.  (One counter for the whole launch costs 45 ns a
// block, an atomic operation on one address from eight XCDs: 16384 tiles took 1441 us.)
//
// A word is 32 bits of a value and a tag, written and read as one 64-bit access at device scope: a word with the right tag is valid by
// itself, with no order between words.  Tags hold the launch's number and are not cleared between launches.  The number comes from the
// host, so a launch must not be replayed from a graph; none can be: the context's stream is its own, and nothing here captures it.
struct Chain {
    uint32_t* tickets;       // one counter a line, 64 bytes apart, 0 between launches
    uint64_t* words;
    uint32_t tiles;          // along the steps
    uint32_t lines;          // sets of columns that are chained on their own
    uint32_t line0;          // the first of them in the operands: a launch takes no more than its lanes can be numbered for
    uint32_t epoch;          // the launch's number, below kEpochs
    uint32_t rounds;         // blocks a line gets: `tiles`, or the next multiple of 8
};
constexpr uint32_t kTicketPitch = 16;
constexpr uint32_t kAgg = 1, kEnd = 2;                           // what a slot holds: (A, H), or the end state in place of H
// A tag: 17 bits of the launch's number, 13 of A's exponent (0 in the words of H), 2 of what the slot holds.
constexpr uint32_t kEpochs = 1u << 17;
constexpr int kTagExponent = 4095;
__device__ __forceinline__ uint32_t tag_of(uint32_t epoch, uint32_t kind, int e = 0) { return epoch << 15 | ((uint32_t)e & 0x1fffu) << 2 | kind; }
__device__ __forceinline__ uint32_t tag_epoch(uint32_t tag) { return tag >> 15; }
__device__ __forceinline__ uint32_t tag_kind(uint32_t tag) { return tag & 3u; }
__device__ __forceinline__ int tag_exponent(uint32_t tag) { return (int)(tag << 17) >> 19; }

__device__ __forceinline__ void put_word(uint64_t* p, uint32_t bits, uint32_t tag) {
    __hip_atomic_store(p, (uint64_t)tag << 32 | bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t get_word(const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

template <class T> struct Slot {
    static constexpr int kHalves = sizeof(T) / 4;
    static constexpr uint32_t kWords = 2 * kHalves * 64;         // per tile: H and A of 64 lanes
    uint64_t w[2 * kHalves];
    static __device__ __forceinline__ uint64_t* at(const Chain& c, uint32_t item) { return c.words + (uint64_t)item * kWords; }
    static __device__ __forceinline__ void put(uint64_t* base, int which, T v, uint32_t tag) {
        if constexpr (kHalves == 1) {
            put_word(base + which * 64, __builtin_bit_cast(uint32_t, v), tag);
        } else {
            const uint64_t b = __builtin_bit_cast(uint64_t, v);
            put_word(base + (which * 2) * 64, (uint32_t)b, tag);
            put_word(base + (which * 2 + 1) * 64, (uint32_t)(b >> 32), tag);
        }
    }
    __device__ __forceinline__ void get(const uint64_t* base) {
#pragma unroll
        for (int k = 0; k < 2 * kHalves; ++k) w[k] = get_word(base + k * 64);
    }
    // 0: not there (yet); the halves of a value may come from two writes, then it is read again
    __device__ __forceinline__ uint32_t kind(uint32_t epoch) const {
        const uint32_t t = (uint32_t)(w[0] >> 32);
        bool ok = tag_epoch(t) == epoch;
        if constexpr (kHalves == 2) ok = ok && (uint32_t)(w[1] >> 32) == t;
        const uint32_t k = tag_kind(t);
        if (k == kAgg) {
#pragma unroll
            for (int j = kHalves; j < 2 * kHalves; ++j) {
                const uint32_t a = (uint32_t)(w[j] >> 32);
                ok = ok && tag_epoch(a) == epoch && tag_kind(a) == kAgg;
            }
        }
        return ok ? k : 0u;
    }
    __device__ __forceinline__ int exponent() const { return tag_exponent((uint32_t)(w[kHalves] >> 32)); }
    __device__ __forceinline__ T value(int which) const {
        if constexpr (kHalves == 1) return __builtin_bit_cast(float, (uint32_t)w[which]);
        else return __builtin_bit_cast(double, (uint64_t)(uint32_t)w[which * 2 + 1] << 32 | (uint32_t)w[which * 2]);
    }
};

// rt_gate_of for f32 in about half the instructions: the hardware's 2^x with the rounding of x log2 e put right (1.5 ulp; results below
// the normal range are 0), and its reciprocal refined once.
__device__ __forceinline__ RtGate<double> gate_of(double g) { return rt_gate_of(g); }
__device__ __forceinline__ RtGate<float> gate_of(float g) {
    float t = g < 0.0f ? g : -g;
    t = t < -200.0f ? -200.0f : t;                               // -inf would make the correction below inf - inf; NaN stays
    const float p = t * 0x1.715476p+0f;                          // log2 e = this + 0x1.4ae0c0p-26
    const float q = __builtin_fmaf(t, 0x1.4ae0c0p-26f, __builtin_fmaf(t, 0x1.715476p+0f, -p));
    const float e0 = __builtin_amdgcn_exp2f(p);
    const float e = __builtin_fmaf(e0, q * 0x1.62e430p-1f, e0);
    const float d = 1.0f + e;
    const float i0 = __builtin_amdgcn_rcpf(d);
    const float inv = __builtin_fmaf(__builtin_fmaf(-d, i0, 1.0f), i0, i0);
    const float low = e * inv;
    return g < 0.0f ? RtGate<float>{low, inv} : RtGate<float>{inv, low};
}

__device__ __forceinline__ float fused(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return __builtin_fma(a, b, c); }
__device__ __forceinline__ bool finite(float v) { return __builtin_fabsf(v) < __builtin_inff(); }
__device__ __forceinline__ bool finite(double v) { return __builtin_fabs(v) < __builtin_inf(); }
__device__ __forceinline__ bool infinite(float v) { return __builtin_fabsf(v) == __builtin_inff(); }
__device__ __forceinline__ bool infinite(double v) { return __builtin_fabs(v) == __builtin_inf(); }

__device__ __forceinline__ float mantissa(float v) { return __builtin_amdgcn_frexp_mantf(v); }
__device__ __forceinline__ double mantissa(double v) { return __builtin_amdgcn_frexp_mant(v); }
__device__ __forceinline__ int exponent(float v) { return __builtin_amdgcn_frexp_expf(v); }
__device__ __forceinline__ int exponent(double v) { return __builtin_amdgcn_frexp_exp(v); }
__device__ __forceinline__ float with_sign(float v, float of) { return __builtin_copysignf(v, of); }
__device__ __forceinline__ double with_sign(double v, double of) { return __builtin_copysign(v, of); }
__device__ __forceinline__ float scaled(float v, int e) { return __builtin_ldexpf(v, e); }
__device__ __forceinline__ double scaled(double v, int e) { return __builtin_ldexp(v, e); }

// The product A of a stretch's factors.
// Those of the sigmoid form are at most 1: nothing lifts a product again that falls below the range, and none goes above it.
template <class T> struct Falling {
    static constexpr bool kApart = false;
    T m;
    static __device__ __forceinline__ Falling of(T f) { return {f}; }
    __device__ __forceinline__ T on(T c, T h) const { return fused(m, c, h); }           // A c + h
};
// Those of the linear form may be above 1 behind others far below it: a state of 2^100 times 2^-200 and then 2^150 is 2^50.  A product below
// the normal range is held as m 2^e, m at the range's lower end and e < 0; any other one as it is, with e = 0.  An infinite m says that a
// prefix of the stretch is above the range, or a factor infinite; such a tile runs step by step.  NaN says that a factor is NaN: behind it the
// plain loop's state is NaN as well.
template <class T> struct Apart {
    static constexpr bool kApart = true;
    static constexpr T kNormal = sizeof(T) == 4 ? (T)0x1p-126 : (T)0x1p-1022;
    static constexpr int kLow = sizeof(T) == 4 ? -125 : -1021, kTop = sizeof(T) == 4 ? 128 : 1024;
    static constexpr int kDead = sizeof(T) == 4 ? -300 : -2200;  // below, A c is 0 for every number c (an infinite one stays infinite)
    T m;
    int e;
    static __device__ __forceinline__ Apart of(T f) { return {f, 0}; }
    // m 2^e of any m and e (above the range, e > 0: where a tile's product sinks below the range first, which no wave's own does)
    static __device__ __forceinline__ Apart from(T m, int e) {
        const int at = m == (T)0 ? 0 : e + exponent(m), near = at < kLow ? kLow : at > kTop ? kTop : at;   // 0 times what leaves the range is NaN
        return {scaled(mantissa(m), near), at - near};
    }
    __device__ __forceinline__ T on(T c, T h) const { return fused(m, scaled(c, e), h); }
};
template <class T, int FORM> using ProductOf = typename std::conditional<FORM == RT_SCAN_LINEAR, Apart<T>, Falling<T>>::type;

// The product of the factors that a lane goes through, multiplied as they come; where a prefix in the wave fell below the range (or a factor
// is 0), once more with the exponents apart.  (Exponents apart in every step: 64 us in place of 51 on (2048, 4097, 1) f64.)
__device__ __forceinline__ float least(float a, float b) { return __builtin_fminf(a, __builtin_fabsf(b)); }
__device__ __forceinline__ double least(double a, double b) { return __builtin_fmin(a, __builtin_fabs(b)); }
template <class T, class P> struct Running {
    T m = (T)1, low = (T)1;
    __device__ __forceinline__ void by(T f) {
        m *= f;
        if constexpr (P::kApart) low = least(low, m);
    }
    // factor(j) and term(j), the first n of L, give the product and the sum H from a start of zero.  odd: a prefix of the product is above the
    // range, or nearly, or a factor is infinite; or, with SUMS, H left the range with finite terms and factors: the plain loop's state
    // need not have.  From a term on that is not finite it has, too; and where the stretch is cut, H is its state.
    template <bool SUMS, int L, class F, class G> __device__ __forceinline__ P whole(T H, bool cut, int n, F factor, G term, bool* odd) const {
        P a = P::of(m);
        bool over = SUMS && !cut && !finite(H), fell = false;
        *odd = false;
        if constexpr (P::kApart) fell = low < P::kNormal || !finite(m);
        if ((SUMS || P::kApart) && __any(over || fell)) {
            if constexpr (P::kApart)
                if (__any(fell)) {
                    T p = (T)1;
                    int e = 0;
#pragma unroll
                    for (int j = 0; j < L; ++j)
                        if (j < n) {
                            p *= mantissa(factor(j));
                            e += exponent(factor(j));
                            *odd = *odd || e > P::kTop || infinite(factor(j));
                        }
                    a = P::from(p, e);
                }
            if (SUMS && __any(over)) {
                T h = (T)0;
                bool first = false;
#pragma unroll
                for (int j = 0; j < L; ++j)
                    if (j < n) {
                        const T q = j == 0 ? term(j) : fused(factor(j), h, term(j));
                        first = first || (j > 0 && finite(factor(j)) && finite(h) && finite(term(j)) && !finite(q));
                        h = q;
                    }
                *odd = *odd || (over && first);
            }
            *odd = *odd && !cut;
        }
        return a;
    }
};

// LN: lanes that hold different columns; with 32 the upper half of a wave repeats the lower one.
template <class T, int W, int LN, class P> struct JoinRoom {
    // tiles before its own that a tile looks at (f64: as many as leave room for the blocks that the registers allow)
    static constexpr int kWindow = W <= 2 ? 1 : sizeof(T) == 4 || W == 16 ? 16 : LN == 32 && W == 8 ? 4 : 8;
    T A[W][LN], H[W][LN];
    union {
        T start[LN];                                             // of serial tiles, which need no products
        int16_t E[P::kApart ? W : 1][LN];
    };
    T winA[kWindow][LN], winH[kWindow][LN];
    int16_t winE[P::kApart ? kWindow : 1][LN];
    uint64_t ends[P::kApart ? 1 : kWindow];
    uint32_t cut[W];                                             // 1: cut, 2: odd, 4: deep
    uint32_t tile;
    int found;
    // a wave's product and its exponent: that of m 2^e as a whole, kNone for 0 and NaN, and those from -2^15 on are all the same: the other
    // waves of a tile lift no state again that far
    static constexpr int kNone = 32767;
    __device__ __forceinline__ void put(int w, int l, const P& a) {
        A[w][l] = a.m;
        if constexpr (P::kApart) {
            const int e = a.m == (T)0 || a.m != a.m ? kNone : a.e + exponent(a.m);
            E[w][l] = (int16_t)(e < -32768 ? -32768 : e);
        }
    }
    __device__ __forceinline__ P get(int w, int l) const {
        if constexpr (P::kApart) {
            const int e = E[w][l] - P::kLow;
            return P{A[w][l], e < 0 ? e : 0};
        } else {
            return P{A[w][l]};
        }
    }
};
constexpr int16_t kEnded = 0x7fff;                               // in place of an exponent: H is the end state

// The end state of tile k - 1 for this lane's column, for all waves of the block.  Waiting is done by one wave on one word of each of the
// tiles in the window, read by one lane each: polling whole slots takes the bandwidth that the tiles being waited for need.  Then the
// waves read the slots between them, again where not all of their words are there yet, and go through them from the farthest.
template <class T, int W, int LN, class P> __device__ __forceinline__ T chain_start(const Chain& ch, JoinRoom<T, W, LN, P>& room, uint32_t item, uint32_t k, int w, int lane) {
    constexpr int kWindow = JoinRoom<T, W, LN, P>::kWindow, kEach = (kWindow + W - 1) / W;
    if (w == 0) {
        const int n = k < (uint32_t)kWindow ? (int)k : kWindow;
        int found;                                               // nearest tile with an end state, all nearer ones having (A, H)
        for (;;) {
            uint32_t tag = 0;
            if (lane < n) tag = (uint32_t)(get_word(Slot<T>::at(ch, item - (uint32_t)(lane + 1) * ch.lines)) >> 32);
            const bool mine = lane < n && tag_epoch(tag) == ch.epoch;
            const uint64_t ends = __ballot(mine && tag_kind(tag) == kEnd), aggs = __ballot(mine && tag_kind(tag) == kAgg);
            found = ends ? (int)__builtin_ctzll(ends) : -1;
            if (found >= 0 && (~aggs & ((1ull << found) - 1)) == 0) break;
            __builtin_amdgcn_s_sleep(2);
        }
        if (lane == 0) room.found = found;
    }
    __syncthreads();
    const int found = __builtin_amdgcn_readfirstlane(room.found);
    Slot<T> s[kEach];
    for (;;) {
        bool ok = true;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (w + i * W <= found) s[i].get(Slot<T>::at(ch, item - (uint32_t)(w + i * W + 1) * ch.lines) + lane);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (w + i * W <= found) {
                const uint32_t kind = s[i].kind(ch.epoch);
                ok = ok && (kind == kEnd || (kind == kAgg && w + i * W < found));
            }
        if (__all(ok)) break;
        __builtin_amdgcn_s_sleep(1);
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int q = w + i * W;
        if (q <= found) {
            // an end state may have taken the place of a nearer tile's (A, H) meanwhile
            const bool ended = s[i].kind(ch.epoch) == kEnd;
            const uint64_t ends = __ballot(ended);
            if (lane < LN) {                                     // the lanes that repeat these may have read it before, these after
                room.winH[q][lane] = s[i].value(0);
                room.winA[q][lane] = s[i].value(1);
                if constexpr (P::kApart) room.winE[q][lane] = ended ? kEnded : (int16_t)s[i].exponent();
            }
            if constexpr (!P::kApart)
                if (lane == 0) room.ends[q] = ends;
        }
    }
    __syncthreads();
    T c = (T)0;
#pragma unroll 1
    for (int q0 = found; q0 >= 0; q0 -= 4) {                     // four at a time are read before the first is used
        T A[4], H[4];
        uint64_t ends[4];
        int e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int q = q0 - i < 0 ? 0 : q0 - i;
            A[i] = room.winA[q][lane & (LN - 1)];
            H[i] = room.winH[q][lane & (LN - 1)];
            if constexpr (P::kApart) e[i] = room.winE[q][lane & (LN - 1)];
            else ends[i] = room.ends[q];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (q0 - i >= 0) {
                if constexpr (P::kApart) c = e[i] == kEnded ? H[i] : P{A[i], e[i]}.on(c, H[i]);
                else c = ends[i] >> (lane & (LN - 1)) & 1 ? H[i] : fused(A[i], c, H[i]);
            }
    }
    return c;
}

// The line a block works on.  Blocks go to the eight XCDs in turn, each with an L2 of its own, and lines that are neighbours in memory
// share the cache lines at their borders (all of them where rows are no multiple of 128 bytes): every XCD goes through all lines in
// order, so that neighbouring lines mostly get the same tile in the same L2.  SPREAD: the XCDs start an eighth of the lines apart, else
// all at the first.  Forward over (1, 65536, 4096) f32 545 us spread, 575 us not; backward over (8, 2048, 2048) 154 and 146 us, over
// (32, 1000, 1500), rows of no whole lines, 246 and 271 us.
template <bool SPREAD> __device__ __forceinline__ uint32_t line_of_block(const Chain& ch) {
    const uint32_t b = blockIdx.x;
    if (ch.rounds % 8 != 0 || ch.tiles == 1) return b % ch.lines;
    return (b / 8 + (SPREAD ? (uint32_t)((uint64_t)(b % 8) * ch.lines / 8) : 0u)) % ch.lines;
}
// The block's tile among those of its line (one that is not there for the blocks too many); whoever takes the last one leaves the counter
// as the next launch needs it.
template <class T, int W, int LN, class P> __device__ __forceinline__ uint32_t take_tile(const Chain& ch, uint32_t line, JoinRoom<T, W, LN, P>& room) {
    if (ch.tiles == 1) return 0;
    if (threadIdx.x == 0) {
        uint32_t* c = ch.tickets + (uint64_t)line * kTicketPitch;
        const uint32_t t = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (t == ch.rounds - 1) __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        room.tile = t;
    }
    __syncthreads();
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)room.tile);
}

// Joins the W stretches of a tile (one a wave, in the order of the waves) with the tiles before it.  (A, H) of the wave's own stretch;
// cut: nothing crosses the stretch (wave-uniform; A has no meaning then); odd: a product inside the stretch left the range (see below);
// first: the state before tile 0.  `run(start, serial)` goes through the stretch from its start state and returns the state it ends at;
// so does this function.
//
// A product of factors above 1 can leave the range while the states stay inside it (a start of zero, say), and so can the sum from a start
// of zero (a state of -c, and x of c twice).  Where one does, the tile's stretches run one after the other and only its end state is
// published: the plain loop's result, at the plain loop's pace.  SUMS: whether the sums are looked at.  Those of the forward sigmoid form are
// averages of x, which leave the range only where x has.  A sum with a term that is not finite does not count: the plain loop has it too.
template <class T, int W, int LN, bool SUMS, class P, class Run>
__device__ __forceinline__ T join_tile(const Chain& ch, JoinRoom<T, W, LN, P>& room, uint32_t item, uint32_t k, const P& A, T H, bool cut, bool odd, T first, Run run) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const bool last = k == ch.tiles - 1;
    room.put(w, lane & (LN - 1), A);
    room.H[w][lane & (LN - 1)] = H;
    bool deep = false;
    if constexpr (P::kApart) deep = !cut && __any(A.e < 0);
    if (lane == 0) room.cut[w] = (cut ? 1u : 0u) | (odd ? 2u : 0u) | (deep ? 4u : 0u);
    __syncthreads();
    const uint32_t epoch = ch.epoch;
    if constexpr (P::kApart) deep = __any((room.cut[lane & (W - 1)] & 4u) != 0);         // from here on: of the tile
    T ta = (T)1, th = (T)0, low = (T)1;
    bool tcut = false, bad = false, wild = false;
    if (!deep) {
#pragma unroll
        for (int v = 0; v < W; ++v) {
            const T av = room.A[v][lane & (LN - 1)], hv = room.H[v][lane & (LN - 1)];
            bad = bad || (room.cut[v] & 2u);
            if (room.cut[v] & 1u) {
                th = hv;
                tcut = true;
            } else {
                th = v == 0 ? hv : fused(av, th, hv);
                bad = bad || infinite(av);
                wild = wild || (SUMS && !finite(th));
                if (!tcut) {
                    ta = v == 0 ? av : ta * av;
                    if constexpr (P::kApart) low = least(low, ta);
                    bad = bad || infinite(ta);
                }
            }
        }
    } else if constexpr (P::kApart) {
#pragma unroll
        for (int v = 0; v < W; ++v) {
            const P av = room.get(v, lane & (LN - 1));
            const T hv = room.H[v][lane & (LN - 1)];
            bad = bad || (room.cut[v] & 2u);
            if (room.cut[v] & 1u) {
                th = hv;
                tcut = true;
            } else {
                th = v == 0 ? hv : av.on(th, hv);
                bad = bad || infinite(av.m);
                wild = wild || (SUMS && !finite(th));
                if (!tcut) {
                    ta = v == 0 ? av.m : ta * av.m;
                    if constexpr (P::kApart) low = least(low, ta);
                    bad = bad || infinite(ta);
                }
            }
        }
    }
    bool serial = __any(bad || wild);                            // the same in all waves: they look at the same numbers
    if (SUMS && serial) {                                        // a sum of finite terms?  A wave's own is looked at by the wave
        T p = (T)0;
#pragma unroll 1
        for (int v = 0; v < W; ++v) {
            const T av = room.A[v][lane & (LN - 1)], hv = room.H[v][lane & (LN - 1)];
            const T q = v == 0 || (room.cut[v] & 1u) ? hv : deep ? room.get(v, lane & (LN - 1)).on(p, hv) : fused(av, p, hv);
            bad = bad || (!finite(q) && finite(p) && finite(hv) && av == av);
            p = q;
        }
        serial = __any(bad);
    }
    uint64_t* slot = last ? nullptr : Slot<T>::at(ch, item) + lane;
    T start = first;
    P whole = P::of(ta);
    if constexpr (P::kApart)
        if (w == 0 && !last && !serial && !tcut && (deep || __any(low < P::kNormal))) {  // with the exponents apart
            int e = 0;
            bool none = false;                                   // 0 or NaN, of which something is left
#pragma unroll
            for (int v = 0; v < W; ++v) {
                const int ev = room.E[v][lane & (LN - 1)];
                e += ev;
                none = none || ev == room.kNone;
            }
            whole = {with_sign(P::kNormal, ta), e};              // nothing is left of any number
            if (__any(e > P::kDead || none)) {
                T p = (T)1;
                e = 0;
#pragma unroll 4
                for (int v = 0; v < W; ++v) {
                    const P av = room.get(v, lane & (LN - 1));
                    p *= mantissa(av.m);
                    e += exponent(av.m) + av.e;
                }
                whole = P::from(p, e);
            }
        }
    if (w == 0 && !last && !serial) {
        if (tcut) Slot<T>::put(slot, 0, th, tag_of(epoch, kEnd));
        else if (k == 0) Slot<T>::put(slot, 0, whole.on(first, th), tag_of(epoch, kEnd));
        else {
            // beyond kTagExponent, exponents are all the same to a state: nothing is left of it, or it is infinite
            int e = 0;
            if constexpr (P::kApart) e = whole.e < -kTagExponent ? -kTagExponent : whole.e > kTagExponent ? kTagExponent : whole.e;
            Slot<T>::put(slot, 1, whole.m, tag_of(epoch, kAgg, e));
            Slot<T>::put(slot, 0, th, tag_of(epoch, kAgg));
        }
    }
    if (W > 1 && k > 0) {                                        // a tile of one wave is the only one of its line
        start = chain_start(ch, room, item, k, w, lane);
        if (w == 0 && !last && !serial && !tcut) Slot<T>::put(slot, 0, whole.on(start, th), tag_of(epoch, kEnd));
    }
    if (serial) {
        __syncthreads();                                         // the room of the start is that of the exponents
        if (w == 0) room.start[lane & (LN - 1)] = start;
        __syncthreads();
    }
    T end = (T)0;
    for (int turn = 0; turn < (serial ? W : 1); ++turn) {
        if (!serial || turn == w) {
            if (serial) start = room.start[lane & (LN - 1)];
            else {
                if (deep) {
                    for (int v = 0; v < w; ++v) start = room.cut[v] & 1u ? room.H[v][lane & (LN - 1)] : room.get(v, lane & (LN - 1)).on(start, room.H[v][lane & (LN - 1)]);
                } else {
                    for (int v = 0; v < w; ++v) start = room.cut[v] & 1u ? room.H[v][lane & (LN - 1)] : fused(room.A[v][lane & (LN - 1)], start, room.H[v][lane & (LN - 1)]);
                }
            }
            end = run(start, serial);
            if (serial) room.start[lane & (LN - 1)] = end;
        }
        if (serial) __syncthreads();
    }
    if (serial && w == 0 && !last) Slot<T>::put(slot, 0, room.start[lane & (LN - 1)], tag_of(epoch, kEnd));
    return end;
}

// Bits 0 .. n - 1: whether the steps at flags[0], flags[stride], ... are reset.  n <= 64, all lanes of the wave.
__device__ __forceinline__ uint64_t reset_bits(const uint8_t* flags, int64_t stride, int n, int lane) {
    return __ballot(lane < n && flags[(int64_t)lane * stride] != 0);
}

// Copies of what a wave's second run through its steps takes from the first, which the compiler does not know to be the same: it would
// keep every address and every condition of the first run in a register until the second.
#define RT_APART                        \
    int rn = n;                         \
    uint64_t rcuts = cuts;              \
    uint32_t rrow = row;                \
    RT_PIN(rn);                         \
    RT_PIN(rcuts);                      \
    RT_PIN(rrow)

// Every wave of the first tile has its state before any of them hands one on: the last tile may write over the state's buffer.
#define RT_PIN_LANE(v) asm volatile("" : "+v"(v))

// W waves of 64 columns, L steps each, in registers: 2 L values a lane, all of them loaded before the first is used, so that the one pass
// over the data is bound by HBM: (1, 65536, 4096) f32 linear 542 us, 5.9 TB/s; (1, 8192, 1024) sigmoid 22 us, of which about 7 are the launch and the
// chain.  Shorter or longer tiles lose to more joins or to fewer blocks.  Lanes behind the last column load what the last column holds, and
// neither use nor store it.
template <class T, int FORM, int W, int L, bool ALIGNED>
__global__ __launch_bounds__(W * 64) void scan_wide_kernel(ScanArgs<T> a, Chain ch, uint32_t col_blocks) {
    typedef ProductOf<T, FORM> P;
    __shared__ JoinRoom<T, W, 64, P> room;
    const uint32_t line = line_of_block<true>(ch), k = take_tile(ch, line, room), item = k * ch.lines + line, at_line = ch.line0 + line, o = at_line / col_blocks;
    if (k >= ch.tiles) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t row = (uint32_t)a.inner, col0 = (at_line - o * col_blocks) * 64, col = col0 + lane;
    const bool in = col < row;
    const uint32_t lc = in ? lane : row - 1 - col0;
    const uint64_t t0 = ((uint64_t)k * W + w) * L;
    const int n = t0 >= a.steps ? 0 : (a.steps - t0 < (uint64_t)L ? (int)(a.steps - t0) : L);   // steps of this wave
    const uint64_t base = ((uint64_t)o * a.steps + t0) * row + col0;                            // wave-uniform
    const uint64_t sc = (uint64_t)o * row + col0 + lc;                                          // the column in (outer, inner)
    T f[L], b[L], H = (T)0;
    P A = P::of((T)1);
    bool odd = false;
    uint64_t cuts = t0 == 0 && !a.state ? 1 : 0;
    if (n) {
        const T *gate = a.gate + base, *x = a.x + base;
        if (n == L) {
#pragma unroll
            for (int j = 0; j < L; ++j) {
                f[j] = once<ALIGNED>(gate + (lc + (uint32_t)j * row));
                b[j] = once<ALIGNED>(x + (lc + (uint32_t)j * row));
            }
        } else {
#pragma unroll
            for (int j = 0; j < L; ++j) {
                f[j] = b[j] = (T)0;
                if (j < n) {
                    f[j] = once<ALIGNED>(gate + (lc + (uint32_t)j * row));
                    b[j] = once<ALIGNED>(x + (lc + (uint32_t)j * row));
                }
            }
        }
        if (a.reset) cuts |= reset_bits(a.reset + (uint64_t)o * a.steps + t0, 1, n, lane);
        Running<T, P> run;
#pragma unroll
        for (int j = 0; j < L; ++j) {
            if constexpr (FORM == RT_SCAN_SIGMOID) {
                const RtGate<T> q = gate_of(f[j]);
                f[j] = q.s;
                b[j] = q.r * b[j];
            }
            if (j < n) {
                H = j == 0 || (cuts >> j & 1) ? b[j] : fused(f[j], H, b[j]);
                run.by(f[j]);
            }
        }
        A = run.template whole<FORM == RT_SCAN_LINEAR, L>(H, cuts != 0, n, [&](int j) { return f[j]; }, [&](int j) { return b[j]; }, &odd);
    }
    T first = k == 0 && a.state ? a.state[sc] : (T)0;
    RT_PIN_LANE(first);
    T* h = a.h + base;
    const T end = join_tile<T, W, 64, FORM == RT_SCAN_LINEAR>(ch, room, item, k, A, H, cuts != 0, __any(odd), first, [&](T p, bool) {
        RT_APART;
        if (in) {
#pragma unroll
            for (int j = 0; j < L; ++j) {
                if (j < rn) {
                    p = rcuts >> j & 1 ? b[j] : fused(f[j], p, b[j]);
                    __builtin_nontemporal_store(p, h + (uint32_t)(lane + j * rrow));
                }
            }
        }
        return p;
    });
    if (a.last && in && n && t0 + n == a.steps) a.last[sc] = end;
}

// What a wave's L rows of 64 columns of a tensor in the 8-bit form take in LDS: the codes, and of each row the exponent bytes of the (at
// most three) groups that its 64 columns lie in.  Four lanes a row load 16 codes and one exponent byte each, so the rows of a wave come
// with two loads instead of two a step, and hold no registers until they are used.
struct HeldRegs {
    rt_u32x4 codes;
    uint32_t exp;
};
template <int L> struct HeldRows {
    alignas(16) uint8_t codes[L][64];
    uint8_t exps[L][4];
    // rows begin at `first + r * row` (wave-uniform; r from `skip` to n - 1); `total` elements in all
    template <class T> static __device__ __forceinline__ HeldRegs load(const Held<T>& h, uint64_t first, uint32_t row, int n, int skip, uint64_t total, int lane) {
        HeldRegs v = {{0u, 0u, 0u, 0u}, 0u};
        const int r = lane >> 2, c = lane & 3;
        if (r >= skip && r < n) {
            const uint64_t start = first + (uint64_t)((uint32_t)r * row), at = start + c * 16, g = start / kP8Group + c;
            if (at + 16 <= total) v.codes = rt_ld16u<int8_t, false>(h.codes + at);
            else
                for (int b = 0; b < 16; ++b)                     // the last rows of the tensor
                    if (at + b < total) v.codes[b >> 2] |= (uint32_t)(uint8_t)h.codes[at + b] << (8 * (b & 3));
            if (g * kP8Group < total) v.exp = h.exps[g];
        }
        return v;
    }
    __device__ __forceinline__ void put(const HeldRegs& v, int lane) {
        const int r = lane >> 2, c = lane & 3;
        if (r < L) {
            *reinterpret_cast<rt_u32x4*>(&codes[r][c * 16]) = v.codes;
            exps[r][c] = (uint8_t)v.exp;
        }
    }
    // element `lane` of row r, which begins at `start` (wave-uniform)
    template <class T> __device__ __forceinline__ T get(int r, uint32_t start, int lane) const {
        return p8_value<T>((int8_t)codes[r][lane], exps[r][(start % kP8Group + lane) / kP8Group]);
    }
};
struct NoRows {};

// The same backward, five values a step in registers, so half the steps: (8, 2048, 2048) f32 sigmoid 147 us, 5.5 TB/s; from the 8-bit form
// (1, 50000, 1088) 196 us, 5.0 TB/s, and (1, 50000, 1111) 277 us: there a wave's 64 columns touch three cache lines a row in place of two, two
// code lines in place of one, and neighbours share few of them (1.7 times the reads).  Position r counts from the last step.  A state's gradient D comes to a step from the one behind it (r - 1) times
// that one's gate.
template <class T, int FORM, class S, int W, int L, bool ALIGNED>
__global__ __launch_bounds__(W * 64) void scan_backward_wide_kernel(BackArgs<T, S> a, Chain ch, uint32_t col_blocks) {
    typedef ProductOf<T, FORM> P;
    __shared__ JoinRoom<T, W, 64, P> room;
    constexpr bool kHeld = S::kHeld, kSigmoid = FORM == RT_SCAN_SIGMOID;
    typedef typename std::conditional<kHeld, HeldRows<L>, NoRows>::type Rows;
    __shared__ Rows hrows[W], xrows[kSigmoid ? W : 1];
    const uint32_t line = line_of_block<!ALIGNED>(ch), k = take_tile(ch, line, room), item = k * ch.lines + line, at_line = ch.line0 + line, o = at_line / col_blocks;
    if (k >= ch.tiles) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t row = (uint32_t)a.inner, col0 = (at_line - o * col_blocks) * 64, col = col0 + lane;
    const bool in = col < row;
    const uint32_t lc = in ? lane : row - 1 - col0;
    const uint64_t r0 = ((uint64_t)k * W + w) * L;
    const int n = r0 >= a.steps ? 0 : (a.steps - r0 < (uint64_t)L ? (int)(a.steps - r0) : L);
    const uint64_t tl = n ? a.steps - 1 - r0 : 0, te = n ? tl + 1 - n : 0;                      // the wave's last and earliest step
    const bool top = te == 0;
    const uint64_t base = ((uint64_t)o * a.steps + te) * row + col0;                            // of the earliest step: j is n - 1 - j rows on
    const uint64_t sc = (uint64_t)o * row + col0 + lc;
    T g[L], up[L], hp[kHeld ? 1 : L], xv[kHeld || !kSigmoid ? 1 : L], s[L], f0 = (T)1, H = (T)0;
    P A = P::of((T)1);
    bool odd = false;
    T st = (T)0;                                                 // the state before step 0
    uint64_t resets = 0, cuts = 0;                               // bit j: step j is reset; the step behind j is
    if (n) {
        const T *gate = a.gate + base, *dh = a.dh + base;
        if (top && a.state) st = a.state[sc];
        HeldRegs hv, xh;
        if constexpr (kHeld) {
            const uint64_t total = a.outer * a.steps * row;
            hv = HeldRows<L>::load(a.h, base - row, row, n, top ? 1 : 0, total, lane);
            if constexpr (kSigmoid) xh = HeldRows<L>::load(a.x, base, row, n, 0, total, lane);
        }
        if (r0 > 0) f0 = gate[lc + (uint32_t)n * row];           // the gate of the step behind j = 0
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const int q = j < n ? n - 1 - j : 0;                 // steps that are not there load the earliest one
            const uint32_t at = lc + (uint32_t)q * row;
            g[j] = once<ALIGNED>(gate + at);
            up[j] = once<ALIGNED>(dh + at);
            if constexpr (!kHeld) {
                if constexpr (kSigmoid) xv[j] = a.x.template at<ALIGNED>(base, at);
                hp[j] = top && q == 0 ? st : a.h.template at<ALIGNED>(base - row, at);
            }
        }
        if (a.reset) {
            resets = reset_bits(a.reset + (uint64_t)o * a.steps + tl, -1, n, lane);
            cuts = resets << 1;
            if (r0 > 0 && a.reset[(uint64_t)o * a.steps + tl + 1]) cuts |= 1;
            cuts &= (2ull << (n - 1)) - 1;
        }
        if constexpr (FORM == RT_SCAN_SIGMOID)
            if (r0 > 0) f0 = gate_of(f0).s;
        T f = f0;
        Running<T, P> run;
#pragma unroll
        for (int j = 0; j < L; ++j) {
            s[j] = g[j];
            if constexpr (FORM == RT_SCAN_SIGMOID) {
                const RtGate<T> q = gate_of(g[j]);
                s[j] = q.s;
                g[j] = q.r;
            }
            if (j < n) {
                H = j == 0 || (cuts >> j & 1) ? up[j] : fused(f, H, up[j]);
                run.by(f);
            }
            f = s[j];
        }
        A = run.template whole<true, L>(H, cuts != 0, n, [&](int j) { return j == 0 ? f0 : s[j ? j - 1 : 0]; }, [&](int j) { return up[j]; }, &odd);
        if constexpr (kHeld) {
            hrows[w].put(hv, lane);
            if constexpr (kSigmoid) xrows[w].put(xh, lane);
        }
    }
    T first = k == 0 && a.dlast ? a.dlast[sc] : (T)0;
    RT_PIN_LANE(first);
    T *dg = a.dgate + base, *dx = a.dx + base;
    const T end = join_tile<T, W, 64, true>(ch, room, item, k, A, H, cuts != 0, __any(odd), first, [&](T d, bool) {
        RT_APART;
        uint64_t rresets = resets;
        RT_PIN(rresets);
        if (in) {
#pragma unroll
            for (int j = 0; j < L; ++j) {
                if (j < rn) {
                    d = rcuts >> j & 1 ? up[j] : fused(j == 0 ? f0 : s[j ? j - 1 : 0], d, up[j]);
                    const bool none = rresets >> j & 1;
                    const int q = rn - 1 - j;                    // row of step j among the wave's, in memory order
                    T hj, xj = (T)0;
                    if constexpr (kHeld) {
                        hj = top && q == 0 ? st : hrows[w].template get<T>(q, (uint32_t)base + (uint32_t)(q - 1) * rrow, lane);
                        if constexpr (kSigmoid) xj = xrows[w].template get<T>(q, (uint32_t)base + (uint32_t)q * rrow, lane);
                    } else {
                        hj = hp[j];
                        if constexpr (kSigmoid) xj = xv[j];
                    }
                    const T p = none ? (T)0 : hj;
                    const uint32_t at = lane + (uint32_t)q * rrow;
                    if constexpr (FORM == RT_SCAN_LINEAR) {
                        const bool unused = none || (top && j == rn - 1 && !a.state);
                        put_once<ALIGNED || sizeof(T) == 8>(unused ? (T)0 : d * p, dg + at);
                        put_once<ALIGNED || sizeof(T) == 8>(d, dx + at);
                    } else {
                        put_once<ALIGNED || sizeof(T) == 8>(d * (p - xj) * (s[j] * g[j]), dg + at);
                        put_once<ALIGNED || sizeof(T) == 8>(g[j] * d, dx + at);
                    }
                }
            }
        }
        return d;
    });
    if (a.dstate && in && n && top) {
        const T g0 = a.gate[(uint64_t)o * a.steps * row + col];
        const bool none = a.reset && a.reset[(uint64_t)o * a.steps];
        a.dstate[sc] = none ? (T)0 : (FORM == RT_SCAN_SIGMOID ? gate_of(g0).s : g0) * end;
    }
}

// ---- few columns: the steps go over the lanes too --------------------------------------------------------------------------------------
// A tile is one contiguous run of memory, `ls` steps for each of the block's segments; it is staged through LDS, a lane takes one column
// of one segment, and the segments of a wave are joined with lane exchanges before the waves and the tiles are.  Short rows are taken
// `rows` at a time as one line with a cut at every row's start.
struct Narrow {
    uint64_t rows;           // of `outer`, in one line
    uint32_t ls;             // steps of a segment, at most kSeg
    uint32_t shift;          // lanes of one segment: 1 << shift >= inner
    FastDiv32 by_inner, by_steps;
};
template <class T> constexpr int seg_steps() { return sizeof(T) == 4 ? 16 : 8; }
template <class T, int W> struct Tile {
    static constexpr uint32_t kMost = W * 64 * seg_steps<T>();   // elements
    static constexpr uint32_t kLine = 64 / sizeof(T);            // one element of padding for each of these: a wave's segments start in
                                                                 // different banks
    static __device__ __forceinline__ uint32_t at(uint32_t e) { return e + e / kLine; }
    static constexpr uint32_t kRoom = kMost + 64 + (kMost + 64) / kLine;             // lanes without a column read up to 62 further
};
// Forward, the gates and then x go through the same room: twice the blocks on a CU.  Backward, both are needed at the end.
template <class T, int W> struct ForwardTile : Tile<T, W> {
    T v[Tile<T, W>::kRoom];
    uint8_t reset[1];                                            // one byte a step and one more, where there are resets
};
template <class T, int W> struct BackwardTile : Tile<T, W> {
    T a[Tile<T, W>::kRoom], b[Tile<T, W>::kRoom];
    uint8_t reset[1];
};
template <class TT, int W> size_t tile_bytes(const Narrow& nw, bool reset) {
    return offsetof(TT, reset) + (reset ? ((size_t)(W * 64) >> nw.shift) * nw.ls + 1 : 0);
}
template <class TT> constexpr size_t most_tile_bytes() { return offsetof(TT, reset) + TT::kMost + 1; }
// What joins a wave's segments: the exclusive prefix of the lane's segment, and the wave's whole.
template <class T, class P> struct Prefix {
    P A, wholeA;
    T H, wholeH;
    bool cut, any_cut, odd;
};
// Whether the wave runs its segments one after the other: `odd` of a lane, or, with SUMS, a sum over several lanes that left the range.  One
// that was not finite on the way has stayed so; unless a lane's own that is not, or NaN among the factors (`given`, and not odd), is part of
// it, its terms are finite.  And one that is NaN without a lane's own that is (`nan`) may have met an infinity that left the range.
template <bool SUMS, class T> __device__ __forceinline__ bool any_odd(bool odd, T H, bool given, bool nan, bool cut, int lane, uint32_t shift) {
    const bool over = SUMS && !finite(H), any = __any(odd || over);
    if (!SUMS || !any) return any;
    for (uint32_t d = 1u << shift; d < 64; d <<= 1) {
        const int below = __shfl_up((nan ? 4 : 0) | (given ? 2 : 0) | (cut ? 1 : 0), d);
        if (lane >= (int)d && !cut) {
            given = given || (below & 2);
            nan = nan || (below & 4);
            cut = below & 1;
        }
    }
    return __any(odd || (over && !given) || (H != H && !nan));
}
template <bool SUMS, class T> __device__ __forceinline__ Prefix<T, Falling<T>> join_lanes(Falling<T> A, T H, bool cut, bool odd, int lane, uint32_t shift) {
    const bool nan = H != H || A.m != A.m, given = nan || !finite(H), own_cut = cut;
    if (cut) A.m = (T)0;
    for (uint32_t d = 1u << shift; d < 64; d <<= 1) {
        const T A1 = __shfl_up(A.m, d), H1 = __shfl_up(H, d);
        const bool c1 = __shfl_up((int)cut, d) != 0;
        if (lane >= (int)d) {
            H = cut ? H : fused(A.m, H1, H);
            cut = cut || c1;
            A.m = cut ? (T)0 : A1 * A.m;
        }
    }
    const int top = 64 - (1 << shift) + (lane & ((1 << shift) - 1));
    Prefix<T, Falling<T>> p;
    p.wholeA = {__shfl(A.m, top)};
    p.wholeH = __shfl(H, top);
    p.any_cut = __any(cut);
    p.odd = any_odd<SUMS>(odd, H, given, nan, own_cut, lane, shift);
    const T A0 = __shfl_up(A.m, 1u << shift), H0 = __shfl_up(H, 1u << shift);
    const bool c0 = __shfl_up((int)cut, 1u << shift) != 0;
    const bool head = lane < (1 << shift);
    p.A = {head ? (T)1 : A0};
    p.H = head ? (T)0 : H0;
    p.cut = !head && c0;
    return p;
}
// The same with the exponents apart: m 2^e, m at least 1, so that scaled(H1, e) leaves the range only where the product does.  Whether the
// stretch is cut goes from lane to lane in the exponent's lowest bit.
template <bool SUMS, class T> __device__ __forceinline__ Prefix<T, Apart<T>> join_lanes(Apart<T> A, T H, bool cut, bool odd, int lane, uint32_t shift) {
    T m = mantissa(A.m) * (T)2;
    int e = exponent(A.m) + A.e - 1;
    odd = odd || (!cut && infinite(m));
    const bool nan = H != H || m != m, given = nan || !finite(H), own_cut = cut;
    for (uint32_t d = 1u << shift; d < 64; d <<= 1) {
        const T m1 = __shfl_up(m, d), H1 = __shfl_up(H, d);
        const int both = __shfl_up(e * 2 + (cut ? 1 : 0), d);
        if (lane >= (int)d) {
            H = cut ? H : fused(m, scaled(H1, e), H);
            cut = cut || (both & 1);
            m *= m1;
            e += both >> 1;
            if (d & 0x12) {                                      // m stays below 2^8: scaled(H1, e) loses at most 2^-142, f64 2^-1067
                e += exponent(m) - 1;
                m = mantissa(m) * (T)2;
            }
        }
    }
    odd = odd || (!cut && e > Apart<T>::kTop);                   // each lane has the product of a prefix
    const int top = 64 - (1 << shift) + (lane & ((1 << shift) - 1));
    const Apart<T> a = Apart<T>::from(m, e);
    Prefix<T, Apart<T>> p;
    p.wholeA = {__shfl(a.m, top), __shfl(a.e, top)};
    p.wholeH = __shfl(H, top);
    p.any_cut = __any(cut);
    p.odd = any_odd<SUMS>(odd, H, given, nan, own_cut, lane, shift);
    const T m0 = __shfl_up(a.m, 1u << shift), H0 = __shfl_up(H, 1u << shift);
    const int both = __shfl_up(a.e * 2 + (cut ? 1 : 0), 1u << shift);
    const bool head = lane < (1 << shift);
    p.A = {head ? (T)1 : m0, head ? 0 : both >> 1};
    p.H = head ? (T)0 : H0;
    p.cut = !head && (both & 1);
    return p;
}
// Runs a wave's segments from the wave's start state: `go(start)` goes through the lane's segment and returns where it ends.
template <class T, class P, class Go> __device__ __forceinline__ T run_lanes(const Prefix<T, P>& p, T start, bool serial, int lane, uint32_t shift, Go go) {
    const int c = lane & ((1 << shift) - 1), seg = lane >> shift;
    T end = start;
    for (int s = 0; s < (serial ? 64 >> shift : 1); ++s) {
        if (!serial) end = go(seg == 0 ? start : p.cut ? p.H : p.A.on(start, p.H));
        else {
            if (seg == s) end = go(start);
            start = __shfl(end, (s << shift) + c);
        }
    }
    return __shfl(end, 64 - (1 << shift) + c);
}

// As RT_APART, of a lane's segment.
#define RT_APART_LANES                          \
    int rls = ls;                               \
    uint32_t rcuts = cuts, rinner = inner;      \
    uint32_t e = v0 * inner + c;                \
    RT_PIN(rls);                                \
    RT_PIN(rinner);                             \
    asm volatile("" : "+v"(rcuts), "+v"(e))

// Segment of a lane: a wave's lanes hold 64 >> shift consecutive ones.
__device__ __forceinline__ int tile_segment(int tid, uint32_t shift) { return (tid >> 6) * (64 >> shift) + ((tid & 63) >> shift); }

// Half of the waves' cycles are waits, neither memory nor LDS nor the arithmetic is full: (2048, 4097, 1) f64 linear 51 us, 3.9 TB/s,
// (64, 2^19, 1) f32 linear 100 us, sigmoid 101 us, 4.0 TB/s.
// Four waves a tile and six on a SIMD, so that there are blocks in every phase; longer tiles for few rows.
template <class T, int FORM, int W>
__global__ __launch_bounds__(W * 64, W == 16 ? 4 : 6) void scan_narrow_kernel(ScanArgs<T> a, Chain ch, Narrow nw) {
    constexpr int kSeg = seg_steps<T>(), kThreads = W * 64;
    typedef ProductOf<T, FORM> P;
    __shared__ JoinRoom<T, W, 32, P> room;                       // inner is below 32
    extern __shared__ __align__(16) char lds[];
    typedef ForwardTile<T, W> TT;
    TT& tile = *reinterpret_cast<TT*>(lds);
    const uint32_t line = line_of_block<true>(ch), k = take_tile(ch, line, room), item = k * ch.lines + line;
    if (k >= ch.tiles) return;
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t inner = (uint32_t)a.inner, segs = kThreads >> nw.shift;
    const uint64_t row0 = (uint64_t)(ch.line0 + line) * nw.rows, rows = a.outer - row0 < nw.rows ? a.outer - row0 : nw.rows, len = rows * a.steps;
    const uint64_t u0 = (uint64_t)k * segs * nw.ls;              // first step of the tile in the line
    const uint32_t cnt = len <= u0 ? 0 : (uint32_t)(len - u0 < (uint64_t)segs * nw.ls ? len - u0 : (uint64_t)segs * nw.ls), E = cnt * inner;
    const uint64_t step0 = row0 * a.steps + u0, base = step0 * inner;
    const uint32_t all = segs * nw.ls * inner;                   // with the steps that are not there: they carry a state on as it is
    T x[kSeg];
    {
        T g[kSeg];                                               // all loads before the first write
#pragma unroll
        for (int q = 0; q < kSeg; ++q) {
            const uint32_t e = tid + q * kThreads;
            g[q] = FORM == RT_SCAN_SIGMOID ? (T)__builtin_inf() : (T)1;
            x[q] = (T)0;
            if (e < E) {
                g[q] = __builtin_nontemporal_load(a.gate + base + e);
                x[q] = __builtin_nontemporal_load(a.x + base + e);
            }
        }
#pragma unroll
        for (int q = 0; q < kSeg; ++q) {
            const uint32_t e = tid + q * kThreads;
            if (e < all) tile.v[TT::at(e)] = g[q];
        }
    }
    if (a.reset)
        for (uint32_t e = tid; e < segs * nw.ls; e += kThreads) tile.reset[e] = e < cnt ? a.reset[step0 + e] : (uint8_t)0;
    __syncthreads();
    const uint32_t c = lane & ((1u << nw.shift) - 1), v0 = (uint32_t)tile_segment(tid, nw.shift) * nw.ls;
    const bool own = c < inner;
    const int ls = (int)nw.ls;
    // the row of the segment's first step and the step's place in it; bit j of `heads`: step j is the first of its row
    const uint64_t row_of = nw.rows == 1 ? 0 : fd_div((uint32_t)u0 + v0, nw.by_steps), rem0 = u0 + v0 - row_of * a.steps;
    const uint32_t steps = a.steps < 64 ? (uint32_t)a.steps : 64u;       // all that a segment can tell
    uint32_t next = rem0 == 0 ? 0u : a.steps - rem0 < 64 ? (uint32_t)(a.steps - rem0) : 64u;
    uint32_t heads = 0, cuts = 0;
    for (; next < (uint32_t)kSeg; next += steps) heads |= 1u << next;
    heads &= v0 >= cnt ? 0u : (1u << (cnt - v0 < nw.ls ? cnt - v0 : nw.ls)) - 1;            // of the segment's own steps
    if (a.reset)
        for (int j = 0; j < ls; ++j) cuts |= (tile.reset[v0 + j] ? 1u : 0u) << j;
    const uint32_t states = a.state && own ? heads & ~cuts : 0u; // steps that begin from a given state
    cuts |= heads;
    const uint64_t place = (row0 + row_of) * inner + c;          // in (outer, inner), of the segment's first row
    T f[kSeg], b[kSeg], H = (T)0;
    Running<T, P> run;
    {
        uint32_t e = v0 * inner + c;
#pragma unroll
        for (int j = 0; j < kSeg; ++j)
            if (j < ls) {
                f[j] = tile.v[TT::at(e)];
                e += inner;
            }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kSeg; ++q) {
        const uint32_t e = tid + q * kThreads;
        if (e < all) tile.v[TT::at(e)] = x[q];
    }
    __syncthreads();
    {
        uint32_t e = v0 * inner + c;
#pragma unroll
        for (int j = 0; j < kSeg; ++j) {
            if (j < ls) {
                b[j] = tile.v[TT::at(e)];
                e += inner;
                if constexpr (FORM == RT_SCAN_SIGMOID) {
                    const RtGate<T> q = gate_of(f[j]);
                    f[j] = q.s;
                    b[j] = q.r * b[j];
                }
                if (states >> j & 1)                             // rows on from the first: heads up to here, the one at 0 being the first's own
                    b[j] = fused(f[j], a.state[place + (uint64_t)__popc(heads & ((2u << j) - 1u) & ~1u) * inner], b[j]);
                H = j == 0 || (cuts >> j & 1) ? b[j] : fused(f[j], H, b[j]);
                run.by(f[j]);
            }
        }
    }
    if (!own) { run = Running<T, P>(); H = (T)0; cuts = 0; }
    bool odd;
    const P A = run.template whole<FORM == RT_SCAN_LINEAR, kSeg>(H, cuts != 0, ls, [&](int j) { return f[j]; }, [&](int j) { return b[j]; }, &odd);
    const Prefix<T, P> pre = join_lanes<FORM == RT_SCAN_LINEAR>(A, H, cuts != 0, own && odd, lane, nw.shift);
    join_tile<T, W, 32, FORM == RT_SCAN_LINEAR>(ch, room, item, k, pre.wholeA, pre.wholeH, pre.any_cut, pre.odd, (T)0, [&](T start, bool serial) {
        return run_lanes(pre, start, serial, lane, nw.shift, [&](T p) {
            RT_APART_LANES;
            if (own) {
#pragma unroll
                for (int j = 0; j < kSeg; ++j) {
                    if (j < rls) {
                        p = rcuts >> j & 1 ? b[j] : fused(f[j], p, b[j]);
                        tile.v[TT::at(e)] = p;
                        e += rinner;
                    }
                }
            }
            return p;
        });
    });
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kSeg; ++q) {
        const uint32_t e = tid + q * kThreads;
        if (e < E) __builtin_nontemporal_store(tile.v[TT::at(e)], a.h + base + e);
    }
    if (a.last && u0 + cnt == len) {                             // the end of a line's rows: all of them, or the one whose last tile this is
        const uint32_t ends = nw.rows == 1 ? inner : (uint32_t)rows * inner, stretch = nw.rows == 1 ? cnt : (uint32_t)a.steps;
        for (uint32_t q = tid; q < ends; q += kThreads) {
            const uint32_t r = fd_div(q, nw.by_inner);
            a.last[row0 * inner + q] = tile.v[TT::at(((r + 1) * stretch - 1) * inner + (q - r * inner))];
        }
    }
}

// Backward: (2048, 8192, 1) f32 linear 82 us, 4.1 TB/s, (100, 50001, 5) f32 sigmoid 187 us, 3.2 TB/s; four waves a tile in place of eight
// make that 216 us.  The segments go through the tile from its end.  Only D comes out of the recurrence; the gradients are formed from it element
// by element afterwards, in memory order.
template <class T, int FORM, class S, int W>
__global__ __launch_bounds__(W * 64) void scan_backward_narrow_kernel(BackArgs<T, S> a, Chain ch, Narrow nw) {
    constexpr int kSeg = seg_steps<T>(), kThreads = W * 64;
    typedef ProductOf<T, FORM> P;
    __shared__ JoinRoom<T, W, 32, P> room;                       // inner is below 32
    extern __shared__ __align__(16) char lds[];
    typedef BackwardTile<T, W> TT;
    TT& tile = *reinterpret_cast<TT*>(lds);
    const uint32_t line = line_of_block<true>(ch), k = take_tile(ch, line, room), item = k * ch.lines + line;
    if (k >= ch.tiles) return;
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t inner = (uint32_t)a.inner, segs = kThreads >> nw.shift;
    const uint64_t row0 = (uint64_t)(ch.line0 + line) * nw.rows, rows = a.outer - row0 < nw.rows ? a.outer - row0 : nw.rows, len = rows * a.steps;
    const uint64_t r0 = (uint64_t)k * segs * nw.ls;              // steps of the line behind the tile
    const uint32_t cnt = len <= r0 ? 0 : (uint32_t)(len - r0 < (uint64_t)segs * nw.ls ? len - r0 : (uint64_t)segs * nw.ls), E = cnt * inner;
    const uint64_t lo = len - r0 - cnt;                          // first step of the tile in the line
    const uint64_t step0 = row0 * a.steps + lo, base = step0 * inner;
    const uint32_t behind = r0 ? inner : 0;                      // the gates of one step more
    // The steps that are not there (they carry a gradient on as it is) lie before the others: step v of the tile is at v + off.
    const uint32_t off = segs * nw.ls - cnt, eoff = off * inner;
    {
        T g[kSeg], d[kSeg];                                      // all loads before the first write
#pragma unroll
        for (int q = 0; q < kSeg; ++q) {
            const uint32_t e = tid + q * kThreads;
            g[q] = FORM == RT_SCAN_SIGMOID ? (T)__builtin_inf() : (T)1;
            d[q] = (T)0;
            if (e >= eoff && e < eoff + E) {
                g[q] = a.gate[base + (e - eoff)];
                d[q] = __builtin_nontemporal_load(a.dh + base + (e - eoff));
            }
        }
        if ((uint32_t)tid < inner) tile.a[TT::at(eoff + E + tid)] = (uint32_t)tid < behind ? a.gate[base + E + tid] : (T)0;
#pragma unroll
        for (int q = 0; q < kSeg; ++q) {
            const uint32_t e = tid + q * kThreads;
            if (e < eoff + E) {
                tile.a[TT::at(e)] = g[q];
                tile.b[TT::at(e)] = d[q];
            }
        }
    }
    if (a.reset)
        for (uint32_t e = tid; e <= segs * nw.ls; e += kThreads)
            tile.reset[e] = e >= off && e < off + cnt + (r0 ? 1 : 0) ? a.reset[step0 + (e - off)] : (uint8_t)0;
    __syncthreads();
    const uint32_t c = lane & ((1u << nw.shift) - 1), q0 = (uint32_t)tile_segment(tid, nw.shift) * nw.ls;
    const bool own = c < inner;
    const int ls = (int)nw.ls;
    const uint32_t v0 = segs * nw.ls - 1 - q0;                   // place of the segment's last step; it goes down from there
    // bit j of `tails`: the step j before the segment's last is the last of its row
    const uint64_t u_last = q0 < cnt ? lo + (cnt - 1 - q0) : 0;
    const uint64_t row_of = nw.rows == 1 ? 0 : fd_div((uint32_t)u_last, nw.by_steps), t_last = u_last - row_of * a.steps;
    const uint32_t steps = a.steps < 64 ? (uint32_t)a.steps : 64u;
    uint32_t next = t_last + 1 == a.steps ? 0u : t_last + 1 < 64 ? (uint32_t)t_last + 1 : 64u;
    uint32_t tails = 0, cuts = 0;
    for (; next < (uint32_t)kSeg; next += steps) tails |= 1u << next;
    tails &= q0 >= cnt ? 0u : (1u << (cnt - q0 < nw.ls ? cnt - q0 : nw.ls)) - 1;
    if (a.reset)                                                 // a reset of the step behind
        for (int j = 0; j < ls; ++j) cuts |= (tile.reset[v0 - j + 1] ? 1u : 0u) << j;
    cuts |= tails;
    const uint32_t lasts = a.dlast && own ? tails : 0u;
    const uint64_t place = (row0 + row_of) * inner + c;          // in (outer, inner), of the segment's last row
    T f[kSeg], b[kSeg], H = (T)0;
    Running<T, P> run;
    {
        uint32_t e = v0 * inner + c;
#pragma unroll
        for (int j = 0; j < kSeg; ++j) {
            if (j < ls) {
                b[j] = tile.b[TT::at(e)];
                f[j] = tile.a[TT::at(e + inner)];
                e -= inner;
                if constexpr (FORM == RT_SCAN_SIGMOID) f[j] = gate_of(f[j]).s;
                if (lasts >> j & 1) b[j] += a.dlast[place - (uint64_t)__popc(tails & ((2u << j) - 1u) & ~1u) * inner];
                H = j == 0 || (cuts >> j & 1) ? b[j] : fused(f[j], H, b[j]);
                run.by(f[j]);
            }
        }
    }
    if (!own) { run = Running<T, P>(); H = (T)0; cuts = 0; }
    bool odd;
    const P A = run.template whole<true, kSeg>(H, cuts != 0, ls, [&](int j) { return f[j]; }, [&](int j) { return b[j]; }, &odd);
    const Prefix<T, P> pre = join_lanes<true>(A, H, cuts != 0, own && odd, lane, nw.shift);
    join_tile<T, W, 32, true>(ch, room, item, k, pre.wholeA, pre.wholeH, pre.any_cut, pre.odd, (T)0, [&](T start, bool serial) {
        return run_lanes(pre, start, serial, lane, nw.shift, [&](T d) {
            RT_APART_LANES;
            if (own) {
#pragma unroll
                for (int j = 0; j < kSeg; ++j) {
                    if (j < rls) {
                        d = rcuts >> j & 1 ? b[j] : fused(f[j], d, b[j]);
                        tile.b[TT::at(e)] = d;
                        e -= rinner;
                    }
                }
            }
            return d;
        });
    });
    __syncthreads();
    const uint32_t head1 = lo == 0 ? 0u : ~0u;                   // the step that begins a row, of a line of one row
    constexpr int kBatch = 4;                                    // elements whose h and x are on their way at once
    for (uint32_t e0 = tid; e0 < E; e0 += kThreads * kBatch) {
        T p[kBatch], x[kBatch];
        uint64_t sc[kBatch];
        bool head[kBatch], reset[kBatch];
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            const uint32_t e = e0 + q * kThreads < E ? e0 + q * kThreads : e0, v = fd_div(e, nw.by_inner);
            const uint32_t row = nw.rows == 1 ? 0u : fd_div((uint32_t)lo + v, nw.by_steps);
            head[q] = nw.rows == 1 ? v == head1 : (uint32_t)lo + v == row * (uint32_t)a.steps;
            reset[q] = a.reset && tile.reset[v + off];
            sc[q] = (row0 + row) * inner + (e - v * inner);
            p[q] = (T)0;
            if (!head[q]) p[q] = a.h.at(base - inner, e);
            else if (a.state) p[q] = a.state[sc[q]];
            if constexpr (FORM == RT_SCAN_SIGMOID) x[q] = a.x.at(base, e);
        }
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            const uint32_t e = e0 + q * kThreads;
            if (e >= E) continue;
            const T d = tile.b[TT::at(e + eoff)], g = tile.a[TT::at(e + eoff)], before = reset[q] ? (T)0 : p[q];
            T factor = g;
            if constexpr (FORM == RT_SCAN_LINEAR) {
                __builtin_nontemporal_store(reset[q] || (head[q] && !a.state) ? (T)0 : d * before, a.dgate + base + e);
                __builtin_nontemporal_store(d, a.dx + base + e);
            } else {
                const RtGate<T> f = gate_of(g);
                factor = f.s;
                __builtin_nontemporal_store(d * (before - x[q]) * (f.s * f.r), a.dgate + base + e);
                __builtin_nontemporal_store(f.r * d, a.dx + base + e);
            }
            if (head[q] && a.dstate) a.dstate[sc[q]] = reset[q] ? (T)0 : factor * d;
        }
    }
}

// dst = src, or zeros: the states of a run of no steps, and copies of states
template <class T> __global__ void scan_no_steps_kernel(const T* src, T* dst, uint64_t n) {
    const uint64_t i = (uint64_t)blockIdx.x * kSBlock + threadIdx.x;
    if (i < n) dst[i] = src ? src[i] : (T)0;
}

constexpr uint64_t kMostLanes = 1ull << 31;     // of one launch: the lanes of a grid are numbered in 32 bits

uint32_t blocks_of(uint64_t n) { return (uint32_t)((n + kSBlock - 1) / kSBlock); }

template <class T> int32_t no_steps(rt_ctx* ctx, const void* src, void* dst, uint64_t n) {
    if (!dst || !n || src == dst) return RT_OK;
    for (uint64_t at = 0; at < n; at += kMostLanes) {
        const uint64_t len = n - at < kMostLanes ? n - at : kMostLanes;
        hipLaunchKernelGGL(scan_no_steps_kernel<T>, dim3(blocks_of(len)), dim3(kSBlock), 0, ctx->stream, src ? (const T*)src + at : nullptr, (T*)dst + at, len);
        RT_HIP(hipGetLastError());
    }
    return RT_OK;
}
// One lane a column, over as many launches as that takes.
template <class Args, class Kernel> int32_t columns_launches(rt_ctx* ctx, Args a, Kernel kernel) {
    const uint64_t cols = a.outer * a.inner;
    for (a.col0 = 0; a.col0 < cols; a.col0 += kMostLanes) {
        const uint64_t len = cols - a.col0 < kMostLanes ? cols - a.col0 : kMostLanes;
        hipLaunchKernelGGL(kernel, dim3(blocks_of(len)), dim3(kSBlock), 0, ctx->stream, a);
        RT_HIP(hipGetLastError());
    }
    return RT_OK;
}

// The chain of a launch: `tiles` along the steps for each of `lines` sets of columns; a workspace only where there is more than one tile.
template <class T> int32_t make_chain(rt_ctx* ctx, uint32_t tiles, uint32_t rounds, uint32_t lines, Chain* out) {
    out->tiles = tiles;
    out->lines = lines;
    out->tickets = nullptr;
    out->words = nullptr;
    out->epoch = 0;
    out->rounds = rounds;
    if (tiles == 1) return RT_OK;
    void *tickets = nullptr, *words = nullptr;
    RT_TRY(rt_chain_room(ctx, 0, (uint64_t)lines * kTicketPitch * sizeof(uint32_t), &tickets));
    RT_TRY(rt_chain_room(ctx, 1, (uint64_t)tiles * lines * Slot<T>::kWords * sizeof(uint64_t), &words));
    // the slots are cleared, and old tags with them, before numbers come round
    if (++ctx->chain_launches == kEpochs) {
        RT_TRY(rt_chain_clear(ctx, 1));
        ctx->chain_launches = 1;
    }
    out->tickets = (uint32_t*)tickets;
    out->words = (uint64_t*)words;
    out->epoch = ctx->chain_launches;
    return RT_OK;
}
// `launch(chain)` for all lines, by blocks of `threads`, over as many launches as that takes.
template <class T, class Launch> int32_t chain_launches(rt_ctx* ctx, uint64_t tiles, uint64_t lines, uint32_t threads, Launch launch) {
    const uint64_t rounds = tiles >= 16 ? (tiles + 7) / 8 * 8 : tiles;
    if (lines >= 1ull << 31 || rounds >= kMostLanes / threads) return rt_fail(RT_E_INVALID, "gated scan: too long for one launch");
    const uint64_t most = kMostLanes / (rounds * threads);
    Chain ch;
    for (uint64_t at = 0; at < lines; at += most) {
        RT_TRY(make_chain<T>(ctx, (uint32_t)tiles, (uint32_t)rounds, (uint32_t)(lines - at < most ? lines - at : most), &ch));
        ch.line0 = (uint32_t)at;
        launch(ch);
        RT_HIP(hipGetLastError());
    }
    return RT_OK;
}

// A lane holds L steps in registers: two values a step forward, five backward.
template <class T> constexpr int forward_steps() { return sizeof(T) == 4 ? 32 : 16; }
template <class T> constexpr int backward_steps() { return sizeof(T) == 4 ? 16 : 8; }
constexpr uint64_t kWideLeast = 32;             // inner: at least half of a wave's lanes have a column
constexpr uint64_t kWideMost = 1ull << 22;      // inner: a wave's rows are addressed with 32-bit offsets; beyond it columns alone fill the card
constexpr uint64_t kFewSteps = 8;               // steps that one lane a column goes through without help

// Rows of few columns that are too few to hide the chain's latency take longer tiles.  Linear, f32 with 16, 8 and 4 waves a tile: one row of
// 2^25 285, 616 and 1386 us; 4 rows of 2^23 168, 177 and 371 us; 8 of 2^22 170, 119 and 201 us; 16 of 2^21 165, 111 and 122 us; 32 of 2^20
// 167, 108 and 108 us.  f64 (16 and 4 waves): 8 rows of 2^21 164 and 317 us; 16 of 2^20 159 and 174 us; 2048 of 4097 104 and 52 us.
constexpr uint64_t kFewRows = 16;

template <class T> bool whole_lines(uint64_t inner) { return inner * sizeof(T) % 128 == 0; }

// One lane a column: few steps (a token), or so many columns that they fill the card.
bool by_columns(uint64_t steps, uint64_t inner) { return steps <= kFewSteps || inner >= kWideMost; }

// Cuts the operands into lines and tiles.
template <class T, int W> void make_narrow(rt_ctx* ctx, uint64_t outer, uint64_t steps, uint64_t inner, Narrow* nw, uint64_t* out_tiles, uint64_t* out_lines) {
    nw->shift = 0;
    while ((1ull << nw->shift) < inner) ++nw->shift;
    const uint64_t segs = (uint64_t)(W * 64) >> nw->shift, most = segs * seg_steps<T>();       // steps of a tile
    nw->rows = steps >= most ? 1 : most / steps;
    if (nw->rows > outer) nw->rows = outer;
    // fewer rows a line where there are too few lines to fill the card
    const uint64_t lines_wanted = (uint64_t)ctx->num_cus * 2;
    if (nw->rows > 1 && (outer + nw->rows - 1) / nw->rows < lines_wanted) nw->rows = (outer + lines_wanted - 1) / lines_wanted;
    const uint64_t len = nw->rows * steps, tiles = (len + most - 1) / most;
    const uint64_t per = (len + tiles - 1) / tiles;
    nw->ls = (uint32_t)((per + segs - 1) / segs);
    nw->by_inner = make_fastdiv((uint32_t)inner);
    nw->by_steps = make_fastdiv(nw->rows > 1 ? (uint32_t)steps : 1u);
    *out_tiles = (len + segs * nw->ls - 1) / (segs * nw->ls);
    *out_lines = (outer + nw->rows - 1) / nw->rows;
}

// More than 64 KiB of LDS has to be asked for, once a device.
int32_t allow_lds(rt_ctx* ctx, const void* kernel, size_t bytes, std::atomic<uint64_t>& allowed) {
    const uint64_t bit = 1ull << (ctx->device & 63);
    if ((allowed.load() & bit) && ctx->device < 64) return RT_OK;
    RT_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    allowed.fetch_or(bit);
    return RT_OK;
}

template <class T, int W, int L, class Args> int32_t wide_launches(rt_ctx* ctx, const Args& a, void (*kernel)(Args, Chain, uint32_t)) {
    const uint64_t cb = (a.inner + 63) / 64;
    return chain_launches<T>(ctx, (a.steps + W * L - 1) / (W * L), a.outer * cb, W * 64, [&](const Chain& ch) {
        hipLaunchKernelGGL(kernel, dim3(ch.rounds * ch.lines), dim3(W * 64), 0, ctx->stream, a, ch, (uint32_t)cb);
    });
}
// Few steps are one tile of as many waves as they need, which leaves room for more blocks: (4000, 33, 512) f32 forward 374 us with eight
// waves, 145 us with two, (500, 100, 2048) 260 us with eight, 221 us with four.
template <int MOST, class Launch> int32_t by_waves(uint64_t steps, int L, Launch launch) {
    if (steps <= (uint64_t)L) return launch(std::integral_constant<int, 1>());
    if (steps <= (uint64_t)L * 2) return launch(std::integral_constant<int, 2>());
    if constexpr (MOST > 4)
        if (steps <= (uint64_t)L * 4) return launch(std::integral_constant<int, 4>());
    return launch(std::integral_constant<int, MOST>());
}

template <class T, int FORM, int W> int32_t forward_narrow(rt_ctx* ctx, const ScanArgs<T>& a) {
    typedef ForwardTile<T, W> TT;
    Narrow nw;
    uint64_t tiles, lines;
    make_narrow<T, W>(ctx, a.outer, a.steps, a.inner, &nw, &tiles, &lines);
    auto kernel = scan_narrow_kernel<T, FORM, W>;
    static std::atomic<uint64_t> allowed{0};
    RT_TRY(allow_lds(ctx, reinterpret_cast<const void*>(kernel), most_tile_bytes<TT>(), allowed));
    const size_t bytes = tile_bytes<TT, W>(nw, a.reset != nullptr);
    return chain_launches<T>(ctx, tiles, lines, W * 64, [&](const Chain& ch) {
        hipLaunchKernelGGL(kernel, dim3(ch.rounds * ch.lines), dim3(W * 64), bytes, ctx->stream, a, ch, nw);
    });
}

template <class T, int FORM> int32_t forward_form(rt_ctx* ctx, const ScanArgs<T>& a) {
    constexpr int kWaves = 8, L = forward_steps<T>();
    if (by_columns(a.steps, a.inner)) return columns_launches(ctx, a, scan_columns_kernel<T, FORM>);
    if (a.inner < kWideLeast) {
        if (a.outer > kFewRows) return forward_narrow<T, FORM, 4>(ctx, a);
        if constexpr (sizeof(T) == 4)
            if (a.outer > kFewRows / 4) return forward_narrow<T, FORM, 8>(ctx, a);
        return forward_narrow<T, FORM, 16>(ctx, a);
    }
    auto launch = [&](auto waves) {
        constexpr int W = decltype(waves)::value;
        return wide_launches<T, W, L>(ctx, a, whole_lines<T>(a.inner) ? scan_wide_kernel<T, FORM, W, L, true> : scan_wide_kernel<T, FORM, W, L, false>);
    };
    return by_waves<kWaves>(a.steps, L, launch);
}
template <class T> int32_t forward_typed(rt_ctx* ctx, int form, const ScanArgs<T>& a) {
    return form == RT_SCAN_LINEAR ? forward_form<T, RT_SCAN_LINEAR>(ctx, a) : forward_form<T, RT_SCAN_SIGMOID>(ctx, a);
}

template <class T, int FORM, class S> int32_t backward_form(rt_ctx* ctx, const BackArgs<T, S>& a) {
    // waves of a wide tile: with the registers of the linear form two blocks of eight fit a CU, of the other one three of four; longer tiles
    // make shorter chains (linear from the 8-bit form over (1, 50000, 1088): 195 us with four, 169 with eight; the other one 199 and 215)
    constexpr int kWaves = FORM == RT_SCAN_LINEAR ? 8 : 4, kNarrowWaves = 8, L = backward_steps<T>();
    if (by_columns(a.steps, a.inner)) return columns_launches(ctx, a, scan_backward_columns_kernel<T, FORM, S>);
    if (a.inner < kWideLeast) {
        Narrow nw;
        uint64_t tiles, lines;
        make_narrow<T, kNarrowWaves>(ctx, a.outer, a.steps, a.inner, &nw, &tiles, &lines);
        auto kernel = scan_backward_narrow_kernel<T, FORM, S, kNarrowWaves>;
        static std::atomic<uint64_t> allowed{0};
        RT_TRY((allow_lds(ctx, reinterpret_cast<const void*>(kernel), most_tile_bytes<BackwardTile<T, kNarrowWaves>>(), allowed)));
        const size_t bytes = tile_bytes<BackwardTile<T, kNarrowWaves>, kNarrowWaves>(nw, a.reset != nullptr);
        return chain_launches<T>(ctx, tiles, lines, kNarrowWaves * 64, [&](const Chain& ch) {
            hipLaunchKernelGGL(kernel, dim3(ch.rounds * ch.lines), dim3(kNarrowWaves * 64), bytes, ctx->stream, a, ch, nw);
        });
    }
    auto launch = [&](auto waves) {
        constexpr int W = decltype(waves)::value;
        return wide_launches<T, W, L>(ctx, a, whole_lines<T>(a.inner) ? scan_backward_wide_kernel<T, FORM, S, W, L, true> : scan_backward_wide_kernel<T, FORM, S, W, L, false>);
    };
    return by_waves<kWaves>(a.steps, L, launch);
}
template <class T, class S> int32_t backward_typed(rt_ctx* ctx, int form, const BackArgs<T, S>& a) {
    return form == RT_SCAN_LINEAR ? backward_form<T, RT_SCAN_LINEAR, S>(ctx, a) : backward_form<T, RT_SCAN_SIGMOID, S>(ctx, a);
}

// A state that is replaced in place: its first tile reads it and its last tile writes it, and where a reset lies between them the last one
// does not wait for the first.  The state is then read from a copy.
template <class T> int32_t apart(rt_ctx* ctx, const void** in, const void* out, const void* reset, uint64_t outer, uint64_t steps, uint64_t inner) {
    if (!*in || *in != out || !reset || by_columns(steps, inner)) return RT_OK;
    void* copy = nullptr;
    RT_TRY(rt_scratch(ctx, outer * inner * sizeof(T), &copy));
    RT_TRY(no_steps<T>(ctx, *in, copy, outer * inner));
    *in = copy;
    return RT_OK;
}

// ---- argument checks ---------------------------------------------------------------------------------------------------------------
struct Operand {
    const char* name;
    const void* p;
    uint64_t len, need;
    int es;
    bool required;
};
int32_t check_operand(const char* what, const Operand& o) {
    if (!o.p) {
        if (o.required && o.need) return rt_fail(RT_E_INVALID, "%s: null %s", what, o.name);
        return RT_OK;
    }
    if (o.len < o.need)
        return rt_fail(RT_E_OUT_OF_BOUNDS, "%s: %s holds %llu of the %llu elements", what, o.name, (unsigned long long)o.len, (unsigned long long)o.need);
    if (reinterpret_cast<uintptr_t>(o.p) % (uintptr_t)o.es) return rt_fail(RT_E_INVALID, "%s: %s is not aligned to its elements", what, o.name);
    return RT_OK;
}
// An output may meet an input only as the very same run (`same`: the inputs for which even that is not allowed are passed with false).
bool meets(const Operand& out, const Operand& in, bool same) {
    if (!out.p || !in.p || !out.need || !in.need) return false;
    if (same && out.p == in.p && out.need == in.need && out.es == in.es) return false;
    return rt_spans_meet(rt_run_span(out.p, out.es, 0, out.need), rt_run_span(in.p, in.es, 0, in.need));
}
int32_t check_sizes(const char* what, int dtype, int form, uint64_t outer, uint64_t steps, uint64_t inner) {
    if (dtype != RT_F32 && dtype != RT_F64) return rt_fail(RT_E_DTYPE, "%s: f32 / f64 only", what);
    if (form != RT_SCAN_LINEAR && form != RT_SCAN_SIGMOID) return rt_fail(RT_E_INVALID, "%s: unknown form %d", what, form);
    const uint64_t most = 1ull << 40;                           // elements: beyond any device memory, and below every overflow here
    const uint64_t s1 = steps ? steps : 1, i1 = inner ? inner : 1, o1 = outer ? outer : 1;
    if (o1 > most || s1 > most / o1 || i1 > most / (o1 * s1))
        return rt_fail(RT_E_INVALID, "%s: %llu x %llu x %llu elements is too long", what, (unsigned long long)outer, (unsigned long long)steps, (unsigned long long)inner);
    return RT_OK;
}

// what both backward entry points share; S holds x and h
struct BackwardCall {
    const char* what;
    rt_ctx* ctx;
    int dtype, form;
    Operand gate, state, reset, dh, dlast, dgate, dx, dstate;
    Operand in[4];                                              // x and h, whole (2) or held (4: codes and exponents of each)
    int nin;
    uint64_t outer, steps, inner;
};
int32_t check_backward(const BackwardCall& c) {
    const Operand* all[12] = {&c.gate, &c.state, &c.reset, &c.dh, &c.dlast, &c.dgate, &c.dx, &c.dstate};
    int n = 8;
    for (int k = 0; k < c.nin; ++k) all[n++] = &c.in[k];
    for (int k = 0; k < n; ++k) RT_TRY(check_operand(c.what, *all[k]));
    const Operand* outs[3] = {&c.dgate, &c.dx, &c.dstate};
    for (int q = 0; q < 3; ++q) {
        for (int k = 0; k < n; ++k) {
            if (all[k] == outs[q]) continue;
            const bool same = (outs[q] == &c.dx && (all[k] == &c.dh || (c.nin == 2 && all[k] == &c.in[0]))) || (outs[q] == &c.dstate && all[k] == &c.dlast);
            if (meets(*outs[q], *all[k], same)) return rt_fail(RT_E_INVALID, "%s: %s overlaps %s", c.what, outs[q]->name, all[k]->name);
        }
    }
    return RT_OK;
}
template <class T, class S> int32_t run_backward(const BackwardCall& c, S x, S h) {
    if (c.steps == 0) return no_steps<T>(c.ctx, c.dlast.p, const_cast<void*>(c.dstate.p), c.outer * c.inner);
    if (c.outer * c.inner == 0) return RT_OK;
    const void* dlast = c.dlast.p;
    RT_TRY(apart<T>(c.ctx, &dlast, c.dstate.p, c.reset.p, c.outer, c.steps, c.inner));
    BackArgs<T, S> a;
    a.gate = (const T*)c.gate.p; a.x = x; a.h = h;
    a.state = (const T*)c.state.p; a.reset = (const uint8_t*)c.reset.p;
    a.dh = (const T*)c.dh.p; a.dlast = (const T*)dlast;
    a.dgate = (T*)const_cast<void*>(c.dgate.p); a.dx = (T*)const_cast<void*>(c.dx.p); a.dstate = (T*)const_cast<void*>(c.dstate.p);
    a.outer = c.outer; a.steps = c.steps; a.inner = c.inner; a.col0 = 0;
    return backward_typed<T, S>(c.ctx, c.form, a);
}

}  // namespace

extern "C" int32_t rt_gated_scan(rt_ctx* ctx, int32_t dtype, int32_t form, const void* gate, uint64_t gate_len, const void* x, uint64_t x_len,
                                 const void* state, uint64_t state_len, const void* reset, uint64_t reset_len, void* h, uint64_t h_len, void* last,
                                 uint64_t last_len, uint64_t outer, uint64_t steps, uint64_t inner) {
    const char* what = "gated scan";
    RT_TRY(check_sizes(what, dtype, form, outer, steps, inner));
    const int es = rt_elem_size(dtype);
    const uint64_t n = outer * steps * inner, cols = outer * inner;
    const Operand og = {"gate", gate, gate_len, n, es, true}, ox = {"x", x, x_len, n, es, true}, os = {"state", state, state_len, cols, es, false},
                  orr = {"reset", reset, reset_len, outer * steps, 1, false}, oh = {"h", h, h_len, n, es, true}, ol = {"last", last, last_len, cols, es, false};
    for (const Operand* o : {&og, &ox, &os, &orr, &oh, &ol}) RT_TRY(check_operand(what, *o));
    for (const Operand* o : {&og, &ox, &os, &orr, &ol})
        if (meets(oh, *o, o == &og || o == &ox)) return rt_fail(RT_E_INVALID, "%s: h overlaps %s", what, o->name);
    for (const Operand* o : {&og, &ox, &os, &orr})
        if (meets(ol, *o, o == &os)) return rt_fail(RT_E_INVALID, "%s: last overlaps %s", what, o->name);
    RT_TRY(rt_ctx_enter(ctx));
    CtxGuard g(ctx);
    if (steps == 0) return dtype == RT_F32 ? no_steps<float>(ctx, state, last, cols) : no_steps<double>(ctx, state, last, cols);
    if (cols == 0) return RT_OK;
    RT_TRY(dtype == RT_F32 ? apart<float>(ctx, &state, last, reset, outer, steps, inner) : apart<double>(ctx, &state, last, reset, outer, steps, inner));
    if (dtype == RT_F32) {
        const ScanArgs<float> a = {(const float*)gate, (const float*)x, (const float*)state, (const uint8_t*)reset, (float*)h, (float*)last, outer, steps, inner, 0};
        return forward_typed<float>(ctx, form, a);
    }
    const ScanArgs<double> a = {(const double*)gate, (const double*)x, (const double*)state, (const uint8_t*)reset, (double*)h, (double*)last, outer, steps, inner, 0};
    return forward_typed<double>(ctx, form, a);
}

extern "C" int32_t rt_gated_scan_backward(rt_ctx* ctx, int32_t dtype, int32_t form, const void* gate, uint64_t gate_len, const void* x, uint64_t x_len,
                                          const void* h, uint64_t h_len, const void* state, uint64_t state_len, const void* reset, uint64_t reset_len,
                                          const void* dh, uint64_t dh_len, const void* dlast, uint64_t dlast_len, void* dgate, uint64_t dgate_len, void* dx,
                                          uint64_t dx_len, void* dstate, uint64_t dstate_len, uint64_t outer, uint64_t steps, uint64_t inner) {
    const char* what = "gated scan backward";
    RT_TRY(check_sizes(what, dtype, form, outer, steps, inner));
    const int es = rt_elem_size(dtype);
    const uint64_t n = outer * steps * inner, cols = outer * inner;
    const bool sig = form == RT_SCAN_SIGMOID;
    const BackwardCall c = {what, ctx, dtype, form,
                            {"gate", gate, gate_len, n, es, true}, {"state", state, state_len, cols, es, false},
                            {"reset", reset, reset_len, outer * steps, 1, false}, {"dh", dh, dh_len, n, es, true}, {"dlast", dlast, dlast_len, cols, es, false},
                            {"dgate", dgate, dgate_len, n, es, true}, {"dx", dx, dx_len, n, es, true}, {"dstate", dstate, dstate_len, cols, es, false},
                            {{"x", sig ? x : nullptr, x_len, n, es, sig}, {"h", h, h_len, n, es, true}, {}, {}}, 2, outer, steps, inner};
    RT_TRY(check_backward(c));
    RT_TRY(rt_ctx_enter(ctx));
    CtxGuard g(ctx);
    if (dtype == RT_F32) return run_backward<float>(c, Whole<float>{(const float*)x}, Whole<float>{(const float*)h});
    return run_backward<double>(c, Whole<double>{(const double*)x}, Whole<double>{(const double*)h});
}

extern "C" int32_t rt_gated_scan_backward_packed8(rt_ctx* ctx, int32_t dtype, int32_t form, const void* gate, uint64_t gate_len, const void* x_codes,
                                                  uint64_t x_codes_len, const void* x_exps, uint64_t x_exps_len, const void* h_codes, uint64_t h_codes_len,
                                                  const void* h_exps, uint64_t h_exps_len, const void* state, uint64_t state_len, const void* reset,
                                                  uint64_t reset_len, const void* dh, uint64_t dh_len, const void* dlast, uint64_t dlast_len, void* dgate,
                                                  uint64_t dgate_len, void* dx, uint64_t dx_len, void* dstate, uint64_t dstate_len, uint64_t outer,
                                                  uint64_t steps, uint64_t inner) {
    const char* what = "gated scan backward (8-bit)";
    RT_TRY(check_sizes(what, dtype, form, outer, steps, inner));
    const int es = rt_elem_size(dtype);
    const uint64_t n = outer * steps * inner, cols = outer * inner, groups = (n + kP8Group - 1) / kP8Group;
    const bool sig = form == RT_SCAN_SIGMOID;
    const BackwardCall c = {what, ctx, dtype, form,
                            {"gate", gate, gate_len, n, es, true}, {"state", state, state_len, cols, es, false},
                            {"reset", reset, reset_len, outer * steps, 1, false}, {"dh", dh, dh_len, n, es, true}, {"dlast", dlast, dlast_len, cols, es, false},
                            {"dgate", dgate, dgate_len, n, es, true}, {"dx", dx, dx_len, n, es, true}, {"dstate", dstate, dstate_len, cols, es, false},
                            {{"x_codes", sig ? x_codes : nullptr, x_codes_len, n, 1, sig}, {"x_exps", sig ? x_exps : nullptr, x_exps_len, groups, 1, sig},
                             {"h_codes", h_codes, h_codes_len, n, 1, true}, {"h_exps", h_exps, h_exps_len, groups, 1, true}}, 4, outer, steps, inner};
    RT_TRY(check_backward(c));
    RT_TRY(rt_ctx_enter(ctx));
    CtxGuard g(ctx);
    const int8_t *xc = (const int8_t*)x_codes, *hc = (const int8_t*)h_codes;
    const uint8_t *xe = (const uint8_t*)x_exps, *he = (const uint8_t*)h_exps;
    if (dtype == RT_F32) return run_backward<float>(c, Held<float>{xc, xe}, Held<float>{hc, he});
    return run_backward<double>(c, Held<double>{xc, xe}, Held<double>{hc, he});
}
