// The element functions that sigmoid, silu and tanh are made of, shared by the elementwise kernels and by the kernels that apply one of
// the three while they hold its argument in 8 bits (rt_pack8.hip), so that both give the same bits.
#pragma once

#include "rt_common.h"
#include "rt_math64.h"

__device__ __forceinline__ float m_exp(float x) { return expf(x); }
__device__ __forceinline__ double m_exp(double x) { return exp(x); }

// 1 / (1 + e) of sigmoid and silu, e = exp(-x) >= 0, and (a - b) / (a + b) of tanh, a = exp(x), b = exp(-x).  f64: the divisor is at
// least 1, so the refined reciprocal (within an ulp) replaces the general division sequence, which is a third of these kernels'
// arithmetic.  The ends of the range are patched by selects, with what the reference's formulas give there: 1 / (1 + inf) = 0;
// (a - b) / (a + b) = +-1 exactly from |x| = 690 on (the smaller exponential is lost in the sum) and inf / inf = NaN once exp overflows.
__device__ __forceinline__ float recip_1p(float e) { return 1.0f / (1.0f + e); }
__device__ __forceinline__ double recip_1p(double e) {
    const double d = 1.0 + e;
    const double r = rt_rcp_f64(d);                              // NaN for d = inf (and for NaN)
    return d == __builtin_inf() ? 0.0 : r;
}
__device__ __forceinline__ float tanh_ratio(float x, float a, float b) { return (a - b) / (a + b); }
__device__ __forceinline__ double tanh_ratio(double x, double a, double b) {
    const double t = a + b;
    const double q = rt_quot_f64(a - b, t);
    const double far = __builtin_copysign(1.0, x) + (t - t);     // t - t: 0 for a finite sum, NaN for inf and NaN
    return __builtin_fabs(x) < 690.0 ? q : far;
}
// exp(-x) next to a = exp(x), for tanh, sinh and cosh.  f64: 1 / a from the refined reciprocal (within an ulp, as the library's
// exponential is) at a quarter of a second exponential's instructions.  Where the refinement has no answer -- a = 0 and a = inf, the
// exponential under- or overflowed -- the raw estimate has the right one (inf, 0).
__device__ __forceinline__ float exp_neg(float x, float a) { return m_exp(-x); }
__device__ __forceinline__ double exp_neg(double x, double a) {
    const double seed = rt_rcp_seed_f64(a);
    double r = __builtin_fma(__builtin_fma(-a, seed, 1.0), seed, seed);
    r = __builtin_fma(__builtin_fma(-a, r, 1.0), r, r);
    return r != r ? seed : r;
}

// sigmoid(g) and 1 - sigmoid(g), each to its own relative precision: both come from e = exp(-|g|) <= 1, so neither is a difference.
template <class T> struct RtGate { T s, r; };
__device__ __forceinline__ float rt_exp_nonpos(float x) { return expf(x); }
__device__ __forceinline__ double rt_exp_nonpos(double x) { return x != x ? x : rt_exp_nonpos_f64(x); }
template <class T> __device__ __forceinline__ RtGate<T> rt_gate_of(T g) {
    const T e = rt_exp_nonpos(g < (T)0 ? g : -g);
    const T inv = (T)1 / ((T)1 + e);
    const T low = e * inv;
    return g < (T)0 ? RtGate<T>{low, inv} : RtGate<T>{inv, low};
}
