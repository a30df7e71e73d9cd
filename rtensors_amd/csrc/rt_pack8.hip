// Activations held in 8 bits: the passes that write the form, restore it, and multiply an upstream gradient by the derivative of an
// activation function taken from it (include/rt_hip.h has the definition).
#include "rt_pack8.h"
#include "rt_unary_math.h"

namespace {

constexpr int kPBlock = 256;
// Vectors of four elements that a lane handles, a block width apart: 2^28 f32 packed and restored take 453, 419, 465 and 463 us with 1, 2, 4
// and 8 (many short-lived waves keep more loads in flight than few long ones; one vector leaves the index arithmetic of a wave too dear).
constexpr int kPVecs = 2;
constexpr uint64_t kPBlockElems = (uint64_t)kPBlock * kPVecs * 4;
constexpr int kNoOp = -1;

// Four consecutive elements, at element alignment
template <class T> struct Four { T e[4]; };
template <class T> __device__ __forceinline__ Four<T> load4(const T* p) {
    Four<T> f;
    if constexpr (sizeof(T) == 4) {
        f = __builtin_bit_cast(Four<T>, rt_ld16u<T, true>(p));
    } else {
        struct Two { T e[2]; };
        const Two a = __builtin_bit_cast(Two, rt_ld16u<T, true>(p)), b = __builtin_bit_cast(Two, rt_ld16u<T, true>(p + 2));
        f = Four<T>{{a.e[0], a.e[1], b.e[0], b.e[1]}};
    }
    return f;
}
template <class T> __device__ __forceinline__ void store4(T* p, const Four<T>& f) {
    if constexpr (sizeof(T) == 4) {
        rt_st16u_nt<T>(p, __builtin_bit_cast(rt_u32x4, f));
    } else {
        struct Two { T e[2]; };
        rt_st16u_nt<T>(p, __builtin_bit_cast(rt_u32x4, Two{{f.e[0], f.e[1]}}));
        rt_st16u_nt<T>(p + 2, __builtin_bit_cast(rt_u32x4, Two{{f.e[2], f.e[3]}}));
    }
}
// Codes are not marked as touched once: they are a fifth of what a pass moves, and a backward pass that follows soon finds them in the
// Infinity Cache (silu of 2^26 f32 forward and backward 192 us with the mark, 179 us without).
typedef uint32_t u32_a1 __attribute__((aligned(1)));
__device__ __forceinline__ uint32_t load_codes(const int8_t* p) { return *reinterpret_cast<const u32_a1*>(p); }
__device__ __forceinline__ void store_codes(int8_t* p, uint32_t w) { *reinterpret_cast<u32_a1*>(p) = w; }

// Largest value over a group's eight lanes: exchanges inside the quad, then with the mirrored lane of the eight.
template <int CTRL> __device__ __forceinline__ uint32_t moved(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
template <int CTRL> __device__ __forceinline__ uint64_t moved(uint64_t v) {
    return (uint64_t)moved<CTRL>((uint32_t)(v >> 32)) << 32 | moved<CTRL>((uint32_t)v);
}
template <class U> __device__ __forceinline__ U group_max(U v) {
    U o = moved<0xB1>(v);  v = v > o ? v : o;       // quad_perm 1 0 3 2
    o = moved<0x4E>(v);    v = v > o ? v : o;       // quad_perm 2 3 0 1
    o = moved<0x141>(v);   return v > o ? v : o;    // row_half_mirror
}

template <int OP, class T> __device__ __forceinline__ T value_of(T x) {
    if constexpr (OP == RT_U_SIGMOID) return recip_1p(m_exp(-x));
    else if constexpr (OP == RT_U_SILU) return x * recip_1p(m_exp(-x));
    else { const T a = m_exp(x), b = exp_neg(x, a); return tanh_ratio(x, a, b); }
}
// sigmoid' = s (1 - s);  silu' = s (1 + x (1 - s));  tanh' = 4 e / (1 + e)^2 with e = exp(-2 |x|): no difference of nearly equal numbers
template <int OP, class T> __device__ __forceinline__ T slope_of(T x) {
    if constexpr (OP == RT_U_TANH) {
        const T e = rt_exp_nonpos(x < (T)0 ? x + x : -(x + x));
        const T inv = (T)1 / ((T)1 + e);
        return (T)4 * e * inv * inv;
    } else {
        const RtGate<T> g = rt_gate_of(x);
        if constexpr (OP == RT_U_SIGMOID) return g.s * g.r;
        else return g.s * ((T)1 + x * g.r);
    }
}

// Codes and exponents of a run, and op of it (OP != kNoOp): a lane has four neighbouring elements a vector, so a group is eight lanes and
// its maximum three lane exchanges.  Bound by HBM: 2^28 f32 200 us in the kernel, 6.7 TB/s; silu of 2^26 f32 forward and backward 179 us,
// 6.8 TB/s of which the Infinity Cache takes the codes; 2^16 elements 2.6 us in the kernel, a launch.
template <class T, int OP>
__global__ __launch_bounds__(kPBlock) void pack8_kernel(const T* src, T* dst, int8_t* __restrict__ codes, uint8_t* __restrict__ exps, uint64_t len) {
    typedef typename std::conditional<sizeof(T) == 4, uint32_t, uint64_t>::type U;
    const uint64_t first = (uint64_t)blockIdx.x * kPBlockElems + (uint64_t)threadIdx.x * 4;
    Four<T> x[kPVecs];
#pragma unroll
    for (int v = 0; v < kPVecs; ++v) {
        const uint64_t e = first + (uint64_t)v * kPBlock * 4;
        if (e + 4 <= len) {
            x[v] = load4(src + e);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[v].e[j] = e + j < len ? src[e + j] : (T)0;
        }
    }
#pragma unroll
    for (int v = 0; v < kPVecs; ++v) {
        const uint64_t e = first + (uint64_t)v * kPBlock * 4;
        U top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) { const U m = p8_magnitude(x[v].e[j]); top = m > top ? m : top; }
        const uint32_t byte = p8_byte_of(group_max(top));
        if (e < len && (threadIdx.x & 7) == 0) exps[e / kP8Group] = (uint8_t)byte;
        const bool fine = byte != kP8NotFinite;
        const T inv = p8_inverse_step<T>(fine ? byte : 127u);
        uint32_t w = 0;
        Four<T> y;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int32_t c = fine ? p8_code(x[v].e[j], inv) : 0;
            w |= ((uint32_t)c & 255u) << (8 * j);
            if constexpr (OP != kNoOp) y.e[j] = value_of<OP, T>(x[v].e[j]);
        }
        if (e + 4 <= len) {
            store_codes(codes + e, w);
            if constexpr (OP != kNoOp) store4(dst + e, y);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (e + j < len) {
                    codes[e + j] = (int8_t)(w >> (8 * j));
                    if constexpr (OP != kNoOp) dst[e + j] = y.e[j];
                }
        }
    }
}

// dst = restored (OP == kNoOp), or upstream * op'(restored).  Bound by HBM: 2^28 f32 200 us in the kernel, 6.7 TB/s; tanh of 2^21 f64 9.1 us, where
// the exponential counts.
template <class T, int OP>
__global__ __launch_bounds__(kPBlock) void unpack8_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ exps, const T* up, T* dst, uint64_t len) {
    const uint64_t first = (uint64_t)blockIdx.x * kPBlockElems + (uint64_t)threadIdx.x * 4;
    uint32_t w[kPVecs], byte[kPVecs];
    Four<T> u[kPVecs];
#pragma unroll
    for (int v = 0; v < kPVecs; ++v) {
        const uint64_t e = first + (uint64_t)v * kPBlock * 4;
        w[v] = 0;
        byte[v] = e < len ? exps[e / kP8Group] : 0;
        if (e + 4 <= len) {
            w[v] = load_codes(codes + e);
            if constexpr (OP != kNoOp) u[v] = load4(up + e);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (e + j < len) w[v] |= (uint32_t)(uint8_t)codes[e + j] << (8 * j);
                if constexpr (OP != kNoOp) u[v].e[j] = e + j < len ? up[e + j] : (T)0;
            }
        }
    }
#pragma unroll
    for (int v = 0; v < kPVecs; ++v) {
        const uint64_t e = first + (uint64_t)v * kPBlock * 4;
        const T step = p8_step<T>(byte[v]);
        Four<T> y;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const T x = (T)(int32_t)(int8_t)(w[v] >> (8 * j)) * step;
            if constexpr (OP == kNoOp) y.e[j] = x;
            else y.e[j] = u[v].e[j] * slope_of<OP, T>(x);
        }
        if (e + 4 <= len) {
            store4(dst + e, y);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (e + j < len) dst[e + j] = y.e[j];
        }
    }
}

// Elements of one launch, whole groups and whole blocks: the lanes of a grid are numbered in 32 bits.
constexpr uint64_t kMostOfLaunch = 1ull << 33;

template <class T, int OP> int32_t pack_launch(rt_ctx* ctx, const T* src, T* dst, void* codes, void* exps, uint64_t len) {
    for (uint64_t at = 0; at < len; at += kMostOfLaunch) {
        const uint64_t n = len - at < kMostOfLaunch ? len - at : kMostOfLaunch;
        hipLaunchKernelGGL((pack8_kernel<T, OP>), dim3((uint32_t)((n + kPBlockElems - 1) / kPBlockElems)), dim3(kPBlock), 0, ctx->stream, src + at,
                           OP == kNoOp ? dst : dst + at, (int8_t*)codes + at, (uint8_t*)exps + at / kP8Group, n);
        RT_HIP(hipGetLastError());
    }
    return RT_OK;
}
template <class T, int OP> int32_t unpack_launch(rt_ctx* ctx, const void* codes, const void* exps, const T* up, T* dst, uint64_t len) {
    for (uint64_t at = 0; at < len; at += kMostOfLaunch) {
        const uint64_t n = len - at < kMostOfLaunch ? len - at : kMostOfLaunch;
        hipLaunchKernelGGL((unpack8_kernel<T, OP>), dim3((uint32_t)((n + kPBlockElems - 1) / kPBlockElems)), dim3(kPBlock), 0, ctx->stream,
                           (const int8_t*)codes + at, (const uint8_t*)exps + at / kP8Group, OP == kNoOp ? up : up + at, dst + at, n);
        RT_HIP(hipGetLastError());
    }
    return RT_OK;
}
template <class T> int32_t pack_typed(rt_ctx* ctx, int op, const T* src, T* dst, void* codes, void* exps, uint64_t len) {
    switch (op) {
        case RT_U_SIGMOID: return pack_launch<T, RT_U_SIGMOID>(ctx, src, dst, codes, exps, len);
        case RT_U_SILU: return pack_launch<T, RT_U_SILU>(ctx, src, dst, codes, exps, len);
        case RT_U_TANH: return pack_launch<T, RT_U_TANH>(ctx, src, dst, codes, exps, len);
        default: return pack_launch<T, kNoOp>(ctx, src, dst, codes, exps, len);
    }
}
template <class T> int32_t unpack_typed(rt_ctx* ctx, int op, const void* codes, const void* exps, const T* up, T* dst, uint64_t len) {
    switch (op) {
        case RT_U_SIGMOID: return unpack_launch<T, RT_U_SIGMOID>(ctx, codes, exps, up, dst, len);
        case RT_U_SILU: return unpack_launch<T, RT_U_SILU>(ctx, codes, exps, up, dst, len);
        case RT_U_TANH: return unpack_launch<T, RT_U_TANH>(ctx, codes, exps, up, dst, len);
        default: return unpack_launch<T, kNoOp>(ctx, codes, exps, up, dst, len);
    }
}

int32_t check_common(const char* what, int dtype, int op, uint64_t len) {
    if (dtype != RT_F32 && dtype != RT_F64) return rt_fail(RT_E_DTYPE, "%s: f32 / f64 only", what);
    if (op != kNoOp && op != RT_U_SIGMOID && op != RT_U_SILU && op != RT_U_TANH)
        return rt_fail(op >= 0 && op < RT_U_EXT_COUNT ? RT_E_DTYPE : RT_E_INVALID, "%s: op %d is not sigmoid, silu or tanh", what, op);
    if (len > (1ull << 40)) return rt_fail(RT_E_INVALID, "%s: %llu elements is too long", what, (unsigned long long)len);
    return RT_OK;
}
int32_t check_run(const char* what, const char* name, const void* p, uint64_t have, uint64_t start, uint64_t need, int es) {
    if (start > have || need > have - start)
        return rt_fail(RT_E_OUT_OF_BOUNDS, "%s: %s holds %llu of the %llu elements from %llu", what, name, (unsigned long long)have, (unsigned long long)need,
                       (unsigned long long)start);
    if (!need) return RT_OK;
    if (!p) return rt_fail(RT_E_INVALID, "%s: null %s", what, name);
    if (reinterpret_cast<uintptr_t>(p) % (uintptr_t)es) return rt_fail(RT_E_INVALID, "%s: %s is not aligned to its elements", what, name);
    return RT_OK;
}

int32_t pack_any(const char* what, rt_ctx* ctx, int32_t dtype, int op, const void* src, uint64_t src_len, uint64_t start, uint64_t len, void* dst,
                 uint64_t dst_len, void* codes, uint64_t codes_len, void* exps, uint64_t exps_len) {
    RT_TRY(check_common(what, dtype, op, len));
    const int es = rt_elem_size(dtype);
    const uint64_t groups = (len + kP8Group - 1) / kP8Group;
    RT_TRY(check_run(what, "src", src, src_len, start, len, es));
    RT_TRY(check_run(what, "codes", codes, codes_len, 0, len, 1));
    RT_TRY(check_run(what, "exps", exps, exps_len, 0, groups, 1));
    if (op != kNoOp) RT_TRY(check_run(what, "dst", dst, dst_len, 0, len, es));
    if (!len) return rt_ctx_enter(ctx);
    const ByteSpan ss = rt_run_span(src, es, start, len), cs = rt_run_span(codes, 1, 0, len), xs = rt_run_span(exps, 1, 0, groups), ds = rt_run_span(dst, es, 0, len);
    if (rt_spans_meet(cs, ss) || rt_spans_meet(xs, ss) || rt_spans_meet(cs, xs)) return rt_fail(RT_E_INVALID, "%s: codes, exps and src overlap", what);
    if (op != kNoOp && ((ds.lo != ss.lo && rt_spans_meet(ds, ss)) || rt_spans_meet(ds, cs) || rt_spans_meet(ds, xs)))
        return rt_fail(RT_E_INVALID, "%s: dst overlaps another operand", what);
    RT_TRY(rt_ctx_enter(ctx));
    CtxGuard g(ctx);
    if (dtype == RT_F32) return pack_typed<float>(ctx, op, (const float*)src + start, (float*)dst, codes, exps, len);
    return pack_typed<double>(ctx, op, (const double*)src + start, (double*)dst, codes, exps, len);
}

int32_t unpack_any(const char* what, rt_ctx* ctx, int32_t dtype, int op, const void* codes, uint64_t codes_len, const void* exps, uint64_t exps_len,
                   const void* up, uint64_t up_len, uint64_t len, void* dst, uint64_t dst_len) {
    RT_TRY(check_common(what, dtype, op, len));
    const int es = rt_elem_size(dtype);
    const uint64_t groups = (len + kP8Group - 1) / kP8Group;
    RT_TRY(check_run(what, "codes", codes, codes_len, 0, len, 1));
    RT_TRY(check_run(what, "exps", exps, exps_len, 0, groups, 1));
    RT_TRY(check_run(what, "dst", dst, dst_len, 0, len, es));
    if (op != kNoOp) RT_TRY(check_run(what, "upstream", up, up_len, 0, len, es));
    if (!len) return rt_ctx_enter(ctx);
    const ByteSpan ds = rt_run_span(dst, es, 0, len), us = rt_run_span(up, es, 0, len);
    if (rt_spans_meet(ds, rt_run_span(codes, 1, 0, len)) || rt_spans_meet(ds, rt_run_span(exps, 1, 0, groups)) || (op != kNoOp && dst != up && rt_spans_meet(ds, us)))
        return rt_fail(RT_E_INVALID, "%s: dst overlaps another operand", what);
    RT_TRY(rt_ctx_enter(ctx));
    CtxGuard g(ctx);
    if (dtype == RT_F32) return unpack_typed<float>(ctx, op, codes, exps, (const float*)up, (float*)dst, len);
    return unpack_typed<double>(ctx, op, codes, exps, (const double*)up, (double*)dst, len);
}

}  // namespace

extern "C" int32_t rt_pack8(rt_ctx* ctx, int32_t dtype, const void* src, uint64_t src_len, uint64_t start, uint64_t len, void* codes, uint64_t codes_len,
                            void* exps, uint64_t exps_len) {
    return pack_any("pack8", ctx, dtype, kNoOp, src, src_len, start, len, nullptr, 0, codes, codes_len, exps, exps_len);
}

extern "C" int32_t rt_unpack8(rt_ctx* ctx, int32_t dtype, const void* codes, uint64_t codes_len, const void* exps, uint64_t exps_len, uint64_t len, void* dst,
                              uint64_t dst_len) {
    return unpack_any("unpack8", ctx, dtype, kNoOp, codes, codes_len, exps, exps_len, nullptr, 0, len, dst, dst_len);
}

extern "C" int32_t rt_pack8_unary(rt_ctx* ctx, int32_t dtype, int32_t op, const void* src, uint64_t src_len, uint64_t start, uint64_t len, void* dst,
                                  uint64_t dst_len, void* codes, uint64_t codes_len, void* exps, uint64_t exps_len) {
    if (op < 0) return rt_fail(RT_E_INVALID, "pack8 unary: unknown op code %d", op);
    return pack_any("pack8 unary", ctx, dtype, op, src, src_len, start, len, dst, dst_len, codes, codes_len, exps, exps_len);
}

extern "C" int32_t rt_pack8_unary_backward(rt_ctx* ctx, int32_t dtype, int32_t op, const void* codes, uint64_t codes_len, const void* exps, uint64_t exps_len,
                                           const void* upstream, uint64_t upstream_len, uint64_t len, void* dst, uint64_t dst_len) {
    if (op < 0) return rt_fail(RT_E_INVALID, "pack8 unary backward: unknown op code %d", op);
    return unpack_any("pack8 unary backward", ctx, dtype, op, codes, codes_len, exps, exps_len, upstream, upstream_len, len, dst, dst_len);
}
