// Gated linear recurrence along a dim and its backward pass (include/rt_hip.h has the formulas).
#include "rt_pack8.h"
#include "rt_unary_math.h"

namespace {

constexpr int kSBlock = 256;

// x and h of the backward pass: whole values or the 8-bit form
template <class T> struct Whole {
    const T* p;
    __device__ __forceinline__ T at(uint64_t i) const { return p[i]; }
};
template <class T> struct Held {
    const int8_t* codes;
    const uint8_t* exps;
    __device__ __forceinline__ T at(uint64_t i) const { return p8_value<T>(codes[i], exps[i / kP8Group]); }
};

template <class T> struct ScanArgs {
    const T *gate, *x, *state;
    const uint8_t* reset;
    T *h, *last;
    uint64_t outer, steps, inner;
};
template <class T, class S> struct BackArgs {
    const T* gate;
    S x, h;
    const T* state;
    const uint8_t* reset;
    const T *dh, *dlast;
    T *dgate, *dx, *dstate;
    uint64_t outer, steps, inner;
};

// One lane per column, the steps one after the other.
template <class T, int FORM>
__global__ __launch_bounds__(kSBlock) void scan_columns_kernel(ScanArgs<T> a) {
    const uint64_t col = (uint64_t)blockIdx.x * kSBlock + threadIdx.x;
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
    const uint64_t col = (uint64_t)blockIdx.x * kSBlock + threadIdx.x;
    if (col >= a.outer * a.inner) return;
    const uint64_t o = col / a.inner, i = col - o * a.inner;
    T carry = a.dlast ? a.dlast[col] : (T)0;          // a[t + 1] * D[t + 1]
    for (uint64_t t = a.steps; t-- > 0;) {
        const uint64_t at = (o * a.steps + t) * a.inner + i;
        const bool cut = a.reset && a.reset[o * a.steps + t];
        const bool none = cut || (t == 0 && !a.state);
        const T d = a.dh[at] + carry;
        const T g = a.gate[at];
        const T p = none ? (T)0 : (t == 0 ? a.state[col] : a.h.at(at - a.inner));
        if constexpr (FORM == RT_SCAN_LINEAR) {
            a.dgate[at] = none ? (T)0 : d * p;
            a.dx[at] = d;
            carry = none ? (T)0 : g * d;
        } else {
            const RtGate<T> q = rt_gate_of(g);
            const T x = a.x.at(at);
            a.dgate[at] = d * (p - x) * (q.s * q.r);
            a.dx[at] = q.r * d;
            carry = cut ? (T)0 : q.s * d;
        }
    }
    if (a.dstate) a.dstate[col] = carry;
}

// dst = src, or zeros: the states of a run of no steps
template <class T> __global__ void scan_no_steps_kernel(const T* src, T* dst, uint64_t n) {
    const uint64_t i = (uint64_t)blockIdx.x * kSBlock + threadIdx.x;
    if (i < n) dst[i] = src ? src[i] : (T)0;
}

uint32_t blocks_of(uint64_t n) { return (uint32_t)((n + kSBlock - 1) / kSBlock); }

template <class T> int32_t no_steps(rt_ctx* ctx, const void* src, void* dst, uint64_t n) {
    if (!dst || !n || src == dst) return RT_OK;
    hipLaunchKernelGGL(scan_no_steps_kernel<T>, dim3(blocks_of(n)), dim3(kSBlock), 0, ctx->stream, (const T*)src, (T*)dst, n);
    RT_HIP(hipGetLastError());
    return RT_OK;
}

template <class T> int32_t forward_typed(rt_ctx* ctx, int form, const ScanArgs<T>& a) {
    const uint64_t cols = a.outer * a.inner;
    if (form == RT_SCAN_LINEAR) hipLaunchKernelGGL((scan_columns_kernel<T, RT_SCAN_LINEAR>), dim3(blocks_of(cols)), dim3(kSBlock), 0, ctx->stream, a);
    else hipLaunchKernelGGL((scan_columns_kernel<T, RT_SCAN_SIGMOID>), dim3(blocks_of(cols)), dim3(kSBlock), 0, ctx->stream, a);
    RT_HIP(hipGetLastError());
    return RT_OK;
}

template <class T, class S> int32_t backward_typed(rt_ctx* ctx, int form, const BackArgs<T, S>& a) {
    const uint64_t cols = a.outer * a.inner;
    if (form == RT_SCAN_LINEAR) hipLaunchKernelGGL((scan_backward_columns_kernel<T, RT_SCAN_LINEAR, S>), dim3(blocks_of(cols)), dim3(kSBlock), 0, ctx->stream, a);
    else hipLaunchKernelGGL((scan_backward_columns_kernel<T, RT_SCAN_SIGMOID, S>), dim3(blocks_of(cols)), dim3(kSBlock), 0, ctx->stream, a);
    RT_HIP(hipGetLastError());
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
    BackArgs<T, S> a;
    a.gate = (const T*)c.gate.p; a.x = x; a.h = h;
    a.state = (const T*)c.state.p; a.reset = (const uint8_t*)c.reset.p;
    a.dh = (const T*)c.dh.p; a.dlast = (const T*)c.dlast.p;
    a.dgate = (T*)const_cast<void*>(c.dgate.p); a.dx = (T*)const_cast<void*>(c.dx.p); a.dstate = (T*)const_cast<void*>(c.dstate.p);
    a.outer = c.outer; a.steps = c.steps; a.inner = c.inner;
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
    if (dtype == RT_F32) {
        const ScanArgs<float> a = {(const float*)gate, (const float*)x, (const float*)state, (const uint8_t*)reset, (float*)h, (float*)last, outer, steps, inner};
        return forward_typed<float>(ctx, form, a);
    }
    const ScanArgs<double> a = {(const double*)gate, (const double*)x, (const double*)state, (const uint8_t*)reset, (double*)h, (double*)last, outer, steps, inner};
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
