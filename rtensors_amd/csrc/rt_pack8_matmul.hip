// Weight gradient of a projection whose input is held in 8 bits: dst[b] (k x n) = restored[b]^T * upstream[b] (m x n).
#include "rt_pack8.h"

namespace {

constexpr int kTile = 16;

// One element of dst per lane, 16 x 16 a block, 16 rows of both operands staged at a time.
template <class T>
__global__ __launch_bounds__(kTile * kTile) void pack8_matmul_plain_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ exps,
                                                                           const T* __restrict__ up, T* __restrict__ dst, uint64_t m, uint64_t k, uint64_t n,
                                                                           uint64_t tiles_k, uint64_t tiles_n) {
    __shared__ T xs[kTile][kTile + 1], ys[kTile][kTile + 1];
    const uint64_t tile = blockIdx.x, batch = tile / (tiles_k * tiles_n), kn = tile - batch * tiles_k * tiles_n;
    const uint64_t k0 = kn / tiles_n * kTile, n0 = kn % tiles_n * kTile;
    const int c = threadIdx.x % kTile, r = threadIdx.x / kTile;
    T acc = (T)0;
    for (uint64_t m0 = 0; m0 < m; m0 += kTile) {
        const uint64_t row = batch * m + m0 + r;
        const bool in = m0 + r < m;
        const uint64_t at = row * k + k0 + c;
        xs[r][c] = in && k0 + c < k ? p8_value<T>(codes[at], exps[at / kP8Group]) : (T)0;
        ys[r][c] = in && n0 + c < n ? up[row * n + n0 + c] : (T)0;
        __syncthreads();
        const int rows = m - m0 < (uint64_t)kTile ? (int)(m - m0) : kTile;
        for (int j = 0; j < rows; ++j) acc += xs[j][r] * ys[j][c];
        __syncthreads();
    }
    if (k0 + r < k && n0 + c < n) dst[(batch * k + k0 + r) * n + n0 + c] = acc;
}

template <class T>
int32_t matmul_typed(rt_ctx* ctx, const void* codes, const void* exps, const void* up, void* dst, uint64_t b, uint64_t m, uint64_t k, uint64_t n) {
    const uint64_t tk = (k + kTile - 1) / kTile, tn = (n + kTile - 1) / kTile;
    if (b * tk * tn >= (1ull << 31)) return rt_fail(RT_E_INVALID, "pack8 matmul backward: the result is too large for one launch");
    hipLaunchKernelGGL(pack8_matmul_plain_kernel<T>, dim3((uint32_t)(b * tk * tn)), dim3(kTile * kTile), 0, ctx->stream, (const int8_t*)codes,
                       (const uint8_t*)exps, (const T*)up, (T*)dst, m, k, n, tk, tn);
    RT_HIP(hipGetLastError());
    return RT_OK;
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
    return dtype == RT_F32 ? matmul_typed<float>(ctx, codes, exps, upstream, dst, b, m, k, n) : matmul_typed<double>(ctx, codes, exps, upstream, dst, b, m, k, n);
}
