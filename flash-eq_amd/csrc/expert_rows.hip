// Rows moved into expert order and back, weights applied.  With the plan of rows x K slots
// (positions[t, k] the slot's place, places from offsets[X] on those of slots without an expert):
//   dispatch  xs[d, positions[t, k]] = x[d, t], zeros at the places without an expert;
//   combine   y[d, t] = sum_k w[t, k] ys[d, positions[t, k]] over the slots with an expert
//             (w = 1: the gradient of dispatch);
//   gradient  gys[d, positions[t, k]] = w[t, k] gy[d, t], zeros at the places without an expert;
//             gw[t, k] = sum over d and columns of gy[d, t] ys[d, positions[t, k]], 0 there.
// Tables are (planes, rows or slots, width).
//
// HBM bounds all three.  A group of lanes takes a row t: it reads the row once and writes its K
// places (or reads K places and writes the row once), where a pass over the slots would read
// the row K times.  Lanes hold 16-byte vectors, narrower where the width or an address asks for it.
// Sums over k and over the row are float32 in a fixed order; the result is rounded once.
#include <algorithm>

#include "elem_types.h"
#include "feq_internal.h"

namespace feq {
namespace {

constexpr int kRowThreads = 256;
constexpr int kMaxRowK = 64;
constexpr int64_t kMaxRowBlocks = 1 << 22;   // workgroups of a plane (they loop over the rows behind)

// Lanes of a row of `chunks` vectors: a power of two up to 64.
int row_lanes(int64_t chunks) {
    int g = 1;
    while (g < 64 && g < chunks) g <<= 1;
    return g;
}

// U: the unit moved (16, 8, 4 or 2 bytes).
template <class U>
__global__ void __launch_bounds__(kRowThreads)
k_rows_dispatch(const U* __restrict__ x, int64_t rows, int K, int64_t chunks, const int32_t* __restrict__ positions,
                const int32_t* __restrict__ placed, U* __restrict__ xs, int GL) {
    const int l = threadIdx.x & (GL - 1);
    const int n = placed[0], per = kRowThreads / GL;
    const int64_t d = blockIdx.y, slots = rows * K;
    U* out = xs + d * slots * chunks;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / GL; t < rows;
         t += static_cast<int64_t>(gridDim.x) * per) {
        const U* xr = x + (d * rows + t) * chunks;
        for (int64_t c = l; c < chunks; c += GL) {
            const U v = xr[c];
            for (int k = 0; k < K; ++k) {
                const int p = positions[t * K + k];
                out[p * chunks + c] = p < n ? v : U{};
            }
        }
    }
}

// KB: slots whose loads are issued together.
template <class T, int V, int KB>
__global__ void __launch_bounds__(kRowThreads)
k_rows_combine(const T* __restrict__ ys, int64_t rows, int K, int64_t width, const int32_t* __restrict__ positions,
               const int32_t* __restrict__ placed, const void* __restrict__ w, int wdt, T* __restrict__ y, int GL) {
    const int l = threadIdx.x & (GL - 1);
    const int n = placed[0], per = kRowThreads / GL;
    const int64_t d = blockIdx.y, chunks = width / V;
    const T* in = ys + d * rows * K * width;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / GL; t < rows;
         t += static_cast<int64_t>(gridDim.x) * per) {
        T* yr = y + (d * rows + t) * width;
        for (int64_t c = l; c < chunks; c += GL) {
            float acc[V];
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] = 0.0f;
            for (int k0 = 0; k0 < K; k0 += KB) {
                float v[KB][V], wk[KB];
                bool on[KB];
#pragma unroll
                for (int i = 0; i < KB; ++i) {
                    const int k = k0 + i;
                    const int p = k < K ? positions[t * K + k] : n;
                    on[i] = p < n;
                    wk[i] = (on[i] && w) ? load_any(w, wdt, t * K + k) : 1.0f;
                    if (on[i]) load_f<T, V>(in + p * width + c * V, v[i]);
                }
#pragma unroll
                for (int i = 0; i < KB; ++i)
                    if (on[i])
#pragma unroll
                        for (int j = 0; j < V; ++j) acc[j] += wk[i] * v[i][j];
            }
            store_f<T, V>(yr + c * V, acc);
        }
    }
}

// A workgroup takes kRowThreads / (GL PS) rows; PS groups of GL lanes share a row, group q the planes q,
// q + PS, ...  gys and gw may be NULL (not both).
template <class T, int V, int KB>
__global__ void __launch_bounds__(kRowThreads)
k_rows_combine_bwd(const T* __restrict__ gy, const T* __restrict__ ys, int64_t rows, int K, int64_t width, int planes,
                   const int32_t* __restrict__ positions, const int32_t* __restrict__ placed,
                   const void* __restrict__ w, int wdt, T* __restrict__ gys, void* __restrict__ gw, int GL, int PS) {
    __shared__ float red[KB][kRowThreads];
    const int l = threadIdx.x & (GL - 1);
    const int group = threadIdx.x / GL, q = group % PS;
    const int n = placed[0], per = kRowThreads / (GL * PS);
    const int64_t chunks = width / V, slots = rows * K;
    for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * per; t0 < rows; t0 += static_cast<int64_t>(gridDim.x) * per)
    for (int k0 = 0; k0 < K; k0 += KB) {
        const int64_t t = t0 + group / PS;
        const bool live = t < rows;
        float dot[KB], wk[KB];
        int p[KB];
#pragma unroll
        for (int i = 0; i < KB; ++i) {
            const int k = k0 + i;
            dot[i] = 0.0f;
            p[i] = (live && k < K) ? positions[t * K + k] : -1;
            wk[i] = p[i] >= 0 ? load_any(w, wdt, t * K + k) : 0.0f;
        }
        if (live)
            for (int d = q; d < planes; d += PS) {
                const T* gr = gy + (d * rows + t) * width;
                const T* in = ys + d * slots * width;
                T* out = gys + d * slots * width;
                for (int64_t c = l; c < chunks; c += GL) {
                    float g[V];
                    load_f<T, V>(gr + c * V, g);
#pragma unroll
                    for (int i = 0; i < KB; ++i) {
                        if (p[i] < 0) continue;
                        const int64_t at = p[i] * width + c * V;
                        const bool on = p[i] < n;
                        if (gw && on) {
                            float v[V];
                            load_f<T, V>(in + at, v);
#pragma unroll
                            for (int j = 0; j < V; ++j) dot[i] += g[j] * v[j];
                        }
                        if (gys) {
                            float o[V];
#pragma unroll
                            for (int j = 0; j < V; ++j) o[j] = on ? wk[i] * g[j] : 0.0f;
                            store_f<T, V>(out + at, o);
                        }
                    }
                }
            }
        if (gw) {
#pragma unroll
            for (int i = 0; i < KB; ++i) {
                for (int o = GL >> 1; o; o >>= 1) dot[i] += __shfl_xor(dot[i], o, 64);
                if (l == 0) red[i][group] = dot[i];
            }
            __syncthreads();
            if (l == 0 && q == 0 && live)
#pragma unroll
                for (int i = 0; i < KB; ++i) {
                    float a = 0.0f;
                    for (int u = 0; u < PS; ++u) a += red[i][group + u];
                    if (k0 + i < K) store_any(gw, wdt, t * K + k0 + i, a);
                }
            __syncthreads();
        }
    }
}

int rows_check(int64_t planes, int64_t rows, int32_t K, int64_t width, int32_t dtype) {
    if (planes < 1 || rows < 0 || K < 1 || width < 1)
        return fail(FEQ_ERR_INVALID, "%lld planes of %lld rows, %d slots a row, width %lld", (long long)planes,
                    (long long)rows, K, (long long)width);
    if (planes > 65535) return fail(FEQ_ERR_UNSUPPORTED, "more than 65535 planes");
    if (K > kMaxRowK) return fail(FEQ_ERR_UNSUPPORTED, "more than %d slots a row", kMaxRowK);
    if (rows * K > INT32_MAX) return fail(FEQ_ERR_UNSUPPORTED, "more than 2^31 - 1 slots");
    if (!dtype_ok(dtype)) return fail(FEQ_ERR_INVALID, "unknown element type %d", dtype);
    return FEQ_OK;
}

// Elements of a vector: 16 bytes where the width and every address allow it, else 1.
template <class T>
bool rows_vec_ok(int64_t width, std::initializer_list<const void*> ptrs) {
    if (width % static_cast<int64_t>(16 / sizeof(T))) return false;
    for (const void* p : ptrs)
        if (p && !aligned_to(p, 16)) return false;
    return true;
}

template <class U>
int dispatch_run(const void* x, int64_t planes, int64_t rows, int K, int64_t bytes, const int32_t* positions,
                 const int32_t* placed, void* xs, hipStream_t s) {
    const int64_t chunks = bytes / static_cast<int64_t>(sizeof(U));
    const int GL = row_lanes(chunks);
    auto kern = k_rows_dispatch<U>;
    FEQ_LAUNCH("k_rows_dispatch", kern, dim3(std::min(ceil_div(rows, kRowThreads / GL), kMaxRowBlocks), planes), dim3(kRowThreads), 0, s,
               static_cast<const U*>(x), rows, K, chunks, positions, placed, static_cast<U*>(xs), GL);
    return FEQ_OK;
}

}  // namespace
}  // namespace feq

using namespace feq;

extern "C" int feq_expert_dispatch(const void* x, int64_t planes, int64_t rows, int32_t top_k, int64_t width,
                                   int32_t dtype, const int32_t* positions, const int32_t* placed, void* xs,
                                   feq_stream_t stream) {
    if (int rc = rows_check(planes, rows, top_k, width, dtype)) return rc;
    if (rows == 0) return FEQ_OK;
    if (!x || !positions || !placed || !xs) return fail(FEQ_ERR_INVALID, "NULL pointer");
    hipStream_t s = stream_of(stream);
    const int64_t bytes = width * elem_size(dtype);
    auto fits = [&](int64_t u) { return bytes % u == 0 && aligned_to(x, u) && aligned_to(xs, u); };
    if (fits(16)) return dispatch_run<uint4>(x, planes, rows, top_k, bytes, positions, placed, xs, s);
    if (fits(8)) return dispatch_run<uint2>(x, planes, rows, top_k, bytes, positions, placed, xs, s);
    if (fits(4)) return dispatch_run<uint32_t>(x, planes, rows, top_k, bytes, positions, placed, xs, s);
    return dispatch_run<uint16_t>(x, planes, rows, top_k, bytes, positions, placed, xs, s);
}

extern "C" int feq_expert_combine(const void* ys, int64_t planes, int64_t rows, int32_t top_k, int64_t width,
                                  int32_t dtype, const int32_t* positions, const int32_t* placed, const void* weights,
                                  int32_t weight_dtype, void* y, feq_stream_t stream) {
    if (int rc = rows_check(planes, rows, top_k, width, dtype)) return rc;
    if (weights && !dtype_ok(weight_dtype)) return fail(FEQ_ERR_INVALID, "unknown weight type %d", weight_dtype);
    if (rows == 0) return FEQ_OK;
    if (!ys || !positions || !placed || !y) return fail(FEQ_ERR_INVALID, "NULL pointer");
    hipStream_t s = stream_of(stream);
    return with_dtype(dtype, [&](auto tt) -> int {
        using T = decltype(tt);
        auto run = [&](auto v, auto kb) -> int {
            constexpr int V = decltype(v)::value, KB = decltype(kb)::value;
            const int GL = row_lanes(width / V);
            auto kern = k_rows_combine<T, V, KB>;
            FEQ_LAUNCH("k_rows_combine", kern, dim3(std::min(ceil_div(rows, kRowThreads / GL), kMaxRowBlocks), planes), dim3(kRowThreads), 0, s,
                       static_cast<const T*>(ys), rows, top_k, width, positions, placed, weights, weight_dtype,
                       static_cast<T*>(y), GL);
            return FEQ_OK;
        };
        auto with_kb = [&](auto v) -> int {
            if (top_k == 1) return run(v, std::integral_constant<int, 1>{});
            if (top_k == 2) return run(v, std::integral_constant<int, 2>{});
            return run(v, std::integral_constant<int, 4>{});
        };
        return rows_vec_ok<T>(width, {ys, y}) ? with_kb(std::integral_constant<int, 16 / sizeof(T)>{})
                                              : with_kb(std::integral_constant<int, 1>{});
    });
}

extern "C" int feq_expert_combine_bwd(const void* grad_y, const void* ys, int64_t planes, int64_t rows, int32_t top_k,
                                      int64_t width, int32_t dtype, const int32_t* positions, const int32_t* placed,
                                      const void* weights, int32_t weight_dtype, void* grad_ys, void* grad_weights,
                                      feq_stream_t stream) {
    if (int rc = rows_check(planes, rows, top_k, width, dtype)) return rc;
    if (!dtype_ok(weight_dtype)) return fail(FEQ_ERR_INVALID, "unknown weight type %d", weight_dtype);
    if (rows == 0 || (!grad_ys && !grad_weights)) return FEQ_OK;
    if (!grad_y || !positions || !placed || !weights || (grad_weights && !ys)) return fail(FEQ_ERR_INVALID, "NULL pointer");
    hipStream_t s = stream_of(stream);
    return with_dtype(dtype, [&](auto tt) -> int {
        using T = decltype(tt);
        auto run = [&](auto v, auto kb) -> int {
            constexpr int V = decltype(v)::value, KB = decltype(kb)::value;
            const int GL = row_lanes(width / V);
            // groups of a row: as many as fill the chip (eight waves a SIMD), no more than planes.  20000 rows of 9
            // planes, 64 float32 columns: one group 43 us, sixteen (seven of them idle) 83
            int PS = 1;
            while (PS * 2 <= planes && GL * PS * 2 <= kRowThreads && rows * GL * PS < 64 * 8192) PS <<= 1;
            auto kern = k_rows_combine_bwd<T, V, KB>;
            FEQ_LAUNCH("k_rows_combine_bwd", kern, dim3(std::min(ceil_div(rows, kRowThreads / (GL * PS)), kMaxRowBlocks)), dim3(kRowThreads), 0,
                       s, static_cast<const T*>(grad_y), static_cast<const T*>(ys), rows, top_k, width,
                       static_cast<int>(planes), positions, placed, weights, weight_dtype, static_cast<T*>(grad_ys),
                       grad_weights, GL, PS);
            return FEQ_OK;
        };
        auto with_kb = [&](auto v) -> int {
            if (top_k == 1) return run(v, std::integral_constant<int, 1>{});
            if (top_k == 2) return run(v, std::integral_constant<int, 2>{});
            return run(v, std::integral_constant<int, 4>{});
        };
        return rows_vec_ok<T>(width, {grad_y, ys, grad_ys}) ? with_kb(std::integral_constant<int, 16 / sizeof(T)>{})
                                                            : with_kb(std::integral_constant<int, 1>{});
    });
}
