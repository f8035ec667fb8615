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
// the row K times.  Lanes hold 16-byte vectors, of rows of any width and alignment (vec_begin; what two vectors
// share is written twice, the same); rows shorter than one take narrower ones.
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

// V: elements (of 16 bits) moved at a time, at most the width.  20000 rows of 9 planes x 64 float32, 2 choices: 25 us,
// 5.5 TB/s.
template <int V>
__global__ void __launch_bounds__(kRowThreads)
k_rows_dispatch(const uint16_t* __restrict__ x, int64_t rows, int K, int width, const int32_t* __restrict__ positions,
                const int32_t* __restrict__ placed, uint16_t* __restrict__ xs, int GL) {
    typedef typename VecOf<uint16_t, V>::type U;
    typedef typename VecOf<uint16_t, V>::any UA;
    const int chunks = (width + V - 1) / V;
    const int l = threadIdx.x & (GL - 1);
    const int n = placed[0], per = kRowThreads / GL;
    const int64_t d = blockIdx.y, slots = rows * K;
    uint16_t* out = xs + d * slots * width;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / GL; t < rows;
         t += static_cast<int64_t>(gridDim.x) * per) {
        const uint16_t* xr = x + (d * rows + t) * width;
        for (int q = l; q < chunks; q += GL) {
            const int c = vec_begin<V>(q, width);
            const U v = *reinterpret_cast<const UA*>(xr + c);
            for (int k = 0; k < K; ++k) {
                const int p = positions[t * K + k];
                *reinterpret_cast<UA*>(out + static_cast<int64_t>(p) * width + c) = p < n ? v : U{};
            }
        }
    }
}

// KB: slots whose loads are issued together.  20000 rows of 9 planes x 64 float32, 2 choices: 24 to 28 us, 5 TB/s.
template <class T, int V, int KB>
__global__ void __launch_bounds__(kRowThreads)
k_rows_combine(const T* __restrict__ ys, int64_t rows, int K, int width, const int32_t* __restrict__ positions,
               const int32_t* __restrict__ placed, const void* __restrict__ w, int wdt, T* __restrict__ y, int GL) {
    const int l = threadIdx.x & (GL - 1);
    const int n = placed[0], per = kRowThreads / GL;
    const int64_t d = blockIdx.y;
    const int chunks = (width + V - 1) / V;
    const T* in = ys + d * rows * K * width;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / GL; t < rows;
         t += static_cast<int64_t>(gridDim.x) * per) {
        T* yr = y + (d * rows + t) * width;
        for (int q = l; q < chunks; q += GL) {
            const int c = vec_begin<V>(q, width);
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
                    if (on[i]) load_f<T, V>(in + static_cast<int64_t>(p) * width + c, v[i]);
                }
#pragma unroll
                for (int i = 0; i < KB; ++i)
                    if (on[i])
#pragma unroll
                        for (int j = 0; j < V; ++j) acc[j] += wk[i] * v[i][j];
            }
            store_f<T, V>(yr + c, acc);
        }
    }
}

// A workgroup takes kRowThreads / (GL PS) rows; PS groups of GL lanes share a row, group q the planes q,
// q + PS, ...  gys and gw may be NULL (not both).  20000 rows of 9 planes x 64 float32, 2 choices: 44 us, 5.2 TB/s.
template <class T, int V, int KB>
__global__ void __launch_bounds__(kRowThreads)
k_rows_combine_bwd(const T* __restrict__ gy, const T* __restrict__ ys, int64_t rows, int K, int width, int planes,
                   const int32_t* __restrict__ positions, const int32_t* __restrict__ placed,
                   const void* __restrict__ w, int wdt, T* __restrict__ gys, void* __restrict__ gw, int GL, int PS) {
    __shared__ float red[KB][kRowThreads];
    const int l = threadIdx.x & (GL - 1);
    const int group = threadIdx.x / GL, q = group % PS;
    const int n = placed[0], per = kRowThreads / (GL * PS);
    const int chunks = (width + V - 1) / V;
    const int64_t slots = rows * K;
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
                for (int q2 = l; q2 < chunks; q2 += GL) {
                    const int c = vec_begin<V>(q2, width), shared = vec_shared<V>(q2, width);
                    float g[V];
                    load_f<T, V>(gr + c, g);
#pragma unroll
                    for (int i = 0; i < KB; ++i) {
                        if (p[i] < 0) continue;
                        const int64_t at = static_cast<int64_t>(p[i]) * width + c;
                        const bool on = p[i] < n;
                        if (gw && on) {
                            float v[V];
                            load_f<T, V>(in + at, v);
#pragma unroll
                            for (int j = 0; j < V; ++j) dot[i] += j >= shared ? g[j] * v[j] : 0.0f;
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
    if (width > (1 << 29)) return fail(FEQ_ERR_UNSUPPORTED, "rows wider than 2^29");
    if (K > kMaxRowK) return fail(FEQ_ERR_UNSUPPORTED, "more than %d slots a row", kMaxRowK);
    if (rows * K > INT32_MAX) return fail(FEQ_ERR_UNSUPPORTED, "more than 2^31 - 1 slots");
    if (!dtype_ok(dtype)) return fail(FEQ_ERR_INVALID, "unknown element type %d", dtype);
    return FEQ_OK;
}

// f(V) for the vector of a row of `width` elements: 16 bytes, less where the row has less.
template <class T, class F>
int with_row_vec(int64_t width, F&& f) {
    constexpr int VV = 16 / sizeof(T);
    if (width >= VV) return f(std::integral_constant<int, VV>{});
    if constexpr (VV == 8) {
        if (width >= 4) return f(std::integral_constant<int, 4>{});
    }
    if (width >= 2) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 1>{});
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
    // moved as 16-bit units
    const int units = static_cast<int>(width) * (elem_size(dtype) / 2);
    return with_row_vec<uint16_t>(units, [&](auto v) -> int {
        constexpr int V = decltype(v)::value;
        const int GL = row_lanes(ceil_div(units, V));
        auto kern = k_rows_dispatch<V>;
        FEQ_LAUNCH("k_rows_dispatch", kern, dim3(std::min(ceil_div(rows, kRowThreads / GL), kMaxRowBlocks), planes),
                   dim3(kRowThreads), 0, s, static_cast<const uint16_t*>(x), rows, top_k, units, positions, placed,
                   static_cast<uint16_t*>(xs), GL);
        return FEQ_OK;
    });
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
            const int GL = row_lanes(ceil_div(width, V));
            auto kern = k_rows_combine<T, V, KB>;
            FEQ_LAUNCH("k_rows_combine", kern, dim3(std::min(ceil_div(rows, kRowThreads / GL), kMaxRowBlocks), planes), dim3(kRowThreads), 0, s,
                       static_cast<const T*>(ys), rows, top_k, static_cast<int>(width), positions, placed, weights,
                       weight_dtype, static_cast<T*>(y), GL);
            return FEQ_OK;
        };
        auto with_kb = [&](auto v) -> int {
            if (top_k == 1) return run(v, std::integral_constant<int, 1>{});
            if (top_k == 2) return run(v, std::integral_constant<int, 2>{});
            return run(v, std::integral_constant<int, 4>{});
        };
        return with_row_vec<T>(width, with_kb);
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
            const int GL = row_lanes(ceil_div(width, V));
            // groups of a row: as many as fill the chip (eight waves a SIMD), no more than planes.  20000 rows of 9
            // planes, 64 float32 columns: one group 43 us, sixteen (seven of them idle) 83
            int PS = 1;
            while (PS * 2 <= planes && GL * PS * 2 <= kRowThreads && rows * GL * PS < 64 * 8192) PS <<= 1;
            auto kern = k_rows_combine_bwd<T, V, KB>;
            FEQ_LAUNCH("k_rows_combine_bwd", kern, dim3(std::min(ceil_div(rows, kRowThreads / (GL * PS)), kMaxRowBlocks)), dim3(kRowThreads), 0,
                       s, static_cast<const T*>(grad_y), static_cast<const T*>(ys), rows, top_k, static_cast<int>(width),
                       static_cast<int>(planes), positions, placed, weights, weight_dtype, static_cast<T*>(grad_ys),
                       grad_weights, GL, PS);
            return FEQ_OK;
        };
        auto with_kb = [&](auto v) -> int {
            if (top_k == 1) return run(v, std::integral_constant<int, 1>{});
            if (top_k == 2) return run(v, std::integral_constant<int, 2>{});
            return run(v, std::integral_constant<int, 4>{});
        };
        return with_row_vec<T>(width, with_kb);
    });
}
