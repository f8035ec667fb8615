// Layer norm over the last axis: for each row of x (rows, width)
//   mu = mean_j x_j,  v = mean_j (x_j - mu)^2,  s = 1 / sqrt(v + eps),
//   y_j = (x_j - mu) s w_j + b_j,
// and, for the gradient g of y with xh = (x - mu) s and h = g w,
//   grad_x = s (h - mean(h) - xh mean(h xh)),
//   grad_w = sum over rows of g xh,  grad_b = sum over rows of g.
//
// HBM bounds both directions (about 20 operations per element), so each reads
// its tables once: a group of G lanes (or a whole workgroup, for wide rows)
// holds a row in registers, forms the mean and then the variance of the
// differences from it (two passes over registers: no cancellation for rows with
// a large mean) and writes the result.  Every value, statistic and sum is
// float32; the only rounding to fewer bits is the one of the stored result.
// In the backward a lane keeps the same columns for all rows of its workgroup,
// so grad_w and grad_b are per-lane sums over rows, summed over the workgroup
// once and over the workgroups by k_ln_wsum in a fixed order (no atomics: the
// same bits on every run).
//
// Rows wider than the register forms hold (32 elements a thread) are read again
// for each pass, from L2 (the _wide kernels).
#include "elem_types.h"
#include "feq_internal.h"
#include "lane_math.h"

namespace feq {
namespace {

constexpr int kLnThreads = 256;
constexpr int kLnWaveElems = 16;    // elements a lane holds in the lane-group form
constexpr int kLnBlockElems = 32;   // and in the workgroup form
constexpr int kLnFwdBlocks = 2048;   // workgroups of the forward: what the chip holds, each over many rows
constexpr int kLnMaxBlocks = 1024;  // workgroups of the backward, and weight-gradient partials
constexpr int64_t kLnMaxWidth = 1 << 24;
constexpr int kLnWide = 1024;       // threads of the _wide kernels
constexpr int kLnWideBlocks = 64;   // their weight-gradient partials
constexpr int kLnOneRows = 8;       // rows of a lane group up to which one workgroup makes the backward

// Sum over the workgroup of NW waves; red holds 2 NW floats, one use per call.
template <int NW>
__device__ __forceinline__ void block_sum2(float& a, float& b, float* red) {
    a = group_sum(a, 64);
    b = group_sum(b, 64);
    const int wave = threadIdx.x >> 6;
    __syncthreads();          // the previous call's readers are done
    if ((threadIdx.x & 63) == 0) {
        red[2 * wave] = a;
        red[2 * wave + 1] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        a += red[2 * w];
        b += red[2 * w + 1];
    }
}

// Vectors of V elements (width >= V; vec_begin, vec_shared); lane `l` of a group of `G` holds vectors l, l + G, ...
// 50000 x 192 float32: 16 us; 160000 x 896 bfloat16: 113 us, 5.1 TB/s.
template <class T, int V, int NV, bool BLK>
__global__ void __launch_bounds__(kLnThreads)
k_ln_fwd(const T* __restrict__ x, int64_t rows, int width, int64_t ldx, const void* __restrict__ w,
         const void* __restrict__ b, int pdt, float eps, T* __restrict__ y, float* __restrict__ mean,
         float* __restrict__ rstd, int G) {
    __shared__ float red[8];
    const int L = BLK ? kLnThreads : G;
    const int l = threadIdx.x & (L - 1);
    const int per = kLnThreads / L;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * per;
    const int nvec = (width + V - 1) / V;
    const float inv = 1.0f / static_cast<float>(width);
    float wv[NV][V], bv[NV][V];
    int at[NV], sh[NV];      // a vector's first column, and how many of its columns the vector before has
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int q = l + v * L;
        at[v] = vec_begin<V>(q, width);
        sh[v] = vec_shared<V>(q, width);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            wv[v][j] = 1.0f;
            bv[v][j] = 0.0f;
        }
        if (w && q < nvec) load_any_v<V>(w, pdt, at[v], wv[v]);
        if (b && q < nvec) load_any_v<V>(b, pdt, at[v], bv[v]);
    }
    float xv[NV][V], xn[NV][V];
    auto load = [&](int64_t r, float (&o)[NV][V]) {
        const T* xr = x + r * ldx;
#pragma unroll
        for (int v = 0; v < NV; ++v) load_f<T, V>(xr + at[v], o[v]);     // a vector of the row in every lane
    };
    int64_t r = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / L;
    if (r < rows) load(r, xv);
    for (; r < rows; r += stride) {
        load(r + stride < rows ? r + stride : r, xn);     // the next row, in flight during this one's sums
        float s = 0.0f, z = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < V; ++j) s += j >= sh[v] ? xv[v][j] : 0.0f;
        if constexpr (BLK) block_sum2<4>(s, z, red);
        else s = group_sum(s, G);
        const float mu = s * inv;
        float q2 = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                xv[v][j] -= mu;
                q2 += j >= sh[v] ? xv[v][j] * xv[v][j] : 0.0f;
            }
        if constexpr (BLK) block_sum2<4>(q2, z, red);
        else q2 = group_sum(q2, G);
        const float rs = 1.0f / sqrtf(q2 * inv + eps);
        T* yr = y + r * width;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int q = l + v * L;
            if (q < nvec) {
                float o[V];
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] = xv[v][j] * rs * wv[v][j] + bv[v][j];
                store_f<T, V>(yr + at[v], o);
            }
        }
        if (l == 0 && mean) {
            mean[r] = mu;
            rstd[r] = rs;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < V; ++j) xv[v][j] = xn[v][j];
    }
}

// The workgroups' sums of grad_w and grad_b go to part (gridDim.x, 2, width), or as gradients to gw and gb where there
// is one workgroup; all NULL: not wanted.  gx may be NULL.  50000 x 192 float32: 22 us; 160000 x 896 bfloat16: 171 us, 5.0
// TB/s.
template <class T, int V, int NV, bool BLK>
__global__ void __launch_bounds__(kLnThreads)
k_ln_bwd(const T* __restrict__ gy, int64_t ldg, const T* __restrict__ x, int64_t rows, int width, int64_t ldx,
         const void* __restrict__ w, int pdt, const float* __restrict__ mean, const float* __restrict__ rstd,
         T* __restrict__ gx, float* __restrict__ part, void* __restrict__ gw, void* __restrict__ gb, int G) {
    __shared__ float red[8];
    // the waves' column sums: 4 waves x (64 lanes x NV V columns) x 2
    __shared__ float sums[BLK ? 1 : 4 * 64 * NV * V * 2];
    const int L = BLK ? kLnThreads : G;
    const int l = threadIdx.x & (L - 1);
    const int per = kLnThreads / L;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * per;
    const int nvec = (width + V - 1) / V;
    const float inv = 1.0f / static_cast<float>(width);
    float wv[NV][V], dw[NV][V], db[NV][V];
    int at[NV], sh[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int q = l + v * L;
        at[v] = vec_begin<V>(q, width);
        sh[v] = vec_shared<V>(q, width);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            wv[v][j] = 1.0f;
            dw[v][j] = db[v][j] = 0.0f;
        }
        if (w && q < nvec) load_any_v<V>(w, pdt, at[v], wv[v]);
    }
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / L; r < rows; r += stride) {
        const T* xr = x + r * ldx;
        const T* gr = gy + r * ldg;
        const float mu = mean[r], rs = rstd[r];
        float xh[NV][V], h[NV][V];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            load_f<T, V>(xr + at[v], xh[v]);
            load_f<T, V>(gr + at[v], h[v]);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                xh[v][j] = (xh[v][j] - mu) * rs;
                dw[v][j] += h[v][j] * xh[v][j];
                db[v][j] += h[v][j];
                h[v][j] *= wv[v][j];
                s1 += j >= sh[v] ? h[v][j] : 0.0f;
                s2 += j >= sh[v] ? h[v][j] * xh[v][j] : 0.0f;
            }
        if (gx) {
            if constexpr (BLK) block_sum2<4>(s1, s2, red);
            else {
                s1 = group_sum(s1, G);
                s2 = group_sum(s2, G);
            }
            s1 *= inv;
            s2 *= inv;
            T* dr = gx + r * width;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int q = l + v * L;
                if (q < nvec) {
                    float o[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) o[j] = rs * (h[v][j] - s1 - xh[v][j] * s2);
                    store_f<T, V>(dr + at[v], o);
                }
            }
        }
    }
    if (!part && !gw && !gb) return;
    float* pw = part + static_cast<int64_t>(blockIdx.x) * 2 * width;
    auto put = [&](int c, float a, float d) {
        if (part) {
            pw[c] = a;
            pw[width + c] = d;
        } else {
            if (gw) store_any(gw, pdt, c, a);
            if (gb) store_any(gb, pdt, c, d);
        }
    };
    if constexpr (BLK) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (j >= sh[v]) put(at[v] + j, dw[v][j], db[v][j]);
            }
    } else {
        // the groups of a wave, then the waves
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int cols = G * NV * V;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float a = dw[v][j], c = db[v][j];
                for (int o = G; o < 64; o <<= 1) {
                    a += __shfl_xor(a, o, 64);
                    c += __shfl_xor(c, o, 64);
                }
                if (lane < G) {
                    const int col = (lane + v * G) * V + j;
                    sums[(wave * cols + col) * 2] = a;
                    sums[(wave * cols + col) * 2 + 1] = c;
                }
            }
        __syncthreads();
        for (int c = threadIdx.x; c < width; c += kLnThreads) {
            const int last = (nvec - 1) * V, place = c < last ? c : last + c - (width - V);
            float a = 0.0f, d = 0.0f;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                a += sums[(u * cols + place) * 2];
                d += sums[(u * cols + place) * 2 + 1];
            }
            put(c, a, d);
        }
    }
}

// grad_w, grad_b (of type pdt) from `groups` partials (2, width): 16 columns a
// workgroup, 64 rows of partials side by side, each summed in order and the 64
// sums in order.
__global__ void __launch_bounds__(1024)
k_ln_wsum(const float* __restrict__ part, int groups, int width, void* __restrict__ gw, void* __restrict__ gb, int pdt) {
    __shared__ float s[64][17];
    const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int64_t n = 2 * static_cast<int64_t>(width);
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 16 + c;
    float a = 0.0f;
    if (col < n) {
#pragma unroll 8
        for (int r = r0; r < groups; r += 64) a += part[r * n + col];
    }
    s[r0][c] = a;
    __syncthreads();
    for (int o = 32; o; o >>= 1) {
        if (r0 < o) s[r0][c] += s[r0 + o][c];
        __syncthreads();
    }
    if (r0 == 0 && col < n) {
        if (col < width) {
            if (gw) store_any(gw, pdt, col, s[0][c]);
        } else if (gb) {
            store_any(gb, pdt, col - width, s[0][c]);
        }
    }
}

// ---- rows wider than a workgroup's registers -----------------------------------
template <class T>
__global__ void __launch_bounds__(kLnWide)
k_ln_fwd_wide(const T* __restrict__ x, int64_t rows, int64_t width, int64_t ldx, const void* __restrict__ w,
              const void* __restrict__ b, int pdt, float eps, T* __restrict__ y, float* __restrict__ mean,
              float* __restrict__ rstd) {
    __shared__ float red[32];
    const float inv = 1.0f / static_cast<float>(width);
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * ldx;
        float s = 0.0f, z = 0.0f, q2 = 0.0f;
        for (int64_t c = threadIdx.x; c < width; c += kLnWide) s += static_cast<float>(xr[c]);
        block_sum2<16>(s, z, red);
        const float mu = s * inv;
        for (int64_t c = threadIdx.x; c < width; c += kLnWide) {
            const float d = static_cast<float>(xr[c]) - mu;
            q2 += d * d;
        }
        block_sum2<16>(q2, z, red);
        const float rs = 1.0f / sqrtf(q2 * inv + eps);
        for (int64_t c = threadIdx.x; c < width; c += kLnWide) {
            const float wv = w ? load_any(w, pdt, c) : 1.0f, bv = b ? load_any(b, pdt, c) : 0.0f;
            y[r * width + c] = static_cast<T>((static_cast<float>(xr[c]) - mu) * rs * wv + bv);
        }
        if (threadIdx.x == 0 && mean) {
            mean[r] = mu;
            rstd[r] = rs;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kLnWide)
k_ln_bwd_wide(const T* __restrict__ gy, int64_t ldg, const T* __restrict__ x, int64_t rows, int64_t width,
              int64_t ldx, const void* __restrict__ w, int pdt, const float* __restrict__ mean,
              const float* __restrict__ rstd, T* __restrict__ gx) {
    __shared__ float red[32];
    const float inv = 1.0f / static_cast<float>(width);
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * ldx;
        const T* gr = gy + r * ldg;
        const float mu = mean[r], rs = rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
        for (int64_t c = threadIdx.x; c < width; c += kLnWide) {
            const float h = static_cast<float>(gr[c]) * (w ? load_any(w, pdt, c) : 1.0f);
            s1 += h;
            s2 += h * ((static_cast<float>(xr[c]) - mu) * rs);
        }
        block_sum2<16>(s1, s2, red);
        s1 *= inv;
        s2 *= inv;
        for (int64_t c = threadIdx.x; c < width; c += kLnWide) {
            const float h = static_cast<float>(gr[c]) * (w ? load_any(w, pdt, c) : 1.0f);
            const float xh = (static_cast<float>(xr[c]) - mu) * rs;
            gx[r * width + c] = static_cast<T>(rs * (h - s1 - xh * s2));
        }
    }
}

// part (gridDim.y, 2, width): a thread per column, a run of rows per blockIdx.y; NULL (one run): gradients to gw, gb.
template <class T>
__global__ void __launch_bounds__(256)
k_ln_cols_wide(const T* __restrict__ gy, int64_t ldg, const T* __restrict__ x, int64_t rows, int64_t width,
               int64_t ldx, const float* __restrict__ mean, const float* __restrict__ rstd, int64_t per,
               float* __restrict__ part, void* __restrict__ gw, void* __restrict__ gb, int pdt) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= width) return;
    const int64_t r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
    float a = 0.0f, d = 0.0f;
    for (int64_t r = r0; r < r1; ++r) {
        const float g = static_cast<float>(gy[r * ldg + c]);
        a += g * ((static_cast<float>(x[r * ldx + c]) - mean[r]) * rstd[r]);
        d += g;
    }
    if (part) {
        float* pw = part + static_cast<int64_t>(blockIdx.y) * 2 * width;
        pw[c] = a;
        pw[width + c] = d;
    } else {
        if (gw) store_any(gw, pdt, c, a);
        if (gb) store_any(gb, pdt, c, d);
    }
}

// ---- which form takes a width ----------------------------------------------------
struct LnForm {
    bool blk;    // a workgroup per row, else a group of G lanes
    int G, NV;
};
bool ln_wide(int64_t width) { return width > kLnThreads * kLnBlockElems; }     // the _wide kernels

// NV of the instances: the smallest that covers (n <= 8: kLnBlockElems elements of at least four a vector).
inline int ln_nv(int64_t n) { return n <= 4 ? static_cast<int>(n) : 8; }

LnForm ln_form(int64_t width, int V) {
    LnForm f{false, 64, 1};
    const int64_t nvec = ceil_div(width, V);
    if (V == 1) {                // a column a lane: fewer columns than a vector
        f.G = 1;
        while (f.G < nvec) f.G <<= 1;
        return f;
    }
    for (int g = 1; g <= 64; g <<= 1) {
        const int nv = ln_nv(ceil_div(nvec, g));
        if (nv * V <= kLnWaveElems) {
            f.G = g;
            f.NV = nv;
            return f;
        }
    }
    f.blk = true;
    f.NV = ln_nv(ceil_div(nvec, kLnThreads));
    return f;
}

// f(NV) for the instance that holds `nv` vectors a lane
template <int V, class F>
int ln_with_nv(int nv, F&& f) {
    if constexpr (V == 1) return f(std::integral_constant<int, 1>{});       // rows narrower than a vector
    switch (nv) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        case 3: return f(std::integral_constant<int, 3>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 8: if constexpr (8 * V <= kLnBlockElems) return f(std::integral_constant<int, 8>{}); else break;
    }
    return fail(FEQ_ERR_INVALID, "internal: layer norm form");
}

template <class T, int V>
int ln_fwd_run(const T* x, int64_t rows, int width, int64_t ldx, const void* w, const void* b, int pdt, float eps,
               T* y, float* mean, float* rstd, const LnForm& f, hipStream_t s) {
    const int per = f.blk ? 1 : kLnThreads / f.G;
    const int64_t blocks = std::min<int64_t>(ceil_div(rows, per), kLnFwdBlocks);
    return ln_with_nv<V>(f.NV, [&](auto nv) -> int {
        constexpr int NV = decltype(nv)::value;
        if (f.blk) {
            auto kern = k_ln_fwd<T, V, NV, true>;
            FEQ_LAUNCH("k_ln_fwd", kern, dim3(blocks), dim3(kLnThreads), 0, s, x, rows, width, ldx, w, b, pdt, eps, y,
                       mean, rstd, f.G);
        } else if constexpr (NV * V <= kLnWaveElems) {
            auto kern = k_ln_fwd<T, V, NV, false>;
            FEQ_LAUNCH("k_ln_fwd", kern, dim3(blocks), dim3(kLnThreads), 0, s, x, rows, width, ldx, w, b, pdt, eps, y,
                       mean, rstd, f.G);
        }
        return FEQ_OK;
    });
}

template <class T, int V>
int ln_bwd_run(const T* gy, int64_t ldg, const T* x, int64_t rows, int width, int64_t ldx, const void* w, int pdt,
               const float* mean, const float* rstd, T* gx, float* part, void* gw, void* gb, int blocks, const LnForm& f,
               hipStream_t s) {
    return ln_with_nv<V>(f.NV, [&](auto nv) -> int {
        constexpr int NV = decltype(nv)::value;
        if (f.blk) {
            auto kern = k_ln_bwd<T, V, NV, true>;
            FEQ_LAUNCH("k_ln_bwd", kern, dim3(blocks), dim3(kLnThreads), 0, s, gy, ldg, x, rows, width, ldx, w, pdt,
                       mean, rstd, gx, part, gw, gb, f.G);
        } else if constexpr (NV * V <= kLnWaveElems) {
            auto kern = k_ln_bwd<T, V, NV, false>;
            FEQ_LAUNCH("k_ln_bwd", kern, dim3(blocks), dim3(kLnThreads), 0, s, gy, ldg, x, rows, width, ldx, w, pdt,
                       mean, rstd, gx, part, gw, gb, f.G);
        }
        return FEQ_OK;
    });
}

int ln_check(int64_t rows, int64_t width, int64_t ldx, int32_t dtype, const void* x, const void* w, const void* b,
             int32_t pdt) {
    if (rows < 0 || width < 1) return fail(FEQ_ERR_INVALID, "layer norm of %lld rows of width %lld", (long long)rows, (long long)width);
    if (width > kLnMaxWidth) return fail(FEQ_ERR_UNSUPPORTED, "layer norm width %lld exceeds 2^24", (long long)width);
    if (ldx < width) return fail(FEQ_ERR_INVALID, "row stride %lld is smaller than the width %lld", (long long)ldx, (long long)width);
    if (!dtype_ok(dtype)) return fail(FEQ_ERR_INVALID, "unknown element type %d", dtype);
    if ((w || b) && !dtype_ok(pdt)) return fail(FEQ_ERR_INVALID, "unknown parameter type %d", pdt);
    if (rows && !x) return fail(FEQ_ERR_INVALID, "NULL pointer");
    return FEQ_OK;
}

// Workgroups of the backward, each with a partial of the weight gradients where `params` wants them.  Few rows
// (kLnOneRows a lane group) then take one workgroup, which writes the gradients itself: launches bound such calls (100
// rows of 192 with their gradients: 60 -> 55 us).  grad_x alone has no launch to save (8 rows of 8000 bfloat16 columns:
// 13.0 us in one workgroup, 4.6 in eight; 128 x 192 float32: 7.8 and 3.5).  Partials of many wide rows would take more memory than the rows: at most kLnWideBlocks.
int ln_bwd_blocks(int64_t rows, int64_t width, int32_t dtype, bool params) {
    if (ln_wide(width)) return static_cast<int>(std::min<int64_t>(rows, kLnWideBlocks));
    const int V = 16 / elem_size(dtype);
    const LnForm f = ln_form(width, width >= V ? V : 1);
    const int64_t rounds = ceil_div(rows, f.blk ? 1 : kLnThreads / f.G);
    return params && rounds <= kLnOneRows ? 1 : static_cast<int>(std::min<int64_t>(rounds, kLnMaxBlocks));
}

}  // namespace
}  // namespace feq

using namespace feq;

extern "C" int feq_layernorm_fwd(const void* x, int64_t rows, int64_t width, int64_t ldx, int32_t dtype,
                                 const void* weight, const void* bias, int32_t param_dtype, float eps, void* y,
                                 float* mean, float* rstd, feq_stream_t stream) {
    if (int rc = ln_check(rows, width, ldx, dtype, x, weight, bias, param_dtype)) return rc;
    if (rows == 0) return FEQ_OK;
    if (!y) return fail(FEQ_ERR_INVALID, "NULL pointer");
    if ((mean == nullptr) != (rstd == nullptr)) return fail(FEQ_ERR_INVALID, "mean and rstd are given together or not at all");
    hipStream_t s = stream_of(stream);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        constexpr int VV = 16 / sizeof(T);
        const T* xt = static_cast<const T*>(x);
        T* yt = static_cast<T*>(y);
        const bool vec = width >= VV;
        const LnForm f = ln_form(width, vec ? VV : 1);
        if (ln_wide(width)) {
            auto kern = k_ln_fwd_wide<T>;
            FEQ_LAUNCH("k_ln_fwd_wide", kern, dim3(std::min<int64_t>(rows, 4096)), dim3(kLnWide), 0, s, xt, rows, width,
                       ldx, weight, bias, param_dtype, eps, yt, mean, rstd);
            return FEQ_OK;
        }
        const int w32 = static_cast<int>(width);
        return vec ? ln_fwd_run<T, VV>(xt, rows, w32, ldx, weight, bias, param_dtype, eps, yt, mean, rstd, f, s)
                   : ln_fwd_run<T, 1>(xt, rows, w32, ldx, weight, bias, param_dtype, eps, yt, mean, rstd, f, s);
    });
}

extern "C" size_t feq_layernorm_bwd_workspace(int64_t rows, int64_t width, int32_t dtype) {
    if (rows < 1 || width < 1 || width > kLnMaxWidth || !dtype_ok(dtype)) return 0;
    const int blocks = ln_bwd_blocks(rows, width, dtype, true);
    return blocks > 1 ? sizeof(float) * 2 * static_cast<size_t>(width) * blocks : 0;
}

extern "C" int feq_layernorm_bwd(const void* grad_y, int64_t ldg, const void* x, int64_t rows, int64_t width,
                                 int64_t ldx, int32_t dtype, const void* weight, int32_t param_dtype,
                                 const float* mean, const float* rstd, void* grad_x, void* grad_w, void* grad_b,
                                 void* workspace, size_t ws_bytes, feq_stream_t stream) {
    if (int rc = ln_check(rows, width, ldx, dtype, x, weight, nullptr, param_dtype)) return rc;
    if (ldg < width) return fail(FEQ_ERR_INVALID, "row stride %lld is smaller than the width %lld", (long long)ldg, (long long)width);
    const bool params = grad_w || grad_b;
    if (params && !dtype_ok(param_dtype)) return fail(FEQ_ERR_INVALID, "unknown parameter type %d", param_dtype);
    if (rows && (!grad_y || !mean || !rstd)) return fail(FEQ_ERR_INVALID, "NULL pointer");
    if (!grad_x && !params) return FEQ_OK;
    const size_t need = params ? feq_layernorm_bwd_workspace(rows, width, dtype) : 0;
    if (need && (!workspace || ws_bytes < need))
        return fail(FEQ_ERR_WORKSPACE, "layer norm workspace of %zu bytes, %zu needed", ws_bytes, need);
    hipStream_t s = stream_of(stream);
    float* part = need ? static_cast<float*>(workspace) : nullptr;
    int blocks = rows ? ln_bwd_blocks(rows, width, dtype, params) : 0;
    if (rows) {
        const int rc = with_dtype(dtype, [&](auto t) -> int {
            using T = decltype(t);
            constexpr int VV = 16 / sizeof(T);
            const T *gt = static_cast<const T*>(grad_y), *xt = static_cast<const T*>(x);
            T* dt = static_cast<T*>(grad_x);
            const bool vec = width >= VV;
            const LnForm f = ln_form(width, vec ? VV : 1);
            if (ln_wide(width)) {
                if (dt) {
                    auto kern = k_ln_bwd_wide<T>;
                    FEQ_LAUNCH("k_ln_bwd_wide", kern, dim3(std::min<int64_t>(rows, 4096)), dim3(kLnWide), 0, s, gt, ldg,
                               xt, rows, width, ldx, weight, param_dtype, mean, rstd, dt);
                }
                if (params) {
                    const int64_t per = ceil_div(rows, blocks);
                    blocks = static_cast<int>(ceil_div(rows, per));
                    auto kern = k_ln_cols_wide<T>;
                    FEQ_LAUNCH("k_ln_cols_wide", kern, dim3(ceil_div(width, 256), blocks), dim3(256), 0, s, gt, ldg, xt,
                               rows, width, ldx, mean, rstd, per, part, grad_w, grad_b, param_dtype);
                }
                return FEQ_OK;
            }
            const int w32 = static_cast<int>(width);
            void *gw = part ? nullptr : grad_w, *gb = part ? nullptr : grad_b;
            return vec ? ln_bwd_run<T, VV>(gt, ldg, xt, rows, w32, ldx, weight, param_dtype, mean, rstd, dt, part, gw, gb, blocks, f, s)
                       : ln_bwd_run<T, 1>(gt, ldg, xt, rows, w32, ldx, weight, param_dtype, mean, rstd, dt, part, gw, gb, blocks, f, s);
        });
        if (rc) return rc;
    }
    if (params && (part || rows == 0))     // with no rows: the sums of no partials, zeros
        FEQ_LAUNCH("k_ln_wsum", k_ln_wsum, dim3(ceil_div(2 * width, 16)), dim3(1024), 0, s, part, blocks,
                   static_cast<int>(width), grad_w, grad_b, param_dtype);
    return FEQ_OK;
}
