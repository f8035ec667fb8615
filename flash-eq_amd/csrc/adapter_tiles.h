// Pieces that the kernels of the adapters share: arguments, rows read where they lie, and the reduced rows as operands.
#pragma once

#include "expert_tiles.h"

namespace feq {
namespace {

constexpr int kAdMaxRank = 64;

// LDS written by the wave is read by its other lanes: no access passes this.
__device__ __forceinline__ void wave_lds() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

}  // namespace

struct AdArgs {
    const void *in, *W, *F, *G, *bias;
    const int32_t *offsets, *order;
    void* out;
    float* low;                  // NULL: not kept
    int X, S, K, N, R, nreps, nbias, dim;
    int rt;                      // rank tiles of 16
    float scale;
};

// Whether one kernel makes grad_x, grad_down and grad_up, and that kernel (a: grad_y, W, up, down, grad_x).
inline bool adapter_fused(int ci, int co, int R) { return ci <= 128 && co <= 128 && R <= 16; }
int adapter_bwd_fused(const int32_t* lvals, int32_t nreps, int32_t X, int64_t S, int32_t ci, int32_t co, int32_t R, int32_t dtype, AdArgs a,
                      const void* x, void* gdown, void* gup, float* parts, hipStream_t s);

namespace {


// The vector of elements k .. of the row at `row`, of which n exist (n <= 0: none); `safe`: any 16 bytes of the table.
template <class T, int HOW>
__device__ __forceinline__ uint4 load_row(const T* row, int k, int n, const T* safe) {
    constexpr int V = 16 / sizeof(T);
    if constexpr (HOW == kWhole) {
        return *reinterpret_cast<const uint4*>(n > 0 ? row + k : safe);
    } else if constexpr (HOW == kRagged) {
        const T* p = n < V ? row + k - (V - n) : row + k;
        const typename VecOf<T, V>::type v = *reinterpret_cast<const typename VecOf<T, V>::any*>(n > 0 ? p : safe);
        return __builtin_bit_cast(uint4, v);
    } else {
        typename VecOf<T, V>::type v;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const T e = n > j ? row[k + j] : *safe;
            v[j] = n > j ? e : static_cast<T>(0.0f);
        }
        return __builtin_bit_cast(uint4, v);
    }
}
// What load_row returned with its elements in place and zeros for those that do not exist.
template <class T, int HOW>
__device__ __forceinline__ uint4 placed_row(uint4 v, int n, int length, const T* safe) {
    if constexpr (HOW == kWhole) return n > 0 ? v : uint4{0, 0, 0, 0};
    else return arrived16<T, HOW>(rows_at(safe, safe, length), v, n);
}

// Largest of a row's values over the lanes (c, 0 .. 3).
__device__ __forceinline__ float row_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The second product's operand of four reduced values.
__device__ __forceinline__ v4f low_frag(v4f t, float) { return t; }
__device__ __forceinline__ b8 low_frag(v4f t, __bf16) {
    b8 f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[j] = static_cast<__bf16>(t[j]);
        f[j + 4] = static_cast<__bf16>(t[j] - static_cast<float>(f[j]));
    }
    return f;
}
__device__ __forceinline__ h8 low_frag(v4f t, _Float16) {
    h8 f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[j] = static_cast<_Float16>(t[j]);
        f[j + 4] = static_cast<_Float16>(t[j] - static_cast<float>(f[j]));
    }
    return f;
}
// G's operand: four elements of a row, in 16-bit types twice.
template <class T>
__device__ __forceinline__ typename Mma<T>::frag twice(const T (&e)[4]) {
    typename Mma<T>::frag f;
#pragma unroll
    for (int j = 0; j < Mma<T>::FE; ++j) f[j] = e[j & 3];
    return f;
}

// The same of column n and ranks r .. r + 3, from memory; zeros for what does not exist.
template <class T, bool TRANS>
__device__ __forceinline__ typename Mma<T>::frag second_frag(const T* ge, int n, int r, int N, int R) {
    T e[4];
    if (!TRANS && R % 4 == 0) {                      // uniform: four ranks at once, aligned as an element
        const bool has = n < N && r < R;
        const typename VecOf<T, 4>::type v = *reinterpret_cast<const typename VecOf<T, 4>::any*>(ge + (has ? static_cast<int64_t>(n) * R + r : 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = has ? v[j] : static_cast<T>(0.0f);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool has = n < N && r + j < R;
            const T v = ge[has ? (TRANS ? static_cast<int64_t>(r + j) * N + n : static_cast<int64_t>(n) * R + r + j) : 0];
            e[j] = has ? v : static_cast<T>(0.0f);
        }
    }
    return twice<T>(e);
}

// The power of two that a row of reduced values is multiplied by (float16), its exponent; 0 for a row of zeros, or one
// that is not finite.  64 at most: the shared map's sum of up to 65536 products of float16 numbers, below 2^48, is multiplied
// too and stays in float32's range.  Rows that would need more lose what is below 2^-14 after the product, so 2^-78 of a reduced
// value: 2^-32 in a sum over 2^30 rows of float16 numbers, where half a step of the smallest result is 2^-25.
constexpr int kAdMaxPower = 64;
__device__ __forceinline__ int low_exponent(float most) {
    const int e = static_cast<int>(__float_as_uint(most) >> 23 & 255u);
    const int p = 127 + 13 - e;
    return e == 0 || e == 255 ? 0 : p < kAdMaxPower ? p : kAdMaxPower;
}
__device__ __forceinline__ float times_power(float v, int e) { return __builtin_amdgcn_ldexpf(v, e); }


struct AdShape {
    const int32_t* lvals;
    int32_t nreps;
    int32_t X;
    int64_t S;
    int32_t ci, co, R, dtype;
};

// Row chunks of a sum over rows, all of about as many row-planes, so that `want` workgroups and the adapters' last, shorter
// chunks run at once; rows are rounded up to `unit`.  Returns the number of partials.
inline int64_t adapter_chunks(const AdShape& p, int want, int unit, XlChunks* ch) {
    int64_t dim = 0;
    for (int r = 0; r < p.nreps; ++r) dim += 2 * p.lvals[r] + 1;
    const int64_t full = std::max<int64_t>(want - static_cast<int64_t>(p.X + 1) * p.nreps, want / 2);
    const int64_t share = ceil_div(std::max<int64_t>(p.S, 1) * dim, full);
    int64_t tiles = 0, slots = 0;
    ch->xcds = 8;
    for (int r = p.nreps - 1; r >= 0; --r) {
        const int64_t rows = std::min<int64_t>(ceil_div(ceil_div(share, 2 * p.lvals[r] + 1), unit) * unit, 1 << 20);
        ch->rows[r] = static_cast<int32_t>(rows);
        ch->tile0[r] = static_cast<int32_t>(tiles);
        ch->slot0[r] = static_cast<int32_t>(slots);
        tiles += ceil_div(p.S / rows + p.X + 1, ch->xcds);
        slots += p.S > rows ? 2 * p.S / rows : 0;
    }
    ch->tile0[p.nreps] = static_cast<int32_t>(tiles);
    ch->slot0[p.nreps] = static_cast<int32_t>(slots);
    return slots;
}
// Those of the kernel that adapter_fused names.
inline int64_t fused_chunks(const AdShape& p, XlChunks* ch) { return adapter_chunks(p, p.dtype == FEQ_F32 && p.ci > 64 && p.co > 64 ? 256 : 512, 16, ch); }

}  // namespace
}  // namespace feq
