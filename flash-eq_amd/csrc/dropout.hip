// Dropout of whole irreps from a counter-based generator (philox.h): y = x where a unit is kept, times the scale, and 0
// where it is dropped, whatever x holds there.  The gradient is the same product with grad_y, so the mask is formed
// again and never stored.
//
// With R = rows x channels, a table holds component d of row-channel rc at rc dim + d (node-major) or d R + rc
// (component-major); the unit of both is rc nreps + irrep of d, so the layouts drop the same.  All components of an irrep
// share one decision: one for each component would not commute with rotations.
//
// A workgroup takes a tile of row-channels, a multiple of eight, so that its units are whole blocks of the generator:
// its threads make a block each and leave the bits in LDS, the bits are spread to the components (node-major: one bit an
// element; component-major: a byte for eight neighbours of a plane, for each irrep), and the elements stream past
// them, eight a thread.  Elementwise dropout (scalars alone) takes the first step's bits as they are.
//
// Memory bounds it: 50000 x 64 x 9 float32 in 51 us, 4.5 TB/s read and written; 160000 x 896 bfloat16 in 112, 5.1 TB/s (the
// 256 MB cache behind the L2s keeps a part).  Numbers have 16 bits, so a block of the generator, ten rounds of four products,
// serves eight units: 32 bits would double its work for the same bytes.
#include <algorithm>

#include "elem_types.h"
#include "feq_internal.h"
#include "philox.h"

namespace feq {
namespace {

constexpr int kDrThreads = 256;
constexpr int kDrElems = 8192;          // elements of a tile, about
constexpr int kDrMaxReps = FEQ_MAX_IRREPS;
constexpr int kDrMaxDim = FEQ_MAX_SLOTS;

struct DrMap {
    int32_t dim, nreps;
    uint32_t bits[kDrMaxReps][kDrMaxDim / 32];   // components of every irrep
    int8_t rep[kDrMaxDim];
};

// `n` <= 8 elements at p times the scale, or 0 where their bit is not set.
template <class T>
__device__ __forceinline__ void drop8(const T* __restrict__ x, T* __restrict__ y, int n, uint32_t bits, float scale) {
    constexpr int V = 16 / sizeof(T);
    if (n >= 8) {
        float v[8 / V][V];
#pragma unroll
        for (int i = 0; i < 8 / V; ++i) load_f<T, V>(x + i * V, v[i]);
#pragma unroll
        for (int i = 0; i < 8 / V; ++i) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] = bits >> (i * V + j) & 1u ? v[i][j] * scale : 0.0f;
            store_f<T, V>(y + i * V, v[i]);
        }
    } else {
        for (int j = 0; j < n; ++j) y[j] = static_cast<T>(bits >> j & 1u ? static_cast<float>(x[j]) * scale : 0.0f);
    }
}

// Scalars alone: eight elements and one block a thread.
template <class T>
__global__ void __launch_bounds__(kDrThreads) k_drop_elems(const T* __restrict__ x, T* __restrict__ y, int64_t n, Drop drop) {
    const uint64_t key = static_cast<uint64_t>(*drop.seed);
    const int64_t step = static_cast<int64_t>(gridDim.x) * kDrThreads, blocks = (n + 7) / 8;
    for (int64_t b = static_cast<int64_t>(blockIdx.x) * kDrThreads + threadIdx.x; b < blocks; b += step) {
        const int64_t at = 8 * b;
        drop8<T>(x + at, y + at, n - at < 8 ? static_cast<int>(n - at) : 8, kept_bits(key, b, drop.limit), drop.scale);
    }
}

// `tile`: row-channels of a workgroup, a multiple of 8.  LDS: the units' bits (tile nreps / 8 bytes), then the
// components' (node-major: tile dim / 8 bytes; component-major: nreps tile / 8).
template <class T, bool CM>
__global__ void __launch_bounds__(kDrThreads)
k_drop_irreps(const T* __restrict__ x, T* __restrict__ y, int64_t R, int tile, DrMap map, Drop drop) {
    extern __shared__ __align__(16) uint32_t lds[];
    const int dim = map.dim, nreps = map.nreps, tid = threadIdx.x;
    const int64_t rc0 = static_cast<int64_t>(blockIdx.x) * tile;
    const int count = R - rc0 < tile ? static_cast<int>(R - rc0) : tile;
    uint8_t* units = reinterpret_cast<uint8_t*>(lds);
    const int unit_words = (tile * nreps / 8 + 3) / 4 + 1;         // one more: 64 bits are read from any byte on
    uint32_t* spread = lds + unit_words;
    const uint64_t key = static_cast<uint64_t>(*drop.seed);
    const int blocks = (count * nreps + 7) / 8;
    const uint64_t block0 = static_cast<uint64_t>(rc0) / 8 * nreps;
    for (int b = tid; b < blocks; b += kDrThreads) units[b] = static_cast<uint8_t>(kept_bits(key, block0 + b, drop.limit));
    if constexpr (!CM)
        for (int i = tid; i < (tile * dim + 31) / 32; i += kDrThreads) spread[i] = 0;
    __syncthreads();
    auto unit_bits = [&](int u, int n) {                            // n <= 32 units from u on
        const int w = u >> 5, s = u & 31;
        const uint64_t two = lds[w] | static_cast<uint64_t>(lds[w + 1]) << 32;
        return static_cast<uint32_t>(two >> s) & (n < 32 ? (1u << n) - 1u : ~0u);
    };
    if constexpr (!CM) {
        for (int rc = tid; rc < count; rc += kDrThreads) {
            uint32_t keep = unit_bits(rc * nreps, nreps);
            const int o = rc * dim, w0 = o >> 5, s = o & 31;
            for (int k = 0; 32 * k < dim; ++k) {
                uint32_t m = 0;
                for (int r = 0; r < nreps; ++r) m |= keep >> r & 1u ? map.bits[r][k] : 0u;
                if (m) {                                            // an OR does not depend on the order
                    atomicOr(&spread[w0 + k], m << s);
                    if (s && m >> (32 - s)) atomicOr(&spread[w0 + k + 1], m >> (32 - s));
                }
            }
        }
        __syncthreads();
        const uint8_t* bits = reinterpret_cast<const uint8_t*>(spread);
        const int64_t e0 = rc0 * dim;
        const int n = count * dim;
        for (int i = 8 * tid; i < n; i += 8 * kDrThreads) drop8<T>(x + e0 + i, y + e0 + i, n - i < 8 ? n - i : 8, bits[i >> 3], drop.scale);
    } else {
        uint8_t* bytes = reinterpret_cast<uint8_t*>(spread);        // of irrep r: from r tile / 8 on
        const int eights = tile / 8, have = (count + 7) / 8;
        for (int i = tid; i < nreps * have; i += kDrThreads) {
            const int r = i / have, q = i % have;
            uint32_t m = 0;
            for (int j = 0; j < 8; ++j) {
                const int u = (8 * q + j) * nreps + r;
                m |= (units[u >> 3] >> (u & 7) & 1u) << j;
            }
            bytes[r * eights + q] = static_cast<uint8_t>(m);
        }
        __syncthreads();
        for (int i = tid; i < dim * have; i += kDrThreads) {
            const int d = i / have, q = i % have;
            const int64_t at = d * R + rc0 + 8 * q;
            drop8<T>(x + at, y + at, count - 8 * q < 8 ? count - 8 * q : 8, bytes[map.rep[d] * eights + q], drop.scale);
        }
    }
}

}  // namespace
}  // namespace feq

using namespace feq;

extern "C" int feq_dropout(const int32_t* lvals, int32_t nreps, int64_t channels, int32_t component_major, int32_t dtype,
                           const void* x, double p, const int64_t* seed, void* y, feq_stream_t stream) {
    if (channels < 0) return fail(FEQ_ERR_INVALID, "%lld channels", (long long)channels);
    if (!(p >= 0.0 && p <= 1.0)) return fail(FEQ_ERR_INVALID, "a dropped share of %g is not in [0, 1]", p);
    if (!dtype_ok(dtype)) return fail(FEQ_ERR_INVALID, "unknown element type %d", dtype);
    if (!lvals || nreps < 1) return fail(FEQ_ERR_INVALID, "lvals must be non-empty");
    if (nreps > kDrMaxReps) return fail(FEQ_ERR_UNSUPPORTED, "more than %d irreps", kDrMaxReps);
    DrMap map{};
    map.nreps = nreps;
    int d = 0;
    for (int r = 0; r < nreps; ++r) {
        if (lvals[r] < 0) return fail(FEQ_ERR_INVALID, "negative degree");
        if (lvals[r] > kDrMaxDim || d + 2 * lvals[r] + 1 > kDrMaxDim)
            return fail(FEQ_ERR_UNSUPPORTED, "representation dimension exceeds %d", kDrMaxDim);
        for (int i = 0; i <= 2 * lvals[r]; ++i, ++d) {
            map.rep[d] = static_cast<int8_t>(r);
            map.bits[r][d / 32] |= 1u << d % 32;
        }
    }
    map.dim = d;
    if (channels > INT64_MAX / 4 / d) return fail(FEQ_ERR_UNSUPPORTED, "%lld channels of %d components", (long long)channels, d);
    if (channels == 0) return FEQ_OK;
    if (!x || !y || !seed) return fail(FEQ_ERR_INVALID, "NULL pointer");
    const Drop drop = make_drop(p, seed);
    hipStream_t s = stream_of(stream);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const T* in = static_cast<const T*>(x);
        T* out = static_cast<T*>(y);
        if (nreps == d && (!component_major || d == 1)) {
            const int64_t n = channels * d, blocks = std::min<int64_t>(ceil_div(n, 8 * kDrThreads), 1 << 20);
            auto kern = k_drop_elems<T>;
            FEQ_LAUNCH("k_drop_elems", kern, dim3(blocks), dim3(kDrThreads), 0, s, in, out, n, drop);
            return FEQ_OK;
        }
        const int tile = static_cast<int>(std::min<int64_t>(align_up(std::max(kDrElems / d, 8), 8), align_up(channels, 8)));
        const int64_t tiles = ceil_div(channels, tile);
        if (tiles > INT32_MAX / kDrThreads) return fail(FEQ_ERR_UNSUPPORTED, "%lld tiles", (long long)tiles);
        const size_t lds = 4 * ((tile * nreps / 8 + 3) / 4 + 1) + (component_major ? tile / 8 * nreps : (tile * d + 31) / 32 * 4 + 4);
        if (component_major) {
            auto kern = k_drop_irreps<T, true>;
            FEQ_LAUNCH("k_drop_irreps_cm", kern, dim3(tiles), dim3(kDrThreads), lds, s, in, out, channels, tile, map, drop);
        } else {
            auto kern = k_drop_irreps<T, false>;
            FEQ_LAUNCH("k_drop_irreps", kern, dim3(tiles), dim3(kDrThreads), lds, s, in, out, channels, tile, map, drop);
        }
        return FEQ_OK;
    });
}
