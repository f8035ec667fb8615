// Tiles of the channel maps whose rows are grouped by expert (or adapter): matrix-core steps, row and column loads of any
// length and alignment, the numbering of an expert's row blocks, and the sums of weight gradients over row chunks.
#pragma once

#include <algorithm>
#include <type_traits>

#include "elem_types.h"
#include "feq_internal.h"
#include "lane_math.h"
#include "tile_math.h"

namespace feq {
namespace {

constexpr int kXlMaxPlanes = FEQ_MAX_SLOTS;
constexpr int kXlMaxReps = FEQ_MAX_IRREPS;
constexpr int kXlMaxExperts = 1024;
constexpr int64_t kXlMaxRows = int64_t{1} << 30;     // a row's number and a chunk's length more fit 32 bits
constexpr int kXlThreads = 256;
constexpr int kXlBM = 128;          // rows of a block
constexpr int kXlStreamK = 128;     // reduction columns of the streaming kernel
constexpr int kXlRowBytes = 128;    // bytes of the reduction staged per row (32 floats, 64 16-bit elements)

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

// Irrep and bias column (-1: none) of every plane; first plane of every irrep.
struct XlMap {
    int8_t rep[kXlMaxPlanes];
    int8_t bcol[kXlMaxPlanes];
    int16_t first[kXlMaxReps + 1];
};

// Weight-gradient chunks, which the irreps of many planes have shorter: rows of a chunk, the first chunk's number over
// `xcds` (irreps in descending order, as launched) and first partial of every irrep; irrep of every bias column.
struct XlChunks {
    int32_t rows[kXlMaxReps];
    int32_t tile0[kXlMaxReps + 1];
    int32_t slot0[kXlMaxReps + 1];
    int8_t brep[kXlMaxReps];
    int32_t xcds;        // XCDs that chunks are dealt to, each with all its tiles; 1: the tiles are
};

// One reduction step of a 16 x 16 tile: KS elements, a lane holding FE of them.
// Lane (c = l % 16, g = l / 16) holds elements FE g .. FE g + FE - 1 of row (or column) c.
template <class T>
struct Mma;
template <>
struct Mma<float> {
    static constexpr int KS = 16, FE = 4;
    typedef v4f frag;
    static __device__ __forceinline__ v4f mul(frag a, frag b, v4f c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = mfma4(a[j], b[j], c);
        return c;
    }
    // tile by tile within a step, so that no product waits for the one before
    template <int NT>
    static __device__ __forceinline__ void mul_all(const frag (&a)[NT], frag b, v4f* acc) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[i] = mfma4(a[i][j], b[j], acc[i]);
    }
    static constexpr int PAD = 4;      // four rows are 16 banks apart
    // element j: row k0 + 4 g + j, column c0 + c of a table with `stride` elements a row
    static __device__ __forceinline__ frag columns(const float* t, int stride, int k0, int g, int c, int c0) {
        const float* p = t + (k0 + 4 * g) * stride + c0 + c;
        return frag{p[0], p[stride], p[2 * stride], p[3 * stride]};
    }
};
// ds_read_b64_tr_b16: in a group of 16 lanes, lane s points at row s / 4 and the four columns of the group's
// quad s % 4 and receives, of column s, the four rows.
template <class T, class F>
struct MmaHalf {
    static constexpr int KS = 32, FE = 8;
    static constexpr int PAD = 16;     // a row is 8 banks on from the one before
    typedef F frag;
    static __device__ __forceinline__ frag columns(const T* t, int stride, int k0, int g, int c, int c0) {
        const T* p = t + (k0 + 8 * g + (c >> 2)) * stride + c0 + 4 * (c & 3);
        const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p));
        const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p + 4 * stride));
        const v8s v = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        return __builtin_bit_cast(frag, v);
    }
};
template <>
struct Mma<_Float16> : MmaHalf<_Float16, h8> {
    static __device__ __forceinline__ v4f mul(h8 a, h8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    template <int NT>
    static __device__ __forceinline__ void mul_all(const frag (&a)[NT], frag b, v4f* acc) {
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i] = mul(a[i], b, acc[i]);
    }
};
template <>
struct Mma<__bf16> : MmaHalf<__bf16, b8> {
    static __device__ __forceinline__ v4f mul(b8 a, b8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    template <int NT>
    static __device__ __forceinline__ void mul_all(const frag (&a)[NT], frag b, v4f* acc) {
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i] = mul(a[i], b, acc[i]);
    }
};

// A table read by buffer loads: an offset past its end gives zeros, so absent rows and columns cost no branch.  (A
// branch around a load makes the compiler wait for every load in flight at the next use: with branches the products of
// 8191 bfloat16 rows, 512 to 1024 columns, took 36 us whatever was prefetched.)  Base and size are uniform.
typedef __amdgpu_buffer_rsrc_t Table;
constexpr uint32_t kTableBytes = 0x7ffffff0u, kOutside = 0x80000000u;
__device__ __forceinline__ Table table(const void* p, bool there = true) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, there ? kTableBytes : 0u, 0x00020000);
}

// How the rows of a table lie: multiples of 16 bytes, aligned to them (kWhole); of any length of at least 16 bytes and
// any alignment (kRagged); shorter (kNarrow).
enum { kWhole, kRagged, kNarrow };

// Rows read in vectors of V elements from multiples of V on.  The last vector of a ragged row (`n` of its elements
// exist, 0 < n < V) is read from `short_by` = V - n elements before its place, inside the row, and shifted to it
// when it has arrived (arrived16); an absent one from `safe`, any 16 bytes of the table.
struct Rows {
    Table t;
    const char* base;
    const char* safe;
    int short_by;
};
template <class T>
__device__ __forceinline__ Rows rows_at(const T* base, const T* safe, int length) {
    constexpr int V = 16 / sizeof(T);
    return Rows{table(base), reinterpret_cast<const char*>(base), reinterpret_cast<const char*>(safe), V - length % V};
}

// The vector at byte offset `at` (below 2^31) of the rows, of which the first `n` elements exist (n <= 0: none).
// ONCE: read past the caches.
template <class T, int HOW, bool ONCE = false>
__device__ __forceinline__ uint4 load16(const Rows& rows, int at, int n) {
    constexpr int V = 16 / sizeof(T), kPast = ONCE ? 2 : 0;
    const Table t = rows.t;
    if constexpr (HOW == kWhole) {
        return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(t, n > 0 ? at : kOutside, 0, kPast));
    } else if constexpr (HOW == kRagged) {
        const char* p = rows.base + (n < V ? at - rows.short_by * static_cast<int>(sizeof(T)) : at);
        const typename VecOf<T, V>::type v = *reinterpret_cast<const typename VecOf<T, V>::any*>(n > 0 ? p : rows.safe);
        return __builtin_bit_cast(uint4, v);
    } else if constexpr (sizeof(T) == 4) {
        uint4 v;
        v.x = __builtin_amdgcn_raw_buffer_load_b32(t, n > 0 ? at : kOutside, 0, kPast);
        v.y = __builtin_amdgcn_raw_buffer_load_b32(t, n > 1 ? at + 4 : kOutside, 0, kPast);
        v.z = __builtin_amdgcn_raw_buffer_load_b32(t, n > 2 ? at + 8 : kOutside, 0, kPast);
        v.w = __builtin_amdgcn_raw_buffer_load_b32(t, n > 3 ? at + 12 : kOutside, 0, kPast);
        return v;
    } else {
        typedef unsigned short us8 __attribute__((ext_vector_type(8)));
        us8 v;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = __builtin_amdgcn_raw_buffer_load_b16(t, n > j ? at + 2 * j : kOutside, 0, kPast);
        return __builtin_bit_cast(uint4, v);
    }
}

// What load16 returned with its elements in place and zeros for those that do not exist.
template <class T, int HOW>
__device__ __forceinline__ uint4 arrived16(const Rows& rows, uint4 v, int n) {
    if constexpr (HOW == kRagged) {
        constexpr int V = 16 / sizeof(T);
        const int s = rows.short_by;             // uniform: 1 .. V - 1, or V where no row has a short vector
        uint4 z = v;
        if constexpr (sizeof(T) == 2) {
            if (s & 4) z = uint4{z.z, z.w, 0, 0};
            if (s & 2) z = uint4{z.y, z.z, z.w, 0};
            if (s & 1) z = uint4{z.x >> 16 | z.y << 16, z.y >> 16 | z.z << 16, z.z >> 16 | z.w << 16, z.w >> 16};
        } else {
            if (s & 2) z = uint4{z.z, z.w, 0, 0};
            if (s & 1) z = uint4{z.y, z.z, z.w, 0};
        }
        const bool none = n <= 0, part = n < V;
        v.x = none ? 0 : part ? z.x : v.x;
        v.y = none ? 0 : part ? z.y : v.y;
        v.z = none ? 0 : part ? z.z : v.z;
        v.w = none ? 0 : part ? z.w : v.w;
    }
    return v;
}

// One element as float32, 0 where it does not exist.
template <class T>
__device__ __forceinline__ float load1(Table t, uint32_t at, bool there) {
    const uint32_t o = there ? at : kOutside;
    if constexpr (sizeof(T) == 4) return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(t, o, 0, 0));
    else return static_cast<float>(__builtin_bit_cast(T, static_cast<unsigned short>(__builtin_amdgcn_raw_buffer_load_b16(t, o, 0, 0))));
}

// A lane's accumulators are four consecutive columns of a tile: 16 bytes of float32, half of that of a 16-bit type,
// whose columns are therefore dealt to pairs of tiles: element m of tile i of a pair is column 8 (m / 4) + 4 i +
// m % 4 of the pair's 32, so the two tiles make one 16-byte store, four lanes' stores 64 bytes of a row (dealt to
// groups of four, a store instruction touches memory in 16-byte pieces: 116 against 107 us for 40000 x 9 float32
// rows, 64 to 128 columns).  LDS holds columns (or the rows of a K-contiguous table) in the dealt order, 16 i + m, so the 16 lanes
// of a read touch neighbours and no bank twice.  Four columns whose first is a multiple of four stay together.
template <class T>
constexpr int kDealt = sizeof(T) == 4 ? 1 : 2;     // tiles of a group
template <class T>
__device__ __forceinline__ int dealt(int n) {
    if constexpr (sizeof(T) == 4) return n;
    const int w = n & 31;
    return (n - w) + 16 * (w >> 2 & 1) + 4 * (w >> 3) + (w & 3);
}

// 16 bytes of consecutive columns from `n` (a multiple of V) at their dealt places in the row at `row`.
template <class T>
__device__ __forceinline__ void put_dealt(T* row, int n, uint4 v) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<uint4*>(row + n) = v;
    } else {
        *reinterpret_cast<uint2*>(row + dealt<T>(n)) = uint2{v.x, v.y};
        *reinterpret_cast<uint2*>(row + dealt<T>(n + 4)) = uint2{v.z, v.w};
    }
}

// A lane's V columns of a tile group (accumulators of tile u at acc[u STEP]) to o, of which `n` exist.
template <class T, int HOW, int STEP>
__device__ __forceinline__ void store_tiles(T* o, int n, const v4f* acc) {
    constexpr int V = 16 / sizeof(T);
    if (HOW == kWhole ? n > 0 : n >= V) {
        float f[V];
#pragma unroll
        for (int v = 0; v < V; ++v) f[v] = acc[v / 4 * STEP][v % 4];
        store_f<T, V>(o, f);
    } else if constexpr (HOW != kWhole) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v < n) o[v] = static_cast<T>(acc[v / 4 * STEP][v % 4]);
    }
}

struct XlTile {
    int expert;      // X: rows without an expert; -1: no such block
    int row0, row1;  // the block's first row, the end of the expert's rows
    int index;       // the block's index among those of the expert
    int before;      // blocks of experts before it that have more than one block
    int count;       // the expert's blocks
};

// The row blocks (of `bm` rows) of the experts in order, the rows behind them last.  A lane has `per` experts next to
// each other, so one sum along the wave numbers the blocks of all.  EMPTY: an expert without rows has one block.
// Built and asked by whole waves; results are uniform.
template <bool EMPTY = false>
struct XlBlocks {
    const int32_t* offsets;
    int X, S, bm, per;
    int own, upto;       // blocks of the lane's experts, and of those up to them
    int many, many_upto; // the same of experts of more than one block

    __device__ __forceinline__ int blocks(int e, int a, int z) const {
        const int n = (z - a + bm - 1) / bm;
        return EMPTY && n == 0 && e < X ? 1 : n;
    }
    __device__ __forceinline__ XlBlocks(const int32_t* __restrict__ offs, int X_, int S_, int bm_)
        : offsets(offs), X(X_), S(S_), bm(bm_), per(X_ / 64 + 1), own(0), many(0) {
        const int lane = threadIdx.x & 63;
#pragma unroll 2
        for (int i = 0; i < per; ++i) {
            const int e = lane * per + i;
            const int n = e <= X ? blocks(e, offsets[e], e < X ? offsets[e + 1] : S) : 0;
            own += n;
            many += e < X && n > 1 ? n : 0;
        }
        upto = inclusive_sum(own);
        many_upto = inclusive_sum(many);
    }
    __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(upto, 63); }
    __device__ __forceinline__ XlTile find(int want) const {
        const uint64_t hit = __ballot(upto > want);
        if (!hit) return XlTile{-1, 0, 0, 0, 0, 0};
        const int f = __ffsll(static_cast<unsigned long long>(hit)) - 1;
        int at = __builtin_amdgcn_readlane(upto - own, f), before = __builtin_amdgcn_readlane(many_upto - many, f);
        int e = f * per, ea, ez, n;
        for (;; ++e) {                           // ends by the lane's last expert
            ea = __builtin_amdgcn_readfirstlane(offsets[e]);
            ez = e < X ? __builtin_amdgcn_readfirstlane(offsets[e + 1]) : S;
            n = blocks(e, ea, ez);
            if (at + n > want || e >= X) break;
            at += n;
            before += n > 1 ? n : 0;
        }
        XlTile t;
        t.expert = e;
        t.index = want - at;
        t.row0 = ea + t.index * bm;
        t.row1 = ez;
        t.before = before;
        t.count = n;
        return t;
    }
};

// Blocks of `bm` rows that X experts and the rows behind them can make of S rows.
inline int64_t tile_bound(int64_t S, int X, int bm) { return S / bm + std::min<int64_t>(S, X + 1); }

// The row block of a workgroup of a grid of 8 ceil(bound / 8) subs workgroups (a plane's), -1: none; `sub` its column
// block.  Workgroups go to the 8 XCDs in turn.  An XCD takes neighbouring row blocks, whole: an expert's weight and
// rows then pass to one L2 and once, where column blocks dealt to the XCDs would bring the rows to all of them.
__device__ __forceinline__ int xcd_tile(int block, int subs, int tiles, int& sub) {
    const int i = block / 8, chunk = (tiles + 7) / 8;
    sub = i % subs;
    const int t = i / subs;
    return t < chunk && block % 8 * chunk + t < tiles ? block % 8 * chunk + t : -1;
}
inline int64_t xcd_grid(int64_t bound, int64_t subs) { return 8 * ceil_div(bound, 8) * subs; }

// Of the experts with several chunks of rc rows, the one of number `want` (-1: there are fewer): its chunks and those of such
// experts before it.  Asked by whole waves; results are uniform.
__device__ __forceinline__ XlTile several_chunks(const int32_t* __restrict__ offsets, int X, int rc, int want) {
    const int lane = threadIdx.x & 63;
    XlTile t{-1, 0, 0, 0, 0, 0};
    int carry = 0, slots = 0;
    for (int e0 = 0; e0 < X; e0 += 64) {
        const int e = e0 + lane;
        const int n = e < X ? (offsets[e + 1] - offsets[e] + rc - 1) / rc : 0;
        const int m = n > 1 ? n : 0;
        const uint64_t many = __ballot(n > 1);
        const int incl = inclusive_sum(m);
        const uint64_t hit = __ballot(n > 1 && carry + static_cast<int>(__popcll(many & ((1ull << lane) - 1ull))) == want);
        if (hit) {
            const int f = __ffsll(static_cast<unsigned long long>(hit)) - 1;
            t.expert = e0 + f;
            t.before = slots + __builtin_amdgcn_readlane(incl - m, f);
            t.count = __builtin_amdgcn_readlane(n, f);
            break;
        }
        carry += static_cast<int>(__popcll(many));
        slots += __builtin_amdgcn_readlane(incl, 63);
    }
    return t;
}

// The gradients of the experts of several chunks: the sum of their partials, in an order that no launch changes.
// blockIdx.y: the expert's number among these, blockIdx.z: the irrep, and behind the irreps the bias columns.
// SPLIT: the four waves of a workgroup take a quarter of the partials each, for experts of many (111 of 34 x 51
// columns: 22 us in one wave, which waits for its loads in turn, 10 in four; one to two of 512 x 1024 columns: 6 us
// and 19).
template <class T, int V, bool SPLIT>
__global__ void __launch_bounds__(256)
k_xl_wsum(const float* __restrict__ pw, const float* __restrict__ pb, const int32_t* __restrict__ offsets, int X,
          XlChunks ch, int64_t wsize, int co, int nreps, T* __restrict__ gw, T* __restrict__ gb, int nbias) {
    __shared__ __align__(16) float part[SPLIT ? 3 : 1][64 * V];
    const int z = blockIdx.z, lane = threadIdx.x & 63, want = blockIdx.y;
    const int rep = z < nreps ? z : ch.brep[z - nreps], rc = ch.rows[rep];
    const XlTile t = several_chunks(offsets, X, rc, want);
    const int expert = t.expert, first = t.before, count = t.count;
    if (expert < 0) return;
    constexpr int EACH = (SPLIT ? 64 : 256) * V;
    const int wave = SPLIT ? threadIdx.x >> 6 : 0;
    const bool w = z < nreps;
    const int64_t size = w ? wsize : co;
    for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * EACH; i0 < size; i0 += static_cast<int64_t>(gridDim.x) * EACH) {
        const int64_t i = i0 + (SPLIT ? lane : threadIdx.x) * V;
        const float* p = (w ? pw : pb) + static_cast<int64_t>(ch.slot0[rep] + first) * size + i;
        float a[V];
#pragma unroll
        for (int v = 0; v < V; ++v) a[v] = 0.0f;
        if (i < size) {
#pragma unroll 8
            for (int q = wave; q < count; q += SPLIT ? 4 : 1) {
                float f[V];
                load_f<float, V>(p + q * size, f);
#pragma unroll
                for (int v = 0; v < V; ++v) a[v] += f[v];
            }
        }
        if constexpr (SPLIT) {
            __syncthreads();                         // the last sums have been read
            if (wave) store_f<float, V>(part[wave - 1] + lane * V, a);
            __syncthreads();
            if (wave) continue;
#pragma unroll
            for (int q = 0; q < 3; ++q)
#pragma unroll
                for (int v = 0; v < V; ++v) a[v] += part[q][lane * V + v];
        }
        if (i >= size) continue;
        if (w) {
            store_f<T, V>(gw + (static_cast<int64_t>(expert) * nreps + z) * wsize + i, a);
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) gb[(static_cast<int64_t>(expert) * co + i + v) * nbias + (z - nreps)] = static_cast<T>(a[v]);
        }
    }
}

int xl_check(const int32_t* lvals, int32_t nreps, int32_t X, int64_t S, int32_t ci, int32_t co, int32_t dtype,
             const int32_t* bias_cols, int32_t nbias, XlMap* map) {
    if (!lvals || nreps < 1) return fail(FEQ_ERR_INVALID, "lvals must be non-empty");
    if (nreps > kXlMaxReps) return fail(FEQ_ERR_UNSUPPORTED, "more than %d irreps", kXlMaxReps);
    if (X < 1 || S < 0 || ci < 1 || co < 1)
        return fail(FEQ_ERR_INVALID, "%lld rows of %d experts, %d to %d channels", (long long)S, X, ci, co);
    if (X > kXlMaxExperts) return fail(FEQ_ERR_UNSUPPORTED, "more than %d experts", kXlMaxExperts);
    if (S > kXlMaxRows) return fail(FEQ_ERR_UNSUPPORTED, "more than 2^30 rows");
    if (ci > 65536 || co > 65536) return fail(FEQ_ERR_UNSUPPORTED, "more than 65536 channels");
    if (!dtype_ok(dtype)) return fail(FEQ_ERR_INVALID, "unknown element type %d", dtype);
    const char* const unused = "%d bias columns, not each of them a scalar irrep's";
    if (bias_cols && nbias > nreps) return fail(FEQ_ERR_INVALID, unused, nbias);     // at most 32: a bit of `used` each
    int d = 0;
    uint32_t used = 0;
    for (int r = 0; r < nreps; ++r) {
        if (lvals[r] < 0) return fail(FEQ_ERR_INVALID, "negative degree");
        const int n = 2 * lvals[r] + 1;
        if (d + n > kXlMaxPlanes) return fail(FEQ_ERR_UNSUPPORTED, "representation dimension exceeds %d", kXlMaxPlanes);
        const int bc = bias_cols ? bias_cols[r] : -1;
        if (bc != -1) {
            if (bc < 0 || bc >= nbias || n != 1 || (used >> bc & 1))
                return fail(FEQ_ERR_INVALID, "bias column %d of irrep %d (degree %d, %d columns)", bc, r, lvals[r], nbias);
            used |= 1u << bc;
        }
        map->first[r] = static_cast<int16_t>(d);
        for (int i = 0; i < n; ++i, ++d) {
            map->rep[d] = static_cast<int8_t>(r);
            map->bcol[d] = static_cast<int8_t>(bc);
        }
    }
    map->first[nreps] = static_cast<int16_t>(d);
    if (bias_cols && nbias > 0 && used != ~0u >> (32 - nbias)) return fail(FEQ_ERR_INVALID, unused, nbias);
    return FEQ_OK;
}

// f(HOW) for rows of ci and co elements at these addresses.
template <class T, class F>
int with_rows(int ci, int co, std::initializer_list<const void*> ptrs, F&& f) {
    constexpr int V = 16 / sizeof(T);
    bool whole = ci % V == 0 && co % V == 0;
    for (const void* p : ptrs) whole = whole && (!p || aligned_to(p, 16));
    if (whole) return f(std::integral_constant<int, kWhole>{});
    if (ci >= V && co >= V) return f(std::integral_constant<int, kRagged>{});
    return f(std::integral_constant<int, kNarrow>{});
}

// Workgroups of a kernel that the chip holds at once (256 CUs).
int resident_blocks(const void* kern, int threads) {
    int n = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, 0) != hipSuccess || n < 1) n = 2;
    return 256 * n;
}

// Weight-gradient chunks: all of about as many row-planes, for about 1024 workgroups, whose partials cost little
// beside the rows.  Rows are rounded up to 64, so that short chunks are uneven: 40000 slots of degrees 0 to 2, 352
// row-planes wanted each, have chunks of 384, 128 x 3 and 128 x 5.  Where the experts' weights alone make half of
// that (64 experts, 512 to 1024 channels: 2048), chunks four times as long: a chunk's partial is written and read at 8
// bytes an element, which 1024 rows are worth and 256 are not (8191 bfloat16 rows: the sums took 166 us beside 44 of
// products).  A partial is needed for an expert of several chunks; those have at most 2 S / rows.  Returns the number
// of partials.
int64_t wgrad_chunks(int64_t S, int X, const int32_t* lvals, int nreps, int ci, int co, XlChunks* ch) {
    const int64_t sub = ceil_div(ci, ci <= 64 ? 64 : 128) * ceil_div(co, 128);
    int64_t dim = 0;
    for (int r = 0; r < nreps; ++r) dim += 2 * lvals[r] + 1;
    const bool heavy = sub * nreps * X >= 512;
    const int64_t want = heavy ? 256 : 1024;
    ch->xcds = heavy ? 1 : 8;
    const int64_t unit = ceil_div(std::max<int64_t>(S, 1) * dim * sub, want);
    int64_t tiles = 0, slots = 0;
    for (int r = nreps - 1; r >= 0; --r) {
        const int64_t rows = std::min<int64_t>(ceil_div(ceil_div(unit, 2 * lvals[r] + 1), 64) * 64, 8192);
        ch->rows[r] = static_cast<int32_t>(rows);
        ch->tile0[r] = static_cast<int32_t>(tiles);
        ch->slot0[r] = static_cast<int32_t>(slots);
        tiles += ceil_div(S / rows + X + 1, ch->xcds);          // the rows without an expert last
        slots += S > rows ? 2 * S / rows : 0;
    }
    ch->tile0[nreps] = static_cast<int32_t>(tiles);      // all
    ch->slot0[nreps] = static_cast<int32_t>(slots);
    return slots;
}

}  // namespace
}  // namespace feq
