// The experts' per-degree channel maps on rows sorted by expert.  With rows offsets[e] ..
// offsets[e + 1] of every plane belonging to expert e, and r(d) the irrep of plane (component) d,
//   y[d, p, n] = sum_k x[d, p, k] W[e, r(d), n, k]  (+ b[e, n, j] on the plane of the j-th scalar irrep),
//   grad_x[d, p, k] = sum_n grad_y[d, p, n] W[e, r(d), n, k],
//   grad_W[e, r, n, k] = sum over the planes d of r and rows p of e of grad_y[d, p, n] x[d, p, k],
//   grad_b[e, n, j] = sum over the rows p of e of grad_y[d_j, p, n];
// rows from offsets[X] on (slots without an expert): y and grad_x are 0, and they enter no sum.
//
// Products run on the matrix cores: v_mfma_f32_16x16x4_f32 for float32, v_mfma_f32_16x16x32_{f16, bf16} for 16-bit
// types, float32 accumulators for both, one rounding at the store.  The expert of a row block is found by every wave
// from the offsets (experts over the lanes, a sum along the wave), so the host never learns the counts and the grid is their
// upper bound.  The weight is the first operand and the rows the second: a lane's accumulators are columns of one row.
//
// Times below are medians of a kernel's launches in training passes unless a comment says otherwise.
#include <algorithm>

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

// out[d, p, :] = in[d, p, :] B (+ bias), B = W[e, r]^T (TRANS false: in has Cin columns, out Cout) or W[e, r]
// (TRANS: in has Cout columns, out Cin).  K: columns of in, N: of out; W rows have wld = Cin elements.
// WR: waves along the output columns (64 each), 4 / WR along the rows.
// 8191 bfloat16 rows of 64 experts, 512 to 1024 columns: 35 us forward, 28 grad_x (246 and 303 TFLOP/s): the
// workgroups run in two rounds of 8 and 16 steps that wait for LDS and for each other.  Steps of half the columns with
// three workgroups on a CU instead of two, against these (31 and 28 us in runs of their own): 45 and 49 us.
template <class T, int HOW, bool TRANS, int WR>
__global__ void __launch_bounds__(kXlThreads, 2)
k_xl_mm(const T* __restrict__ in, const T* __restrict__ W, const int32_t* __restrict__ offsets, int X, int S, int K,
        int N, int nreps, XlMap map, const T* __restrict__ bias, int nbias, T* __restrict__ out) {
    using M = Mma<T>;
    constexpr int V = 16 / sizeof(T), BK = kXlRowBytes / sizeof(T), CH = BK / V;   // 8 vectors of a staged row
    constexpr int BN = 64 * WR, WC = 4 / WR, PT = kXlBM / (16 * WC);
    constexpr int LD = BK + V;                       // stride of a K-contiguous row: 144 bytes
    constexpr int LDT = BN + M::PAD;                 // stride of a W row staged as it lies (TRANS)
    constexpr int NIN = kXlBM * CH / kXlThreads;     // vectors a thread stages
    constexpr int NW = BN * CH / kXlThreads;
    __shared__ __align__(16) T sIn[2][kXlBM * LD];
    __shared__ __align__(16) T sW[2][TRANS ? BK * LDT : BN * LD];
    const int d = blockIdx.y;
    int sub;
    const XlBlocks<> experts(offsets, X, S, kXlBM);
    const int tile = xcd_tile(blockIdx.x, (N + BN - 1) / BN, experts.total(), sub);
    if (tile < 0) return;
    const XlTile t = experts.find(tile);
    const int n0 = sub * BN;
    const int rows = t.row1 - t.row0 < kXlBM ? t.row1 - t.row0 : kXlBM;
    T* od = out + (static_cast<int64_t>(d) * S + t.row0) * N;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave % WR, wc = wave / WR;
    const bool none = t.expert == X;                 // uniform: rows without an expert
    const Rows rows_in = rows_at(in + (static_cast<int64_t>(d) * S + t.row0) * K, in, K);
    const T* we = W + (static_cast<int64_t>(none ? 0 : t.expert) * nreps + __builtin_amdgcn_readfirstlane(map.rep[d])) * K * N;

    auto load = [&](int k0, uint4 (&vin)[NIN], uint4 (&vw)[NW]) {
#pragma unroll
        for (int i = 0; i < NIN; ++i) {
            const int q = tid + kXlThreads * i, r = q / CH, k = k0 + (q % CH) * V;
            vin[i] = load16<T, HOW>(rows_in, (r * K + k) * static_cast<int>(sizeof(T)), r < rows ? K - k : 0);
        }
        const Rows w = rows_at(TRANS ? we + static_cast<int64_t>(k0) * N + n0 : we + static_cast<int64_t>(n0) * K, W, TRANS ? N : K);
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const int q = tid + kXlThreads * i;
            if constexpr (TRANS) {                   // W rows are k, columns n
                const int r = q / (BN / V), n = (q % (BN / V)) * V;
                vw[i] = load16<T, HOW>(w, (r * N + n) * static_cast<int>(sizeof(T)), k0 + r < K ? N - n0 - n : 0);
            } else {
                const int r = q / CH, k = k0 + (q % CH) * V;
                vw[i] = load16<T, HOW>(w, (r * K + k) * static_cast<int>(sizeof(T)), n0 + r < N ? K - k : 0);
            }
        }
    };
    const Rows w_rows = rows_at(W, W, TRANS ? N : K);
    auto stage = [&](int u, int k0, const uint4 (&vin)[NIN], const uint4 (&vw)[NW]) {
#pragma unroll
        for (int i = 0; i < NIN; ++i) {
            const int q = tid + kXlThreads * i, r = q / CH, k = (q % CH) * V;
            *reinterpret_cast<uint4*>(sIn[u] + r * LD + k) = arrived16<T, HOW>(rows_in, vin[i], r < rows ? K - k0 - k : 0);
        }
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const int q = tid + kXlThreads * i;
            if constexpr (TRANS) {
                const int r = q / (BN / V), n = (q % (BN / V)) * V;
                put_dealt<T>(sW[u] + r * LDT, n, arrived16<T, HOW>(w_rows, vw[i], k0 + r < K ? N - n0 - n : 0));
            } else {
                const int r = q / CH, k = (q % CH) * V;
                *reinterpret_cast<uint4*>(sW[u] + dealt<T>(r) * LD + k) =
                    arrived16<T, HOW>(w_rows, vw[i], n0 + r < N ? K - k0 - k : 0);
            }
        }
    };

    // lane (c, g): row c of row tile j, columns 16 i + V g + 0 .. V - 1 of the wave's 64 for tile group i; the sums
    // begin with the bias
    const int nw = n0 + 64 * wr + V * g;
    const int bc = __builtin_amdgcn_readfirstlane(map.bcol[d]);
    const bool biased = !TRANS && bias && bc >= 0 && !none;
    const Table be = table(biased ? bias + static_cast<int64_t>(t.expert) * N * nbias : nullptr, biased);
    v4f acc[4][PT];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = nw + 16 * (i - i % kDealt<T>) + 4 * (i % kDealt<T>) + r;
            const float bv = load1<T>(be, (n * nbias + bc) * sizeof(T), n < N);
#pragma unroll
            for (int j = 0; j < PT; ++j) acc[i][j][r] = bv;
        }
    // step k0 from LDS buffer u: meanwhile the next step goes to the other buffer and the registers take the one
    // after it
    uint4 vin[NIN], vw[NW];
    auto step = [&](int k0, int u) {
        stage(u ^ 1, k0 + BK, vin, vw);
        load(k0 + 2 * BK, vin, vw);                  // nothing behind K
#pragma unroll
        for (int ks = 0; ks < BK; ks += M::KS) {
            typename M::frag a[4], b[PT];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int q0 = 64 * wr + 16 * i;
                if constexpr (TRANS) a[i] = M::columns(sW[u], LDT, ks, g, c, q0);
                else a[i] = *reinterpret_cast<const typename M::frag*>(sW[u] + (q0 + c) * LD + ks + M::FE * g);
            }
#pragma unroll
            for (int j = 0; j < PT; ++j)
                b[j] = *reinterpret_cast<const typename M::frag*>(sIn[u] + (16 * (wc * PT + j) + c) * LD + ks + M::FE * g);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < PT; ++j) acc[i][j] = M::mul(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    };
    if (!none) {
        load(0, vin, vw);
        stage(0, 0, vin, vw);
        load(BK, vin, vw);
        __syncthreads();
        for (int k0 = 0; k0 < K; k0 += 2 * BK) {
            step(k0, 0);
            if (k0 + BK >= K) break;
            step(k0 + BK, 1);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i += kDealt<T>) {
        const int n = nw + 16 * i;
#pragma unroll
        for (int j = 0; j < PT; ++j) {
            const int r = 16 * (wc * PT + j) + c;
            if (r < rows) store_tiles<T, HOW, PT>(od + static_cast<int64_t>(r) * N + n, N - n, &acc[i][j]);
        }
    }
}

// The same product for a reduction of at most 128 columns: a block of the weight stays in LDS, the rows stream.  The
// 16-row blocks of all planes (and, for wide outputs, of their groups of NB columns) lie in one line; every
// workgroup takes an equal run of it, as many workgroups as fit the chip at once, and stages the weight again
// where its run comes to another expert or plane.  Its waves take the run's blocks in turn, straight from memory
// in the matrix cores' layout (lane (c, g): FE elements of row c), the next block's rows in flight during this
// one's products.  Nothing but the weight passes through LDS and no barrier stands between blocks of an
// expert.  NS: reduction steps held (K <= NS KS).
// Forward and grad_x alone, against the tile kernel: 93 and 90 us (107 and 105) for 40000 x 9 float32 rows, 64 x 128 (3.0
// TB/s; the matrix cores' share is 38 us); 122 and 121 (140 and 141) for 20011 x 49 bfloat16 rows, 128 x 128 (4.1 TB/s;
// 137, 3.7 TB/s, where the fused gradients run between the calls).  Column blocks no wider than the output: 16 columns
// take 28 us in blocks of 32, 52 in blocks of 128.
template <class T, int HOW, bool TRANS, int NB, int NS>
__global__ void __launch_bounds__(kXlThreads, NB * NS * Mma<T>::KS * sizeof(T) > 40000 ? 2 : NS == 8 || HOW != kWhole ? 3 : 4)
k_xl_stream(const T* __restrict__ in, const T* __restrict__ W, const int32_t* __restrict__ offsets, int X, int S, int K,
            int N, int nreps, XlMap map, int dim, const T* __restrict__ bias, int nbias, T* __restrict__ out) {
    using M = Mma<T>;
    typedef typename M::frag frag;
    constexpr int V = 16 / sizeof(T), KM = NS * M::KS;
    constexpr int NT = NB / 16, NA = NT < 4 ? NT : 4;   // tiles; those whose weight fragments are held at a time
    constexpr int LD = KM + V, LDT = NB + M::PAD;
    __shared__ __align__(16) T sW[TRANS ? KM * LDT : NB * LD];
    __shared__ __align__(16) float sBias[NB];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nb = (N + NB - 1) / NB;
    const XlBlocks<> experts(offsets, X, S, 16);
    const int per_plane = experts.total();
    const int64_t total = static_cast<int64_t>(per_plane) * dim * nb;
    const int64_t share = total / gridDim.x, more = total % gridDim.x;
    int64_t at = blockIdx.x * share + (blockIdx.x < more ? blockIdx.x : more);
    const int64_t end = at + share + (blockIdx.x < more ? 1 : 0);
    while (at < end) {
        const int line = static_cast<int>(at / per_plane), d = line / nb, n0 = line % nb * NB;
        const XlTile t = experts.find(static_cast<int>(at % per_plane));
        const int expert = t.expert, row0 = t.row0, rows = t.row1 - t.row0, left = t.count - t.index;
        const int nblocks = static_cast<int>(end - at < left ? end - at : left);
        at += nblocks;
        const T* id = in + (static_cast<int64_t>(d) * S + row0) * K;
        T* od = out + (static_cast<int64_t>(d) * S + row0) * N + n0;

        frag b0[NS], b1[NS];
        auto load = [&](int blk, frag (&b)[NS]) {
            const Rows p = rows_at(id + static_cast<int64_t>(16 * blk) * K, in, K);
            const bool there = 16 * blk + c < rows;
#pragma unroll
            for (int ks = 0; ks < NS; ++ks) {
                const int k = ks * M::KS + M::FE * g;
                b[ks] = __builtin_bit_cast(frag, load16<T, HOW>(p, (c * K + k) * static_cast<int>(sizeof(T)), there ? K - k : 0));
            }
        };
        auto arrived = [&](int blk, const frag (&b)[NS]) {
            const Rows p = rows_at(in, in, K);
#pragma unroll
            for (int ks = 0; ks < NS; ++ks)
                b0[ks] = __builtin_bit_cast(frag, arrived16<T, HOW>(p, __builtin_bit_cast(uint4, b[ks]),
                                                                    16 * blk + c < rows ? K - ks * M::KS - M::FE * g : 0));
        };
        auto store = [&](int blk, const v4f (&acc)[NT]) {
            const int r = 16 * blk + c;
            if (r >= rows) return;
            T* o = od + static_cast<int64_t>(r) * N;
#pragma unroll
            for (int i = 0; i < NT; i += kDealt<T>) {
                const int n = 16 * i + V * g;
                store_tiles<T, HOW, 1>(o + n, N - n0 - n, &acc[i]);
            }
        };
        if (expert == X) {                           // rows without an expert
            v4f zero[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) zero[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            for (int blk = wave; blk < nblocks; blk += 4) store(blk, zero);
            continue;
        }
        load(wave, b1);                              // nothing behind the last row
        __syncthreads();                             // the last expert's weight has been read
        const T* wm = W + (static_cast<int64_t>(expert) * nreps + __builtin_amdgcn_readfirstlane(map.rep[d])) * K * N;
        const Rows we = rows_at(TRANS ? wm + n0 : wm + static_cast<int64_t>(n0) * K, W, TRANS ? N : K);
#pragma unroll
        for (int i = 0; i < KM * NB / V / kXlThreads; ++i) {
            const int q = tid + kXlThreads * i;
            if constexpr (TRANS) {
                const int k = q / (NB / V), n = (q % (NB / V)) * V;
                const int there = k < K ? N - n0 - n : 0;
                put_dealt<T>(sW + k * LDT, n,
                             arrived16<T, HOW>(we, load16<T, HOW>(we, (k * N + n) * static_cast<int>(sizeof(T)), there), there));
            } else {
                const int n = q / (KM / V), k = (q % (KM / V)) * V;
                const int there = n0 + n < N ? K - k : 0;
                *reinterpret_cast<uint4*>(sW + dealt<T>(n) * LD + k) =
                    arrived16<T, HOW>(we, load16<T, HOW>(we, (n * K + k) * static_cast<int>(sizeof(T)), there), there);
            }
        }
        const int bc = __builtin_amdgcn_readfirstlane(map.bcol[d]);
        const bool biased = !TRANS && bias && bc >= 0;
        if (tid < NB)
            sBias[tid] = load1<T>(table(biased ? bias + static_cast<int64_t>(expert) * N * nbias : nullptr, biased),
                                  ((n0 + tid) * nbias + bc) * sizeof(T), n0 + tid < N);
        __syncthreads();
        arrived(wave, b1);
        for (int blk = wave; blk < nblocks; blk += 4) {
            load(blk + 4, b1);                       // nothing behind the last row
            // the weight is read from LDS for every block: kept in registers it would take them from the rows in flight
            asm volatile("" ::: "memory");
            v4f acc[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i)
                acc[i] = *reinterpret_cast<const v4f*>(sBias + 16 * (i - i % kDealt<T>) + V * g + 4 * (i % kDealt<T>));
#pragma unroll
            for (int ks = 0; ks < NS; ++ks) {
#pragma unroll
                for (int i0 = 0; i0 < NT; i0 += NA) {
                    frag a[NA];
#pragma unroll
                    for (int i = 0; i < NA; ++i) {
                        if constexpr (TRANS) a[i] = M::columns(sW, LDT, ks * M::KS, g, c, 16 * (i0 + i));
                        else a[i] = *reinterpret_cast<const frag*>(sW + (16 * (i0 + i) + c) * LD + ks * M::KS + M::FE * g);
                    }
                    M::template mul_all<NA>(a, b0[ks], acc + i0);
                }
            }
            store(blk, acc);
            arrived(blk + 4, b1);
        }
    }
}

// grad_W and grad_b over row chunks.  A workgroup takes a chunk of one expert, one irrep r (all its
// planes), 16 TI WR columns k of x and BN columns n of grad_y (tiles of k first).  An expert of one chunk gets its
// gradient written (zeros without rows), one of several a float32 partial per chunk: pw[slot N K + n K + k],
// pb[slot N + n], summed by k_xl_wsum.
// GX: grad_x too, from the same rows of grad_y, where one tile covers the weight (20011 x 49 bfloat16 rows, 128 x 128:
// 164 us, where grad_x took 121 and grad_W 105; 40000 x 9 float32 rows, 64 x 128: 145, where they took 84 and 75).  HBM
// bounds the first (4.6 TB/s).  The second has 78 us of bytes and 77 of products; its chunks, whose rows are rounded up
// (wgrad_chunks), are no even load.  A second pair of row buffers, filled during the products, gained nothing.
// ONCE: one tile covers the weight, so every row is read once; the rows then go past the caches, which leaves them to
// the kernels around (grad_W alone for 20011 x 49 bfloat16 rows, 128 x 128: 137 -> 97 us).  Rows that several tiles read
// lose by it (42 -> 52 us for 512 x 1024).
template <class T, int HOW, int WR, int TI, int BN, bool ONCE, bool GX>
__global__ void __launch_bounds__(kXlThreads, GX ? 2 : 1)
k_xl_wgrad(const T* __restrict__ gy, const T* __restrict__ x, const T* __restrict__ W, const int32_t* __restrict__ offsets,
           int X, int S, int ci, int co, int nreps, XlMap map, XlChunks ch, T* __restrict__ gx, T* __restrict__ gw,
           T* __restrict__ gb, int nbias, float* __restrict__ pw, float* __restrict__ pb) {
    using M = Mma<T>;
    constexpr int V = 16 / sizeof(T), BP = kXlRowBytes / sizeof(T);   // rows staged at a time
    constexpr int BK = 16 * TI * WR, WC = 4 / WR, NT = BN / (16 * WC);
    constexpr int LX = BK + M::PAD, LG = BN + M::PAD;
    constexpr int NX = BP * (BK / V) / kXlThreads, NG = BP * (BN / V) / kXlThreads;
    constexpr int SIZE = BP * (LX + LG), WSIZE = GX ? BN * LX : 0;
    __shared__ __align__(16) T lds[SIZE > WSIZE ? SIZE : WSIZE];
    T *sX = lds, *sG = lds + BP * LX;
    const int nk = (ci + BK - 1) / BK, nn = (co + BN - 1) / BN;
    // workgroups go to the 8 XCDs in turn; the tiles of a chunk go to one, whose L2 passes its rows to all of them
    // (20000 x 9 bfloat16 rows, 256 x 256: 93 -> 86 us; float32: 279 -> 262), unless chunks are long and few
    // (wgrad_chunks): those leave XCDs idle.  A map with all its gradients, dealt by tiles and by chunks: 15000 x 400 x
    // 1000 float32 of 32 experts 606 and 633 us, bfloat16 8191 x 1024 x 512 of 64 101 and 104, 4000 x 1024 x 1024 of 8 85 and
    // 91; where there are more chunks, 20000 x 4 x 256 x 256 of 64 129 and 121, 60000 x 256 x 512 146 and 142
    const int xcds = ch.xcds, block = blockIdx.x / (xcds * nk * nn);
    int rep = nreps - 1;                             // the irreps of most planes first
    while (rep > 0 && block >= ch.tile0[rep - 1]) --rep;
    const int rc = ch.rows[rep];
    const int i0 = blockIdx.x / xcds - ch.tile0[rep] * nk * nn, sub = i0 % (nk * nn);
    const XlTile t = XlBlocks<true>(offsets, X, S, rc).find(i0 / (nk * nn) * xcds + blockIdx.x % xcds);
    if (t.expert < 0 || (!GX && t.expert == X)) return;
    const int k0 = (sub % nk) * BK, n0 = (sub / nk) * BN;
    const int rend = t.row1 - t.row0 < rc ? t.row1 : t.row0 + rc;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave % WR, wc = wave / WR;
    const int d0 = __builtin_amdgcn_readfirstlane(map.first[rep]), d1 = __builtin_amdgcn_readfirstlane(map.first[rep + 1]);
    // GX: a wave takes CT column tiles of grad_x, the weight's fragments of which it keeps, and RP row tiles of a step
    constexpr int KT = BK / 16, CT = KT / 4 > kDealt<T> ? KT / 4 : kDealt<T>, CW = KT / CT, RP = BP / 16 * CW / 4;
    constexpr int GS = GX ? BN / M::KS : 1;
    const int gc = wave % CW, gr = wave / CW * RP;
    typename M::frag wf[GS][CT];
    if constexpr (GX) {
        if (t.expert == X) {                         // rows without an expert: grad_x is 0
            const int n = (rend - t.row0) * ci;      // of a plane, in one piece
            for (int d = d0; d < d1; ++d) {
                T* o = gx + (static_cast<int64_t>(d) * S + t.row0) * ci;
                const float zero[V] = {};
                for (int i = tid * V; i < n; i += kXlThreads * V) {
                    if (i + V <= n) store_f<T, V>(o + i, zero);
                    else
                        for (int j = i; j < n; ++j) o[j] = static_cast<T>(0.0f);
                }
            }
            return;
        }
        const Rows w = rows_at(W + (static_cast<int64_t>(t.expert) * nreps + rep) * co * ci, W, ci);
#pragma unroll
        for (int i = 0; i < BN * (BK / V) / kXlThreads; ++i) {
            const int q = tid + kXlThreads * i, r = q / (BK / V), k = (q % (BK / V)) * V;
            const int there = r < co ? ci - k : 0;
            put_dealt<T>(lds + r * LX, k, arrived16<T, HOW>(w, load16<T, HOW>(w, (r * ci + k) * static_cast<int>(sizeof(T)), there), there));
        }
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < GS; ++ks)
#pragma unroll
            for (int j = 0; j < CT; ++j) wf[ks][j] = M::columns(lds, LX, ks * M::KS, g, c, 16 * (gc * CT + j));
    }
    const int steps = (rend - t.row0 + BP - 1) / BP, total = steps * (d1 - d0);
    const int bc = __builtin_amdgcn_readfirstlane(map.bcol[d0]);
    const bool sums = gb && bc >= 0 && k0 == 0;                    // uniform

    uint4 vx[NX], vg[NG];
    auto load = [&](int it) {
        const int d = it < total ? d0 + it / steps : d0, r0 = t.row0 + (it % steps) * BP;
        const int64_t base = static_cast<int64_t>(d) * S + r0;
        const Rows tx = rows_at(x + base * ci + k0, x, ci), tg = rows_at(gy + base * co + n0, gy, co);
        const int there = it < total ? rend - r0 : 0;
#pragma unroll
        for (int i = 0; i < NX; ++i) {
            const int q = tid + kXlThreads * i, r = q / (BK / V), k = (q % (BK / V)) * V;
            vx[i] = load16<T, HOW, ONCE>(tx, (r * ci + k) * static_cast<int>(sizeof(T)), r < there ? ci - k0 - k : 0);
        }
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int q = tid + kXlThreads * i, r = q / (BN / V), n = (q % (BN / V)) * V;
            vg[i] = load16<T, HOW, ONCE>(tg, (r * co + n) * static_cast<int>(sizeof(T)), r < there ? co - n0 - n : 0);
        }
    };
    v4f acc[TI][NT];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float bsum = 0.0f;                                             // thread n < BN: column n0 + n
    if (total) load(0);
    for (int it = 0; it < total; ++it) {
        __syncthreads();
        const int there = rend - (t.row0 + (it % steps) * BP);
        const Rows tx = rows_at(x, x, ci), tg = rows_at(gy, gy, co);
#pragma unroll
        for (int i = 0; i < NX; ++i) {
            const int q = tid + kXlThreads * i, r = q / (BK / V), k = (q % (BK / V)) * V;
            put_dealt<T>(sX + r * LX, k, arrived16<T, HOW>(tx, vx[i], r < there ? ci - k0 - k : 0));
        }
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int q = tid + kXlThreads * i, r = q / (BN / V), n = (q % (BN / V)) * V;
            *reinterpret_cast<uint4*>(sG + r * LG + n) = arrived16<T, HOW>(tg, vg[i], r < there ? co - n0 - n : 0);
        }
        __syncthreads();
        load(it + 1);
#pragma unroll
        for (int ks = 0; ks < BP; ks += M::KS) {
            typename M::frag a[TI], b[NT];
#pragma unroll
            for (int i = 0; i < TI; ++i) a[i] = M::columns(sX, LX, ks, g, c, 16 * (wr * TI + i));
#pragma unroll
            for (int j = 0; j < NT; ++j) b[j] = M::columns(sG, LG, ks, g, c, 16 * (wc * NT + j));
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = M::mul(a[i], b[j], acc[i][j]);
        }
        if constexpr (GX) {
            v4f o[RP][CT];
#pragma unroll
            for (int r = 0; r < RP; ++r)
#pragma unroll
                for (int j = 0; j < CT; ++j) o[r][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < GS; ++ks)
#pragma unroll
                for (int r = 0; r < RP; ++r)
                    M::template mul_all<CT>(wf[ks], *reinterpret_cast<const typename M::frag*>(
                                                sG + (16 * (gr + r) + c) * LG + ks * M::KS + M::FE * g), o[r]);
#pragma unroll
            for (int r = 0; r < RP; ++r) {
                const int row = 16 * (gr + r) + c;
                if (row >= there) continue;
                T* at = gx + (static_cast<int64_t>(d0 + it / steps) * S + t.row0 + (it % steps) * BP + row) * ci;
#pragma unroll
                for (int j = 0; j < CT; j += kDealt<T>) {
                    const int n = 16 * (gc * CT + j) + V * g;
                    store_tiles<T, HOW, 1>(at + n, ci - n, &o[r][j]);
                }
            }
        }
        if (sums && tid < BN)
            for (int p = 0; p < BP; ++p) bsum += static_cast<float>(sG[p * LG + tid]);
    }
    const bool direct = t.count == 1;
    const int64_t slot = ch.slot0[rep] + t.before + t.index;
    const int kw = k0 + 16 * TI * wr + V * g;
    const int64_t base = direct ? (static_cast<int64_t>(t.expert) * nreps + rep) * co
                                : slot * co;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int n = n0 + 16 * (wc * NT + j) + c;
        if (n >= co) continue;
#pragma unroll
        for (int i = 0; i < TI; i += kDealt<T>) {
            const int k = kw + 16 * i;
            if (direct) {
                store_tiles<T, HOW, NT>(gw + (base + n) * ci + k, ci - k, &acc[i][j]);
            } else {
                float* o = pw + (base + n) * ci + k;
#pragma unroll
                for (int u = 0; u < kDealt<T>; ++u) store_tiles<float, HOW, 1>(o + 4 * u, ci - k - 4 * u, &acc[i + u][j]);
            }
        }
    }
    if (sums && tid < BN && n0 + tid < co) {
        if (direct) gb[(static_cast<int64_t>(t.expert) * co + n0 + tid) * nbias + bc] = static_cast<T>(bsum);
        else pb[slot * co + n0 + tid] = bsum;
    }
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
    int expert = -1, first = 0, count = 0, carry = 0, slots = 0;
    for (int e0 = 0; e0 < X; e0 += 64) {
        const int e = e0 + lane;
        const int n = e < X ? (offsets[e + 1] - offsets[e] + rc - 1) / rc : 0;
        const int m = n > 1 ? n : 0;
        const uint64_t many = __ballot(n > 1);
        const int incl = inclusive_sum(m);
        const uint64_t hit = __ballot(n > 1 && carry + static_cast<int>(__popcll(many & ((1ull << lane) - 1ull))) == want);
        if (hit) {
            const int f = __ffsll(static_cast<unsigned long long>(hit)) - 1;
            expert = e0 + f;
            first = slots + __builtin_amdgcn_readlane(incl - m, f);
            count = __builtin_amdgcn_readlane(n, f);
            break;
        }
        carry += static_cast<int>(__popcll(many));
        slots += __builtin_amdgcn_readlane(incl, 63);
    }
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

template <class T, bool TRANS>
int mm_run(const void* in, const void* W, const int32_t* offsets, int X, int64_t S, int ci, int co, int nreps,
           const XlMap& map, const void* bias, int nbias, void* out, hipStream_t s) {
    const int K = TRANS ? co : ci, N = TRANS ? ci : co;
    const int dim = map.first[nreps];
    return with_rows<T>(ci, co, {in, W, out}, [&](auto how) -> int {
        constexpr int HOW = decltype(how)::value;
        auto stream = [&](auto nn, auto ns) -> int {
            constexpr int NB = decltype(nn)::value;
            auto kern = k_xl_stream<T, HOW, TRANS, NB, decltype(ns)::value>;
            // as many workgroups as run at once
            static const int resident = resident_blocks(reinterpret_cast<const void*>(kern), kXlThreads);
            const int64_t blocks = std::min<int64_t>(resident, tile_bound(S, X, 16) * dim * ceil_div(N, NB));
            FEQ_LAUNCH(TRANS ? "k_xl_stream_t" : "k_xl_stream", kern, dim3(blocks), dim3(kXlThreads), 0, s,
                       static_cast<const T*>(in), static_cast<const T*>(W), offsets, X, static_cast<int>(S), K, N, nreps, map,
                       dim, static_cast<const T*>(bias), nbias, static_cast<T*>(out));
            return FEQ_OK;
        };
        auto tile = [&](auto wr) -> int {
            constexpr int WR = decltype(wr)::value;
            const int64_t blocks = xcd_grid(tile_bound(S, X, kXlBM), ceil_div(N, 64 * WR));
            if (blocks > INT32_MAX / kXlThreads) return fail(FEQ_ERR_UNSUPPORTED, "%lld blocks", (long long)blocks);
            auto kern = k_xl_mm<T, HOW, TRANS, WR>;
            FEQ_LAUNCH(TRANS ? "k_xl_mm_t" : "k_xl_mm", kern, dim3(blocks, dim), dim3(kXlThreads), 0, s,
                       static_cast<const T*>(in), static_cast<const T*>(W), offsets, X, static_cast<int>(S), K, N, nreps, map,
                       static_cast<const T*>(bias), nbias, static_cast<T*>(out));
            return FEQ_OK;
        };
        constexpr int H = 64 / Mma<T>::KS;           // steps of 64 columns
        auto with_ns = [&](auto nn) -> int {
            if (K <= 64) return stream(nn, std::integral_constant<int, H>{});
            if constexpr (HOW == kNarrow && decltype(nn)::value > 32) return FEQ_ERR_INVALID;        // neither is narrow
            else return stream(nn, std::integral_constant<int, 2 * H>{});
        };
        if (K > kXlStreamK) {
            if (N <= 64) return tile(std::integral_constant<int, 1>{});
            if constexpr (HOW == kNarrow) return FEQ_ERR_INVALID;
            else return tile(std::integral_constant<int, 2>{});
        }
        if (N <= 32) return with_ns(std::integral_constant<int, 32>{});
        if (N <= 64) return with_ns(std::integral_constant<int, 64>{});
        return with_ns(std::integral_constant<int, 128>{});
    });
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

// Whether one kernel makes grad_x and grad_W: where one tile covers the weight.
bool bwd_fused(int ci, int co) { return ci <= 128 && co <= 128; }

// grad_W, grad_b (gb NULL: not wanted) and, for gx, with the weight W, grad_x in the same kernel.
int bwd_w_run(const int32_t* lvals, int nreps, int experts, int64_t slots, int cin, int cout, int dtype, const XlMap& map,
              const void* grad_y, const void* x, const void* weight, const int32_t* offsets, int nb, const int32_t* bias_cols,
              void* grad_x, void* grad_weight, void* grad_bias, void* workspace, size_t ws_bytes, hipStream_t s) {
    const size_t need = feq_expert_linear_bwd_workspace(lvals, nreps, experts, slots, cin, cout, nb);
    if (ws_bytes < need) return fail(FEQ_ERR_WORKSPACE, "weight-gradient workspace of %zu bytes, %zu needed", ws_bytes, need);
    if (need && !workspace) return fail(FEQ_ERR_INVALID, "NULL pointer");
    XlChunks ch;
    const int64_t nslots = wgrad_chunks(slots, experts, lvals, nreps, cin, cout, &ch);
    for (int r = 0; r < nreps; ++r)
        if (nb && bias_cols[r] >= 0) ch.brep[bias_cols[r]] = static_cast<int8_t>(r);
    Carver c(workspace);
    float* pw = c.take<float>(static_cast<size_t>(nslots) * cin * cout);
    float* pb = c.take<float>(nb ? static_cast<size_t>(nslots) * cout : 0);
    return with_dtype(dtype, [&](auto tt) -> int {
        using T = decltype(tt);
        T *gx = static_cast<T*>(grad_x), *gw = static_cast<T*>(grad_weight), *gb = static_cast<T*>(grad_bias);
        return with_rows<T>(cin, cout, {grad_y, x, weight, grad_x, grad_weight}, [&](auto how) -> int {
            constexpr int HOW = decltype(how)::value;
            auto run = [&](auto wr, auto ti, auto bn) -> int {
                constexpr int WR = decltype(wr)::value, TI = decltype(ti)::value, BN = decltype(bn)::value;
                constexpr int BK = 16 * TI * WR;
                const int64_t blocks = ch.xcds * static_cast<int64_t>(ch.tile0[nreps]) * ceil_div(cin, BK) * ceil_div(cout, BN);
                if (blocks > INT32_MAX / kXlThreads) return fail(FEQ_ERR_UNSUPPORTED, "%lld blocks", (long long)blocks);
                auto go = [&](auto once, auto with_gx) -> int {
                    constexpr bool GX = decltype(with_gx)::value;
                    auto kern = k_xl_wgrad<T, HOW, WR, TI, BN, decltype(once)::value, GX>;
                    FEQ_LAUNCH(GX ? "k_xl_bwd" : "k_xl_wgrad", kern, dim3(blocks), dim3(kXlThreads), 0, s,
                               static_cast<const T*>(grad_y), static_cast<const T*>(x), static_cast<const T*>(weight),
                               offsets, experts, static_cast<int>(slots), cin, cout, nreps, map, ch, gx, gw, gb, nb, pw, pb);
                    return FEQ_OK;
                };
                constexpr std::integral_constant<bool, HOW == kWhole> past{};
                if (gx) return go(past, std::true_type{});
                if constexpr (HOW == kWhole) {
                    if (cin <= BK && cout <= BN) return go(past, std::false_type{});
                }
                return go(std::false_type{}, std::false_type{});
            };
            auto with_bn = [&](auto wr, auto ti) -> int {
                if (cout <= 64) return run(wr, ti, std::integral_constant<int, 64>{});
                if constexpr (HOW == kNarrow && decltype(ti)::value > 2) return FEQ_ERR_INVALID;     // neither is narrow
                else return run(wr, ti, std::integral_constant<int, 128>{});
            };
            constexpr std::integral_constant<int, 1> one{};
            constexpr std::integral_constant<int, 2> two{};
            constexpr std::integral_constant<int, 4> four{};
            if (const int err = cin <= 32 ? with_bn(one, two) : cin <= 64 ? with_bn(one, four) : with_bn(two, four)) return err;
            if (nslots == 0) return FEQ_OK;               // every expert in one chunk
            const int64_t wsize = static_cast<int64_t>(cin) * cout;
            int least = ch.rows[0];
            for (int r = 1; r < nreps; ++r) least = std::min(least, static_cast<int>(ch.rows[r]));
            const int64_t many = std::min<int64_t>(experts, slots / least);  // experts of several chunks, at most
            const bool split = slots / least > 8 * experts;                  // more than eight chunks an expert, on average
            auto sum = [&](auto vv, auto sp) -> int {
                constexpr int V = decltype(vv)::value;
                constexpr bool SPLIT = decltype(sp)::value;
                auto kern = k_xl_wsum<T, V, SPLIT>;
                // a grid of 2^32 threads and more loses its last workgroups without an error
                const int64_t blocks = std::min<int64_t>(ceil_div(std::max<int64_t>(wsize, cout), (SPLIT ? 64 : 256) * V), 1 << 20);
                FEQ_LAUNCH("k_xl_wsum", kern, dim3(blocks, many, nreps + nb), dim3(256), 0, s, pw, pb, offsets, experts, ch,
                           wsize, cout, nreps, gw, gb, nb);
                return FEQ_OK;
            };
            auto with_split = [&](auto vv) -> int { return split ? sum(vv, std::true_type{}) : sum(vv, std::false_type{}); };
            return HOW == kWhole ? with_split(four) : with_split(one);
        });
    });
}

}  // namespace
}  // namespace feq

using namespace feq;

extern "C" int feq_expert_linear_fwd(const int32_t* lvals, int32_t nreps, int32_t experts, int64_t slots, int32_t cin,
                                     int32_t cout, int32_t dtype, const void* x, const void* weight,
                                     const int32_t* offsets, const void* bias, int32_t nbias, const int32_t* bias_cols,
                                     void* y, feq_stream_t stream) {
    XlMap map;
    if (int rc = xl_check(lvals, nreps, experts, slots, cin, cout, dtype, bias ? bias_cols : nullptr, nbias, &map)) return rc;
    if (bias && (!bias_cols || nbias < 1)) return fail(FEQ_ERR_INVALID, "a bias needs bias columns");
    if (slots == 0) return FEQ_OK;
    if (!x || !weight || !offsets || !y) return fail(FEQ_ERR_INVALID, "NULL pointer");
    return with_dtype(dtype, [&](auto t) -> int {
        return mm_run<decltype(t), false>(x, weight, offsets, experts, slots, cin, cout, nreps, map, bias, nbias, y,
                                          stream_of(stream));
    });
}

extern "C" int feq_expert_linear_bwd_x(const int32_t* lvals, int32_t nreps, int32_t experts, int64_t slots, int32_t cin,
                                       int32_t cout, int32_t dtype, const void* grad_y, const void* weight,
                                       const int32_t* offsets, void* grad_x, feq_stream_t stream) {
    XlMap map;
    if (int rc = xl_check(lvals, nreps, experts, slots, cin, cout, dtype, nullptr, 0, &map)) return rc;
    if (slots == 0) return FEQ_OK;
    if (!grad_y || !weight || !offsets || !grad_x) return fail(FEQ_ERR_INVALID, "NULL pointer");
    return with_dtype(dtype, [&](auto t) -> int {
        return mm_run<decltype(t), true>(grad_y, weight, offsets, experts, slots, cin, cout, nreps, map, nullptr, 0,
                                         grad_x, stream_of(stream));
    });
}

extern "C" size_t feq_expert_linear_bwd_workspace(const int32_t* lvals, int32_t nreps, int32_t experts, int64_t slots,
                                                  int32_t cin, int32_t cout, int32_t nbias) {
    if (!lvals || nreps < 1 || nreps > kXlMaxReps || experts < 1 || slots < 1 || cin < 1 || cout < 1 || nbias < 0) return 0;
    for (int r = 0; r < nreps; ++r)
        if (lvals[r] < 0 || lvals[r] > kXlMaxPlanes) return 0;
    XlChunks ch;
    const int64_t n = wgrad_chunks(slots, experts, lvals, nreps, cin, cout, &ch);
    Carver c(nullptr);                                   // the partials
    c.take<float>(static_cast<size_t>(n) * cin * cout);
    c.take<float>(nbias ? static_cast<size_t>(n) * cout : 0);
    return c.used;
}

extern "C" int feq_expert_linear_bwd_w(const int32_t* lvals, int32_t nreps, int32_t experts, int64_t slots, int32_t cin,
                                       int32_t cout, int32_t dtype, const void* grad_y, const void* x,
                                       const int32_t* offsets, int32_t nbias, const int32_t* bias_cols, void* grad_weight,
                                       void* grad_bias, void* workspace, size_t ws_bytes, feq_stream_t stream) {
    XlMap map;
    if (int rc = xl_check(lvals, nreps, experts, slots, cin, cout, dtype, grad_bias ? bias_cols : nullptr, nbias, &map)) return rc;
    if (!grad_weight || !offsets || (slots && (!grad_y || !x))) return fail(FEQ_ERR_INVALID, "NULL pointer");
    if (grad_bias && (!bias_cols || nbias < 1)) return fail(FEQ_ERR_INVALID, "a bias gradient needs bias columns");
    return bwd_w_run(lvals, nreps, experts, slots, cin, cout, dtype, map, grad_y, x, nullptr, offsets, grad_bias ? nbias : 0,
                     bias_cols, nullptr, grad_weight, grad_bias, workspace, ws_bytes, stream_of(stream));
}

extern "C" int feq_expert_linear_bwd(const int32_t* lvals, int32_t nreps, int32_t experts, int64_t slots, int32_t cin,
                                     int32_t cout, int32_t dtype, const void* grad_y, const void* x, const void* weight,
                                     const int32_t* offsets, int32_t nbias, const int32_t* bias_cols, void* grad_x,
                                     void* grad_weight, void* grad_bias, void* workspace, size_t ws_bytes,
                                     feq_stream_t stream) {
    XlMap map;
    if (int rc = xl_check(lvals, nreps, experts, slots, cin, cout, dtype, grad_bias ? bias_cols : nullptr, nbias, &map)) return rc;
    if (!grad_weight || !offsets || (slots && (!grad_y || !x || !weight || !grad_x))) return fail(FEQ_ERR_INVALID, "NULL pointer");
    if (grad_bias && (!bias_cols || nbias < 1)) return fail(FEQ_ERR_INVALID, "a bias gradient needs bias columns");
    const bool fused = slots && bwd_fused(cin, cout);
    if (const int rc = bwd_w_run(lvals, nreps, experts, slots, cin, cout, dtype, map, grad_y, x, fused ? weight : nullptr,
                                 offsets, grad_bias ? nbias : 0, bias_cols, fused ? grad_x : nullptr, grad_weight, grad_bias,
                                 workspace, ws_bytes, stream_of(stream)))
        return rc;
    if (fused || slots == 0) return FEQ_OK;
    return feq_expert_linear_bwd_x(lvals, nreps, experts, slots, cin, cout, dtype, grad_y, weight, offsets, grad_x, stream);
}
