// Edge attention with a learned bias for each head and bucket of the edges, and dropout of the weights.  For the edges e
// into node n, with Q read at n and K at the edge's source (node form) or both at the edge (edge form),
//   z[e, h] = exp(log_scale) <Q[., h], K[., h]> - r[e] / decay + b[bucket(e), h]
//   w[e, h] = exp(z - max) / (sum over the edges into n of exp(z - max) + 1e-8),    out = w f(e H + h),
// f the dropout's factors (philox.h).  An edge whose z is -inf (a bias of -inf: a forbidden bucket, whatever K holds) has
// weight 0 and passes no gradient; a node with no other edges has none.  A NaN or +inf makes the weights of its node's head NaN.
// With g = f grad_out,
//   grad_z = w (g - sum w g),  grad_Q = scale sum over e of grad_z K,  grad_K = scale sum over the edges out of m of grad_z Q,
//   grad_b[j, h] = sum over the edges of bucket j of grad_z,  grad_log_scale = sum over n of <Q, grad_Q>,
//   grad_r = -sum over h of grad_z / decay.
//
// One wave per destination (or, for grad_K, source) node and group of heads, over the CSR of the edges.  L = 64 / NH lanes
// serve each of the NH heads of a group and own a chunk of L edges: lane p of them holds edge p's index, row, logit,
// weight and gradient, so exponentials, random numbers and stores are work of all lanes.  Rows are read by subgroups of G
// lanes, lane j holding vectors j, j + G, ... (NT of them) of the head; subgroup s serves the edges whose place is
// s modulo L / G, so short segments still keep all subgroups busy.  Heads too long for NT G vectors take several slices.
// Where a head's runs are shorter than its lanes (component-major tables), the lanes of a run of all heads are neighbours:
// a load then touches memory in pieces of 64 bytes and more (neighbouring lanes on different runs: 50000 x 24 edges,
// eight heads of 8 channels, 212 us against 204 for the forward).
// Sums run in the CSR's order, those of grad_b in the edges' (k_ea_bias: additions in LDS that no two lanes share): the same bits
// on every run.
//
// What bounds a pass is the gather of a row for each edge: 640000 random edges of 2304-byte rows take 203 us forward, 214 and
// 219 in the two backward passes (by destination, by source), 6.7 to 7.3 TB/s from behind the L2s, where a kernel that only
// gathers reaches 8.1.  Along a chain the L2s hold the rows: 186 us for 1.2 million edges, where gathers alone take 116, and no
// unit is full (vector units 51 of 100, scalar ones 39).  Of a wave's time 47 in 100 go to waiting for loads, a segment of
// 24 edges beginning with four that depend on each other (offsets, edge, source and bucket, rows), and 29 to waiting for a
// place to issue from, 4.4 waves to a vector unit: latency bounds it.
// Tried without gain: two rows in flight and the next two loading, rows' addresses formed by lanes, more waves on a unit.
#include <algorithm>

#include "elem_types.h"
#include "feq_internal.h"
#include "lane_math.h"
#include "philox.h"

namespace feq {
namespace {

constexpr int kEaWaves = 4;            // segments of a workgroup
constexpr int kEaMaxHeadLanes = 16;    // heads of a group
constexpr int kEaMaxBuckets = 4096;
constexpr int64_t kEaMaxNodes = int64_t{1} << 25;     // a grid of 2^32 threads and more loses its last workgroups
constexpr int kEaBiasLds = 65536;      // bytes of the bias gradient's tables in LDS
constexpr int kEaBiasThreads = 256;
constexpr int kEaBiasRun = 2048;        // edges of a slot between two sums of the tables

// A head of a row is `segs` runs of `len` elements, `cs` apart, the runs in vectors of V elements (the last one of a run
// begins V before its end).
struct EaHead {
    int64_t hs, cs;        // from head to head, from run to run
    int len, cpd, vecs;    // vectors of a run, of a head
    int ragged;            // whether a run's last vector shares elements with the one before
};

struct EaBias {
    const void* table;     // (buckets, heads) of dtype
    const void* bucket;    // of every edge
    int dtype, count, wide;   // wide: 64-bit indices
};

template <class T>
struct EaArgs {
    const T *q, *k;
    int64_t ldq, ldk;
    const int64_t* kidx;
    int64_t nk;
    const int32_t *perm, *offsets;
    int64_t N, E;
    int H;
    int lgL, lgG, lgC, slices;      // lanes of a head, of a row, of a row's run where these are neighbours; slices of a row
    EaHead head;
    const void* log_scale;
    int scale_dtype;
    const float* dist;
    float decay;
    EaBias bias;
    Drop drop;
};

// Bucket of edge e, -1 outside the table.
__device__ __forceinline__ int bucket_of(const EaBias& b, int64_t e) {
    const int64_t i = b.wide ? static_cast<const int64_t*>(b.bucket)[e] : static_cast<const int32_t*>(b.bucket)[e];
    return i >= 0 && i < b.count ? static_cast<int>(i) : -1;
}

// Workgroups go to the 8 XCDs in turn; an XCD takes neighbouring segments, whose rows its L2 then shares (graphs number
// near nodes alike).  The grid has 8 ceil(blocks / 8) workgroups along x.
__device__ __forceinline__ int64_t ea_block(int64_t blocks) {
    const int64_t chunk = (blocks + 7) / 8;
    const int64_t i = blockIdx.x / 8;
    return i < chunk ? blockIdx.x % 8 * chunk + i : blocks;
}

// The lane's place: head, position in a chunk, subgroup and place in it.  UNI (one subgroup): the lowest lgC bits of j are the
// lane's lowest, the others its highest, the head between them.
struct EaLane {
    int h, pos, j, hg;
    bool hv;
    __device__ __forceinline__ EaLane(int H, int lgL, int lgG, int lgC, bool uni) {
        const int lane = threadIdx.x & 63, L = 1 << lgL, G = 1 << lgG, lgH = 6 - lgL;
        if (uni) {
            hg = (lane >> lgC) & ((1 << lgH) - 1);
            j = (lane >> (lgC + lgH) << lgC) | (lane & ((1 << lgC) - 1));
            pos = j;
        } else {
            const int p = lane & (L - 1);
            hg = lane >> lgL;
            j = p & (G - 1);
            pos = (j << (lgL - lgG)) + (p >> lgG);
        }
        h = static_cast<int>(blockIdx.y) * (1 << lgH) + hg;
        hv = h < H;
    }
};

// Sums and maxima over lanes that differ in their `low` lowest and `high` highest bits (uniform), of N values at once; the
// moves of a level are the same instruction for all.  Neighbours within 16 lanes by data-parallel moves: exchanges for the
// low bits, rotations (of values that are equal in the bits above) for the high ones.
struct EaReduce {
    int low, high;
    template <int N, class Op>
    __device__ __forceinline__ void run(float (&v)[N], Op op) const {
        auto move = [&](auto c) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = op(v[i], __uint_as_float(dpp_u<decltype(c)::value>(__float_as_uint(v[i]))));
        };
        auto swap16 = [&] {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
                v[i] = op(__uint_as_float(p[0]), __uint_as_float(p[1]));
            }
        };
        auto swap32 = [&] {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
                v[i] = op(__uint_as_float(p[0]), __uint_as_float(p[1]));
            }
        };
        if (low > 0) move(std::integral_constant<int, 0xB1>{});      // quad_perm [1, 0, 3, 2]
        if (low > 1) move(std::integral_constant<int, 0x4E>{});      // quad_perm [2, 3, 0, 1]
        if (low > 2) move(std::integral_constant<int, 0x141>{});     // row_half_mirror
        if (low > 3) move(std::integral_constant<int, 0x140>{});     // row_mirror
        if (low > 4) swap16();
        if (low > 5) swap32();
        if (high > 0) swap32();
        if (high > 1) swap16();
        if (high > 2) move(std::integral_constant<int, 0x128>{});    // row_ror 8
        if (high > 3) move(std::integral_constant<int, 0x124>{});    // 4
        if (high > 4) move(std::integral_constant<int, 0x122>{});    // 2
        if (high > 5) move(std::integral_constant<int, 0x121>{});    // 1
    }
    template <int N>
    __device__ __forceinline__ void sums(float (&v)[N]) const { run(v, [](float a, float b) { return a + b; }); }
    __device__ __forceinline__ float sum(float v) const {
        float a[1] = {v};
        sums(a);
        return a[0];
    }
    __device__ __forceinline__ float most(float v) const {
        float a[1] = {v};
        run(a, [](float x, float y) { return fmaxf(x, y); });
        return a[0];
    }
};

// Offsets of the lane's vectors of a slice within a row, and how many of their first elements belong to the vector
// before (V: there is no such vector, and the head's first is read in its place).
template <int V, int NT>
struct EaVecs {
    int64_t off[NT];
    int shared[NT];
    __device__ __forceinline__ EaVecs(const EaHead& hd, int64_t h, int j, int G, int slice) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int c = j + G * (t + NT * slice);
            const int run = c / hd.cpd, i = (c - run * hd.cpd) * V;
            const bool there = c < hd.vecs;
            const int last = hd.len - V;
            off[t] = h * hd.hs + (there ? run * hd.cs + (i < last ? i : last) : 0);
            shared[t] = there ? (i > last ? i - last : 0) : V;
        }
    }
};

// A row that all lanes read, by buffer loads: the base is a scalar, the lane's offsets are 32 bits, and what lies outside (a
// lane's absent vectors, all of an absent row) is 0 without a memory access or a select.
typedef __amdgpu_buffer_rsrc_t EaTable;
constexpr uint32_t kEaInside = 0x7ffffff0u, kEaOutside = 0x80000000u;

// A row's vectors, in the table's type until they are used (16-bit rows in flight take half the registers).
template <class T, int V, int NT>
struct EaRow {
    typedef typename VecOf<T, V>::type vec;
    vec v[NT];
    __device__ __forceinline__ void load(const T* __restrict__ row, const EaVecs<V, NT>& vecs) {
#pragma unroll
        for (int t = 0; t < NT; ++t) v[t] = *reinterpret_cast<const typename VecOf<T, V>::any*>(row + vecs.off[t]);
    }
    __device__ __forceinline__ void load_uniform(const T* row, bool there, const uint32_t (&at)[NT]) {
        const EaTable r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(row), 0, there ? kEaInside : 0u, 0x00020000);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if constexpr (sizeof(vec) == 16) v[t] = __builtin_bit_cast(vec, __builtin_amdgcn_raw_buffer_load_b128(r, at[t], 0, 0));
            else if constexpr (sizeof(vec) == 8) v[t] = __builtin_bit_cast(vec, __builtin_amdgcn_raw_buffer_load_b64(r, at[t], 0, 0));
            else if constexpr (sizeof(vec) == 4) v[t] = __builtin_bit_cast(vec, __builtin_amdgcn_raw_buffer_load_b32(r, at[t], 0, 0));
            else v[t] = __builtin_bit_cast(vec, __builtin_amdgcn_raw_buffer_load_b16(r, at[t], 0, 0));
        }
    }
    __device__ __forceinline__ float get(int t, int u) const {
        if constexpr (V == 1) return static_cast<float>(v[t]);
        else return static_cast<float>(v[t][u]);
    }
};

// The part of a dot product that the lane's vectors make.
template <bool UNI, class T, int V, int NT>
__device__ __forceinline__ float ea_dot(const float (&a)[NT][V], const EaRow<T, V, NT>& b, const EaVecs<V, NT>& v, int ragged) {
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float d = 0.0f;
        if (!UNI && ragged) {                    // uniform
#pragma unroll
            for (int u = 0; u < V; ++u) d += u < v.shared[t] ? 0.0f : a[t][u] * b.get(t, u);
        } else {
#pragma unroll
            for (int u = 0; u < V; ++u) d += a[t][u] * b.get(t, u);
        }
        sum += UNI || v.shared[t] < V ? d : 0.0f;
    }
    return sum;
}
template <class T, int V, int NT>
__device__ __forceinline__ void ea_floats(const EaRow<T, V, NT>& r, float (&o)[NT][V]) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < V; ++u) o[t][u] = r.get(t, u);
}

// The lane's offsets in bytes for load_uniform.
template <class T, int V, int NT>
__device__ __forceinline__ void ea_bytes(const EaVecs<V, NT>& v, uint32_t (&at)[NT]) {
#pragma unroll
    for (int t = 0; t < NT; ++t) at[t] = v.shared[t] < V ? static_cast<uint32_t>(v.off[t]) * static_cast<uint32_t>(sizeof(T)) : kEaOutside;
}

constexpr int kEaLgRows = 2, kEaRows = 1 << kEaLgRows;      // rows in flight

__device__ __forceinline__ bool ea_segment(const int32_t* __restrict__ offsets, int64_t N, int64_t E, int64_t& n, int& b, int& cnt) {
    n = ea_block((N + kEaWaves) / kEaWaves) * kEaWaves + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    if (n > N) return false;
    b = offsets[n];
    cnt = (n < N ? offsets[n + 1] : static_cast<int>(E)) - b;
    return true;
}

// The edges of 64 places of a segment, one a lane: number, row (-1: outside the table) and bucket (-1: none).
template <class T>
struct EaEdges {
    int e, row, bucket;
    template <bool NODE, bool BUCKETS>
    __device__ __forceinline__ void load(const EaArgs<T>& a, int b, int cnt, int s0) {
        const int at = s0 + static_cast<int>(threadIdx.x & 63);
        const bool there = at < cnt;
        e = a.perm[b + (there ? at : 0)];
        row = e;
        bucket = -1;
        if constexpr (NODE) {
            const int64_t r = a.kidx[e];
            row = r >= 0 && r < a.nk ? static_cast<int>(r) : -1;
        }
        if (!there) row = -1;
        if (BUCKETS && a.bias.table) bucket = bucket_of(a.bias, e);
    }
    __device__ __forceinline__ int edge(int i) const { return __shfl(e, i, 64); }
};

// w (float32; out where that is NULL is the result itself) holds the logits between the two passes of a segment of more than
// 64 edges, LDS those (and then their exponentials) of a shorter one.
template <class T, int V, int NT, bool NODE, bool UNI>
__global__ void __launch_bounds__(64 * kEaWaves)
k_ea_fwd(EaArgs<T> a, float* __restrict__ w, T* __restrict__ out) {
    __shared__ float kept_z[kEaWaves][64 * kEaMaxHeadLanes];
    int64_t n;
    int b, cnt;
    if (!ea_segment(a.offsets, a.N, a.E, n, b, cnt)) return;
    const int H = a.H, lgL = a.lgL, L = 1 << lgL, G = 1 << a.lgG, lgE = lgL - a.lgG, lane = threadIdx.x & 63;
    const EaLane me(H, lgL, a.lgG, a.lgC, UNI);
    const EaReduce all{UNI ? a.lgC : lgL, UNI ? lgL - a.lgC : 0}, row{UNI ? a.lgC : a.lgG, UNI ? lgL - a.lgC : 0};
    const int64_t h = me.hv ? me.h : 0;
    if (n == a.N) {                              // destinations outside the graph
        for (int i = me.pos; i < cnt; i += L) {
            const int64_t at = static_cast<int64_t>(a.perm[b + i]) * H + h;
            if (!me.hv) continue;
            w[at] = 0.0f;
            if (out) out[at] = static_cast<T>(0.0f);
        }
        return;
    }
    if (cnt == 0) return;
    float* const zs = kept_z[threadIdx.x >> 6];
    const float scale = expf(load_any(a.log_scale, a.scale_dtype, 0));
    constexpr int UE = kEaRows;
    const int sub = UNI ? 0 : (lane & (L - 1)) >> a.lgG, per = UE << lgE;      // subgroup; places of a step
    const int lg_per = lgE + kEaLgRows;
    const bool one = UNI || a.slices == 1;
    float q[NT][V];
    const EaVecs<V, NT> first(a.head, h, me.j, G, 0);
    uint32_t bytes[NT];
    if constexpr (UNI) ea_bytes<T>(first, bytes);
    auto load_row = [&](EaRow<T, V, NT>& k, const T* table, int64_t ld, int64_t r, const EaVecs<V, NT>& vecs) {
        if constexpr (UNI) k.load_uniform(table + (r < 0 ? 0 : r) * ld, r >= 0, bytes);
        else k.load(table + (r < 0 ? 0 : r) * ld, vecs);
    };
    auto queries = [&](const EaVecs<V, NT>& vecs) {
        EaRow<T, V, NT> own;
        load_row(own, a.q, a.ldq, n, vecs);
        ea_floats(own, q);
    };
    float top = -INFINITY, sum = 0.0f;
    EaEdges<T> ed;
    for (int s0 = 0; s0 < cnt; s0 += 64) {
        ed.template load<NODE, true>(a, b, cnt, s0);
        const int left = cnt - s0 < 64 ? cnt - s0 : 64, steps = (left + per - 1) >> lg_per;
        float z = 0.0f, bias = 0.0f;
        bool there = false;
        int64_t e = 0;
        auto begin = [&](int c0) {               // the lane's edge of the chunk at place c0
            there = c0 + me.pos < left;
            e = ed.edge((c0 + me.pos) & 63);
            const int j = __shfl(ed.bucket, (c0 + me.pos) & 63, 64);
            bias = j >= 0 ? load_any(a.bias.table, a.bias.dtype, static_cast<int64_t>(j) * H + h) : 0.0f;
            if (a.decay > 0.0f) bias -= a.dist[e] / a.decay;
            z = 0.0f;
        };
        auto finish = [&](int c0) {
            const int from = __shfl(ed.row, (c0 + me.pos) & 63, 64);
            z = from < 0 ? 0.0f : z * scale;      // an edge from outside the graph: a row of zeros
            z = !there || bias == -INFINITY ? -INFINITY : z + bias;
            // the lane's own maximum and sum: the lanes meet once, at the segment's end (a reduction for every chunk:
            // 204 us against 184 for 50000 x 24 edges of eight heads)
            if (cnt <= 64) {
                zs[(c0 >> lgL) * 64 + lane] = z;
                top = fmaxf(z, top);
                return;
            }
            if (there && me.hv) w[e * H + h] = z;
            const float most = fmaxf(z, top), base = most == -INFINITY ? 0.0f : most;
            sum = sum * expf(top - base) + expf(z - base);
            top = most;
        };
        auto row_at = [&](int i) {               // of the edge at place i of the 64
            return UNI ? __builtin_amdgcn_readlane(ed.row, i & 63) : __shfl(ed.row, i & 63, 64);
        };
        auto rows_of = [&](const EaVecs<V, NT>& vecs, int t, EaRow<T, V, NT> (&k)[UE]) {
#pragma unroll
            for (int u = 0; u < UE; ++u) load_row(k[u], a.k, a.ldk, row_at(t * per + (u << lgE) + sub), vecs);
        };
        auto dots = [&](const EaVecs<V, NT>& vecs, int t, const EaRow<T, V, NT> (&k)[UE]) {
            float d[UE];
#pragma unroll
            for (int u = 0; u < UE; ++u) {
                if constexpr (!NODE) {
                    EaRow<T, V, NT> own;
                    load_row(own, a.q, a.ldq, row_at(t * per + (u << lgE) + sub), vecs);
                    ea_floats(own, q);
                }
                d[u] = ea_dot<UNI>(q, k[u], vecs, a.head.ragged);
            }
            row.sums(d);
            const int u0 = t * UE & (G - 1);
#pragma unroll
            for (int u = 0; u < UE; ++u)
                if (me.j == u0 + u) z += d[u];
        };
        const int su = G >> kEaLgRows;   // steps of a chunk
        if (one) {
            if (NODE && s0 == 0) queries(first);
            for (int t = 0; t < steps; ++t) {
                EaRow<T, V, NT> k[UE];
                rows_of(first, t, k);
                if ((t & (su - 1)) == 0) begin(t * per);
                dots(first, t, k);
                if (((t + 1) & (su - 1)) == 0 || t + 1 == steps) finish((t * per) & ~(L - 1));
            }
        } else {
            for (int t0 = 0; t0 < steps; t0 += su) {
                begin(t0 * per);
                for (int sl = 0; sl < a.slices; ++sl) {
                    const EaVecs<V, NT> vecs(a.head, h, me.j, G, sl);
                    if (NODE) queries(vecs);
                    for (int t = t0; t < steps && t < t0 + su; ++t) {
                        EaRow<T, V, NT> k[UE];
                        rows_of(vecs, t, k);
                        dots(vecs, t, k);
                    }
                }
                finish(t0 * per);
            }
        }
    }
    const float most = all.most(top), base = most == -INFINITY ? 0.0f : most;
    if (cnt <= 64) {
        for (int c0 = 0; c0 < cnt; c0 += L) {        // by the lane that stored them
            float& z = zs[(c0 >> lgL) * 64 + lane];
            z = expf(z - base);
            sum += z;
        }
    } else {
        sum *= expf(top - base);
    }
    const float inv = 1.0f / (all.sum(sum) + 1e-8f);
    const uint64_t key = a.drop.limit ? static_cast<uint64_t>(*a.drop.seed) : 0;
    for (int s0 = 0; s0 < cnt; s0 += 64) {
        if (cnt > 64) ed.e = a.perm[b + (s0 + lane < cnt ? s0 + lane : 0)];
        for (int c0 = 0; c0 < 64 && s0 + c0 < cnt; c0 += L) {
            const int64_t at = static_cast<int64_t>(ed.edge((c0 + me.pos) & 63)) * H + h;
            if (s0 + c0 + me.pos >= cnt || !me.hv) continue;
            const float v = (cnt <= 64 ? zs[(c0 >> lgL) * 64 + lane] : expf(w[at] - base)) * inv;
            w[at] = v;
            if (out) {
                const bool keep = !a.drop.limit || kept(key, at, a.drop.limit);
                out[at] = static_cast<T>(a.drop.limit ? (keep ? v * a.drop.scale : 0.0f) : v);
            }
        }
    }
}

// The gradient of weight w, whose dropout's factor it gets.
template <class T>
__device__ __forceinline__ float ea_grad(const T* __restrict__ g, int64_t at, const Drop& drop, uint64_t key) {
    if (!drop.limit) return static_cast<float>(g[at]);
    return kept(key, at, drop.limit) ? static_cast<float>(g[at]) * drop.scale : 0.0f;
}

// Rows of a segment summed with grad_z: out[n] = scale sum of grad_z[e] rows[.].  DST: by destination, grad_z is formed from w and
// the gradient and written, rows are K's; else by source, it is read, rows are Q's.  ROWS false: grad_z alone (edge form).
// dots (DST): the wave's share of sum over n of <Q[n], grad_Q[n]>, one for every node and group of heads.
template <class T, int V, int NT, bool DST, bool ROWS, bool UNI>
__global__ void __launch_bounds__(64 * kEaWaves)
k_ea_bwd(EaArgs<T> a, const float* __restrict__ w, const T* __restrict__ g, float* __restrict__ gz, T* __restrict__ out,
         int64_t ldo, float* __restrict__ dots) {
    int64_t n;
    int b, cnt;
    if (!ea_segment(a.offsets, a.N, a.E, n, b, cnt)) return;
    const int H = a.H, L = 1 << a.lgL, G = 1 << a.lgG, lgE = a.lgL - a.lgG, lane = threadIdx.x & 63;
    const EaLane me(H, a.lgL, a.lgG, a.lgC, UNI);
    const EaReduce all{UNI ? a.lgC : a.lgL, UNI ? a.lgL - a.lgC : 0};
    // the lane that holds the edge of row step j
    const int lgH = 6 - a.lgL;
    auto holder = [&](int j) {
        if constexpr (UNI) return (j >> a.lgC << (a.lgC + lgH)) | (me.hg << a.lgC) | (j & ((1 << a.lgC) - 1));
        else return (lane & ~(G - 1)) | j;
    };
    const int64_t h = me.hv ? me.h : 0;
    if (n == a.N) {
        if (DST)
            for (int i = me.pos; i < cnt; i += L)
                if (me.hv) gz[static_cast<int64_t>(a.perm[b + i]) * H + h] = 0.0f;
        return;
    }
    const uint64_t key = DST && a.drop.limit ? static_cast<uint64_t>(*a.drop.seed) : 0;
    const float scale = ROWS ? expf(load_any(a.log_scale, a.scale_dtype, 0)) : 0.0f;
    // an edge of weight 0 passes no gradient, whatever the gradient of its weight holds
    float total = 0.0f;
    EaEdges<T> ed;
    if constexpr (DST) {
        for (int s0 = 0; s0 < cnt; s0 += 64) {
            ed.template load<ROWS, false>(a, b, cnt, s0);
            const int left = cnt - s0 < 64 ? cnt - s0 : 64;
#pragma unroll 4
            for (int c0 = 0; c0 < left; c0 += L) {
                const int64_t at = static_cast<int64_t>(ed.edge((c0 + me.pos) & 63)) * H + h;
                const float v = c0 + me.pos < left && me.hv ? w[at] : 0.0f;
                if (v != 0.0f) total += v * ea_grad(g, at, a.drop, key);
            }
        }
        total = all.sum(total);
    }
    constexpr int UE = kEaRows;
    const int per = UE << lgE, lg_per = lgE + kEaLgRows, su = G >> kEaLgRows, sub = UNI ? 0 : (lane & (L - 1)) >> a.lgG;
    float dot = 0.0f;
    for (int sl = 0; sl < (ROWS && !UNI ? a.slices : 1); ++sl) {
        const EaVecs<V, NT> vecs(a.head, h, me.j, G, sl);
        uint32_t bytes[NT];
        if constexpr (UNI) ea_bytes<T>(vecs, bytes);
        float acc[NT][V];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < V; ++u) acc[t][u] = 0.0f;
        for (int s0 = 0; s0 < cnt; s0 += 64) {
            if (cnt > 64 || (sl == 0 && !DST)) ed.template load<ROWS, false>(a, b, cnt, s0);
            const int left = cnt - s0 < 64 ? cnt - s0 : 64, steps = (left + per - 1) >> lg_per;
            float c = 0.0f;
            auto begin = [&](int c0) {           // the lane's edge of the chunk at place c0
                const int at = c0 + me.pos;
                const int64_t e = ed.edge(at & 63);
                c = 0.0f;
                if (at < left && me.hv) {
                    if constexpr (DST) {
                        const float v = w[e * H + h];
                        if (v != 0.0f) c = v * (ea_grad(g, e * H + h, a.drop, key) - total);
                        if (sl == 0) gz[e * H + h] = c;
                    } else {
                        c = gz[e * H + h];
                    }
                }
                c = __shfl(ed.row, at & 63, 64) < 0 ? 0.0f : c * scale;
            };
            if constexpr (ROWS) {
                auto rows_of = [&](int t, EaRow<T, V, NT> (&k)[UE]) {
#pragma unroll
                    for (int u = 0; u < UE; ++u) {
                        const int i = (t * per + (u << lgE) + sub) & 63;
                        const int r = UNI ? __builtin_amdgcn_readlane(ed.row, i) : __shfl(ed.row, i, 64);
                        const T* at = a.k + static_cast<int64_t>(r < 0 ? 0 : r) * a.ldk;
                        if constexpr (UNI) k[u].load_uniform(at, r >= 0, bytes);
                        else k[u].load(at, vecs);
                    }
                };
                auto add = [&](int t, const EaRow<T, V, NT> (&k)[UE]) {
                    const int u0 = t * UE & (G - 1);
                    float cu[UE];
#pragma unroll
                    for (int u = 0; u < UE; ++u) cu[u] = __shfl(c, holder(u0 + u), 64);
#pragma unroll
                    for (int u = 0; u < UE; ++u) {
                        if (__any(cu[u] == 0.0f)) {      // 0 times what an absent or forbidden edge's row holds may be NaN
#pragma unroll
                            for (int i = 0; i < NT; ++i)
#pragma unroll
                                for (int v = 0; v < V; ++v) acc[i][v] += cu[u] == 0.0f ? 0.0f : cu[u] * k[u].get(i, v);
                        } else {
#pragma unroll
                            for (int i = 0; i < NT; ++i)
#pragma unroll
                                for (int v = 0; v < V; ++v) acc[i][v] += cu[u] * k[u].get(i, v);
                        }
                    }
                };
                for (int t = 0; t < steps; ++t) {
                    EaRow<T, V, NT> k[UE];
                    rows_of(t, k);
                    if ((t & (su - 1)) == 0) begin(t * per);
                    add(t, k);
                }
            } else {
                for (int c0 = 0; c0 < left; c0 += L) begin(c0);
            }
        }
        if constexpr (ROWS) {
            if constexpr (!UNI)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int v = 0; v < V; ++v)
                        for (int o = G; o < L; o <<= 1) acc[t][v] += __shfl_xor(acc[t][v], o, 64);
            if (me.hv && (UNI || (me.pos & ((1 << lgE) - 1)) == 0)) {      // the first subgroup
                T* o = out + n * ldo;
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    if (vecs.shared[t] < V) store_f<T, V>(o + vecs.off[t], acc[t]);
                if (DST && dots) {
                    EaRow<T, V, NT> own;
                    own.load(a.q + n * a.ldq, vecs);
                    float q[NT][V];
                    ea_floats(own, q);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int v = 0; v < V; ++v)
                            if (v >= vecs.shared[t] && acc[t][v] != 0.0f) dot += q[t][v] * acc[t][v];
                }
            }
        }
    }
    if (DST && ROWS && dots) {
        dot = group_sum(dot, 64);
        if ((threadIdx.x & 63) == 0) dots[static_cast<int64_t>(blockIdx.y) * a.N + n] = dot;
    }
}

// The edge form's rows: grad_Q[e] = scale grad_z K[e], grad_K[e] = scale grad_z Q[e], dots[workgroup] its share of the
// sum of grad_z scale <Q, K>.  A thread takes a vector of V elements of a head.
template <class T, int V>
__global__ void __launch_bounds__(256)
k_ea_edge_rows(EaArgs<T> a, const float* __restrict__ gz, T* __restrict__ gq, int64_t ldgq, T* __restrict__ gk, int64_t ldgk,
               float* __restrict__ dots) {
    __shared__ float part[4];
    const float scale = expf(load_any(a.log_scale, a.scale_dtype, 0));
    const int64_t total = a.E * a.H * a.head.vecs;
    float dot = 0.0f;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t eh = i / a.head.vecs, e = eh / a.H;
        const int c = static_cast<int>(i % a.head.vecs), h = static_cast<int>(eh % a.H);
        const EaVecs<V, 1> vec(a.head, h, c, 1, 0);
        const float s = gz[eh] * scale;
        EaRow<T, V, 1> q, k;
        q.load(a.q + e * a.ldq, vec);
        k.load(a.k + e * a.ldk, vec);
        float o[V], p[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            o[v] = s == 0.0f ? 0.0f : s * k.get(0, v);
            p[v] = s == 0.0f ? 0.0f : s * q.get(0, v);
            if (v >= vec.shared[0] && s != 0.0f) dot += q.get(0, v) * o[v];
        }
        store_f<T, V>(gq + e * ldgq + vec.off[0], o);
        store_f<T, V>(gk + e * ldgk + vec.off[0], p);
    }
    if (!dots) return;
    dot = group_sum(dot, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = dot;
    __syncthreads();
    if (threadIdx.x == 0) dots[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

// grad_b over an equal share of the edges a workgroup.  Every slot (a lane for each of 2^lgP heads) adds its edges to a
// table of its own in LDS, one edge after another: no two lanes meet in it, so the order is fixed although the additions
// are LDS's own (which a lane need not wait for: read, add and write took 45 us where these take 32, 640000 edges of 8
// heads and 100 buckets).  Latency bounds it: 64 KB of tables leave a vector unit two waves, of whose time half goes to waiting for
// loads, in eight rounds a slot, and 38 in 100 to waiting for a place to issue from, with no bank conflict and every unit below a
// tenth.  Larger tables leave fewer slots: of 16 heads and 512 buckets two fit (32 of 256 lanes), 77 us, of 8 heads and 4096
// buckets one for each half of the heads (4 lanes), 277 us.  After at most kEaBiasRun edges of a slot the tables are summed in order and added to the workgroup's
// partial: a sum of n numbers one after another may be off by n 2^-24 of them, and the largest tables leave a slot a quarter
// million of two million edges.  Slots beyond the `tables` that fit take no edges.
// blockIdx.y: heads from hn blockIdx.y on.
template <bool WIDE>
__global__ void __launch_bounds__(kEaBiasThreads)
k_ea_bias(const float* __restrict__ gz, EaBias bias, int64_t E, int H, int hn, int lgP, int tables, float* __restrict__ part) {
    extern __shared__ __align__(16) float tab[];
    const int h0 = blockIdx.y * hn, heads = H - h0 < hn ? H - h0 : hn, size = bias.count * heads;
    const int slot = threadIdx.x >> lgP, hl = threadIdx.x & ((1 << lgP) - 1);
    const int share = static_cast<int>((E + gridDim.x - 1) / gridDim.x);      // below 2^31 / 8 where there are so many
    const int64_t e0 = static_cast<int64_t>(blockIdx.x) * share;
    const int count = static_cast<int>(e0 + share < E ? share : E > e0 ? E - e0 : 0);
    const float* mine = gz + e0 * H + h0;
    int from = 0;
    do {
        const int upto = count - from < kEaBiasRun * tables ? count : from + kEaBiasRun * tables;
        for (int i = threadIdx.x; i < tables * size; i += kEaBiasThreads) tab[i] = 0.0f;
        __syncthreads();
        if (slot < tables) {
            for (int h = hl; h < heads; h += 1 << lgP) {
                constexpr int AT = 8;            // edges whose loads are on their way together
                for (int e = from + slot; e < upto; e += AT * tables) {
                    int64_t j[AT];
                    float v[AT];
#pragma unroll
                    for (int i = 0; i < AT; ++i) {
                        const int at = e + i * tables < upto ? e + i * tables : e;
                        if constexpr (WIDE) j[i] = static_cast<const int64_t*>(bias.bucket)[e0 + at];
                        else j[i] = static_cast<const int32_t*>(bias.bucket)[e0 + at];
                        v[i] = mine[static_cast<int64_t>(at) * H + h];
                    }
#pragma unroll
                    for (int i = 0; i < AT; ++i)
                        if (j[i] >= 0 && j[i] < bias.count && e + i * tables < upto)
                            unsafeAtomicAdd(&tab[slot * size + static_cast<int>(j[i]) * heads + h], v[i]);
                }
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < size; i += kEaBiasThreads) {
            float s = 0.0f;
#pragma unroll 8
            for (int t = 0; t < tables; ++t) s += tab[t * size + i];
            const int j = i / heads, h = i % heads;
            float& to = part[(static_cast<int64_t>(blockIdx.x) * bias.count + j) * H + h0 + h];
            to = from ? to + s : s;
        }
        from = upto;
        __syncthreads();                         // the tables have been read
    } while (from < count);
}

// The last sums, in float64 and a fixed order.  grad_b = the workgroups' partials (groups, n): a workgroup for each 64
// of its elements; grad_log_scale = the sum of ndots shares: the last workgroup.
__global__ void __launch_bounds__(1024)
k_ea_finish(const float* __restrict__ part, int groups, int n, void* gb, int bias_dtype, const float* __restrict__ dots, int64_t ndots,
            void* gls, int scale_dtype) {
    __shared__ double sums[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool last = gls && blockIdx.x == gridDim.x - 1;
    const int i = blockIdx.x * 64 + lane;
    double s = 0.0;
    if (last) {
#pragma unroll 4
        for (int64_t k = threadIdx.x; k < ndots; k += 1024) s += static_cast<double>(dots[k]);
    } else if (i < n) {
#pragma unroll 4
        for (int g = wave; g < groups; g += 16) s += static_cast<double>(part[static_cast<int64_t>(g) * n + i]);
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < 16; ++w) s += sums[w][lane];
    if (last) {
        for (int o = 32; o > 0; o >>= 1) s += __shfl_down(s, o, 64);
        if (lane == 0) store_any(gls, scale_dtype, 0, static_cast<float>(s));
    } else if (i < n) {
        store_any(gb, bias_dtype, i, static_cast<float>(s));
    }
}

// grad_r[e] = -sum over the heads of grad_z / decay.
__global__ void __launch_bounds__(256)
k_ea_dist(const float* __restrict__ gz, int64_t E, int H, float decay, float* __restrict__ gd) {
    for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < E; e += static_cast<int64_t>(gridDim.x) * 256) {
        float s = 0.0f;
        for (int h = 0; h < H; ++h) s += gz[e * H + h];
        gd[e] = -s / decay;
    }
}

// bucket[e] = the number of bounds that are at most r[e] (a NaN: 0), by halves.
__global__ void __launch_bounds__(256)
k_buckets(const float* __restrict__ r, int64_t E, const float* __restrict__ bounds, int n, int32_t* __restrict__ bucket) {
    for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < E; e += static_cast<int64_t>(gridDim.x) * 256) {
        const float v = r[e];
        int lo = 0, hi = n;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (bounds[mid] <= v) lo = mid + 1;
            else hi = mid;
        }
        bucket[e] = lo;
    }
}

// ---- host ------------------------------------------------------------------------------

struct EaShape {
    int V, NT, lgL, lgG, lgC, slices, groups;     // groups of heads
    bool uni;                                // a wave reads one row at a time, in one slice of whole, aligned vectors within 31 bits
    EaHead head;
};

int lg(int v) {
    int n = 0;
    while ((1 << n) < v) ++n;
    return n;
}

// Vectors as long as a run allows (16 bytes at most), at most 16 elements a lane.  A group has as many heads as lanes
// and rows allow: fewer where a head would otherwise need slices.
EaShape ea_shape(const feq_edge_attn& a, int size) {
    EaShape s{};
    const int most = 16 / size;
    s.V = a.head_len >= 8 && most == 8 ? 8 : a.head_len >= 4 ? 4 : 1;
    s.head.hs = a.head_stride;
    s.head.cs = a.run_stride;
    s.head.len = a.head_len;
    s.head.cpd = static_cast<int>(ceil_div(a.head_len, s.V));
    s.head.vecs = s.head.cpd * a.head_runs;
    s.head.ragged = a.head_len % s.V != 0;
    const int nt = s.V == 8 ? 2 : 4;
    int nh = std::min(1 << lg(a.heads), kEaMaxHeadLanes);
    while (nh > 1 && 64 / nh * nt < s.head.vecs) nh >>= 1;
    s.lgL = lg(64 / nh);
    s.lgG = 2;
    while (s.lgG < s.lgL && (nt << s.lgG) < s.head.vecs) ++s.lgG;
    const int per = static_cast<int>(ceil_div(s.head.vecs, 1 << s.lgG));
    s.slices = static_cast<int>(ceil_div(per, nt));
    s.NT = static_cast<int>(ceil_div(per, s.slices));
    s.groups = static_cast<int>(ceil_div(a.heads, nh));
    const int64_t span = (a.heads - 1) * a.head_stride + (a.head_runs - 1) * a.run_stride + a.head_len;
    const int64_t vec = s.V * size;          // buffer loads from multiples of a vector
    bool whole = aligned_to(a.q, vec) && aligned_to(a.k, vec);
    for (const int64_t stride : {a.ldq, a.ldk, a.head_stride, a.run_stride}) whole = whole && stride % s.V == 0;
    // short runs of neighbouring heads: their lanes lie together (EaLane)
    const bool together = s.head.cpd == 1 << lg(s.head.cpd) && lg(s.head.cpd) < s.lgL && a.head_stride == a.head_len;
    s.lgC = a.head_runs > 1 && together ? lg(s.head.cpd) : s.lgL;
    s.uni = s.lgL == s.lgG && s.slices == 1 && !s.head.ragged && whole && span < (int64_t{1} << 31) / size - s.V;
    return s;
}

template <class F>
int ea_with(const EaShape& s, F&& f) {
    auto nt = [&](auto v) -> int {
        if constexpr (decltype(v)::value == 8) {
            if (s.NT == 1) return f(v, std::integral_constant<int, 1>{});
            return f(v, std::integral_constant<int, 2>{});
        } else {
            if (s.NT == 1) return f(v, std::integral_constant<int, 1>{});
            if (s.NT == 2) return f(v, std::integral_constant<int, 2>{});
            if (s.NT == 3) return f(v, std::integral_constant<int, 3>{});
            return f(v, std::integral_constant<int, 4>{});
        }
    };
    if (s.V == 8) return nt(std::integral_constant<int, 8>{});
    if (s.V == 4) return nt(std::integral_constant<int, 4>{});
    return nt(std::integral_constant<int, 1>{});
}

int ea_check(const feq_edge_attn* a) {
    if (!a) return fail(FEQ_ERR_INVALID, "NULL pointer");
    if (a->num_edges < 0 || a->num_nodes < 1) return fail(FEQ_ERR_INVALID, "invalid graph sizes");
    if (a->num_edges > INT32_MAX) return fail(FEQ_ERR_UNSUPPORTED, "more than 2^31 - 1 edges");
    if (a->num_nodes > kEaMaxNodes || a->num_k > kEaMaxNodes) return fail(FEQ_ERR_UNSUPPORTED, "more than 2^25 nodes");
    if (a->heads < 1 || a->heads > 1024) return fail(FEQ_ERR_INVALID, "num_heads must be 1 to 1024, got %d", a->heads);
    if (a->head_len < 1 || a->head_runs < 1 || a->head_len > 1 << 20 || a->head_runs > FEQ_MAX_SLOTS)
        return fail(FEQ_ERR_INVALID, "heads of %d runs of %d elements", a->head_runs, a->head_len);
    if (!dtype_ok(a->dtype) || !dtype_ok(a->scale_dtype)) return fail(FEQ_ERR_INVALID, "unknown element type");
    if (a->bias) {
        if (!dtype_ok(a->bias_dtype)) return fail(FEQ_ERR_INVALID, "unknown element type %d", a->bias_dtype);
        if (a->num_buckets < 1 || a->num_buckets > kEaMaxBuckets)
            return fail(FEQ_ERR_UNSUPPORTED, "%d buckets, 1 to %d are supported", a->num_buckets, kEaMaxBuckets);
        if (a->num_edges && !a->buckets) return fail(FEQ_ERR_INVALID, "a bias needs the edges' buckets");
    }
    if (!(a->dropout >= 0.0 && a->dropout <= 1.0)) return fail(FEQ_ERR_INVALID, "a dropped share of %g is not in [0, 1]", a->dropout);
    if (a->dropout > 0.0 && !a->seed) return fail(FEQ_ERR_INVALID, "a dropout needs a seed");
    if (!(a->decay >= 0.0f)) return fail(FEQ_ERR_INVALID, "negative distance decay");
    if (a->decay > 0.0f && a->num_edges && !a->dist) return fail(FEQ_ERR_INVALID, "distance decay needs distances");
    if ((a->k_idx != nullptr) != (a->q_idx != nullptr))
        return fail(FEQ_ERR_INVALID, "q_idx and k_idx must both be given or both be NULL");
    if (a->k_idx && a->num_k < 1) return fail(FEQ_ERR_INVALID, "the node form needs the rows of k");
    if (!a->log_scale || !a->offsets) return fail(FEQ_ERR_INVALID, "NULL pointer");
    if (a->num_edges && (!a->q || !a->k || !a->perm)) return fail(FEQ_ERR_INVALID, "NULL pointer");
    return FEQ_OK;
}

template <class T>
EaArgs<T> ea_args(const feq_edge_attn& a, const EaShape& s) {
    EaArgs<T> r{};
    r.q = static_cast<const T*>(a.q);
    r.k = static_cast<const T*>(a.k);
    r.ldq = a.ldq;
    r.ldk = a.ldk;
    r.kidx = a.k_idx;
    r.nk = a.k_idx ? a.num_k : a.num_edges;
    r.perm = a.perm;
    r.offsets = a.offsets;
    r.N = a.num_nodes;
    r.E = a.num_edges;
    r.H = a.heads;
    r.lgL = s.lgL;
    r.lgG = s.lgG;
    r.lgC = s.lgC;
    r.slices = s.slices;
    r.head = s.head;
    r.log_scale = a.log_scale;
    r.scale_dtype = a.scale_dtype;
    r.dist = a.dist;
    r.decay = a.decay;
    r.bias = EaBias{a.bias, a.buckets, a.bias_dtype, a.num_buckets, a.wide_buckets};
    r.drop = make_drop(a.dropout, a.seed);
    return r;
}

// Workgroups of the segments 0 .. n (the last: the edges outside the graph).
dim3 ea_grid(int64_t n, int groups) { return dim3(8 * ceil_div(ceil_div(n + 1, kEaWaves), 8), groups); }

// Workgroups, tables and heads of the bias gradient.
struct EaBiasPlan {
    int blocks, tables, hn, lgP, parts;
};
EaBiasPlan ea_bias_plan(int64_t E, int H, int B) {
    EaBiasPlan p;
    p.hn = std::min(H, std::max(1, kEaBiasLds / 4 / B));
    p.lgP = std::min(lg(p.hn), 6);
    p.tables = std::min(kEaBiasThreads >> p.lgP, std::max(1, kEaBiasLds / 4 / (B * p.hn)));
    const int64_t most = std::max<int64_t>(8, std::min<int64_t>(512, (int64_t{1} << 24) / (static_cast<int64_t>(B) * H)));
    p.blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, ceil_div(E, 8 * p.tables))));
    p.parts = static_cast<int>(ceil_div(H, p.hn));
    return p;
}

constexpr int kEaEdgeBlocks = 2048;

size_t ea_workspace(const feq_edge_attn& a, bool bias, bool scale, Carver* c, float** part, float** dots, int64_t* ndots) {
    if (bias) *part = c->take<float>(static_cast<size_t>(ea_bias_plan(a.num_edges, a.heads, a.num_buckets).blocks) * a.num_buckets * a.heads);
    if (scale) {
        *ndots = a.k_idx ? a.num_nodes * ea_shape(a, elem_size(a.dtype)).groups : kEaEdgeBlocks;
        *dots = c->take<float>(static_cast<size_t>(*ndots));
    }
    return c->used;
}

}  // namespace
}  // namespace feq

using namespace feq;

extern "C" int feq_distance_buckets(const float* dist, int64_t num_edges, const float* bounds, int32_t num_bounds, int32_t* buckets,
                                    feq_stream_t stream) {
    if (num_edges < 0 || num_bounds < 0) return fail(FEQ_ERR_INVALID, "negative sizes");
    if (num_edges == 0) return FEQ_OK;
    if (!dist || !buckets || (num_bounds && !bounds)) return fail(FEQ_ERR_INVALID, "NULL pointer");
    auto kern = k_buckets;
    FEQ_LAUNCH("k_buckets", kern, dim3(std::min<int64_t>(ceil_div(num_edges, 256), 1 << 20)), dim3(256), 0, stream_of(stream), dist,
               num_edges, bounds, num_bounds, buckets);
    return FEQ_OK;
}

extern "C" int feq_edge_attn_fwd(const feq_edge_attn* a, float* weights, void* out, feq_stream_t stream) {
    if (int rc = ea_check(a)) return rc;
    if (a->num_edges == 0) return FEQ_OK;
    if (!weights) return fail(FEQ_ERR_INVALID, "NULL pointer");
    if (!out && (a->dtype != FEQ_F32 || a->dropout > 0.0)) return fail(FEQ_ERR_INVALID, "float32 weights without dropout alone are the result");
    return with_dtype(a->dtype, [&](auto t) -> int {
        using T = decltype(t);
        const EaShape s = ea_shape(*a, sizeof(T));
        const EaArgs<T> args = ea_args<T>(*a, s);
        return ea_with(s, [&](auto v, auto nt) -> int {
            constexpr int V = decltype(v)::value, NT = decltype(nt)::value;
            if constexpr (V * sizeof(T) > 16) {
                return fail(FEQ_ERR_INVALID, "vectors of %d bytes", V * (int)sizeof(T));
            } else {
                auto go = [&](auto node, auto uni) -> int {
                    auto kern = k_ea_fwd<T, V, NT, decltype(node)::value, decltype(uni)::value>;
                    FEQ_LAUNCH("k_ea_fwd", kern, ea_grid(a->num_nodes, s.groups), dim3(64 * kEaWaves), 0, stream_of(stream), args,
                               weights, static_cast<T*>(out));
                    return FEQ_OK;
                };
                if (s.uni) return a->k_idx ? go(std::true_type{}, std::true_type{}) : go(std::false_type{}, std::true_type{});
                return a->k_idx ? go(std::true_type{}, std::false_type{}) : go(std::false_type{}, std::false_type{});
            }
        });
    });
}

extern "C" size_t feq_edge_attn_bwd_workspace(const feq_edge_attn* a, int32_t want_bias, int32_t want_scale) {
    if (ea_check(a) || a->num_edges == 0) return 0;
    Carver c(nullptr);
    float *part, *dots;
    int64_t n;
    return ea_workspace(*a, want_bias && a->bias, want_scale, &c, &part, &dots, &n);
}

extern "C" int feq_edge_attn_bwd(const feq_edge_attn* a, const int32_t* perm_k, const int32_t* offsets_k, const float* weights,
                                 const void* grad_out, float* grad_logits, void* grad_q, int64_t ldgq, void* grad_k, int64_t ldgk,
                                 void* grad_bias, void* grad_log_scale, float* grad_dist, void* workspace, size_t ws_bytes,
                                 feq_stream_t stream) {
    if (int rc = ea_check(a)) return rc;
    if (a->num_edges == 0) return fail(FEQ_ERR_INVALID, "no edges");
    if (!weights || !grad_out || !grad_logits) return fail(FEQ_ERR_INVALID, "NULL pointer");
    if ((grad_q != nullptr) != (grad_k != nullptr)) return fail(FEQ_ERR_INVALID, "grad_q and grad_k must both be given or both be NULL");
    if (grad_log_scale && !grad_q) return fail(FEQ_ERR_INVALID, "the scale's gradient comes with those of q and k");
    if (grad_q && a->k_idx && (!perm_k || !offsets_k)) return fail(FEQ_ERR_INVALID, "the node form needs the CSR of the edges by k_idx");
    if (grad_bias && !a->bias) return fail(FEQ_ERR_INVALID, "no bias");
    if (grad_dist && !(a->decay > 0.0f)) return fail(FEQ_ERR_INVALID, "no distance decay");
    Carver c(workspace);
    float *part = nullptr, *dots = nullptr;
    int64_t ndots = 0;
    const size_t need = ea_workspace(*a, grad_bias, grad_log_scale, &c, &part, &dots, &ndots);
    if (ws_bytes < need) return fail(FEQ_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", ws_bytes, need);
    if (need && !workspace) return fail(FEQ_ERR_INVALID, "NULL pointer");
    hipStream_t st = stream_of(stream);
    const int rc = with_dtype(a->dtype, [&](auto t) -> int {
        using T = decltype(t);
        const EaShape s = ea_shape(*a, sizeof(T));
        EaArgs<T> args = ea_args<T>(*a, s);
        const T* g = static_cast<const T*>(grad_out);
        T *gq = static_cast<T*>(grad_q), *gk = static_cast<T*>(grad_k);
        return ea_with(s, [&](auto v, auto nt) -> int {
            constexpr int V = decltype(v)::value, NT = decltype(nt)::value;
            if constexpr (V * sizeof(T) > 16) {
                return fail(FEQ_ERR_INVALID, "vectors of %d bytes", V * (int)sizeof(T));
            } else {
                const dim3 grid = ea_grid(a->num_nodes, s.groups), block(64 * kEaWaves);
                if (!gq || !a->k_idx) {
                    auto kern = k_ea_bwd<T, V, NT, true, false, false>;
                    FEQ_LAUNCH("k_ea_bwd_z", kern, grid, block, 0, st, args, weights, g, grad_logits, static_cast<T*>(nullptr),
                               int64_t{0}, static_cast<float*>(nullptr));
                    if (!gq) return FEQ_OK;
                    auto rows = k_ea_edge_rows<T, V>;
                    FEQ_LAUNCH("k_ea_edge_rows", rows, dim3(kEaEdgeBlocks), dim3(256), 0, st, args, grad_logits, gq, ldgq, gk, ldgk, dots);
                    return FEQ_OK;
                }
                auto go = [&](auto uni) -> int {
                    auto dst = k_ea_bwd<T, V, NT, true, true, decltype(uni)::value>;
                    FEQ_LAUNCH("k_ea_bwd_dst", dst, grid, block, 0, st, args, weights, g, grad_logits, gq, ldgq, dots);
                    args.perm = perm_k;
                    args.offsets = offsets_k;
                    args.k = args.q;
                    args.ldk = args.ldq;
                    args.kidx = a->q_idx;
                    args.nk = a->num_nodes;
                    args.N = a->num_k;
                    auto src = k_ea_bwd<T, V, NT, false, true, decltype(uni)::value>;
                    FEQ_LAUNCH("k_ea_bwd_src", src, ea_grid(a->num_k, s.groups), block, 0, st, args, static_cast<const float*>(nullptr),
                               static_cast<const T*>(nullptr), grad_logits, gk, ldgk, static_cast<float*>(nullptr));
                    return FEQ_OK;
                };
                return s.uni ? go(std::true_type{}) : go(std::false_type{});
            }
        });
    });
    if (rc) return rc;
    if (grad_bias) {
        const EaBiasPlan p = ea_bias_plan(a->num_edges, a->heads, a->num_buckets);
        const EaBias b{a->bias, a->buckets, a->bias_dtype, a->num_buckets, a->wide_buckets};
        auto go = [&](auto wide) -> int {
            auto kern = k_ea_bias<decltype(wide)::value>;
            FEQ_LAUNCH("k_ea_bias", kern, dim3(p.blocks, p.parts), dim3(kEaBiasThreads),
                       static_cast<size_t>(p.tables) * a->num_buckets * p.hn * 4, st, grad_logits, b, a->num_edges, a->heads, p.hn, p.lgP,
                       p.tables, part);
            return FEQ_OK;
        };
        if (int err = b.wide ? go(std::true_type{}) : go(std::false_type{})) return err;
    }
    if (grad_bias || grad_log_scale) {
        const int n = grad_bias ? a->num_buckets * a->heads : 0;
        const int groups = grad_bias ? ea_bias_plan(a->num_edges, a->heads, a->num_buckets).blocks : 0;
        auto kern = k_ea_finish;
        FEQ_LAUNCH("k_ea_finish", kern, dim3(ceil_div(n, 64) + (grad_log_scale ? 1 : 0)), dim3(1024), 0, st, part, groups, n, grad_bias,
                   a->bias_dtype, dots, ndots, grad_log_scale, a->scale_dtype);
    }
    if (grad_dist) {
        auto kern = k_ea_dist;
        FEQ_LAUNCH("k_ea_dist", kern, dim3(std::min<int64_t>(ceil_div(a->num_edges, 256), 1 << 20)), dim3(256), 0, st, grad_logits,
                   a->num_edges, a->heads, a->decay, grad_dist);
    }
    return FEQ_OK;
}
