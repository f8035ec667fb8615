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
// Sums run in the CSR's order: no atomics, the same bits on every run.
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

// A head of a row is `segs` runs of `len` elements, `cs` apart, the runs in vectors of V elements (the last one of a run
// begins V before its end).
struct EaHead {
    int64_t hs, cs;        // from head to head, from run to run
    int len, cpd, vecs;    // vectors of a run, of a head
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
    int lgL, lgG, slices;      // lanes of a head, of a row; slices of a row
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

// The lane's place: head, position in a chunk, subgroup and place in it.
struct EaLane {
    int h, pos, j, base;       // base: first lane of the subgroup
    bool hv;
    __device__ __forceinline__ EaLane(int H, int lgL, int lgG) {
        const int lane = threadIdx.x & 63, L = 1 << lgL, G = 1 << lgG, p = lane & (L - 1);
        h = static_cast<int>(blockIdx.y) * (64 >> lgL) + (lane >> lgL);
        hv = h < H;
        j = p & (G - 1);
        pos = (j << (lgL - lgG)) + (p >> lgG);
        base = lane & ~(G - 1);
    }
};

// Offsets of the lane's vectors of a slice within a head, and how many of their first elements belong to the vector
// before (V: there is no such vector, and the head's first is read in its place).
template <int V, int NT>
struct EaVecs {
    int64_t off[NT];
    int shared[NT];
    __device__ __forceinline__ EaVecs(const EaHead& hd, int j, int G, int slice) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int c = j + G * (t + NT * slice);
            const int run = c / hd.cpd, i = (c - run * hd.cpd) * V;
            const bool there = c < hd.vecs;
            const int last = hd.len - V;
            off[t] = there ? run * hd.cs + (i < last ? i : last) : 0;
            shared[t] = there ? (i > last ? i - last : 0) : V;
        }
    }
};

template <class T, int V, int NT>
__device__ __forceinline__ void ea_load(const T* __restrict__ row, const EaVecs<V, NT>& v, float (&o)[NT][V]) {
#pragma unroll
    for (int t = 0; t < NT; ++t) load_f<T, V>(row + v.off[t], o[t]);
}

// The part of a dot product that the lane's vectors make.
template <int V, int NT>
__device__ __forceinline__ float ea_dot(const float (&a)[NT][V], const float (&b)[NT][V], const EaVecs<V, NT>& v) {
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float d = 0.0f;
#pragma unroll
        for (int u = 0; u < V; ++u) d += u < v.shared[t] ? 0.0f : a[t][u] * b[t][u];
        sum += d;
    }
    return sum;
}

template <int V, int NT>
constexpr int kEaRows = V * NT <= 8 ? 4 : V * NT <= 16 ? 4 : 2;      // rows in flight

__device__ __forceinline__ bool ea_segment(const int32_t* __restrict__ offsets, int64_t N, int64_t E, int64_t& n, int& b, int& cnt) {
    n = ea_block((N + kEaWaves) / kEaWaves) * kEaWaves + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    if (n > N) return false;
    b = offsets[n];
    cnt = (n < N ? offsets[n + 1] : static_cast<int>(E)) - b;
    return true;
}

// w (float32; out where that is NULL is the result itself) holds the logits between the two passes.
template <class T, int V, int NT, bool NODE>
__global__ void __launch_bounds__(64 * kEaWaves)
k_ea_fwd(EaArgs<T> a, float* __restrict__ w, T* __restrict__ out) {
    int64_t n;
    int b, cnt;
    if (!ea_segment(a.offsets, a.N, a.E, n, b, cnt)) return;
    const int H = a.H, L = 1 << a.lgL, G = 1 << a.lgG, lgE = a.lgL - a.lgG;
    const EaLane me(H, a.lgL, a.lgG);
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
    const float scale = expf(load_any(a.log_scale, a.scale_dtype, 0));
    constexpr int UE = kEaRows<V, NT>;
    float q[NT][V];
    float top = -INFINITY, sum = 0.0f;
    for (int c0 = 0; c0 < cnt; c0 += L) {
        const int at = c0 + me.pos;
        const bool there = at < cnt;
        const int64_t e = there ? a.perm[b + at] : 0;
        int row = -1;
        float bias = 0.0f;
        if (there) {
            if constexpr (NODE) {
                const int64_t r = a.kidx[e];
                row = r >= 0 && r < a.nk ? static_cast<int>(r) : -1;
            } else {
                row = static_cast<int>(e);
            }
            if (a.bias.table) {
                const int j = bucket_of(a.bias, e);
                if (j >= 0) bias = load_any(a.bias.table, a.bias.dtype, static_cast<int64_t>(j) * H + h);
            }
            if (a.decay > 0.0f) bias -= a.dist[e] / a.decay;
        }
        float z = 0.0f;
        for (int sl = 0; sl < a.slices; ++sl) {
            const EaVecs<V, NT> vecs(a.head, me.j, G, sl);
            if (NODE && (a.slices > 1 || c0 == 0)) ea_load<T, V, NT>(a.q + n * a.ldq + h * a.head.hs, vecs, q);
            for (int u0 = 0; u0 < G && c0 + (u0 << lgE) < cnt; u0 += UE) {
                float k[UE][NT][V];
#pragma unroll
                for (int u = 0; u < UE; ++u) {
                    const int r = __shfl(row, me.base | (u0 + u), 64);
                    ea_load<T, V, NT>(a.k + static_cast<int64_t>(r < 0 ? 0 : r) * a.ldk + h * a.head.hs, vecs, k[u]);
                }
#pragma unroll
                for (int u = 0; u < UE; ++u) {
                    if constexpr (!NODE) {
                        const int r = __shfl(row, me.base | (u0 + u), 64);
                        ea_load<T, V, NT>(a.q + static_cast<int64_t>(r < 0 ? 0 : r) * a.ldq + h * a.head.hs, vecs, q);
                    }
                    const float d = group_sum(ea_dot<V, NT>(q, k[u], vecs), G);
                    if (me.j == u0 + u) z += d;
                }
            }
        }
        z = row < 0 ? 0.0f : z * scale;          // an edge from outside the graph: a row of zeros
        z = !there || bias == -INFINITY ? -INFINITY : z + bias;
        if (there && me.hv) w[e * H + h] = z;
        const float most = group_max(fmaxf(z, top), L);
        const float base = most == -INFINITY ? 0.0f : most;
        sum = sum * expf(top - base) + group_sum(expf(z - base), L);
        top = most;
    }
    const float base = top == -INFINITY ? 0.0f : top;
    const float inv = 1.0f / (sum + 1e-8f);
    const uint64_t key = a.drop.limit ? static_cast<uint64_t>(*a.drop.seed) : 0;
    if (!me.hv) return;
    for (int i = me.pos; i < cnt; i += L) {      // by the lane that stored them
        const int64_t at = static_cast<int64_t>(a.perm[b + i]) * H + h;
        const float v = expf(w[at] - base) * inv;
        w[at] = v;
        if (out) {
            const bool keep = !a.drop.limit || kept(key, at, a.drop.limit);
            out[at] = static_cast<T>(a.drop.limit ? (keep ? v * a.drop.scale : 0.0f) : v);
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
template <class T, int V, int NT, bool DST, bool ROWS>
__global__ void __launch_bounds__(64 * kEaWaves)
k_ea_bwd(EaArgs<T> a, const float* __restrict__ w, const T* __restrict__ g, float* __restrict__ gz, T* __restrict__ out,
         int64_t ldo, float* __restrict__ dots) {
    int64_t n;
    int b, cnt;
    if (!ea_segment(a.offsets, a.N, a.E, n, b, cnt)) return;
    const int H = a.H, L = 1 << a.lgL, G = 1 << a.lgG, lgE = a.lgL - a.lgG;
    const EaLane me(H, a.lgL, a.lgG);
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
    if constexpr (DST) {
        for (int i = me.pos; i < cnt; i += L) {
            const int64_t at = static_cast<int64_t>(a.perm[b + i]) * H + h;
            const float v = me.hv ? w[at] : 0.0f;
            if (v != 0.0f) total += v * ea_grad(g, at, a.drop, key);
        }
        total = group_sum(total, L);
    }
    constexpr int UE = kEaRows<V, NT>;
    float dot = 0.0f;
    for (int sl = 0; sl < (ROWS ? a.slices : 1); ++sl) {
        const EaVecs<V, NT> vecs(a.head, me.j, G, sl);
        float acc[NT][V];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < V; ++u) acc[t][u] = 0.0f;
        for (int c0 = 0; c0 < cnt; c0 += L) {
            const int at = c0 + me.pos;
            const bool there = at < cnt && me.hv;
            const int64_t e = at < cnt ? a.perm[b + at] : 0;
            float c = 0.0f;
            if (there) {
                if constexpr (DST) {
                    const float v = w[e * H + h];
                    if (v != 0.0f) c = v * (ea_grad(g, e * H + h, a.drop, key) - total);
                    if (sl == 0) gz[e * H + h] = c;
                } else {
                    c = gz[e * H + h];
                }
            }
            if constexpr (ROWS) {
                int row = -1;
                if (at < cnt) {
                    const int64_t r = a.kidx[e];
                    row = r >= 0 && r < a.nk ? static_cast<int>(r) : -1;
                }
                c = row < 0 ? 0.0f : c * scale;
                for (int u0 = 0; u0 < G && c0 + (u0 << lgE) < cnt; u0 += UE) {
                    float k[UE][NT][V], cu[UE];
#pragma unroll
                    for (int u = 0; u < UE; ++u) {
                        const int r = __shfl(row, me.base | (u0 + u), 64);
                        cu[u] = __shfl(c, me.base | (u0 + u), 64);
                        ea_load<T, V, NT>(a.k + static_cast<int64_t>(r < 0 ? 0 : r) * a.ldk + h * a.head.hs, vecs, k[u]);
                    }
#pragma unroll
                    for (int u = 0; u < UE; ++u)
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int v = 0; v < V; ++v) acc[t][v] += cu[u] == 0.0f ? 0.0f : cu[u] * k[u][t][v];
                }
            }
        }
        if constexpr (ROWS) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    for (int o = G; o < L; o <<= 1) acc[t][v] += __shfl_xor(acc[t][v], o, 64);
            if (me.hv && (me.pos & ((1 << lgE) - 1)) == 0) {      // the first subgroup
                T* o = out + n * ldo + h * a.head.hs;
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    if (vecs.shared[t] < V) store_f<T, V>(o + vecs.off[t], acc[t]);
                if (DST && dots) {
                    float q[NT][V];
                    ea_load<T, V, NT>(a.q + n * a.ldq + h * a.head.hs, vecs, q);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int v = 0; v < V; ++v) q[t][v] = acc[t][v] == 0.0f ? 0.0f : q[t][v];
                    dot += ea_dot<V, NT>(q, acc, vecs);
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
        const EaVecs<V, 1> vec(a.head, c, 1, 0);
        const int64_t at = h * a.head.hs + vec.off[0];
        const float s = gz[eh] * scale;
        float q[1][V], k[1][V], o[V], p[V];
        load_f<T, V>(a.q + e * a.ldq + at, q[0]);
        load_f<T, V>(a.k + e * a.ldk + at, k[0]);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            o[v] = s == 0.0f ? 0.0f : s * k[0][v];
            p[v] = s == 0.0f ? 0.0f : s * q[0][v];
        }
        store_f<T, V>(gq + e * ldgq + at, o);
        store_f<T, V>(gk + e * ldgk + at, p);
        if (s != 0.0f) dot += s * ea_dot<V, 1>(q, k, vec);
    }
    if (!dots) return;
    dot = group_sum(dot, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = dot;
    __syncthreads();
    if (threadIdx.x == 0) dots[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

// out[0] = the sum of n floats, in float64 and a fixed order.
__global__ void __launch_bounds__(1024) k_ea_total(const float* __restrict__ in, int64_t n, void* out, int dtype) {
    __shared__ double part[1024];
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) sum += static_cast<double>(in[i]);
    part[threadIdx.x] = sum;
    __syncthreads();
    for (int o = 512; o > 0; o >>= 1) {
        if (threadIdx.x < static_cast<unsigned>(o)) part[threadIdx.x] += part[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) store_any(out, dtype, 0, static_cast<float>(part[0]));
}

// grad_b over an equal share of the edges a workgroup.  Every slot (a lane for each of `hp` heads) adds its edges to a
// table of its own in LDS, one edge after another, so that no two lanes meet and the order is fixed; the tables are
// then summed in order.  Slots beyond the `tables` that fit take no edges.  blockIdx.y: heads from hn blockIdx.y on.
__global__ void __launch_bounds__(kEaBiasThreads)
k_ea_bias(const float* __restrict__ gz, EaBias bias, int64_t E, int H, int hn, int lgP, int tables, float* __restrict__ part) {
    extern __shared__ __align__(16) float tab[];
    const int h0 = blockIdx.y * hn, heads = H - h0 < hn ? H - h0 : hn, size = bias.count * heads;
    for (int i = threadIdx.x; i < tables * size; i += kEaBiasThreads) tab[i] = 0.0f;
    __syncthreads();
    const int slot = threadIdx.x >> lgP, hl = threadIdx.x & ((1 << lgP) - 1);
    const int64_t share = (E + gridDim.x - 1) / gridDim.x;
    const int64_t e0 = blockIdx.x * share, e1 = e0 + share < E ? e0 + share : E;
    if (slot < tables) {
        float* mine = tab + slot * size;
#pragma unroll 4
        for (int64_t e = e0 + slot; e < e1; e += tables) {
            const int j = bucket_of(bias, e);
            for (int h = hl; h < heads; h += 1 << lgP) {
                const float v = gz[e * H + h0 + h];
                if (j >= 0) mine[j * heads + h] += v;
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < size; i += kEaBiasThreads) {
        float s = 0.0f;
        for (int t = 0; t < tables; ++t) s += tab[t * size + i];
        const int j = i / heads, h = i % heads;
        part[(static_cast<int64_t>(blockIdx.x) * bias.count + j) * H + h0 + h] = s;
    }
}

// grad_b = the workgroups' partials summed in order: a wave for each 64 of its elements.
__global__ void __launch_bounds__(256) k_ea_bias_sum(const float* __restrict__ part, int groups, int n, void* out, int dtype) {
    __shared__ double sums[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = blockIdx.x * 64 + lane;
    double s = 0.0;
    if (i < n)
#pragma unroll 8
        for (int g = wave; g < groups; g += 4) s += static_cast<double>(part[static_cast<int64_t>(g) * n + i]);
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && i < n) store_any(out, dtype, i, static_cast<float>(sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane]));
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
    int V, NT, lgL, lgG, slices, groups;     // groups of heads
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
                auto go = [&](auto node) -> int {
                    auto kern = k_ea_fwd<T, V, NT, decltype(node)::value>;
                    FEQ_LAUNCH("k_ea_fwd", kern, ea_grid(a->num_nodes, s.groups), dim3(64 * kEaWaves), 0, stream_of(stream), args,
                               weights, static_cast<T*>(out));
                    return FEQ_OK;
                };
                return a->k_idx ? go(std::true_type{}) : go(std::false_type{});
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
                    auto kern = k_ea_bwd<T, V, NT, true, false>;
                    FEQ_LAUNCH("k_ea_bwd_z", kern, grid, block, 0, st, args, weights, g, grad_logits, static_cast<T*>(nullptr),
                               int64_t{0}, static_cast<float*>(nullptr));
                    if (!gq) return FEQ_OK;
                    auto rows = k_ea_edge_rows<T, V>;
                    FEQ_LAUNCH("k_ea_edge_rows", rows, dim3(kEaEdgeBlocks), dim3(256), 0, st, args, grad_logits, gq, ldgq, gk, ldgk, dots);
                    return FEQ_OK;
                }
                auto dst = k_ea_bwd<T, V, NT, true, true>;
                FEQ_LAUNCH("k_ea_bwd_dst", dst, grid, block, 0, st, args, weights, g, grad_logits, gq, ldgq, dots);
                args.perm = perm_k;
                args.offsets = offsets_k;
                args.k = args.q;
                args.ldk = args.ldq;
                args.kidx = a->q_idx;
                args.nk = a->num_nodes;
                args.N = a->num_k;
                auto src = k_ea_bwd<T, V, NT, false, true>;
                FEQ_LAUNCH("k_ea_bwd_src", src, ea_grid(a->num_k, s.groups), block, 0, st, args, static_cast<const float*>(nullptr),
                           static_cast<const T*>(nullptr), grad_logits, gk, ldgk, static_cast<float*>(nullptr));
                return FEQ_OK;
            }
        });
    });
    if (rc) return rc;
    if (grad_bias) {
        const EaBiasPlan p = ea_bias_plan(a->num_edges, a->heads, a->num_buckets);
        const EaBias b{a->bias, a->buckets, a->bias_dtype, a->num_buckets, a->wide_buckets};
        const int n = a->num_buckets * a->heads;
        auto kern = k_ea_bias;
        FEQ_LAUNCH("k_ea_bias", kern, dim3(p.blocks, p.parts), dim3(kEaBiasThreads), static_cast<size_t>(p.tables) * a->num_buckets * p.hn * 4,
                   st, grad_logits, b, a->num_edges, a->heads, p.hn, p.lgP, p.tables, part);
        auto sum = k_ea_bias_sum;
        FEQ_LAUNCH("k_ea_bias_sum", sum, dim3(ceil_div(n, 64)), dim3(256), 0, st, part, p.blocks, n, grad_bias, a->bias_dtype);
    }
    if (grad_log_scale) {
        auto kern = k_ea_total;
        FEQ_LAUNCH("k_ea_total", kern, dim3(1), dim3(1024), 0, st, dots, ndots, grad_log_scale, a->scale_dtype);
    }
    if (grad_dist) {
        auto kern = k_ea_dist;
        FEQ_LAUNCH("k_ea_dist", kern, dim3(std::min<int64_t>(ceil_div(a->num_edges, 256), 1 << 20)), dim3(256), 0, st, grad_logits,
                   a->num_edges, a->heads, a->decay, grad_dist);
    }
    return FEQ_OK;
}
