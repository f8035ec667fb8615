// The choice of each row's experts (top-k of the logits with softmax weights) and the plan
// that sorts the chosen (row, expert) slots by expert.
//
// Top-k.  For the logits l (rows, X) of a row: e_i = exp(l_i - max l), p = e / sum e; the K
// experts of the largest logits are chosen (equal logits: the lowest index first; a NaN counts
// as the largest), an expert whose logit is -inf never (its place holds id -1, weight 0).
// Weights: e_sel / sum of the chosen e (normalized) or p_sel.  Also mean_i = the mean of p_i
// over the rows, for a balancing loss.  Gradient, with g the weights' and m the mean's:
//   normalized:  dl_sel += w (g - sum w g)
//   otherwise:   dl_i += p_i (gp_i - sum p gp), gp_sel = g, 0 elsewhere
//   the mean:    dl_i += p_i (m_i - sum p m) / rows.
// All sums are float32.  A group of G lanes takes a row, each lane NE of its logits in
// registers: reductions over a row are a few lane exchanges, and the K maxima are K rounds of
// (value, index) maxima over the lanes.  HBM bounds the largest calls, issue the ordinary ones;
// a lane keeps the same experts for all rows of its workgroup, so the mean is a register
// sum per lane, summed over lanes, waves and workgroups in a fixed order.
//
// Plan.  A stable counting sort: per 2048-slot tile a histogram (k_plan_hist), per bucket the
// tiles' exclusive sums (k_plan_scan; few tiles sum them themselves), then every tile ranks
// its slots (k_plan_place).  Up to 8192 slots one workgroup does all three (k_plan_one).  Lanes
// with equal keys find each other by one ballot per key bit, so a slot's rank needs no atomics and
// the order is the slots' own.  Slots whose expert lies outside [0, X) fill a last bucket.  The
// plan is integer work on 8 bytes per slot: launches and latency bound it.
#include <algorithm>

#include "elem_types.h"
#include "feq_internal.h"
#include "lane_math.h"

namespace feq {
namespace {

constexpr int kTopkThreads = 256;
constexpr int kTopkMaxBlocks = 1024;
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopk = 64;

constexpr int kPlanTile = 2048;       // slots of a k_plan_hist / k_plan_place workgroup
constexpr int kPlanOne = 8192;        // slots of k_plan_one: 200 take it 4 us, the tiles' launches 8; 8191 either 8.5
constexpr int kPlanRounds = 8;        // 64-slot rounds of a wave
// Up to these many tiles and buckets every tile sums the others' histograms itself, a launch less (16000 slots of 8
// experts 9 us, with k_plan_scan 11; 130000 of 512 experts 19 and 16).
constexpr int kPlanOwnSums = 64, kPlanOwnBuckets = 256;

// Larger key = earlier choice: bits of the logit in an order-preserving form, a NaN above all, +0 and -0 equal.
// Keys up to kNever (that of -inf) are never chosen; 0 marks what has been.
constexpr uint32_t kNever = 0x007fffffu;
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    const uint32_t k = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
    return v != v ? 0xffffffffu : k;
}
// The logit of a key (any NaN for a NaN's).
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

// A lane's logits: NC vectors of V, vector c of lane l at expert at[c] (vec_begin), the first sh[c] of them another
// lane's (vec_shared).
template <int V, int NC>
__device__ __forceinline__ void lane_vectors(int l, int G, int X, int (&at)[NC], int (&sh)[NC]) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        at[c] = vec_begin<V>(c * G + l, X);
        sh[c] = vec_shared<V>(c * G + l, X);
    }
}

// The row's logits, -inf for those that are not the lane's.
template <class T, int V, int NC>
__device__ __forceinline__ void load_row(const T* row, const int (&at)[NC], const int (&sh)[NC], float (&x)[NC][V]) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        load_f<T, V>(row + at[c], x[c]);         // at[c] is a vector of the row in every lane
#pragma unroll
        for (int j = 0; j < V; ++j) x[c][j] = j >= sh[c] ? x[c][j] : -__builtin_inff();
    }
}

// e = exp(l - max) of the row; returns sum e.  A row of -inf alone gives e = 0 and the sum 0.  The exponential
// is 2^((l - max) log2 e): rounding that product costs |l - max| steps of the result, no more than rounding l - max
// itself has.
__device__ __forceinline__ float exp_below(float v, float m) { return __builtin_amdgcn_exp2f((v - m) * 1.44269504f); }
template <int V, int NC>
__device__ __forceinline__ float row_exp(const float (&x)[NC][V], int G, float (&e)[NC][V], float& m) {
    m = -__builtin_inff();
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) m = fmaxf(m, x[c][j]);
    m = group_max(m, G);
    m = m == -__builtin_inff() ? 0.0f : m;       // nothing left: e = exp(-inf) = 0, not exp(-inf + inf)
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            e[c][j] = exp_below(x[c][j], m);
            s += e[c][j];
        }
    return group_sum(s, G);
}

// X >= V.  KMAX: the choices are kept in registers until the weights' sum is known (K <= KMAX); 0: they wait in
// memory.  200003 float32 rows of 64, 4 choices: 28 us, 2.2 TB/s; a round over the lanes for every choice makes issue
// the bound.  The workgroups' sums of probabilities go to part (gridDim.x, X), or as means to mean (X) where there is
// one workgroup (a launch of 4 us less); neither: not wanted.
template <class T, int V, int NC, int KMAX>
__global__ void __launch_bounds__(kTopkThreads)
k_topk_fwd(const T* __restrict__ logits, int64_t rows, int X, int K, int normalize, int64_t* __restrict__ ids,
           float* __restrict__ weights, float* __restrict__ part, float* __restrict__ mean_out, float inv_rows, int G) {
    __shared__ float sums[4 * kMaxExperts];
    const int l = threadIdx.x & (G - 1);
    const int per = kTopkThreads / G;
    int at[NC], sh[NC];
    lane_vectors<V, NC>(l, G, X, at, sh);
    float mean[NC][V];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) mean[c][j] = 0.0f;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * per;
    int64_t r = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / G;
    float x[NC][V], next[NC][V], e[NC][V];
    if (r < rows) load_row<T, V, NC>(logits + r * X, at, sh, x);
    for (; r < rows; r += stride) {
        load_row<T, V, NC>(logits + (r + stride < rows ? r + stride : r) * X, at, sh, next);   // in flight meanwhile
        float m;
        const float s = row_exp<V, NC>(x, G, e, m);
        const float inv = s == 0.0f ? 0.0f : 1.0f / s;
        uint32_t key[NC][V];
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                mean[c][j] += e[c][j] * inv;
                key[c][j] = order_key(x[c][j]);
            }
        // the next choice: its expert (none: -1) and e, the same in the group's lanes
        auto choose = [&](int& id, float& ek) {
            uint32_t best = 0;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < V; ++j) best = key[c][j] > best ? key[c][j] : best;
            best = group_max_u(best, G);
            // its lowest index: the lane's first element that holds it, then the lowest over the lanes
            int mine = NC * V;
#pragma unroll
            for (int c = NC - 1; c >= 0; --c)
#pragma unroll
                for (int j = V - 1; j >= 0; --j) mine = key[c][j] == best ? c * V + j : mine;
            uint32_t index = 0xffffffffu;
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (mine / V == c) index = at[c] + mine % V;
            const uint32_t first = group_min_u(index, G);
            const bool got = best > kNever;
            mine = index == first ? mine : NC * V;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < V; ++j) key[c][j] = mine == c * V + j ? 0u : key[c][j];
            ek = got ? exp_below(key_value(best), m) : 0.0f;
            id = got ? static_cast<int>(first) : -1;
        };
        float total = 0.0f;
        // a row without a choice has weights 0, not 0 / 0
        auto inverse = [](float den) { return den == 0.0f ? 0.0f : 1.0f / den; };
        if constexpr (KMAX > 0) {
            int id[KMAX];
            float ek[KMAX];
#pragma unroll
            for (int k = 0; k < KMAX; ++k)
                if (k < K) {
                    choose(id[k], ek[k]);
                    total += ek[k];
                }
            const float scale = inverse(normalize ? total : s);
#pragma unroll
            for (int k = 0; k < KMAX; ++k)
                if (k < K && l == (k & (G - 1))) {
                    ids[r * K + k] = id[k];
                    weights[r * K + k] = ek[k] * scale;
                }
        } else {
            for (int k = 0; k < K; ++k) {
                int id;
                float ek;
                choose(id, ek);
                total += ek;
                if (l == 0) {
                    ids[r * K + k] = id;
                    weights[r * K + k] = ek;
                }
            }
            const float scale = inverse(normalize ? total : s);
            if (l == 0)
                for (int k = 0; k < K; ++k) weights[r * K + k] *= scale;
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) x[c][j] = next[c][j];
    }
    if (!part && !mean_out) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float a = mean[c][j];
            for (int o = G; o < 64; o <<= 1) a += __shfl_xor(a, o, 64);
            if (lane < G && j >= sh[c]) sums[wave * X + at[c] + j] = a;
        }
    __syncthreads();
    for (int i = threadIdx.x; i < X; i += kTopkThreads) {
        const float a = (sums[i] + sums[X + i]) + (sums[2 * X + i] + sums[3 * X + i]);
        if (part) part[static_cast<int64_t>(blockIdx.x) * X + i] = a;
        else mean_out[i] = a * inv_rows;
    }
}

// mean[i] = (sum of the workgroups' sums) / rows, 16 experts a workgroup.
__global__ void __launch_bounds__(1024)
k_topk_mean(const float* __restrict__ part, int groups, int X, float inv_rows, float* __restrict__ mean) {
    __shared__ float s[64][17];
    const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4, i = blockIdx.x * 16 + c;
    float a = 0.0f;
    if (i < X)
#pragma unroll 8
        for (int r = r0; r < groups; r += 64) a += part[static_cast<int64_t>(r) * X + i];
    s[r0][c] = a;
    __syncthreads();
    for (int o = 32; o; o >>= 1) {
        if (r0 < o) s[r0][c] += s[r0 + o][c];
        __syncthreads();
    }
    if (r0 == 0 && i < X) mean[i] = s[0][c] * inv_rows;
}

// gw (rows, K) or NULL, gmean (X) or NULL.  200003 float32 rows of 64, 4 choices: 26 us, 4.4 TB/s.
template <class T, int V, int NC>
__global__ void __launch_bounds__(kTopkThreads)
k_topk_bwd(const T* __restrict__ logits, const int64_t* __restrict__ ids, const float* __restrict__ weights,
           const float* __restrict__ gw, const float* __restrict__ gmean, int64_t rows, int X, int K, int normalize,
           float inv_rows, T* __restrict__ gl, int G) {
    const int l = threadIdx.x & (G - 1);
    const int per = kTopkThreads / G;
    int at[NC], sh[NC];
    lane_vectors<V, NC>(l, G, X, at, sh);
    float gm[NC][V];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) gm[c][j] = (gmean && j >= sh[c]) ? gmean[at[c] + j] * inv_rows : 0.0f;
    const bool full = gmean || (gw && !normalize);      // uniform: the probabilities enter
    const int64_t stride = static_cast<int64_t>(gridDim.x) * per;
    int64_t r = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / G;
    float x[NC][V], next[NC][V];
    if (r < rows && full) load_row<T, V, NC>(logits + r * X, at, sh, x);
    for (; r < rows; r += stride) {
        if (full) load_row<T, V, NC>(logits + (r + stride < rows ? r + stride : r) * X, at, sh, next);
        float gp[NC][V], d[NC][V];
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                gp[c][j] = gm[c][j];
                d[c][j] = 0.0f;
            }
        if (gw) {
            float dot = 0.0f;
            if (normalize)
#pragma unroll 4
                for (int k = 0; k < K; ++k)      // a place without an expert is no function of the logits: not 0 g
                    dot += ids[r * K + k] >= 0 ? weights[r * K + k] * gw[r * K + k] : 0.0f;
#pragma unroll 4
            for (int k = 0; k < K; ++k) {
                const int id = static_cast<int>(ids[r * K + k]);
                const float g = gw[r * K + k];
                const float a = normalize ? weights[r * K + k] * (g - dot) : g;
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const bool here = at[c] + j == id && j >= sh[c];
                        if (normalize) d[c][j] += here ? a : 0.0f;
                        else gp[c][j] += here ? a : 0.0f;
                    }
            }
        }
        if (full) {
            float e[NC][V];
            float m;
            const float s = row_exp<V, NC>(x, G, e, m);
            const float inv = s == 0.0f ? 0.0f : 1.0f / s;
            float dot = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    e[c][j] *= inv;
                    dot += e[c][j] * gp[c][j];
                }
            dot = group_sum(dot, G);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < V; ++j) d[c][j] += e[c][j] * (gp[c][j] - dot);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            T* o = gl + r * X + at[c];
            if (sh[c] == 0) {
                store_f<T, V>(o, d[c]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j >= sh[c]) o[j] = static_cast<T>(d[c][j]);
            }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) x[c][j] = next[c][j];
    }
}

int topk_check(int64_t rows, int32_t X, int32_t K, int32_t dtype) {
    if (rows < 0 || X < 1 || K < 1) return fail(FEQ_ERR_INVALID, "top-k of %lld rows: %d of %d experts", (long long)rows, K, X);
    if (K > X) return fail(FEQ_ERR_INVALID, "top-k chooses %d of %d experts", K, X);
    if (X > kMaxExperts) return fail(FEQ_ERR_UNSUPPORTED, "more than %d experts", kMaxExperts);
    if (K > kMaxTopk) return fail(FEQ_ERR_UNSUPPORTED, "more than %d choices a row", kMaxTopk);
    if (!dtype_ok(dtype)) return fail(FEQ_ERR_INVALID, "unknown element type %d", dtype);
    return FEQ_OK;
}

// A lane holds up to 8 logits of rows up to these many, above them up to 16: the forward's work is per lane and choice
// (top-6 of 233 bfloat16 for 59000 rows: 34 us with 16, 42 with 8), the backward's per logit (58342 rows of 201
// float16: 31 us with 16, 27 with 8).
constexpr int kForwardNarrow = 64, kBackwardNarrow = 512;
// Lanes of a row.
int topk_lanes(int X, int narrow) {
    int g = 1;
    while (g < 64 && g * (X <= narrow ? 8 : 16) < X) g <<= 1;
    return g;
}
int topk_blocks(int64_t rows, int X) {
    return static_cast<int>(std::min<int64_t>(ceil_div(rows, kTopkThreads / topk_lanes(X, kForwardNarrow)), kTopkMaxBlocks));
}

// f(V, NC) for the instance of X experts
template <class T, class F>
int with_topk_form(int X, int narrow, F&& f) {
    constexpr int VV = 16 / sizeof(T);
    if (X < VV) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});     // fewer than a vector
    return X <= narrow ? f(std::integral_constant<int, VV>{}, std::integral_constant<int, 8 / VV>{})
                       : f(std::integral_constant<int, VV>{}, std::integral_constant<int, 16 / VV>{});
}

// ---- plan ------------------------------------------------------------------------

// Bucket of slot i: its expert, X where it has none, X + 1 behind the last slot.
__device__ __forceinline__ int slot_key(const int64_t* ids, int64_t i, int64_t n, int X) {
    if (i >= n) return X + 1;
    const int64_t e = ids[i];
    return (e >= 0 && e < X) ? static_cast<int>(e) : X;
}

__device__ __forceinline__ uint64_t lanes_with(int key, int bits) {
    uint64_t m = ~0ull;
    for (int b = 0; b < bits; ++b) {
        const bool on = (key >> b) & 1;
        const uint64_t v = __ballot(on);
        m &= on ? v : ~v;
    }
    return m;
}

// A wave's slots [beg, beg + 64 rounds) in order: key[i] and rank[i] of this lane's slot of round i among
// the wave's equal keys; cnt (X + 2 ints, zero) receives the wave's histogram.  rounds is uniform, at most 8.
__device__ __forceinline__ void rank_wave(const int64_t* ids, int64_t beg, int rounds, int64_t n, int X, int bits, int* cnt,
                                          int (&key)[kPlanRounds], int (&rank)[kPlanRounds]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < kPlanRounds; ++i) key[i] = slot_key(ids, i < rounds ? beg + 64 * i + lane : n, n, X);
#pragma unroll
    for (int i = 0; i < kPlanRounds; ++i) {
        if (i >= rounds) break;
        const uint64_t m = lanes_with(key[i], bits);
        const int before = __popcll(m & ((1ull << lane) - 1ull));
        const int base = cnt[key[i]];
        rank[i] = base + before;
        // every lane has read before a lane writes, and the write comes before the next round's reads
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (before == 0) cnt[key[i]] = base + static_cast<int>(__popcll(m));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// Exclusive sums of v[0..X) in place (X <= 1024), the total returned, by a workgroup of NT threads.
template <int NT>
__device__ __forceinline__ int scan_buckets(int* v, int X, int* tmp) {
    constexpr int PER = kMaxExperts / NT;
    int own[PER], s = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int b = threadIdx.x * PER + i;
        own[i] = b < X ? v[b] : 0;
        s += own[i];
    }
    const int incl = inclusive_sum(s);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 63) tmp[wave] = incl;
    __syncthreads();
    int base = 0, total = 0;
    for (int w = 0; w < NT / 64; ++w) {
        if (w < wave) base += tmp[w];
        total += tmp[w];
    }
    int run = base + incl - s;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int b = threadIdx.x * PER + i;
        if (b < X) v[b] = run;
        run += own[i];
    }
    __syncthreads();
    return total;
}

// Up to 8192 slots in one workgroup.  LDS: cnt[16][X + 2], base[X + 2].
__global__ void __launch_bounds__(1024)
k_plan_one(const int64_t* __restrict__ ids, int n, int X, int bits, int32_t* __restrict__ order,
           int32_t* __restrict__ positions, int32_t* __restrict__ offsets) {
    extern __shared__ int lds[];
    __shared__ int tmp[16];
    const int nb = X + 2, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int* base = lds + 16 * nb;
    for (int i = threadIdx.x; i < 16 * nb; i += 1024) lds[i] = 0;
    __syncthreads();
    int key[kPlanRounds], rank[kPlanRounds];
    const int rounds = (n + 1023) / 1024, beg = wave * 64 * rounds;      // the slots spread over the waves
    if (beg < n) rank_wave(ids, beg, rounds, n, X, bits, lds + wave * nb, key, rank);
    __syncthreads();
    for (int b = threadIdx.x; b < nb; b += 1024) {      // the waves' exclusive sums per bucket
        int run = 0;
        for (int w = 0; w < 16; ++w) {
            const int c = lds[w * nb + b];
            lds[w * nb + b] = run;
            run += c;
        }
        base[b] = run;
    }
    __syncthreads();
    const int total = scan_buckets<1024>(base, X, tmp);
    if (threadIdx.x == 0) base[X] = total;
    __syncthreads();
    for (int b = threadIdx.x; b <= X; b += 1024) offsets[b] = base[b];
    if (beg < n) {
#pragma unroll
        for (int i = 0; i < kPlanRounds; ++i) {
            const int slot = beg + 64 * i + lane;
            if (i < rounds && slot < n) {
                const int p = base[key[i]] + lds[wave * nb + key[i]] + rank[i];
                order[p] = slot;
                positions[slot] = p;
            }
        }
    }
}

// hist[bucket][tile].  20000 rows of 2 choices, 8 experts: 5 us, and k_plan_place 7.
__global__ void __launch_bounds__(256)
k_plan_hist(const int64_t* __restrict__ ids, int64_t n, int X, int64_t ntiles, int32_t* __restrict__ hist) {
    __shared__ int cnt[kMaxExperts + 2];
    for (int i = threadIdx.x; i < X + 2; i += 256) cnt[i] = 0;
    __syncthreads();
    const int64_t beg = static_cast<int64_t>(blockIdx.x) * kPlanTile;
#pragma unroll
    for (int i = 0; i < kPlanTile / 256; ++i) atomicAdd(&cnt[slot_key(ids, beg + 256 * i + threadIdx.x, n, X)], 1);
    __syncthreads();
    for (int i = threadIdx.x; i <= X; i += 256) hist[i * ntiles + blockIdx.x] = cnt[i];
}

// Exclusive sums over the tiles of each bucket; total[bucket].
__global__ void __launch_bounds__(256)
k_plan_scan(int32_t* __restrict__ hist, int64_t ntiles, int32_t* __restrict__ total) {
    __shared__ int tmp[4];
    int32_t* h = hist + static_cast<int64_t>(blockIdx.x) * ntiles;
    int carry = 0;
    for (int64_t t0 = 0; t0 < ntiles; t0 += 256) {
        const int64_t t = t0 + threadIdx.x;
        const int v = t < ntiles ? h[t] : 0;
        const int incl = inclusive_sum(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 63) tmp[threadIdx.x >> 6] = incl;
        __syncthreads();
        int before = carry, all = 0;
        for (int w = 0; w < 4; ++w) {
            if (w < static_cast<int>(threadIdx.x >> 6)) before += tmp[w];
            all += tmp[w];
        }
        if (t < ntiles) h[t] = before + incl - v;
        carry += all;
    }
    if (threadIdx.x == 0) total[blockIdx.x] = carry;
}

__global__ void __launch_bounds__(256)
k_plan_place(const int64_t* __restrict__ ids, int64_t n, int X, int bits, int64_t ntiles,
             const int32_t* __restrict__ hist, const int32_t* __restrict__ total, int scanned, int32_t* __restrict__ order,
             int32_t* __restrict__ positions, int32_t* __restrict__ offsets) {
    __shared__ int cnt[4 * (kMaxExperts + 2)];
    __shared__ int base[kMaxExperts + 2], before[kMaxExperts + 2];
    __shared__ int tmp[4];
    const int nb = X + 2, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int i = threadIdx.x; i < 4 * nb; i += 256) cnt[i] = 0;
    for (int i = threadIdx.x; i <= X; i += 256) {
        int all = 0, mine = 0;                // slots of the bucket, and those in the tiles before
        if (scanned) {
            all = total[i];
            mine = hist[i * ntiles + blockIdx.x];
        } else {
#pragma unroll 8
            for (int t = 0; t < ntiles; ++t) {
                const int h = hist[i * ntiles + t];
                all += h;
                mine += t < static_cast<int>(blockIdx.x) ? h : 0;
            }
        }
        base[i] = all;
        before[i] = mine;
    }
    __syncthreads();
    const int all = scan_buckets<256>(base, X, tmp);
    if (threadIdx.x == 0) base[X] = all;
    __syncthreads();
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= X; b += 256) offsets[b] = base[b];
    int key[kPlanRounds], rank[kPlanRounds];
    const int64_t beg = static_cast<int64_t>(blockIdx.x) * kPlanTile + wave * 512;
    rank_wave(ids, beg, kPlanRounds, n, X, bits, cnt + wave * nb, key, rank);
    __syncthreads();
    for (int b = threadIdx.x; b <= X; b += 256) {
        int run = base[b] + before[b];
        for (int w = 0; w < 4; ++w) {
            const int c = cnt[w * nb + b];
            cnt[w * nb + b] = run;
            run += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPlanRounds; ++i) {
        const int64_t slot = beg + 64 * i + lane;
        if (slot < n) {
            const int p = cnt[wave * nb + key[i]] + rank[i];
            order[p] = static_cast<int32_t>(slot);
            positions[slot] = p;
        }
    }
}

__global__ void k_plan_empty(int32_t* offsets, int X) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i <= X) offsets[i] = 0;
}

// The one-workgroup form: its counters, 17 (X + 2) and 16, fit 64 KB.
bool plan_one(int64_t slots, int X) { return slots <= kPlanOne && (17 * (X + 2) + 16) * sizeof(int) <= 64 * 1024; }

}  // namespace
}  // namespace feq

using namespace feq;

extern "C" size_t feq_expert_topk_workspace(int64_t rows, int32_t experts) {
    if (rows < 1 || experts < 1 || experts > kMaxExperts) return 0;
    const int blocks = topk_blocks(rows, experts);
    return blocks > 1 ? sizeof(float) * static_cast<size_t>(experts) * blocks : 0;
}

extern "C" int feq_expert_topk_fwd(const void* logits, int64_t rows, int32_t experts, int32_t dtype, int32_t top_k,
                                   int32_t normalize, int64_t* ids, float* weights, float* mean, void* workspace,
                                   size_t ws_bytes, feq_stream_t stream) {
    if (int rc = topk_check(rows, experts, top_k, dtype)) return rc;
    if (rows && (!logits || !ids || !weights)) return fail(FEQ_ERR_INVALID, "NULL pointer");
    const size_t need = mean ? feq_expert_topk_workspace(rows, experts) : 0;
    if (need && (!workspace || ws_bytes < need))
        return fail(FEQ_ERR_WORKSPACE, "top-k workspace of %zu bytes, %zu needed", ws_bytes, need);
    hipStream_t s = stream_of(stream);
    const int G = topk_lanes(experts, kForwardNarrow), blocks = rows ? topk_blocks(rows, experts) : 0;
    float* part = need ? static_cast<float*>(workspace) : nullptr;
    const float inv_rows = rows ? 1.0f / static_cast<float>(rows) : 0.0f;
    if (rows) {
        const int rc = with_dtype(dtype, [&](auto t) -> int {
            using T = decltype(t);
            return with_topk_form<T>(experts, kForwardNarrow, [&](auto v, auto nc) -> int {
                auto run = [&](auto km) -> int {
                    auto kern = k_topk_fwd<T, decltype(v)::value, decltype(nc)::value, decltype(km)::value>;
                    FEQ_LAUNCH("k_topk_fwd", kern, dim3(blocks), dim3(kTopkThreads), 0, s, static_cast<const T*>(logits),
                               rows, experts, top_k, normalize, ids, weights, part, part ? nullptr : mean, inv_rows, G);
                    return FEQ_OK;
                };
                if (top_k <= 2) return run(std::integral_constant<int, 2>{});
                if (top_k <= 8) return run(std::integral_constant<int, 8>{});
                return run(std::integral_constant<int, 0>{});
            });
        });
        if (rc) return rc;
    }
    if (mean && blocks != 1)     // of no rows: 0
        FEQ_LAUNCH("k_topk_mean", k_topk_mean, dim3(ceil_div(experts, 16)), dim3(1024), 0, s, part, blocks, experts,
                   inv_rows, mean);
    return FEQ_OK;
}

extern "C" int feq_expert_topk_bwd(const void* logits, const int64_t* ids, const float* weights, const float* grad_weights,
                                   const float* grad_mean, int64_t rows, int32_t experts, int32_t dtype, int32_t top_k,
                                   int32_t normalize, void* grad_logits, feq_stream_t stream) {
    if (int rc = topk_check(rows, experts, top_k, dtype)) return rc;
    if (rows == 0) return FEQ_OK;
    if (!logits || !ids || !weights || !grad_logits) return fail(FEQ_ERR_INVALID, "NULL pointer");
    hipStream_t s = stream_of(stream);
    const int G = topk_lanes(experts, kBackwardNarrow);
    const int64_t blocks = std::min<int64_t>(ceil_div(rows, kTopkThreads / G), 2048);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        return with_topk_form<T>(experts, kBackwardNarrow, [&](auto v, auto nc) -> int {
            auto kern = k_topk_bwd<T, decltype(v)::value, decltype(nc)::value>;
            FEQ_LAUNCH("k_topk_bwd", kern, dim3(blocks), dim3(kTopkThreads), 0, s, static_cast<const T*>(logits), ids,
                       weights, grad_weights, grad_mean, rows, experts, top_k, normalize,
                       1.0f / static_cast<float>(rows), static_cast<T*>(grad_logits), G);
            return FEQ_OK;
        });
    });
}

extern "C" size_t feq_expert_plan_workspace(int64_t slots, int32_t experts) {
    if (slots < 1 || experts < 1 || experts > kMaxExperts || plan_one(slots, experts)) return 0;
    return sizeof(int32_t) * static_cast<size_t>(experts + 1) * (ceil_div(slots, kPlanTile) + 1);
}

extern "C" int feq_expert_plan(const int64_t* ids, int64_t slots, int32_t experts, int32_t* order, int32_t* positions,
                               int32_t* offsets, void* workspace, size_t ws_bytes, feq_stream_t stream) {
    if (slots < 0 || experts < 1) return fail(FEQ_ERR_INVALID, "plan of %lld slots over %d experts", (long long)slots, experts);
    if (experts > kMaxExperts) return fail(FEQ_ERR_UNSUPPORTED, "more than %d experts", kMaxExperts);
    if (slots > INT32_MAX) return fail(FEQ_ERR_UNSUPPORTED, "more than 2^31 - 1 slots");
    if (!offsets || (slots && (!ids || !order || !positions))) return fail(FEQ_ERR_INVALID, "NULL pointer");
    hipStream_t s = stream_of(stream);
    if (slots == 0) {
        FEQ_LAUNCH("k_plan_empty", k_plan_empty, dim3(ceil_div(experts + 1, 256)), dim3(256), 0, s, offsets, experts);
        return FEQ_OK;
    }
    int bits = 1;
    while ((1 << bits) < experts + 2) ++bits;
    if (plan_one(slots, experts)) {
        FEQ_LAUNCH("k_plan_one", k_plan_one, dim3(1), dim3(1024), 17 * (experts + 2) * sizeof(int), s, ids,
                   static_cast<int>(slots), experts, bits, order, positions, offsets);
        return FEQ_OK;
    }
    if (!workspace || ws_bytes < feq_expert_plan_workspace(slots, experts))
        return fail(FEQ_ERR_WORKSPACE, "plan workspace of %zu bytes, %zu needed", ws_bytes,
                    feq_expert_plan_workspace(slots, experts));
    const int64_t ntiles = ceil_div(slots, kPlanTile);
    int32_t* hist = static_cast<int32_t*>(workspace);
    int32_t* total = hist + (experts + 1) * ntiles;
    FEQ_LAUNCH("k_plan_hist", k_plan_hist, dim3(ntiles), dim3(256), 0, s, ids, slots, experts, ntiles, hist);
    const bool scan = ntiles > kPlanOwnSums || experts + 1 > kPlanOwnBuckets;
    if (scan) FEQ_LAUNCH("k_plan_scan", k_plan_scan, dim3(experts + 1), dim3(256), 0, s, hist, ntiles, total);
    FEQ_LAUNCH("k_plan_place", k_plan_place, dim3(ntiles), dim3(256), 0, s, ids, slots, experts, bits, ntiles, hist,
               total, scan, order, positions, offsets);
    return FEQ_OK;
}
