// A channel map shared by all rows beside low-rank maps of which every row has its own.  With a = the adapter of row i,
// r(d) the irrep of plane (component) d and s the scale,
//   t[d, i, q] = s sum_k x[d, i, k] down[a, r, q, k],
//   y[d, i, n] = sum_k x[d, i, k] W[r, n, k] + sum_q t[d, i, q] up[a, r, n, q]  (+ b[n, j] on the plane of the j-th scalar irrep),
//   u[d, i, q] = s sum_n grad_y[d, i, n] up[a, r, n, q],
//   grad_x[d, i, k] = sum_n grad_y[d, i, n] W[r, n, k] + sum_q u[d, i, q] down[a, r, q, k],
//   grad_down[a, r, q, k] = sum over the planes d of r and rows i of a of u[d, i, q] x[d, i, k],
//   grad_up[a, r, n, q] = sum over the same of t[d, i, q] grad_y[d, i, n];
// a row without an adapter has the shared map alone.  Forward and grad_x are one product of the form
//   out = in B + ((s in F^T) G^T) with (B, F, G) = (W^T, down, up) or (W, up^T, down^T), and the reduced rows s in F^T are kept in
// float32 for the sums over rows (`low`, (dim, rows, 16 rt), in the plan's order).
//
// Rows are taken in the plan's order, so that those of an adapter are neighbours, and read and written where they lie: the
// order's entries are the rows' numbers.  The reduced row is the first product's accumulator and goes into the second product
// without leaving the registers: rank q = 4 g + m of a tile of 16 is what lane (c, g) holds of row c, which are the four
// elements that the second operand's lane (c, g) needs.  16-bit types enter it as the sum of two 16-bit numbers (elements
// 0 to 3 the rounded values, 4 to 7 what is left), with up's elements twice: 2^-16 (bfloat16) or 2^-21 of the value is lost,
// where one number would lose 2^-8 or 2^-11 of a sum that the result rounds only once.  float16's narrow range: every row is
// multiplied by a power of two that brings its largest reduced value to 2^13 .. 2^14, and so is its accumulator meanwhile.
#include "adapter_tiles.h"

namespace feq {
namespace {

// A reduction of at most 128 columns: the shared map and the maps of one adapter stay in LDS, the rows stream (see
// k_xl_stream, whose division of the work this is).  20011 x 49 bfloat16 rows of 128 to 128 columns, 16 adapters of rank
// 16, take 132 us, 3.8 TB/s; 20000 x 9 float32 rows of 64 to 128 take 65, memory's 28 and the products' 27 overlapped in part.
template <class T, int HOW, bool TRANS, int NB, int NS, int RT>
__global__ void __launch_bounds__(kXlThreads, NB * NS * Mma<T>::KS * sizeof(T) > 40000 || RT > 1 ? 2 : 3)
k_ad_stream(AdArgs a, XlMap map) {
    using M = Mma<T>;
    typedef typename M::frag frag;
    constexpr int V = 16 / sizeof(T), KM = NS * M::KS;
    constexpr int NT = NB / 16, NA = NT < 4 ? NT : 4;
    constexpr int LD = KM + V, LDT = NB + M::PAD;
    const int rt = RT == 1 ? 1 : a.rt, rp = 16 * rt, K = a.K, N = a.N, X = a.X, S = a.S, R = a.R, nreps = a.nreps;
    const int LDF = TRANS ? rp + M::PAD : LD, LDG = TRANS ? LDT : rp + 4;
    extern __shared__ __align__(16) char smem[];
    T* sW = reinterpret_cast<T*>(smem);
    float* sBias = reinterpret_cast<float*>(sW + (TRANS ? KM * LDT : NB * LD));
    T* sF = reinterpret_cast<T*>(sBias + NB);
    T* sG = sF + (TRANS ? KM * LDF : rp * LDF);
    const T *in = static_cast<const T*>(a.in), *W = static_cast<const T*>(a.W);
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nb = (N + NB - 1) / NB;
    const XlBlocks<> experts(a.offsets, X, S, 16);
    const int per_plane = experts.total();
    const int64_t total = static_cast<int64_t>(per_plane) * a.dim * nb;
    const int64_t share = total / gridDim.x, more = total % gridDim.x;
    int64_t at = blockIdx.x * share + (blockIdx.x < more ? blockIdx.x : more);
    const int64_t end = at + share + (blockIdx.x < more ? 1 : 0);
    int staged = -1;
    while (at < end) {
        const int line = static_cast<int>(at / per_plane), d = line / nb, n0 = line % nb * NB;
        const XlTile t = experts.find(static_cast<int>(at % per_plane));
        const int rows = t.row1 - t.row0, left = t.count - t.index;
        const int nblocks = static_cast<int>(end - at < left ? end - at : left);
        at += nblocks;
        const int rep = __builtin_amdgcn_readfirstlane(map.rep[d]);
        const bool own = t.expert < X;               // uniform
        const T* id = in + static_cast<int64_t>(d) * S * K;
        T* od = static_cast<T*>(a.out) + static_cast<int64_t>(d) * S * N + n0;

        auto number = [&](int blk) {                 // the row at this lane's place, -1: none
            const int r = 16 * blk + c;
            return r < rows && blk < nblocks ? a.order[t.row0 + r] : -1;
        };
        frag b0[NS], b1[NS];
        auto load = [&](int64_t row, frag (&b)[NS]) {
            const T* p = id + (row < 0 ? 0 : row) * K;
#pragma unroll
            for (int ks = 0; ks < NS; ++ks) {
                const int k = ks * M::KS + M::FE * g;
                b[ks] = __builtin_bit_cast(frag, load_row<T, HOW>(p, k, K - k, in));
            }
        };
        auto arrived = [&](const frag (&b)[NS]) {
#pragma unroll
            for (int ks = 0; ks < NS; ++ks)
                b0[ks] = __builtin_bit_cast(frag, placed_row<T, HOW>(__builtin_bit_cast(uint4, b[ks]), K - ks * M::KS - M::FE * g, K, in));
        };
        int row = number(wave), next = number(wave + 4);
        load(row, b1);
        __syncthreads();                             // what the last run read
        if (staged != line) {
            staged = line;
            const T* wm = W + static_cast<int64_t>(rep) * K * N;
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
            const bool biased = !TRANS && a.bias && bc >= 0;
            if (tid < NB)
                sBias[tid] = load1<T>(table(a.bias, biased), ((n0 + tid) * a.nbias + bc) * sizeof(T), n0 + tid < N);
        }
        if (own) {
            const int64_t map0 = (static_cast<int64_t>(t.expert) * nreps + rep) * R;
            const T *fe = static_cast<const T*>(a.F) + map0 * K, *ge = static_cast<const T*>(a.G) + map0 * N;
            for (int i = tid; i < rp * KM; i += kXlThreads) {        // F: down (R, K) as it lies, or up (K, R) as it lies
                const int q = TRANS ? i % rp : i / KM, k = TRANS ? i / rp : i % KM;
                const bool there = q < R && k < K;
                const T v = fe[there ? (TRANS ? k * R + q : q * K + k) : 0];
                sF[TRANS ? k * LDF + q : q * LDF + k] = there ? v : static_cast<T>(0.0f);
            }
            for (int i = tid; i < rp * NB; i += kXlThreads) {        // G: up (N, R) as it lies, or down (R, N) as it lies
                const int q = TRANS ? i / NB : i % rp, n = TRANS ? i % NB : i / rp;
                const bool there = q < R && n0 + n < N;
                const T v = ge[there ? (TRANS ? q * N + n0 + n : static_cast<int64_t>(n0 + n) * R + q) : 0];
                sG[TRANS ? q * LDG + dealt<T>(n) : dealt<T>(n) * LDG + q] = there ? v : static_cast<T>(0.0f);
            }
        }
        __syncthreads();
        arrived(b1);
        for (int blk = wave; blk < nblocks; blk += 4) {
            const int after = number(blk + 8);
            load(next, b1);
            asm volatile("" ::: "memory");           // the maps are read from LDS for every block (k_xl_stream)
            v4f acc[NT], low[RT];
#pragma unroll
            for (int i = 0; i < NT; ++i)
                acc[i] = *reinterpret_cast<const v4f*>(sBias + 16 * (i - i % kDealt<T>) + V * g + 4 * (i % kDealt<T>));
#pragma unroll
            for (int ks = 0; ks < NS; ++ks) {
#pragma unroll
                for (int i0 = 0; i0 < NT; i0 += NA) {
                    frag f[NA];
#pragma unroll
                    for (int i = 0; i < NA; ++i) {
                        if constexpr (TRANS) f[i] = M::columns(sW, LDT, ks * M::KS, g, c, 16 * (i0 + i));
                        else f[i] = *reinterpret_cast<const frag*>(sW + (16 * (i0 + i) + c) * LD + ks * M::KS + M::FE * g);
                    }
                    M::template mul_all<NA>(f, b0[ks], acc + i0);
                }
            }
            if (own) {
                float most = 0.0f;
#pragma unroll
                for (int q = 0; q < RT; ++q) {
                    if (q >= rt) break;
                    low[q] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int ks = 0; ks < NS; ++ks) {
                        frag f;
                        if constexpr (TRANS) f = M::columns(sF, LDF, ks * M::KS, g, c, 16 * q);
                        else f = *reinterpret_cast<const frag*>(sF + (16 * q + c) * LDF + ks * M::KS + M::FE * g);
                        low[q] = M::mul(f, b0[ks], low[q]);
                    }
                    low[q] *= a.scale;
                    if (a.low && n0 == 0 && row >= 0)
                        *reinterpret_cast<v4f*>(a.low + (static_cast<int64_t>(d) * S + t.row0 + 16 * blk + c) * rp + 16 * q + 4 * g) = low[q];
                    if constexpr (std::is_same<T, _Float16>::value)
#pragma unroll
                        for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(low[q][j]));
                }
                int power = 0;
                if constexpr (std::is_same<T, _Float16>::value) {
                    power = low_exponent(row_max(most));
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[i][j] = times_power(acc[i][j], power);
                }
#pragma unroll
                for (int q = 0; q < RT; ++q) {
                    if (q >= rt) break;
                    v4f v = low[q];
                    if constexpr (std::is_same<T, _Float16>::value)
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[j] = times_power(v[j], power);
                    const frag b = low_frag(v, T{});
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        T e[4];
                        if constexpr (!TRANS) {
                            const typename VecOf<T, 4>::type x = *reinterpret_cast<const typename VecOf<T, 4>::type*>(sG + (16 * i + c) * LDG + 16 * q + 4 * g);
#pragma unroll
                            for (int j = 0; j < 4; ++j) e[j] = x[j];
                        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) e[j] = sG[(16 * q + 4 * g + j) * LDG + 16 * i + c];
                        } else {
                            const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(sG + (16 * q + 4 * g + (c >> 2)) * LDG + 16 * i + 4 * (c & 3)));
#pragma unroll
                            for (int j = 0; j < 4; ++j) e[j] = __builtin_bit_cast(T, static_cast<short>(x[j]));
                        }
                        acc[i] = M::mul(twice<T>(e), b, acc[i]);
                    }
                }
                if constexpr (std::is_same<T, _Float16>::value)
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[i][j] = times_power(acc[i][j], -power);
            }
            if (row >= 0) {
                T* o = od + static_cast<int64_t>(row) * N;
#pragma unroll
                for (int i = 0; i < NT; i += kDealt<T>) {
                    const int n = 16 * i + V * g;
                    store_tiles<T, HOW, 1>(o + n, N - n0 - n, &acc[i]);
                }
            }
            arrived(b1);
            row = next;
            next = after;
        }
    }
}

// The reduced rows of a wide reduction, s in F^T, 16 rows of an adapter a workgroup, whose waves take a quarter of the
// reduction each.  blockIdx.y: the plane.  8191 bfloat16 rows, rank 32: 8 us for 512 columns, 13 for 1024 (1.0 and 1.3 TB/s: a
// wave has 2 to 8 steps, and their loads' latency bounds it).
template <class T, int HOW, bool TRANS>
__global__ void __launch_bounds__(kXlThreads)
k_ad_low(AdArgs a, XlMap map) {
    using M = Mma<T>;
    typedef typename M::frag frag;
    __shared__ __align__(16) v4f part[3][kAdMaxRank / 16][64];
    const int d = blockIdx.y, K = a.K, R = a.R, rp = 16 * a.rt;
    const XlTile t = XlBlocks<>(a.offsets, a.X, a.S, 16).find(blockIdx.x);
    if (t.expert < 0 || t.expert == a.X) return;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const bool there = t.row0 + c < t.row1;
    const T* in = static_cast<const T*>(a.in);
    const T* row = in + (static_cast<int64_t>(d) * a.S + a.order[there ? t.row0 + c : t.row0]) * K;
    const T* fe = static_cast<const T*>(a.F) + (static_cast<int64_t>(t.expert) * a.nreps + map.rep[d]) * R * K;
    v4f acc[kAdMaxRank / 16];
#pragma unroll
    for (int q = 0; q < kAdMaxRank / 16; ++q) acc[q] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int steps = (K + M::KS - 1) / M::KS;
    for (int ks = wave; ks < steps; ks += 4) {
        const int k = ks * M::KS + M::FE * g;
        const frag b = __builtin_bit_cast(frag, placed_row<T, HOW>(load_row<T, HOW>(row, k, K - k, in), K - k, K, in));
#pragma unroll
        for (int q = 0; q < kAdMaxRank / 16; ++q) {
            if (q >= a.rt) break;
            const int r = 16 * q + c;
            frag f;
            if constexpr (!TRANS) {
                const int n = r < R ? K - k : 0;
                f = __builtin_bit_cast(frag, placed_row<T, HOW>(load_row<T, HOW>(fe + (r < R ? r : 0) * static_cast<int64_t>(K), k, n, in), n, K, in));
            } else {
#pragma unroll
                for (int j = 0; j < M::FE; ++j) {
                    const bool has = r < R && k + j < K;
                    const T v = fe[has ? static_cast<int64_t>(k + j) * R + r : 0];
                    f[j] = has ? v : static_cast<T>(0.0f);
                }
            }
            acc[q] = M::mul(f, b, acc[q]);
        }
    }
    if (wave)
        for (int q = 0; q < a.rt; ++q) part[wave - 1][q][lane] = acc[q];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int q = 0; q < kAdMaxRank / 16; ++q) {
        if (q >= a.rt) break;
        v4f v = acc[q];
#pragma unroll
        for (int w = 0; w < 3; ++w) v += part[w][q][lane];
        if (there) *reinterpret_cast<v4f*>(a.low + (static_cast<int64_t>(d) * a.S + t.row0 + c) * rp + 16 * q + 4 * g) = v * a.scale;
    }
}

// The product for a wider reduction: blocks of 128 rows in the plan's order, whatever their adapters, through LDS (k_xl_mm's
// tiles); then, for the adapters of the block in turn, the reduced rows (k_ad_low's) times G, whose operands come from
// memory in the matrix cores' layout.  8191 bfloat16 rows, 512 to 1024 columns, 64 adapters: 32 us, 270 TFLOP/s; 64 row blocks
// by 8 column blocks are one round of the chip, of 8 steps whose LDS and barrier latency bounds it.
template <class T, int HOW, bool TRANS, int WR>
__global__ void __launch_bounds__(kXlThreads, 2)
k_ad_mm(AdArgs a, XlMap map) {
    using M = Mma<T>;
    typedef typename M::frag frag;
    constexpr int V = 16 / sizeof(T), BK = kXlRowBytes / sizeof(T), CH = BK / V;
    constexpr int BN = 64 * WR, WC = 4 / WR, PT = kXlBM / (16 * WC);
    constexpr int LD = BK + V, LDT = BN + M::PAD;
    constexpr int NIN = kXlBM * CH / kXlThreads, NW = BN * CH / kXlThreads;
    __shared__ __align__(16) T sIn[2][kXlBM * LD];
    __shared__ __align__(16) T sW[2][TRANS ? BK * LDT : BN * LD];
    const int d = blockIdx.y, K = a.K, N = a.N, X = a.X, S = a.S, R = a.R;
    int sub;
    const int tile = xcd_tile(blockIdx.x, (N + BN - 1) / BN, (S + kXlBM - 1) / kXlBM, sub);
    if (tile < 0) return;
    const int row0 = tile * kXlBM, n0 = sub * BN, rows = S - row0 < kXlBM ? S - row0 : kXlBM;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave % WR, wc = wave / WR;
    const int rep = __builtin_amdgcn_readfirstlane(map.rep[d]);
    const T *in = static_cast<const T*>(a.in), *W = static_cast<const T*>(a.W);
    const T* id = in + static_cast<int64_t>(d) * S * K;
    const T* we = W + static_cast<int64_t>(rep) * K * N;
    const T* from[NIN];
#pragma unroll
    for (int i = 0; i < NIN; ++i) {
        const int r = (tid + kXlThreads * i) / CH;
        from[i] = id + static_cast<int64_t>(a.order[row0 + (r < rows ? r : 0)]) * K;
    }
    const int kin = tid % CH * V;                    // kXlThreads is a multiple of CH
    auto load = [&](int k0, uint4 (&vin)[NIN], uint4 (&vw)[NW]) {
#pragma unroll
        for (int i = 0; i < NIN; ++i) vin[i] = load_row<T, HOW>(from[i], k0 + kin, K - k0 - kin, in);
        const Rows w = rows_at(TRANS ? we + static_cast<int64_t>(k0) * N + n0 : we + static_cast<int64_t>(n0) * K, W, TRANS ? N : K);
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const int q = tid + kXlThreads * i;
            if constexpr (TRANS) {
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
            const int r = (tid + kXlThreads * i) / CH;
            *reinterpret_cast<uint4*>(sIn[u] + r * LD + kin) = placed_row<T, HOW>(vin[i], K - k0 - kin, K, in);
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
    // lane (c, g): row c of row tile j, columns 16 i + V g + 0 .. V - 1 of the wave's 64 for tile group i
    const int nw = n0 + 64 * wr + V * g;
    const int bc = __builtin_amdgcn_readfirstlane(map.bcol[d]);
    const bool biased = !TRANS && a.bias && bc >= 0;
    const Table be = table(a.bias, biased);
    v4f acc[4][PT];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = nw + 16 * (i - i % kDealt<T>) + 4 * (i % kDealt<T>) + r;
            const float bv = load1<T>(be, (n * a.nbias + bc) * sizeof(T), n < N);
#pragma unroll
            for (int j = 0; j < PT; ++j) acc[i][j][r] = bv;
        }
    uint4 vin[NIN], vw[NW];
    auto step = [&](int k0, int u) {
        stage(u ^ 1, k0 + BK, vin, vw);
        load(k0 + 2 * BK, vin, vw);                  // nothing behind K
#pragma unroll
        for (int ks = 0; ks < BK; ks += M::KS) {
            frag f[4], b[PT];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int q0 = 64 * wr + 16 * i;
                if constexpr (TRANS) f[i] = M::columns(sW[u], LDT, ks, g, c, q0);
                else f[i] = *reinterpret_cast<const frag*>(sW[u] + (q0 + c) * LD + ks + M::FE * g);
            }
#pragma unroll
            for (int j = 0; j < PT; ++j)
                b[j] = *reinterpret_cast<const frag*>(sIn[u] + (16 * (wc * PT + j) + c) * LD + ks + M::FE * g);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < PT; ++j) acc[i][j] = M::mul(f[i], b[j], acc[i][j]);
        }
        __syncthreads();
    };
    load(0, vin, vw);
    stage(0, 0, vin, vw);
    load(BK, vin, vw);
    __syncthreads();
    for (int k0 = 0; k0 < K; k0 += 2 * BK) {
        step(k0, 0);
        if (k0 + BK >= K) break;
        step(k0 + BK, 1);
    }
    // the adapters of the wave's rows
    const int r0 = row0 + 16 * wc * PT, r1 = r0 + 16 * PT < row0 + rows ? r0 + 16 * PT : row0 + rows;
    int power[PT];
#pragma unroll
    for (int j = 0; j < PT; ++j) power[j] = 0;
    if constexpr (std::is_same<T, _Float16>::value) {
#pragma unroll
        for (int j = 0; j < PT; ++j) {
            const int row = r0 + 16 * j + c;
            float most = 0.0f;
            if (row < r1 && row < a.offsets[X]) {
                const float* lo = a.low + (static_cast<int64_t>(d) * S + row) * 16 * a.rt + 4 * g;
                for (int q = 0; q < a.rt; ++q)
#pragma unroll
                    for (int m = 0; m < 4; ++m) most = fmaxf(most, fabsf(lo[16 * q + m]));
            }
            power[j] = low_exponent(row_max(most));
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int m = 0; m < 4; ++m) acc[i][j][m] = times_power(acc[i][j][m], power[j]);
        }
    }
    int lo_e = 0, hi_e = X;                          // the adapter of row r0: the last whose rows begin at or before it
    while (hi_e - lo_e > 1) {
        const int mid = (lo_e + hi_e) >> 1;
        if (a.offsets[mid] <= r0) lo_e = mid;
        else hi_e = mid;
    }
    for (int e = lo_e; e < X; ++e) {
        const int ea = a.offsets[e], ez = a.offsets[e + 1];          // uniform
        if (ea >= r1) break;
        if (ez <= ea || ez <= r0) continue;
        const T* ge = static_cast<const T*>(a.G) + (static_cast<int64_t>(e) * a.nreps + rep) * R * N;
        for (int q = 0; q < a.rt; ++q) {
            frag f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // the column that row 16 i + c of the dealt tile is
                const int m = 16 * i + c, p = m & 31;
                const int n = n0 + 64 * wr + (kDealt<T> == 1 ? m : (m - p) + 8 * (p >> 2 & 3) + 4 * (p >> 4) + (p & 3));
                f[i] = second_frag<T, TRANS>(ge, n, 16 * q + 4 * g, N, R);
            }
#pragma unroll
            for (int j = 0; j < PT; ++j) {
                const int ta = r0 + 16 * j;
                if (ta + 16 <= ea || ta >= ez || ta >= r1) continue;                 // uniform
                const int row = ta + c;
                v4f v = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                if (row >= ea && row < ez && row < r1)
                    v = *reinterpret_cast<const v4f*>(a.low + (static_cast<int64_t>(d) * S + row) * 16 * a.rt + 16 * q + 4 * g);
                if constexpr (std::is_same<T, _Float16>::value)
#pragma unroll
                    for (int m = 0; m < 4; ++m) v[m] = times_power(v[m], power[j]);
                const frag b = low_frag(v, T{});
                if (ta >= ea && ta + 16 <= ez) {                                     // uniform
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[i][j] = M::mul(f[i], b, acc[i][j]);
                } else {                             // rows of other adapters too: 0 times what this one's maps hold may be NaN
                    const bool mine = row >= ea && row < ez;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const v4f sum = M::mul(f[i], b, v4f{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                        for (int m = 0; m < 4; ++m) acc[i][j][m] += mine ? sum[m] : 0.0f;
                    }
                }
            }
        }
    }
    T* od = static_cast<T*>(a.out) + static_cast<int64_t>(d) * S * N;
#pragma unroll
    for (int j = 0; j < PT; ++j) {
        const int r = r0 + 16 * j + c;
        if constexpr (std::is_same<T, _Float16>::value)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int m = 0; m < 4; ++m) acc[i][j][m] = times_power(acc[i][j][m], -power[j]);
        if (r >= r1) continue;
        T* o = od + static_cast<int64_t>(a.order[r]) * N;
#pragma unroll
        for (int i = 0; i < 4; i += kDealt<T>) {
            const int n = nw + 16 * i;
            store_tiles<T, HOW, PT>(o + n, N - n, &acc[i][j]);
        }
    }
}

// The same product for few rows, whose 128-row blocks would leave the chip idle: a wave takes 16 rows and 32 columns, all
// operands straight from memory in the matrix cores' layout, the reduction in steps of four loads each.
template <class T, int HOW, bool TRANS>
__global__ void __launch_bounds__(64)
k_ad_few(AdArgs a, XlMap map) {
    using M = Mma<T>;
    typedef typename M::frag frag;
    constexpr int V = 16 / sizeof(T), CT = 2, NU = 4;            // column tiles; reduction steps on their way together
    const int d = blockIdx.z, K = a.K, N = a.N, X = a.X, S = a.S, R = a.R;
    const int lane = threadIdx.x, c = lane & 15, g = lane >> 4;
    const int row0 = blockIdx.y * 16, n0 = blockIdx.x * 16 * CT, rows = S - row0 < 16 ? S - row0 : 16;
    const int rep = __builtin_amdgcn_readfirstlane(map.rep[d]);
    const T *in = static_cast<const T*>(a.in), *we = static_cast<const T*>(a.W) + static_cast<int64_t>(rep) * K * N;
    const int mine = a.order[row0 + (c < rows ? c : 0)];
    const T* row = in + (static_cast<int64_t>(d) * S + mine) * K;
    // the column that row c of tile i is: as stored, 16 bytes of a row of the result are a lane's
    int col[CT];
#pragma unroll
    for (int i = 0; i < CT; ++i) col[i] = n0 + (kDealt<T> == 1 ? 16 * i + c : 8 * (c >> 2) + 4 * i + (c & 3));
    const int bc = __builtin_amdgcn_readfirstlane(map.bcol[d]);
    const bool biased = !TRANS && a.bias && bc >= 0;
    const Table be = table(a.bias, biased);
    v4f acc[CT];
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const int n = n0 + V * g + 16 * (i - i % kDealt<T>) + 4 * (i % kDealt<T>) + m;
            acc[i][m] = load1<T>(be, (n * a.nbias + bc) * sizeof(T), n < N);
        }
    const int steps = (K + M::KS - 1) / M::KS;
    for (int s0 = 0; s0 < steps; s0 += NU) {
        uint4 vb[NU];
        frag fw[NU][CT];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int k = (s0 + u) * M::KS + M::FE * g;
            vb[u] = load_row<T, HOW>(row, k, K - k, in);
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                if constexpr (!TRANS) {
                    const int n = col[i] < N ? K - k : 0;
                    fw[u][i] = __builtin_bit_cast(frag, placed_row<T, HOW>(load_row<T, HOW>(we + static_cast<int64_t>(col[i] < N ? col[i] : 0) * K, k, n, we), n, K, we));
                } else {
#pragma unroll
                    for (int j = 0; j < M::FE; ++j) {
                        const bool has = col[i] < N && k + j < K;
                        const T v = we[has ? static_cast<int64_t>(k + j) * N + col[i] : 0];
                        fw[u][i][j] = has ? v : static_cast<T>(0.0f);
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int k = (s0 + u) * M::KS + M::FE * g;
            const frag b = __builtin_bit_cast(frag, placed_row<T, HOW>(vb[u], K - k, K, in));
#pragma unroll
            for (int i = 0; i < CT; ++i) acc[i] = M::mul(fw[u][i], b, acc[i]);
        }
    }
    const int placed = a.offsets[X];
    int power = 0;
    const float* lo = a.low + (static_cast<int64_t>(d) * S + row0 + c) * 16 * a.rt + 4 * g;
    const bool own = c < rows && row0 + c < placed;
    if constexpr (std::is_same<T, _Float16>::value) {
        float most = 0.0f;
        if (own)
            for (int q = 0; q < a.rt; ++q)
#pragma unroll
                for (int m = 0; m < 4; ++m) most = fmaxf(most, fabsf(lo[16 * q + m]));
        power = low_exponent(row_max(most));
#pragma unroll
        for (int i = 0; i < CT; ++i)
#pragma unroll
            for (int m = 0; m < 4; ++m) acc[i][m] = times_power(acc[i][m], power);
    }
    // the row's adapter: the last whose rows begin at or before it
    int lo_e = 0, hi_e = X;
    while (hi_e - lo_e > 1) {
        const int mid = (lo_e + hi_e) >> 1;
        if (a.offsets[mid] <= row0 + (c < rows ? c : 0)) lo_e = mid;
        else hi_e = mid;
    }
    const int adapter = own ? lo_e : -1;
    for (int q = 0; q < a.rt; ++q) {
        v4f v = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (own) v = *reinterpret_cast<const v4f*>(lo + 16 * q);
        if constexpr (std::is_same<T, _Float16>::value)
#pragma unroll
            for (int m = 0; m < 4; ++m) v[m] = times_power(v[m], power);
        const frag b = low_frag(v, T{});
        // the adapters of the rows, four at a time; a row takes the sums of its own
        for (int p0 = 0; p0 < rows; p0 += 4) {
            frag f[4][CT];
            int e[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                e[u] = p0 + u < rows ? __builtin_amdgcn_readlane(adapter, p0 + u) : -1;
                const int before = p0 + u > 0 ? __builtin_amdgcn_readlane(adapter, (p0 + u - 1) & 15) : -1;
                if (e[u] == before) e[u] = -1;                   // uniform: rows of an adapter are neighbours
                const T* ge = static_cast<const T*>(a.G) + (static_cast<int64_t>(e[u] < 0 ? 0 : e[u]) * a.nreps + rep) * R * N;
#pragma unroll
                for (int i = 0; i < CT; ++i) f[u][i] = second_frag<T, TRANS>(ge, e[u] < 0 ? N : col[i], 16 * q + 4 * g, N, R);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (e[u] < 0) continue;
#pragma unroll
                for (int i = 0; i < CT; ++i) {
                    const v4f sum = M::mul(f[u][i], b, v4f{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                    for (int m = 0; m < 4; ++m) acc[i][m] += adapter == e[u] ? sum[m] : 0.0f;
                }
            }
        }
    }
    if constexpr (std::is_same<T, _Float16>::value)
#pragma unroll
        for (int i = 0; i < CT; ++i)
#pragma unroll
            for (int m = 0; m < 4; ++m) acc[i][m] = times_power(acc[i][m], -power);
    if (c >= rows) return;
    T* o = static_cast<T*>(a.out) + (static_cast<int64_t>(d) * S + mine) * N;
#pragma unroll
    for (int i = 0; i < CT; i += kDealt<T>) {
        const int n = n0 + 16 * i + V * g;
        store_tiles<T, HOW, 1>(o + n, N - n, &acc[i]);
    }
}

// Sums over an adapter's rows of a reduced row and a whole one, out[q, k] = sum of z[q] v[k] (UP: out[k, q]), over row
// chunks as the experts' weight gradients (k_xl_wgrad): an adapter of one chunk gets its gradient written, one of several
// a float32 partial per chunk.  float32 products for all types: the reduced rows are float32.  8191 bfloat16 rows of 64 adapters
// of rank 32 take 12 us for 512 columns and 26 for 1024, most of it latency: two or three steps a chunk.  (16-bit products from
// the waves' own LDS and both sums in one launch made the pass no shorter.)
template <class T, int HOW, int BC, bool UP>
__global__ void __launch_bounds__(kXlThreads)
k_ad_sums(const T* __restrict__ v, const float* __restrict__ z, const int32_t* __restrict__ offsets,
          const int32_t* __restrict__ order, int X, int S, int C, int R, int rt, int nreps, XlMap map, XlChunks ch,
          T* __restrict__ out, float* __restrict__ parts) {
    using M = Mma<float>;
    constexpr int V = 16 / sizeof(T), BP = 32;
    constexpr int NT = BC / 64;                                  // column tiles of a wave
    constexpr int LV = BC + M::PAD, LZ = kAdMaxRank + M::PAD;
    constexpr int NV = BP * (BC / V) / kXlThreads;
    __shared__ __align__(16) float sV[BP * LV];
    __shared__ __align__(16) float sZ[BP * LZ];
    const int nc = (C + BC - 1) / BC, xcds = ch.xcds, block = blockIdx.x / (xcds * nc);
    int rep = nreps - 1;
    while (rep > 0 && block >= ch.tile0[rep - 1]) --rep;
    const int rc = ch.rows[rep];
    const int i0 = blockIdx.x / xcds - ch.tile0[rep] * nc, sub = i0 % nc;
    const XlTile t = XlBlocks<true>(offsets, X, S, rc).find(i0 / nc * xcds + blockIdx.x % xcds);
    if (t.expert < 0 || t.expert == X) return;
    const int c0 = sub * BC, rp = 16 * rt;
    const int rend = t.row1 - t.row0 < rc ? t.row1 : t.row0 + rc;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int d0 = __builtin_amdgcn_readfirstlane(map.first[rep]), d1 = __builtin_amdgcn_readfirstlane(map.first[rep + 1]);
    const int steps = (rend - t.row0 + BP - 1) / BP, total = steps * (d1 - d0);
    const int zq = rp / 4;                                       // vectors of a reduced row: 32 rows have 32 zq of them
    uint4 vv[NV];
    v4f vz[2];
    auto load = [&](int it) {
        const int d = it < total ? d0 + it / steps : d0, r0 = it < total ? t.row0 + (it % steps) * BP : t.row0;
        const int there = it < total ? rend - r0 : 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int q = tid + kXlThreads * i, r = q / (BC / V), k = c0 + (q % (BC / V)) * V;
            const bool has = r < there;
            const T* p = v + (static_cast<int64_t>(d) * S + (has ? order[r0 + r] : 0)) * C;
            vv[i] = load_row<T, HOW>(p, k, has ? C - k : 0, v);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int q = tid + kXlThreads * i, r = q / zq, k = (q % zq) * 4;
            const bool has = r < BP && r < there;
            vz[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            if (has) vz[i] = *reinterpret_cast<const v4f*>(z + (static_cast<int64_t>(d) * S + r0 + r) * rp + k);
        }
    };
    v4f acc[kAdMaxRank / 16][NT];
#pragma unroll
    for (int q = 0; q < kAdMaxRank / 16; ++q)
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[q][i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (total) load(0);
    for (int it = 0; it < total; ++it) {
        const int there = rend - (t.row0 + (it % steps) * BP);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int q = tid + kXlThreads * i, r = q / (BC / V), k = (q % (BC / V)) * V;
            const uint4 w = placed_row<T, HOW>(vv[i], r < there ? C - c0 - k : 0, C, v);
            const typename VecOf<T, V>::type e = __builtin_bit_cast(typename VecOf<T, V>::type, w);
#pragma unroll
            for (int j = 0; j < V; ++j) sV[r * LV + k + j] = static_cast<float>(e[j]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int q = tid + kXlThreads * i, r = q / zq, k = (q % zq) * 4;
            if (r < BP) *reinterpret_cast<v4f*>(sZ + r * LZ + k) = vz[i];
        }
        __syncthreads();
        load(it + 1);
#pragma unroll
        for (int ks = 0; ks < BP; ks += M::KS) {
            v4f b[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) b[i] = M::columns(sV, LV, ks, g, c, 16 * (wave * NT + i));
#pragma unroll
            for (int q = 0; q < kAdMaxRank / 16; ++q) {
                if (q >= rt) break;
                const v4f f = M::columns(sZ, LZ, ks, g, c, 16 * q);
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[q][i] = M::mul(f, b[i], acc[q][i]);
            }
        }
    }
    const bool direct = t.count == 1;
    const int64_t slot = ch.slot0[rep] + t.before + t.index;
    const int64_t base = (direct ? static_cast<int64_t>(t.expert) * nreps + rep : slot) * R * C;
#pragma unroll
    for (int q = 0; q < kAdMaxRank / 16; ++q) {
        if (q >= rt) break;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int k = c0 + 16 * (wave * NT + i) + c;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const int r = 16 * q + 4 * g + m;
                if (k >= C || r >= R) continue;
                const int64_t o = base + (UP ? static_cast<int64_t>(k) * R + r : static_cast<int64_t>(r) * C + k);
                if (direct) out[o] = static_cast<T>(acc[q][i][m]);
                else parts[o] = acc[q][i][m];
            }
        }
    }
}

// The ends of one expert that has all S rows.
__global__ void k_ad_all(int32_t* offsets, int S) {
    if (threadIdx.x < 2) offsets[threadIdx.x] = threadIdx.x ? S : 0;
}

int ad_check(const AdShape& p, const int32_t* bias_cols, int32_t nbias, float scale, XlMap* map) {
    if (p.R < 1) return fail(FEQ_ERR_INVALID, "adapters of rank %d", p.R);
    if (p.R > kAdMaxRank) return fail(FEQ_ERR_UNSUPPORTED, "adapters of a rank above %d", kAdMaxRank);
    if (!(scale - scale == 0.0f)) return fail(FEQ_ERR_INVALID, "scale %g is not finite", scale);
    return xl_check(p.lvals, p.nreps, p.X, p.S, p.ci, p.co, p.dtype, bias_cols, nbias, map);
}

int ad_tiles(int R) { return static_cast<int>(ceil_div(R, 16)); }

template <class T, bool TRANS>
int ad_run(const AdShape& p, const XlMap& map, AdArgs a, std::initializer_list<const void*> ptrs, hipStream_t s) {
    a.X = p.X;
    a.S = static_cast<int>(p.S);
    a.K = TRANS ? p.co : p.ci;
    a.N = TRANS ? p.ci : p.co;
    a.R = p.R;
    a.nreps = p.nreps;
    a.dim = map.first[p.nreps];
    a.rt = ad_tiles(p.R);
    const int K = a.K, N = a.N, dim = a.dim;
    return with_rows<T>(p.ci, p.co, ptrs, [&](auto how) -> int {
        constexpr int HOW = decltype(how)::value;
        if (K > kXlStreamK) {
            if (!a.low) return fail(FEQ_ERR_INVALID, "no room for the reduced rows");
            const int64_t blocks = tile_bound(p.S, p.X, 16);
            if (blocks > INT32_MAX / kXlThreads) return fail(FEQ_ERR_UNSUPPORTED, "%lld blocks", (long long)blocks);
            auto low = k_ad_low<T, HOW, TRANS>;
            FEQ_LAUNCH(TRANS ? "k_ad_low_t" : "k_ad_low", low, dim3(blocks, dim), dim3(kXlThreads), 0, s, a, map);
            // blocks of 128 rows for fewer than half of the CUs: a call of 64 bfloat16 rows, 512 to 1024 columns, 15 us against 88
            if (ceil_div(p.S, kXlBM) * ceil_div(N, 128) * dim < 128) {
                auto few = k_ad_few<T, HOW, TRANS>;
                FEQ_LAUNCH(TRANS ? "k_ad_few_t" : "k_ad_few", few, dim3(ceil_div(N, 32), ceil_div(p.S, 16), dim), dim3(64), 0, s, a, map);
                return FEQ_OK;
            }
            auto tile = [&](auto wr) -> int {
                constexpr int WR = decltype(wr)::value;
                const int64_t tiles = xcd_grid(ceil_div(p.S, kXlBM), ceil_div(N, 64 * WR));
                if (tiles > INT32_MAX / kXlThreads) return fail(FEQ_ERR_UNSUPPORTED, "%lld blocks", (long long)tiles);
                auto kern = k_ad_mm<T, HOW, TRANS, WR>;
                FEQ_LAUNCH(TRANS ? "k_ad_mm_t" : "k_ad_mm", kern, dim3(tiles, dim), dim3(kXlThreads), 0, s, a, map);
                return FEQ_OK;
            };
            if (N <= 64) return tile(std::integral_constant<int, 1>{});
            if constexpr (HOW == kNarrow) return FEQ_ERR_INVALID;              // N is narrow
            else return tile(std::integral_constant<int, 2>{});
        }
        auto stream_rt = [&](auto nn, auto ns, auto rts) -> int {
            constexpr int NB = decltype(nn)::value, NS = decltype(ns)::value;
            using M = Mma<T>;
            constexpr int V = 16 / sizeof(T), KM = NS * M::KS, LD = KM + V, LDT = NB + M::PAD;
            const int rp = 16 * a.rt;
            const size_t lds = sizeof(T) * ((TRANS ? KM * LDT : NB * LD) + (TRANS ? KM * (rp + M::PAD) : rp * LD) +
                                            (TRANS ? rp * LDT : NB * (rp + 4))) + sizeof(float) * NB;
            auto kern = k_ad_stream<T, HOW, TRANS, NB, NS, decltype(rts)::value>;
            const int fit = static_cast<int>(std::min<size_t>(163840 / lds, 4));
            const int64_t blocks = std::min<int64_t>(256 * fit, tile_bound(p.S, p.X, 16) * dim * ceil_div(N, NB));
            if (lds > 65536)
                FEQ_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
            FEQ_LAUNCH(TRANS ? "k_ad_stream_t" : "k_ad_stream", kern, dim3(blocks), dim3(kXlThreads), lds, s, a, map);
            return FEQ_OK;
        };
        auto stream = [&](auto nn, auto ns) -> int {
            if (a.rt == 1) return stream_rt(nn, ns, std::integral_constant<int, 1>{});
            return stream_rt(nn, ns, std::integral_constant<int, kAdMaxRank / 16>{});
        };
        constexpr int H = 64 / Mma<T>::KS;
        auto with_ns = [&](auto nn) -> int {
            if (K <= 64) return stream(nn, std::integral_constant<int, H>{});
            if constexpr (HOW == kNarrow && decltype(nn)::value > 32) return FEQ_ERR_INVALID;
            else return stream(nn, std::integral_constant<int, 2 * H>{});
        };
        if (N <= 32) return with_ns(std::integral_constant<int, 32>{});
        if (N <= 64) return with_ns(std::integral_constant<int, 64>{});
        return with_ns(std::integral_constant<int, 128>{});
    });
}

// grad_down (UP false: v = x) or grad_up (v = grad_y).
template <class T, bool UP>
int ad_sums(const AdShape& p, const XlMap& map, const void* v, const float* z, const int32_t* offsets, const int32_t* order,
            void* out, float* parts, hipStream_t s) {
    const int C = UP ? p.co : p.ci;
    XlChunks ch;
    const int64_t nslots = wgrad_chunks(p.S, p.X, p.lvals, p.nreps, C, p.R, &ch);
    return with_rows<T>(C, C, {v}, [&](auto how) -> int {
        constexpr int HOW = decltype(how)::value;
        auto run = [&](auto bc) -> int {
            constexpr int BC = decltype(bc)::value;
            const int64_t blocks = ch.xcds * static_cast<int64_t>(ch.tile0[p.nreps]) * ceil_div(C, BC);
            if (blocks > INT32_MAX / kXlThreads) return fail(FEQ_ERR_UNSUPPORTED, "%lld blocks", (long long)blocks);
            auto kern = k_ad_sums<T, HOW, BC, UP>;
            FEQ_LAUNCH(UP ? "k_ad_sums_up" : "k_ad_sums", kern, dim3(blocks), dim3(kXlThreads), 0, s, static_cast<const T*>(v), z,
                       offsets, order, p.X, static_cast<int>(p.S), C, p.R, ad_tiles(p.R), p.nreps, map, ch, static_cast<T*>(out), parts);
            return FEQ_OK;
        };
        int rc;
        if (C <= 64) rc = run(std::integral_constant<int, 64>{});
        else if constexpr (HOW == kNarrow) rc = FEQ_ERR_INVALID;
        else rc = run(std::integral_constant<int, 128>{});
        if (rc || nslots == 0) return rc;
        const int64_t size = static_cast<int64_t>(C) * p.R;
        int least = ch.rows[0];
        for (int r = 1; r < p.nreps; ++r) least = std::min(least, static_cast<int>(ch.rows[r]));
        const int64_t many = std::min<int64_t>(p.X, p.S / least);
        auto sum = [&](auto split) -> int {
            constexpr bool SPLIT = decltype(split)::value;
            auto kern = k_xl_wsum<T, 1, SPLIT>;
            const int64_t blocks = std::min<int64_t>(ceil_div(size, SPLIT ? 64 : 256), 1 << 20);
            FEQ_LAUNCH("k_xl_wsum", kern, dim3(blocks, many, p.nreps), dim3(256), 0, s, parts, static_cast<const float*>(nullptr),
                       offsets, p.X, ch, size, p.co, p.nreps, static_cast<T*>(out), static_cast<T*>(nullptr), 0);
            return FEQ_OK;
        };
        return p.S / least > 8 * p.X ? sum(std::true_type{}) : sum(std::false_type{});
    });
}

struct AdScratch {
    float *low, *parts_down, *parts_up;
    int32_t* all;
    void* shared;
    size_t shared_bytes;
};
// Of a backward: the reduced gradient rows, the partial sums, the shared map's.
size_t ad_scratch(const AdShape& p, int dim, bool shared, int nbias, void* base, AdScratch* out) {
    Carver c(base);
    XlChunks ch;
    if (adapter_fused(p.ci, p.co, p.R)) {
        out->low = out->parts_up = nullptr;
        out->parts_down = c.take<float>(static_cast<size_t>(fused_chunks(p, &ch)) * p.R * (p.ci + p.co));
    } else {
        out->low = c.take<float>(static_cast<size_t>(dim) * p.S * 16 * ad_tiles(p.R));
        out->parts_down = c.take<float>(static_cast<size_t>(wgrad_chunks(p.S, p.X, p.lvals, p.nreps, p.ci, p.R, &ch)) * p.ci * p.R);
        out->parts_up = c.take<float>(static_cast<size_t>(wgrad_chunks(p.S, p.X, p.lvals, p.nreps, p.co, p.R, &ch)) * p.co * p.R);
    }
    out->all = c.take<int32_t>(2);
    out->shared_bytes = shared ? feq_expert_linear_bwd_workspace(p.lvals, p.nreps, 1, p.S, p.ci, p.co, nbias) : 0;
    out->shared = c.take<char>(out->shared_bytes);
    return c.used;
}

}  // namespace
}  // namespace feq

using namespace feq;

extern "C" int feq_adapter_linear_fwd(const int32_t* lvals, int32_t nreps, int32_t adapters, int64_t rows, int32_t cin, int32_t cout,
                                      int32_t rank, int32_t dtype, const void* x, const void* weight, const void* down,
                                      const void* up, float scale, const int32_t* order, const int32_t* offsets,
                                      const void* bias, int32_t nbias, const int32_t* bias_cols, void* y, float* low,
                                      feq_stream_t stream) {
    XlMap map;
    const AdShape p{lvals, nreps, adapters, rows, cin, cout, rank, dtype};
    if (int rc = ad_check(p, bias ? bias_cols : nullptr, nbias, scale, &map)) return rc;
    if (bias && (!bias_cols || nbias < 1)) return fail(FEQ_ERR_INVALID, "a bias needs bias columns");
    if (rows == 0) return FEQ_OK;
    if (!x || !weight || !down || !up || !order || !offsets || !y) return fail(FEQ_ERR_INVALID, "NULL pointer");
    return with_dtype(dtype, [&](auto t) -> int {
        AdArgs a{x, weight, down, up, bias, offsets, order, y, low};
        a.nbias = nbias;
        a.scale = scale;
        return ad_run<decltype(t), false>(p, map, a, {x, weight, down, y}, stream_of(stream));
    });
}

extern "C" size_t feq_adapter_linear_low_floats(const int32_t* lvals, int32_t nreps, int64_t rows, int32_t cin, int32_t cout, int32_t rank,
                                                int32_t train) {
    if (!lvals || nreps < 1 || nreps > kXlMaxReps || rows < 1 || cin < 1 || cout < 1 || rank < 1 || rank > kAdMaxRank) return 0;
    int64_t dim = 0;
    for (int r = 0; r < nreps; ++r) {
        if (lvals[r] < 0 || lvals[r] > kXlMaxPlanes) return 0;
        dim += 2 * lvals[r] + 1;
    }
    if (cin <= kXlStreamK && (!train || adapter_fused(cin, cout, rank))) return 0;
    return static_cast<size_t>(dim) * rows * 16 * ad_tiles(rank);
}

extern "C" size_t feq_adapter_linear_bwd_workspace(const int32_t* lvals, int32_t nreps, int32_t adapters, int64_t rows, int32_t cin,
                                                   int32_t cout, int32_t rank, int32_t dtype, int32_t shared, int32_t nbias) {
    XlMap map;
    const AdShape p{lvals, nreps, adapters, rows, cin, cout, rank, dtype};
    if (ad_check(p, nullptr, 0, 1.0f, &map) || rows == 0 || nbias < 0) return 0;
    AdScratch s;
    return ad_scratch(p, map.first[nreps], shared, nbias, nullptr, &s);
}

extern "C" int feq_adapter_linear_bwd(const int32_t* lvals, int32_t nreps, int32_t adapters, int64_t rows, int32_t cin, int32_t cout,
                                      int32_t rank, int32_t dtype, const void* grad_y, const void* x, const void* weight,
                                      const void* down, const void* up, float scale, const int32_t* order,
                                      const int32_t* offsets, const float* low, int32_t nbias, const int32_t* bias_cols,
                                      void* grad_x, void* grad_down, void* grad_up, void* grad_weight, void* grad_bias,
                                      void* workspace, size_t ws_bytes, feq_stream_t stream) {
    XlMap map;
    const AdShape p{lvals, nreps, adapters, rows, cin, cout, rank, dtype};
    if (int rc = ad_check(p, grad_bias ? bias_cols : nullptr, nbias, scale, &map)) return rc;
    if (rows == 0) return fail(FEQ_ERR_INVALID, "no rows");
    if (!grad_y || !x || !weight || !down || !up || !order || !offsets) return fail(FEQ_ERR_INVALID, "NULL pointer");
    const bool fused = adapter_fused(cin, cout, rank);
    if (grad_up && !low && !fused) return fail(FEQ_ERR_INVALID, "the gradient of up needs the forward's reduced rows");
    if ((grad_down || grad_up) && !grad_x) return fail(FEQ_ERR_INVALID, "the adapters' gradients come with that of x");
    if (grad_bias && (!grad_weight || !bias_cols || nbias < 1)) return fail(FEQ_ERR_INVALID, "a bias gradient needs bias columns and comes with the weight's");
    AdScratch w;
    const size_t need = ad_scratch(p, map.first[nreps], grad_weight, grad_bias ? nbias : 0, workspace, &w);
    if (ws_bytes < need) return fail(FEQ_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", ws_bytes, need);
    if (!workspace) return fail(FEQ_ERR_INVALID, "NULL pointer");
    hipStream_t s = stream_of(stream);
    const int rc = with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (grad_x) {
            AdArgs a{grad_y, weight, up, down, nullptr, offsets, order, grad_x, w.low};
            a.scale = scale;
            if (fused && (grad_down || grad_up)) return adapter_bwd_fused(lvals, nreps, adapters, rows, cin, cout, rank, dtype, a, x, grad_down, grad_up, w.parts_down, s);
            if (int err = ad_run<T, true>(p, map, a, {grad_y, weight, down, grad_x}, s)) return err;
        }
        if (grad_down)
            if (int err = ad_sums<T, false>(p, map, x, w.low, offsets, order, grad_down, w.parts_down, s)) return err;
        if (grad_up)
            if (int err = ad_sums<T, true>(p, map, grad_y, low, offsets, order, grad_up, w.parts_up, s)) return err;
        return FEQ_OK;
    });
    if (rc || !grad_weight) return rc;
    auto all = k_ad_all;
    FEQ_LAUNCH("k_ad_all", all, dim3(1), dim3(64), 0, s, w.all, static_cast<int>(rows));
    return feq_expert_linear_bwd_w(lvals, nreps, 1, rows, cin, cout, dtype, grad_y, x, w.all, grad_bias ? nbias : 0, bias_cols,
                                   grad_weight, grad_bias, w.shared, w.shared_bytes, stream);
}
