// The backward of the adapters (adapter_linear.hip) in one pass over the rows, for narrow maps.
#include "adapter_tiles.h"

namespace feq {
namespace {

// grad_x, grad_down and grad_up in one pass over grad_y and x: channels of at most 128 both ways and ranks of at most 16.  A
// workgroup takes a chunk of rows of one adapter (or of none) and one irrep, all its planes, as k_xl_wgrad; the shared map
// and the adapter's stay in LDS, and a wave takes RB rows at a time straight from memory in the matrix cores' layout, the next
// ones in flight meanwhile.  Both reduced rows are formed here: u as in k_ad_stream for grad_x, and again with the operands
// exchanged, which leaves lane (c, g) rank c of rows 4 g .. 4 g + 3, the first operand of the sums over rows; t likewise.  Their
// second operands are columns of x and grad_y: the wave writes its rows to LDS and reads them transposed.  16-bit types
// sum 32 rows a product: element j < 4 is row 4 g + j of the first 16, j >= 4 of the next.  The waves' sums are added at
// the chunk's end.
template <class T, int HOW, int NB, int KB>
__global__ void __launch_bounds__(kXlThreads, 1)
k_ad_bwd(AdArgs a, const T* __restrict__ x, XlMap map, XlChunks ch, T* __restrict__ gdown, T* __restrict__ gup,
         float* __restrict__ parts) {
    using M = Mma<T>;
    typedef typename M::frag frag;
    constexpr bool F16 = std::is_same<T, _Float16>::value;
    constexpr int V = 16 / sizeof(T), RT = sizeof(T) == 4 ? 1 : 2, RB = 16 * RT;      // row tiles and rows of a step
    constexpr int NT = NB / 16, KT = KB / 16, NA = NT < 4 ? NT : 4, NSK = KB / M::KS, NSX = NB / M::KS;
    constexpr int LDT = NB + M::PAD, LDF = 16 + M::PAD, LDX = NB + V, LC = (NB > KB ? NB : KB) + M::PAD;
    const int K = a.K, N = a.N, X = a.X, S = a.S, R = a.R, nreps = a.nreps;
    extern __shared__ __align__(16) char smem[];
    T* sW = reinterpret_cast<T*>(smem);              // W as it lies (co, ci), its columns dealt
    T* sF = sW + KB * LDT;                           // up (co, R)
    T* sG = sF + KB * LDF;                           // down (R, ci), its columns dealt
    T* sD = sG + 16 * LDT;                           // down (R, ci)
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    T* buf = sD + 16 * LDX + wave * RB * LC;
    const int xcds = ch.xcds, block = blockIdx.x / xcds;
    int rep = nreps - 1;                             // the irreps of most planes first
    while (rep > 0 && block >= ch.tile0[rep - 1]) --rep;
    const int rc = ch.rows[rep];
    const XlTile t = XlBlocks<true>(a.offsets, X, S, rc).find((block - ch.tile0[rep]) * xcds + blockIdx.x % xcds);
    if (t.expert < 0) return;
    const bool own = t.expert < X;                   // uniform
    const int rows = t.row1 - t.row0 < rc ? t.row1 - t.row0 : rc;
    const int d0 = __builtin_amdgcn_readfirstlane(map.first[rep]), d1 = __builtin_amdgcn_readfirstlane(map.first[rep + 1]);
    const int steps = (rows + RB - 1) / RB, total = steps * (d1 - d0);
    const T *gy = static_cast<const T*>(a.in), *W = static_cast<const T*>(a.W);

    auto number = [&](int it, int r) {               // row tile r's row at this lane's place, -1: none
        const int i = it < total ? it % steps * RB + 16 * r + c : rows;
        return i < rows ? a.order[t.row0 + i] : -1;
    };
    uint4 vg[RT][NSK], vx[RT][NSX];                  // in flight
    int row[RT], next[RT];
    auto load = [&](int it, const int (&at)[RT]) {
        const int d = it < total ? d0 + it / steps : d0;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int64_t i = static_cast<int64_t>(d) * S + (at[r] < 0 ? 0 : at[r]);
#pragma unroll
            for (int ks = 0; ks < NSK; ++ks) {
                const int k = ks * M::KS + M::FE * g;
                vg[r][ks] = load_row<T, HOW>(gy + i * K, k, at[r] < 0 ? 0 : K - k, gy);
            }
#pragma unroll
            for (int ks = 0; ks < NSX; ++ks) {
                const int k = ks * M::KS + M::FE * g;
                vx[r][ks] = load_row<T, HOW>(x + i * N, k, at[r] < 0 || !own ? 0 : N - k, x);
            }
        }
    };
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        row[r] = number(wave, r);
        next[r] = number(wave + 4, r);
    }
    load(wave, row);
    const T* wm = W + static_cast<int64_t>(rep) * K * N;
    const Rows we = rows_at(wm, W, N);
#pragma unroll
    for (int i = 0; i < KB * NB / V / kXlThreads; ++i) {
        const int q = tid + kXlThreads * i, k = q / (NB / V), n = (q % (NB / V)) * V;
        const int there = k < K ? N - n : 0;
        put_dealt<T>(sW + k * LDT, n, arrived16<T, HOW>(we, load16<T, HOW>(we, (k * N + n) * static_cast<int>(sizeof(T)), there), there));
    }
    if (own) {
        const int64_t map0 = (static_cast<int64_t>(t.expert) * nreps + rep) * R;
        const T *fe = static_cast<const T*>(a.F) + map0 * K, *ge = static_cast<const T*>(a.G) + map0 * N;
        for (int i = tid; i < 16 * KB; i += kXlThreads) {
            const int q = i % 16, k = i / 16;
            const bool there = q < R && k < K;
            const T v = fe[there ? k * R + q : 0];
            sF[k * LDF + q] = there ? v : static_cast<T>(0.0f);
        }
        for (int i = tid; i < 16 * NB; i += kXlThreads) {
            const int q = i / NB, n = i % NB;
            const bool there = q < R && n < N;
            const T v = ge[there ? q * N + n : 0];
            const T e = there ? v : static_cast<T>(0.0f);
            sG[q * LDT + dealt<T>(n)] = e;
            sD[q * LDX + n] = e;
        }
    }
    __syncthreads();
    v4f ga[NT], gb[KT];                              // grad_down, grad_up: ranks 4 g .. 4 g + 3 of column c of the tile
#pragma unroll
    for (int i = 0; i < NT; ++i) ga[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < KT; ++i) gb[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    int pa = 0, pb = 0;                              // the powers of two that float16's sums are multiplied by
    bool have_a = false, have_b = false;
    // columns of the wave's rows in `buf`
    auto columns = [&](int c0) -> frag {
        if constexpr (sizeof(T) == 4) {
            return M::columns(buf, LC, 0, g, c, c0);
        } else {
            const T* p = buf + (4 * g + (c >> 2)) * LC + c0 + 4 * (c & 3);
            const v4s u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p));
            const v4s w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p + 16 * LC));
            const v8s v = {u[0], u[1], u[2], u[3], w[0], w[1], w[2], w[3]};
            return __builtin_bit_cast(frag, v);
        }
    };
    // sums += z^T (columns of the rows in `buf`)
    auto add = [&](v4f (&z)[RT], auto& sums, int& power, bool& have) {
        constexpr int TILES = sizeof(sums) / sizeof(v4f);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < TILES; ++i) sums[i] = M::mul(z[0], columns(16 * i), sums[i]);
        } else {
            if constexpr (F16) {                     // the sums' power follows the largest reduced value so far
                float most = 0.0f;
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int m = 0; m < 4; ++m) most = fmaxf(most, fabsf(z[r][m]));
                most = group_max(most, 64);
                const int p = low_exponent(most);
                if (most > 0.0f && (!have || p < power)) {           // uniform
                    if (have)
#pragma unroll
                        for (int i = 0; i < TILES; ++i)
#pragma unroll
                            for (int m = 0; m < 4; ++m) sums[i][m] = times_power(sums[i][m], p - power);
                    power = p;
                    have = true;
                }
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int m = 0; m < 4; ++m) z[r][m] = times_power(z[r][m], power);
            }
            frag hi, lo;
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const float v = z[r % RT][m];
                    const T h = static_cast<T>(v);
                    hi[4 * r + m] = h;
                    lo[4 * r + m] = static_cast<T>(v - static_cast<float>(h));
                }
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                const frag b = columns(16 * i);
                sums[i] = M::mul(hi, b, sums[i]);
                sums[i] = M::mul(lo, b, sums[i]);
            }
        }
    };
    for (int it = wave; it < total; it += 4) {
        frag gf[RT][NSK], xf[RT][NSX];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
#pragma unroll
            for (int ks = 0; ks < NSK; ++ks)
                gf[r][ks] = __builtin_bit_cast(frag, placed_row<T, HOW>(vg[r][ks], row[r] < 0 ? 0 : K - ks * M::KS - M::FE * g, K, gy));
#pragma unroll
            for (int ks = 0; ks < NSX; ++ks)
                xf[r][ks] = __builtin_bit_cast(frag, placed_row<T, HOW>(vx[r][ks], row[r] < 0 || !own ? 0 : N - ks * M::KS - M::FE * g, N, x));
        }
        int after[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) after[r] = number(it + 8, r);
        load(it + 4, next);
        asm volatile("" ::: "memory");               // the maps are read from LDS for every step
        v4f u[RT], v[RT];
        T* od = static_cast<T*>(a.out) + static_cast<int64_t>(d0 + it / steps) * S * N;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            v4f acc[NT], low = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < NSK; ++ks)
#pragma unroll
                for (int i0 = 0; i0 < NT; i0 += NA) {
                    frag f[NA];
#pragma unroll
                    for (int i = 0; i < NA; ++i) f[i] = M::columns(sW, LDT, ks * M::KS, g, c, 16 * (i0 + i));
                    M::template mul_all<NA>(f, gf[r][ks], acc + i0);
                }
            if (own) {
                u[r] = v[r] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < NSK; ++ks) {
                    const frag f = M::columns(sF, LDF, ks * M::KS, g, c, 0);
                    low = M::mul(f, gf[r][ks], low);
                    u[r] = M::mul(gf[r][ks], f, u[r]);
                }
#pragma unroll
                for (int ks = 0; ks < NSX; ++ks)
                    v[r] = M::mul(xf[r][ks], *reinterpret_cast<const frag*>(sD + c * LDX + ks * M::KS + M::FE * g), v[r]);
                low *= a.scale;
                u[r] *= a.scale;
                v[r] *= a.scale;
                int power = 0;
                if constexpr (F16) {
                    float most = 0.0f;
#pragma unroll
                    for (int m = 0; m < 4; ++m) most = fmaxf(most, fabsf(low[m]));
                    power = low_exponent(row_max(most));
#pragma unroll
                    for (int m = 0; m < 4; ++m) low[m] = times_power(low[m], power);
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int m = 0; m < 4; ++m) acc[i][m] = times_power(acc[i][m], power);
                }
                const frag b = low_frag(low, T{});
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    T e[4];
                    if constexpr (sizeof(T) == 4) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) e[j] = sG[(4 * g + j) * LDT + 16 * i + c];
                    } else {
                        const v4s w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(sG + (4 * g + (c >> 2)) * LDT + 16 * i + 4 * (c & 3)));
#pragma unroll
                        for (int j = 0; j < 4; ++j) e[j] = __builtin_bit_cast(T, static_cast<short>(w[j]));
                    }
                    acc[i] = M::mul(twice<T>(e), b, acc[i]);
                }
                if constexpr (F16)
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int m = 0; m < 4; ++m) acc[i][m] = times_power(acc[i][m], -power);
            }
            if (row[r] >= 0) {
                T* o = od + static_cast<int64_t>(row[r]) * N;
#pragma unroll
                for (int i = 0; i < NT; i += kDealt<T>) {
                    const int n = 16 * i + V * g;
                    store_tiles<T, HOW, 1>(o + n, N - n, &acc[i]);
                }
            }
        }
        if (own) {
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int ks = 0; ks < NSX; ++ks) *reinterpret_cast<frag*>(buf + (16 * r + c) * LC + ks * M::KS + M::FE * g) = xf[r][ks];
            wave_lds();
            add(u, ga, pa, have_a);
            wave_lds();
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int ks = 0; ks < NSK; ++ks) *reinterpret_cast<frag*>(buf + (16 * r + c) * LC + ks * M::KS + M::FE * g) = gf[r][ks];
            wave_lds();
            add(v, gb, pb, have_b);
            wave_lds();
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            row[r] = next[r];
            next[r] = after[r];
        }
    }
    if (!own) return;
    __syncthreads();                                 // the maps have been read
    constexpr int LP = NB + KB;
    float* sum = reinterpret_cast<float*>(smem) + wave * 16 * LP;
#pragma unroll
    for (int i = 0; i < NT + KT; ++i) {
        const v4f v = i < NT ? ga[i < NT ? i : 0] : gb[i < NT ? 0 : i - NT];
#pragma unroll
        for (int m = 0; m < 4; ++m) sum[(4 * g + m) * LP + 16 * i + c] = F16 ? times_power(v[m], -(i < NT ? pa : pb)) : v[m];
    }
    __syncthreads();
    const float* sums = reinterpret_cast<const float*>(smem);
    const bool direct = t.count == 1;
    const int64_t slot = ch.slot0[rep] + t.before + t.index, one = static_cast<int64_t>(t.expert) * nreps + rep;
    for (int i = tid; i < R * (N + K); i += kXlThreads) {
        const bool up = i >= R * N;                  // grad_down (R, ci), then grad_up (co, R)
        const int j = up ? i - R * N : i, q = up ? j % R : j / N, k = up ? j / R : j % N;
        const float* p = sums + q * LP + (up ? NB + k : k);
        const float v = p[0] + p[16 * LP] + p[32 * LP] + p[48 * LP];
        if (!direct) parts[slot * R * (N + K) + i] = v;
        else if (up && gup) gup[one * R * K + j] = static_cast<T>(v);
        else if (!up && gdown) gdown[one * R * N + j] = static_cast<T>(v);
    }
}

// The sums of the adapters of several chunks of k_ad_bwd, in order: blockIdx.y the adapter's number among these,
// blockIdx.z the irrep; the four waves take a quarter of the chunks each.
template <class T>
__global__ void __launch_bounds__(256)
k_ad_parts(const float* __restrict__ parts, const int32_t* __restrict__ offsets, int X, XlChunks ch, int N, int K, int R, int nreps,
           T* __restrict__ gdown, T* __restrict__ gup) {
    __shared__ float part[3][64];
    const int rep = blockIdx.z, rc = ch.rows[rep], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const XlTile t = several_chunks(offsets, X, rc, blockIdx.y);
    if (t.expert < 0) return;
    const int size = R * (N + K);
    const int64_t one = static_cast<int64_t>(t.expert) * nreps + rep;
    for (int i0 = blockIdx.x * 64; i0 < size; i0 += gridDim.x * 64) {
        const int i = i0 + lane;
        const float* p = parts + static_cast<int64_t>(ch.slot0[rep] + t.before) * size + i;
        float s = 0.0f;
        if (i < size)
#pragma unroll 8
            for (int q = wave; q < t.count; q += 4) s += p[static_cast<int64_t>(q) * size];
        __syncthreads();                             // the last sums have been read
        if (wave) part[wave - 1][lane] = s;
        __syncthreads();
        if (wave || i >= size) continue;
        s += part[0][lane];
        s += part[1][lane];
        s += part[2][lane];
        if (i < R * N) {
            if (gdown) gdown[one * R * N + i] = static_cast<T>(s);
        } else if (gup) {
            gup[one * R * K + i - R * N] = static_cast<T>(s);
        }
    }
}

template <class T>
int run_bwd(const AdShape& p, const XlMap& map, AdArgs a, const void* x, void* gdown, void* gup, float* parts, hipStream_t s) {
    a.X = p.X;
    a.S = static_cast<int>(p.S);
    a.K = p.co;
    a.N = p.ci;
    a.R = p.R;
    a.nreps = p.nreps;
    a.dim = map.first[p.nreps];
    a.rt = 1;
    XlChunks ch;
    const int64_t nslots = wgrad_chunks(p.S, p.X, p.lvals, p.nreps, p.ci, p.co, &ch);
    const int64_t blocks = ch.xcds * static_cast<int64_t>(ch.tile0[p.nreps]);
    if (blocks > INT32_MAX / kXlThreads) return fail(FEQ_ERR_UNSUPPORTED, "%lld blocks", (long long)blocks);
    return with_rows<T>(p.ci, p.co, {a.in, x, a.W, a.G, a.out}, [&](auto how) -> int {
        constexpr int HOW = decltype(how)::value;
        auto run = [&](auto nn, auto kk) -> int {
            using M = Mma<T>;
            constexpr int NB = decltype(nn)::value, KB = decltype(kk)::value, V = 16 / sizeof(T), RB = sizeof(T) == 4 ? 16 : 32;
            constexpr size_t maps = KB * (NB + M::PAD) + KB * (16 + M::PAD) + 16 * (NB + M::PAD) + 16 * (NB + V);
            constexpr size_t lds = std::max(sizeof(T) * (maps + 4 * RB * (std::max(NB, KB) + M::PAD)), sizeof(float) * 64 * (NB + KB));
            auto kern = k_ad_bwd<T, HOW, NB, KB>;
            if (lds > 65536)
                FEQ_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
            FEQ_LAUNCH("k_ad_bwd", kern, dim3(blocks), dim3(kXlThreads), lds, s, a, static_cast<const T*>(x), map, ch,
                       static_cast<T*>(gdown), static_cast<T*>(gup), parts);
            if (nslots == 0) return FEQ_OK;
            int least = ch.rows[0];
            for (int r = 1; r < p.nreps; ++r) least = std::min(least, static_cast<int>(ch.rows[r]));
            const int64_t many = std::min<int64_t>(p.X, p.S / least);
            auto sum = k_ad_parts<T>;
            FEQ_LAUNCH("k_ad_parts", sum, dim3(ceil_div(p.R * (p.ci + p.co), 64), many, p.nreps), dim3(256), 0, s, parts, a.offsets, p.X, ch,
                       p.ci, p.co, p.R, p.nreps, static_cast<T*>(gdown), static_cast<T*>(gup));
            return FEQ_OK;
        };
        constexpr std::integral_constant<int, 32> c32{};
        constexpr std::integral_constant<int, 64> c64{};
        constexpr std::integral_constant<int, 128> c128{};
        auto with_k = [&](auto nn) -> int {
            if (p.co <= 64) return run(nn, c64);
            if constexpr (HOW == kNarrow && decltype(nn)::value > 32) return FEQ_ERR_INVALID;      // neither is narrow
            else return run(nn, c128);
        };
        if (p.ci <= 32) return with_k(c32);
        if (p.ci <= 64) return with_k(c64);
        return with_k(c128);
    });
}

}  // namespace

int adapter_bwd_fused(const int32_t* lvals, int32_t nreps, int32_t X, int64_t S, int32_t ci, int32_t co, int32_t R, int32_t dtype, AdArgs a,
                      const void* x, void* gdown, void* gup, float* parts, hipStream_t s) {
    XlMap map;
    const AdShape p{lvals, nreps, X, S, ci, co, R, dtype};
    if (int rc = xl_check(lvals, nreps, X, S, ci, co, dtype, nullptr, 0, &map)) return rc;
    return with_dtype(dtype, [&](auto t) -> int { return run_bwd<decltype(t)>(p, map, a, x, gdown, gup, parts, s); });
}

}  // namespace feq
