// The backward of the adapters (adapter_linear.hip) in one pass over the rows, for narrow maps.
#include "adapter_tiles.h"

namespace feq {
namespace {

// grad_x, grad_down and grad_up in one pass over grad_y and x: channels of at most 128 both ways and ranks of at most 16.  A
// workgroup takes a chunk of rows of one adapter (or of none) and one irrep, all its planes, as k_xl_wgrad; the shared map
// and the adapter's stay in LDS, and a wave takes 16 rows at a time straight from memory in the matrix cores' layout, the next
// ones in flight meanwhile.  Both reduced rows are formed here: u as in k_ad_stream for grad_x, and again with the operands
// exchanged, which leaves lane (c, g) rank c of rows 4 g .. 4 g + 3, the first operand of the sums over rows; t likewise.  Their
// second operands are columns of x and grad_y: the wave writes its rows to LDS, 64 columns at a time, and reads them
// transposed.  16-bit types take a reduced row as two numbers, as in k_ad_stream, so 16 rows fill a product.  The waves' sums
// are added at the chunk's end.
//
// 20011 x 49 bfloat16 rows of 128 columns both ways, 16 adapters of rank 16: 195 us, 3.9 TB/s, where grad_x and the two
// sums in kernels of their own took 410; float32, 20000 x 9 rows of 64 to 128: 88 us, memory's 37 and the products' 41 overlapped
// in part.
template <class T, int NB, int KB>
constexpr size_t kAdBwdLds =
    sizeof(T) * (KB * (NB + Mma<T>::PAD) + KB * (16 + Mma<T>::PAD) + 16 * (NB + Mma<T>::PAD) + 16 * (NB + 16 / sizeof(T)) + 4 * 16 * (64 + Mma<T>::PAD));

template <class T, int HOW, int NB, int KB>
__global__ void __launch_bounds__(kXlThreads, (2 * kAdBwdLds<T, NB, KB> <= 163840 ? 2 : 1))
k_ad_bwd(AdArgs a, const T* __restrict__ x, XlMap map, XlChunks ch, T* __restrict__ gdown, T* __restrict__ gup,
         float* __restrict__ parts) {
    using M = Mma<T>;
    typedef typename M::frag frag;
    constexpr bool F16 = std::is_same<T, _Float16>::value;
    constexpr int V = 16 / sizeof(T);
    constexpr int NT = NB / 16, KT = KB / 16, NA = NT < 4 ? NT : 4, NSK = KB / M::KS, NSX = NB / M::KS;
    constexpr int LDT = NB + M::PAD, LDF = 16 + M::PAD, LDX = NB + V, LC = 64 + M::PAD;
    const int K = a.K, N = a.N, X = a.X, S = a.S, R = a.R, nreps = a.nreps;
    extern __shared__ __align__(16) char smem[];
    T* sW = reinterpret_cast<T*>(smem);              // W as it lies (co, ci), its columns dealt
    T* sF = sW + KB * LDT;                           // up (co, R)
    T* sG = sF + KB * LDF;                           // down (R, ci), its columns dealt
    T* sD = sG + 16 * LDT;                           // down (R, ci)
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    T* buf = sD + 16 * LDX + wave * 16 * LC;
    const int xcds = ch.xcds, block = blockIdx.x / xcds;
    int rep = nreps - 1;                             // the irreps of most planes first
    while (rep > 0 && block >= ch.tile0[rep - 1]) --rep;
    const int rc = ch.rows[rep];
    const XlTile t = XlBlocks<true>(a.offsets, X, S, rc).find((block - ch.tile0[rep]) * xcds + blockIdx.x % xcds);
    if (t.expert < 0) return;
    const bool own = t.expert < X;                   // uniform
    const int rows = t.row1 - t.row0 < rc ? t.row1 - t.row0 : rc;
    const int d0 = __builtin_amdgcn_readfirstlane(map.first[rep]), d1 = __builtin_amdgcn_readfirstlane(map.first[rep + 1]);
    const int steps = (rows + 15) / 16, total = steps * (d1 - d0);
    const T *gy = static_cast<const T*>(a.in), *W = static_cast<const T*>(a.W);

    auto number = [&](int it) {                      // the row at this lane's place, -1: none
        const int i = it < total ? it % steps * 16 + c : rows;
        return i < rows ? a.order[t.row0 + i] : -1;
    };
    uint4 vg[NSK], vx[NSX];                          // in flight
    auto load = [&](int it, int at) {
        const int64_t i = static_cast<int64_t>(it < total ? d0 + it / steps : d0) * S + (at < 0 ? 0 : at);
#pragma unroll
        for (int ks = 0; ks < NSK; ++ks) {
            const int k = ks * M::KS + M::FE * g;
            vg[ks] = load_row<T, HOW>(gy + i * K, k, at < 0 ? 0 : K - k, gy);
        }
#pragma unroll
        for (int ks = 0; ks < NSX; ++ks) {
            const int k = ks * M::KS + M::FE * g;
            vx[ks] = load_row<T, HOW>(x + i * N, k, at < 0 || !own ? 0 : N - k, x);
        }
    };
    int row = number(wave), next = number(wave + 4);
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
    // sums += z^T r for reduced rows z and the wave's rows r
    auto add = [&](v4f z, const auto& r, auto& sums, int& power, bool& have) {
        constexpr int TILES = sizeof(sums) / sizeof(v4f), PIECE = TILES < 4 ? TILES : 4;
        if constexpr (F16) {                         // the sums' power follows the largest reduced value so far
            float most = 0.0f;
#pragma unroll
            for (int m = 0; m < 4; ++m) most = fmaxf(most, fabsf(z[m]));
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
            for (int m = 0; m < 4; ++m) z[m] = times_power(z[m], power);
        }
        const frag f = low_frag(z, T{});
#pragma unroll
        for (int i0 = 0; i0 < TILES; i0 += PIECE) {
#pragma unroll
            for (int k = 0; k < 16 * PIECE; k += M::KS)
                *reinterpret_cast<frag*>(buf + c * LC + k + M::FE * g) = r[(16 * i0 + k) / M::KS];
            wave_lds();
#pragma unroll
            for (int i = 0; i < PIECE; ++i) {
                frag b;
                if constexpr (sizeof(T) == 4) {
                    b = M::columns(buf, LC, 0, g, c, 16 * i);
                } else {
                    const v4s w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(buf + (4 * g + (c >> 2)) * LC + 16 * i + 4 * (c & 3)));
                    const v8s v = {w[0], w[1], w[2], w[3], w[0], w[1], w[2], w[3]};
                    b = __builtin_bit_cast(frag, v);
                }
                sums[i0 + i] = M::mul(f, b, sums[i0 + i]);
            }
            wave_lds();
        }
    };
    for (int it = wave; it < total; it += 4) {
        frag gf[NSK], xf[NSX];
#pragma unroll
        for (int ks = 0; ks < NSK; ++ks)
            gf[ks] = __builtin_bit_cast(frag, placed_row<T, HOW>(vg[ks], row < 0 ? 0 : K - ks * M::KS - M::FE * g, K, gy));
#pragma unroll
        for (int ks = 0; ks < NSX; ++ks)
            xf[ks] = __builtin_bit_cast(frag, placed_row<T, HOW>(vx[ks], row < 0 || !own ? 0 : N - ks * M::KS - M::FE * g, N, x));
        const int after = number(it + 8);
        load(it + 4, next);
        asm volatile("" ::: "memory");               // the maps are read from LDS for every step
        v4f acc[NT], low = v4f{0.0f, 0.0f, 0.0f, 0.0f}, u = low, v = low;
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < NSK; ++ks)
#pragma unroll
            for (int i0 = 0; i0 < NT; i0 += NA) {
                frag f[NA];
#pragma unroll
                for (int i = 0; i < NA; ++i) f[i] = M::columns(sW, LDT, ks * M::KS, g, c, 16 * (i0 + i));
                M::template mul_all<NA>(f, gf[ks], acc + i0);
            }
        if (own) {
#pragma unroll
            for (int ks = 0; ks < NSK; ++ks) {
                const frag f = M::columns(sF, LDF, ks * M::KS, g, c, 0);
                low = M::mul(f, gf[ks], low);
                u = M::mul(gf[ks], f, u);
            }
#pragma unroll
            for (int ks = 0; ks < NSX; ++ks)
                v = M::mul(xf[ks], *reinterpret_cast<const frag*>(sD + c * LDX + ks * M::KS + M::FE * g), v);
            low *= a.scale;
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
        if (row >= 0) {
            T* o = static_cast<T*>(a.out) + (static_cast<int64_t>(d0 + it / steps) * S + row) * N;
#pragma unroll
            for (int i = 0; i < NT; i += kDealt<T>) {
                const int n = 16 * i + V * g;
                store_tiles<T, HOW, 1>(o + n, N - n, &acc[i]);
            }
        }
        if (own) {
            add(u * a.scale, xf, ga, pa, have_a);
            add(v * a.scale, gf, gb, pb, have_b);
        }
        row = next;
        next = after;
    }
    if (!own) return;
    __syncthreads();                                 // the maps have been read
    constexpr int LP = NB + KB;
    float* sum = reinterpret_cast<float*>(smem) + wave * 16 * LP;
#pragma unroll
    for (int i = 0; i < NT + KT; ++i) {
        const v4f s = i < NT ? ga[i < NT ? i : 0] : gb[i < NT ? 0 : i - NT];
#pragma unroll
        for (int m = 0; m < 4; ++m) sum[(4 * g + m) * LP + 16 * i + c] = F16 ? times_power(s[m], -(i < NT ? pa : pb)) : s[m];
    }
    __syncthreads();
    const float* sums = reinterpret_cast<const float*>(smem);
    const bool direct = t.count == 1;
    const int64_t slot = ch.slot0[rep] + t.before + t.index, one = static_cast<int64_t>(t.expert) * nreps + rep;
    for (int i = tid; i < R * (N + K); i += kXlThreads) {
        const bool up = i >= R * N;                  // grad_down (R, ci), then grad_up (co, R)
        const int j = up ? i - R * N : i, q = up ? j % R : j / N, k = up ? j / R : j % N;
        const float* p = sums + q * LP + (up ? NB + k : k);
        const float s = p[0] + p[16 * LP] + p[32 * LP] + p[48 * LP];
        if (!direct) parts[slot * R * (N + K) + i] = s;
        else if (up && gup) gup[one * R * K + j] = static_cast<T>(s);
        else if (!up && gdown) gdown[one * R * N + j] = static_cast<T>(s);
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
    const int64_t nslots = fused_chunks(p, &ch);
    const int64_t blocks = ch.xcds * static_cast<int64_t>(ch.tile0[p.nreps]);
    if (blocks > INT32_MAX / kXlThreads) return fail(FEQ_ERR_UNSUPPORTED, "%lld blocks", (long long)blocks);
    return with_rows<T>(p.ci, p.co, {a.in, x, a.W, a.G, a.out}, [&](auto how) -> int {
        constexpr int HOW = decltype(how)::value;
        auto run = [&](auto nn, auto kk) -> int {
            constexpr int NB = decltype(nn)::value, KB = decltype(kk)::value;
            constexpr size_t lds = std::max(kAdBwdLds<T, NB, KB>, sizeof(float) * 64 * (NB + KB));       // the maps and rows, or the sums
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
