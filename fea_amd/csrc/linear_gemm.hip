// The fp32 products of the many-class loss heads on the exact fp32 matrix rate, any alignment, and the choice of a product's kernel.
//
//   z[m][n] = (sum_k a[m][k] b[n][k] + bias[n]) / T
//   LIN_LSE:   per row and column tile (max, sum exp(z - max)); z itself is stored, in fp32, where the caller keeps it for the backward
//   LIN_DZ:    q = exp(z - lse_m), stored row-major; the label's entries are corrected behind it.  The upstream gradient is not in it: in the
//              bf16 form a common factor would round the labels' entries, all close to it, the same way in every row (2,048 rows:
//              3.2e-3 off in dw and dh instead of 1.8e-3)
//   LIN_STORE: out = scale * (a . b), or fp32 slabs of a split reduction (joined by the caller in split order: no atomics)
//
// 128 x 128 tile, 4 waves of 64 x 64 (2 x 2 accumulators of 32 x 32), reduction in steps of 32 channels, two LDS stages filled through
// registers, two steps ahead, so that rows, columns and reduction of any length are cut by a guard on the load.  The operands
// of the MFMA are swapped (classes as its rows), so a lane holds one label row and 32 of its classes: the softmax sums are
// in-lane sums and one exchange between wave halves.  An operand with its rows along the reduction keeps them in LDS, and a
// fragment is four reads down a column.
// Bound by the fp32 matrix rate: 1,531 x 643 x 10,007 takes 204 us (96 TFLOP/s), as planes (linear_gemm256.hip) 120 us and 19 us of copies;
// this kernel serves what the planes' copies do not pay for: with 2 rows x 1,472 x 119,936 the products take 180 to 220 us each, bound
// by the weight's bytes (706 MB), as planes 400 us and 290 us of copies.
#include "linear_loss.h"

static constexpr int LG_T = 128, LG_CK = 32;

// TM: label rows of a tile, 128 or, for 64 rows and less in all, 64 with the four waves along the classes (64 x 32 each)
template <int EPI, bool ALN, bool TA, int TM>
__global__ __launch_bounds__(256, 2) void lin_gemm_kernel(const LinGemm g) {
    constexpr bool TB = EPI == LIN_STORE;
    constexpr int WM = TM / 64, WN = 4 / WM, NJ = 4 / WN, WC = 32 * NJ, LG_STAGE = (TM + LG_T) * 128;      // waves along labels and classes, class tiles and classes of a wave
    __shared__ __attribute__((aligned(128))) char smem[2 * LG_STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = WM == 2 ? wave & 1 : 0, wn = WM == 2 ? wave >> 1 : wave, l32 = lane & 31, hf = lane >> 5;
    // consecutive tiles of an XCD share the class tile and walk the label rows: the larger operand is read once
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int tm = id % g.ntm, rest = id / g.ntm, tn = rest % g.ntn, sp = rest / g.ntn;
    const int m0 = tm * TM, n0 = tn * LG_T;
    const int k0 = EPI == LIN_STORE ? sp * g.kper : 0, k1 = EPI == LIN_STORE ? min(k0 + g.kper, g.K) : g.K;

    // staging.  Rows along the tile: thread -> rows r + 32 i, 16-byte chunk c of 128 bytes, XOR-swizzled by the row.  Rows along the reduction:
    // thread -> rows of 32, 4 columns each, columns XORed so that the two halves of a wave read different banks.
    const int r = tid >> 3, c = tid & 7;
    const float *const ap = (const float*)g.a, *const bp = (const float*)g.b;
    u32x4 ra[2][TM / 32], rb[2][4];          // two steps on the way: the first is needed a whole step after it was asked for
    auto fetch1 = [&](const float* p, long long ld, int x0, int X, int k, int i, bool t, int W) {      // W: rows of the tile
        const int kr = k + tid / (W / 4) + 1024 / W * i, x = x0 + tid % (W / 4) * 4;
        if (t) return kr < k1 ? lin_load16<float, ALN>(p + kr * ld + x, X - x) : u32x4{0, 0, 0, 0};
        return x0 + r + 32 * i < X ? lin_load16<float, ALN>(p + (x0 + r + 32 * i) * ld + k + 4 * c, k1 - k - 4 * c) : u32x4{0, 0, 0, 0};
    };
    auto fetch = [&](int u, int k) {
#pragma unroll
        for (int i = 0; i < TM / 32; ++i) ra[u][i] = fetch1(ap, g.lda, m0, g.M, k, i, TA, TM);
#pragma unroll
        for (int i = 0; i < 4; ++i) rb[u][i] = fetch1(bp, g.ldb, n0, g.N, k, i, TB, LG_T);
    };
    auto put1 = [&](char* op, const u32x4& v, int i, bool t, int W) {
        const int row = t ? tid / (W / 4) + 1024 / W * i : r + 32 * i;
        *reinterpret_cast<u32x4*>(op + (t ? row * 4 * W + ((tid % (W / 4) ^ (((row >> 2) & 1) << 3)) << 4) : row * 128 + ((c ^ (row & 7)) << 4))) = v;
    };
    // fragment of 32 rows from x: lane l32 -> row, channels 8 s + 4 hf .. + 3
    auto frag = [&](const char* op, int x, int s, bool t, int W) {
        if (!t) return *reinterpret_cast<const u32x4*>(op + (x + l32) * 128 + (((2 * s + hf) ^ (l32 & 7)) << 4));
        const uint32_t* p = reinterpret_cast<const uint32_t*>(op) + (8 * s + 4 * hf) * W + ((x + l32) ^ (hf << 5));
        return u32x4{p[0], p[W], p[2 * W], p[3 * W]};
    };
    f32x16 acc[2][NJ];                 // [label tile][class tile]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    if (k0 < k1) fetch(0, k0);
    if (k0 + LG_CK < k1) fetch(1, k0 + LG_CK);
    const int live = g.M - m0 - __builtin_amdgcn_readfirstlane(wm) * 64;        // of few rows only the half or quarter that holds them is computed
    auto step = [&](int st, int k) {   // stage and register set of the same parity
        char* const sa = smem + st * LG_STAGE;
        char* const sb = sa + TM * 128;
#pragma unroll
        for (int i = 0; i < TM / 32; ++i) put1(sa, ra[st][i], i, TA, TM);
#pragma unroll
        for (int i = 0; i < 4; ++i) put1(sb, rb[st][i], i, TB, LG_T);
        __syncthreads();              // one barrier per step: the other stage was last read in front of the previous one
        if (k + 2 * LG_CK < k1) fetch(st, k + 2 * LG_CK);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            u32x4 b[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j) b[j] = frag(sb, wn * WC + j * 32, s, TB, LG_T);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (32 * i >= live) break;
                const u32x4 a = frag(sa, wm * 64 + i * 32, s, TA, TM);
#pragma unroll
                for (int j = 0; j < NJ; ++j) mma16(acc[i][j], b[j], a, (const float*)nullptr);
            }
        }
    };
    for (int k = k0; k < k1; k += 2 * LG_CK) {
        step(0, k);
        if (k + LG_CK < k1) step(1, k + LG_CK);
    }
    __syncthreads();

    // lane: label row mrow(i), register e of class tile j: class ncol(j, e)
    auto mrow = [&](int i) { return m0 + wm * 64 + i * 32 + l32; };
    auto ncol = [&](int j, int e) { return n0 + wn * WC + j * 32 + 8 * (e >> 2) + 4 * hf + (e & 3); };

    if constexpr (EPI == LIN_STORE) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int m = mrow(i);
            if (m >= g.M) continue;
            const float sc = g.scale == 1 ? lin_row_scale(g.gout, g.gstride, g.count, g.t, g.stat[m].y, m)
                           : g.scale == 2 ? lin_row_scale(g.gout, 0, g.count, g.t, 1.f, 0) : 1.f;
            float* const o = g.slab ? g.slab + ((long long)sp * g.M + m) * g.ldo : (float*)g.out + m * g.ldo;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const int n = ncol(j, e);         // (rows of the output are whole 16 bytes)
                    if (n < g.N) *reinterpret_cast<f32x4*>(o + n) = f32x4{acc[i][j][e] * sc, acc[i][j][e + 1] * sc, acc[i][j][e + 2] * sc, acc[i][j][e + 3] * sc};
                }
        }
        return;
    }

    // z in place; classes behind the last are -inf
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int n = ncol(j, e);
            const float b = g.bias && n < g.N ? g.bias[n] : 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) acc[i][j][e] = n < g.N ? (acc[i][j][e] + b) * g.inv_t : -INFINITY;
        }

    if constexpr (EPI == LIN_LSE) {
        float2* const red = reinterpret_cast<float2*>(smem);       // [wn][rows]
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, acc[i][j][e]);
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float base = mx == -INFINITY ? 0.f : mx;         // every class masked by a -inf bias: the sum is 0, not NaN
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) sum += __expf(acc[i][j][e] - base);
            sum += __shfl_xor(sum, 32);
            if (hf == 0) red[wn * TM + wm * 64 + i * 32 + l32] = make_float2(mx, sum);
        }
        __syncthreads();
        if (tid < TM && m0 + tid < g.M) {
            float mx = red[tid].x, sum = 0.f;
#pragma unroll
            for (int w = 1; w < WN; ++w) mx = fmaxf(mx, red[w * TM + tid].x);
            const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
            for (int w = 0; w < WN; ++w) sum += red[w * TM + tid].y * __expf(red[w * TM + tid].x - base);
            g.part[(long long)(m0 + tid) * g.ntn + tn] = make_float2(mx, sum);
        }
        if (g.keep)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int m = mrow(i);
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const int n = ncol(j, e);
                        if (m < g.M && n < g.ldkeep) *reinterpret_cast<f32x4*>((float*)g.keep + m * g.ldkeep + n) = f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
                    }
            }
    }

    if constexpr (EPI == LIN_DZ) {
        float sc[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int m = mrow(i);
            const float2 st2 = m < g.M ? g.stat[m] : make_float2(0.f, 0.f);
            const bool dead = st2.y == 0.f;                        // the row does not count: 0 whatever its hidden state holds
            const float lse = st2.x;
            sc[i] = dead ? 0.f : lin_row_scale(g.gout, g.gstride, g.count, g.t, st2.y, m);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float q = __expf(acc[i][j][e] - lse);
                    acc[i][j][e] = dead || ncol(j, e) >= g.N ? 0.f : q;
                }
        }
        if (g.colsum) {
            float* const red = reinterpret_cast<float*>(smem);     // [wm][128 classes]
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float s = acc[0][j][e] * sc[0] + acc[1][j][e] * sc[1];
#pragma unroll
                    for (int d = 16; d; d >>= 1) s += __shfl_xor(s, d);
                    if (l32 == 0) red[wm * LG_T + ncol(j, e) - n0] = s;
                }
            __syncthreads();
            if (tid < LG_T && n0 + tid < g.N) g.colsum[tm * g.ldcol + n0 + tid] = WM == 2 ? red[tid] + red[LG_T + tid] : red[tid];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int m = mrow(i);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const int n = ncol(j, e);
                    if (m < g.M && n < g.Npad) *reinterpret_cast<f32x4*>((float*)g.dz + m * g.lddz + n) = f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
                }
        }
    }
}

// Tile and split of a product: the one whose modelled time is least, from the rates that the kernels reach on full chips (fp32 100, bf16 700
// and 1,300 TFLOP/s) and from the bytes of operands and result at 4 TB/s.  Both take whole rounds of the chip (256 workgroups of the large
// tile, 512 of the small one); the parts of a split reduction are written and read once more, at least 512 (bf16) or 256 (fp32)
// channels each.  Of up to 64 or 32 rows the fp32 kernel computes no more.  dtype FEA_PL: K is six times the planes'.
LinTile fea_lin_tile(int dtype, long long M, long long N, long long K, bool split) {
    LinTile best{128, 1, 1e30};
    const double size = dtype == FEA_F32 ? 4 : dtype == FEA_BF16 ? 2 : 1;      // bytes per element of K: a plane pair's share is 6 of 6 K
    const double bytes = ((double)M * K + (double)N * K) * size + (split ? (double)M * N * (dtype == FEA_BF16 ? 2 : 4) : 0.0);
    for (int tile = 128; tile <= (dtype == FEA_F32 ? 128 : 256); tile += 128) {
        const double slots = tile == 256 ? 256 : 512;
        const double rate = dtype == FEA_F32 ? 100e12 : tile == 256 ? 1300e12 : 700e12;
        const double rows = dtype == FEA_F32 && M <= 64 ? (M <= 32 ? 32 : 64) : tile;      // that are computed
        const long long tiles = ((M + tile - 1) / tile) * ((N + tile - 1) / tile);
        for (int sp = 1; sp <= (split ? 32 : 1); ++sp) {
            if (sp > 1 && K / sp < (dtype == FEA_F32 ? 256 : 512)) break;
            // (a workgroup of the small tile that has a CU to itself takes 0.6 of the time of two)
            const long long n = tiles * sp, full = n / (long long)slots, rest = n % (long long)slots;
            const double rounds = (double)full + (rest == 0 ? 0.0 : tile == 128 && rest <= 256 ? 0.6 : 1.0);
            double t = rounds * (2.0 * rows * tile * ((double)K / sp + 128) / (rate / slots));
            if (t < bytes / 4e12) t = bytes / 4e12;
            t += sp > 1 ? 2.0 * sp * M * N * 4 / 4e12 + 3e-6 : 0.0;
            if (t < best.time * 0.999) best = LinTile{tile, sp, t};
        }
    }
    return best;
}

template <int EPI, bool TA> static void lg_launch(const LinGemm& g, bool aln, unsigned grid, hipStream_t s) {
    if (g.M <= 64) {
        if (aln) hipLaunchKernelGGL((lin_gemm_kernel<EPI, true, TA, 64>), dim3(grid), dim3(256), 0, s, g);
        else     hipLaunchKernelGGL((lin_gemm_kernel<EPI, false, TA, 64>), dim3(grid), dim3(256), 0, s, g);
    } else {
        if (aln) hipLaunchKernelGGL((lin_gemm_kernel<EPI, true, TA, 128>), dim3(grid), dim3(256), 0, s, g);
        else     hipLaunchKernelGGL((lin_gemm_kernel<EPI, false, TA, 128>), dim3(grid), dim3(256), 0, s, g);
    }
}

int fea_lin_gemm(int epi, int dtype, int tile, LinGemm g, hipStream_t s) {
    const int epc = dtype == FEA_F32 ? 4 : 8;
    const bool aln = g.lda % epc == 0 && g.ldb % epc == 0 && ((uintptr_t)g.a | (uintptr_t)g.b) % 16 == 0 && (epi == LIN_STORE ? g.N % epc == 0 || dtype != FEA_F32 : g.K % epc == 0);
    const long long k = dtype == FEA_PL ? 3ll * g.Kp : g.K;
    FEA_CHECK(g.M > 0 && g.N > 0 && g.K > 0 && g.lda >= (epi == LIN_STORE && g.ta ? g.M : k) && g.ldb >= (epi == LIN_STORE ? g.N : k), FEA_E_BADARG,
              "lin_gemm: operands of %d x %d x %d", g.M, g.N, g.K);
    FEA_CHECK(dtype == FEA_F32 ? tile == 128 : aln && g.lda < (1 << 21) && g.ldb < (1 << 21), FEA_E_UNSUPPORTED_SHAPE, "lin_gemm: tile %d, strides %lld, %lld", tile, g.lda, g.ldb);
    FEA_CHECK(dtype != FEA_PL || (g.Kp > 0 && g.Kp % 64 == 0 && g.K == 6 * g.Kp && g.Kr <= g.Kp && (epi != LIN_STORE || g.slab)), FEA_E_BADARG, "lin_gemm: planes of %d, K %d", g.Kp, g.K);
    FEA_CHECK(epi != LIN_LSE || (g.slab != nullptr) == (g.splits > 1), FEA_E_BADARG, "lin_gemm: %d parts", g.splits);
    // what the stores take: whole 16 bytes of a row (slabs' rows are padded; gradients of other widths go through slabs)
    const int epo = g.slab || dtype == FEA_F32 ? 4 : 8;
    if (epi == LIN_STORE)
        FEA_CHECK((g.slab || g.N % epo == 0) && g.ldo >= g.N && g.ldo % epo == 0 && (uintptr_t)(g.slab ? (void*)g.slab : g.out) % 16 == 0, FEA_E_BADARG,
                  "lin_gemm: result of %d columns in rows of %lld", g.N, g.ldo);
    if (epi == LIN_DZ)
        FEA_CHECK(g.Npad >= g.N && g.Npad % 64 == 0 && g.lddz % 8 == 0 && (uintptr_t)g.dz % 16 == 0, FEA_E_BADARG, "lin_gemm: dz of %d columns in rows of %lld", g.Npad, g.lddz);
    FEA_CHECK(epi != LIN_STORE || dtype == FEA_F32 || (g.Kr > 0 && g.Kr <= (dtype == FEA_PL ? g.Kp : g.K)), FEA_E_BADARG, "lin_gemm: reduction of %d of %d", g.Kr, g.K);
    g.ntm = (g.M + tile - 1) / tile; g.ntn = (g.N + tile - 1) / tile;
    if (g.splits < 1) { g.splits = 1; g.kper = g.K; }
    const long long grid = (long long)g.ntm * g.ntn * g.splits;
    FEA_CHECK(grid > 0 && grid <= (1 << 23), FEA_E_UNSUPPORTED_SHAPE, "lin_gemm: %lld tiles", grid);
    if (dtype != FEA_F32) fea_lin_gemm256(epi, tile, dtype == FEA_PL, g, (unsigned)grid, s);
    else if (epi == LIN_LSE) lg_launch<LIN_LSE, false>(g, aln, (unsigned)grid, s);
    else if (epi == LIN_DZ)  lg_launch<LIN_DZ, false>(g, aln, (unsigned)grid, s);
    else if (g.ta)           lg_launch<LIN_STORE, true>(g, aln, (unsigned)grid, s);
    else                     lg_launch<LIN_STORE, false>(g, aln, (unsigned)grid, s);
    FEA_LAUNCH_CHECK();
    return FEA_OK;
}
