// Tiled product of the many-class loss heads with its three epilogues: log-sum-exp partials, softmax gradient, store.
//
//   z[m][n] = (sum_k a[m][k] b[n][k] + bias[n]) / T
//   LIN_LSE:   per row and column tile (max, sum exp(z - max)); no z leaves the registers
//   LIN_DZ:    q = exp(z - lse_m), rounded once to the storage type (it is the operand of the next two products on the
//              matrix pipe; the sums there are fp32), stored row-major and transposed so that both products find their
//              reduction axis contiguous.  The upstream gradient is not in it: a common factor rounds the labels' entries, all
//              close to it, the same way in every row (bf16, 2,048 rows: 3.2e-3 off in dw and dh instead of 2.3e-3)
//   LIN_STORE: out = scale * (a . b), or fp32 slabs of a split reduction (joined by the caller in split order: no atomics)
//
// 128 x 128 tile, 4 waves of 64 x 64 (2 x 2 accumulators of 32 x 32), reduction in 128-byte steps of every row (64 bf16 / 32 fp32),
// two LDS stages filled through registers, two steps ahead, so that rows, columns and reduction of any length are cut by a guard on the load.
// The operands of the MFMA are swapped (classes as its rows), so a lane holds one label row and 32 of its classes: the softmax
// sums are in-lane sums and one exchange between wave halves.
#include "linear_loss.h"

static constexpr int LG_T = 128, LG_STAGE = 2 * LG_T * 128;

template <typename T> __device__ __forceinline__ void lg_store4(T* p, const float (&v)[4], int n) {
    if (n >= 4 && (((uintptr_t)p) & (4 * sizeof(T) - 1)) == 0) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
        else { const bf16x4 x = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]}; *reinterpret_cast<bf16x4*>(p) = x; }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) if (i < n) p[i] = from_f32<T>(v[i]);
    }
}

template <typename T, int EPI, bool ALN, bool PL>
__global__ __launch_bounds__(256, 2) void lin_gemm_kernel(const LinGemm g) {
    constexpr int EPC = Elem<T>::EPC, CK = Elem<T>::CK;
    __shared__ __attribute__((aligned(128))) char smem[2 * LG_STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave & 1, wn = wave >> 1, l32 = lane & 31, hf = lane >> 5;
    // consecutive tiles of an XCD share the class tile and walk the label rows: the larger operand is read once
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int tm = id % g.ntm, rest = id / g.ntm, tn = rest % g.ntn, sp = rest / g.ntn;
    const int m0 = tm * LG_T, n0 = tn * LG_T;
    const int k0 = EPI == LIN_STORE ? sp * g.kper : 0, k1 = EPI == LIN_STORE ? min(k0 + g.kper, g.K) : g.K;

    // staging: thread -> rows r + 32 i, 16-byte chunk c of the 128-byte row, XOR-swizzled by the row
    const int r = tid >> 3, c = tid & 7;
    const T* const ap = (const T*)g.a;
    const T* const bp = (const T*)g.b;
    u32x4 ra[2][4], rb[2][4];          // two steps on the way: the first is needed a whole step after it was asked for
    int pair = PL ? k0 / g.Kp : 0, pk = PL ? k0 - pair * g.Kp : 0;
    auto fetch = [&](int u, int k) {
        const int left = k1 - k - c * EPC;
        int ka = k + c * EPC, kb = ka;
        if constexpr (PL) {
            ka = lin_plane_a(pair) * g.Kp + pk + c * EPC; kb = lin_plane_b(pair) * g.Kp + pk + c * EPC;
            pk += CK;
            if (pk >= g.Kp) { pk = 0; ++pair; }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = m0 + r + 32 * i, n = n0 + r + 32 * i;
            ra[u][i] = m < g.M ? lin_load16<T, ALN>(ap + m * g.lda + ka, left) : u32x4{0, 0, 0, 0};
            rb[u][i] = n < g.N ? lin_load16<T, ALN>(bp + n * g.ldb + kb, left) : u32x4{0, 0, 0, 0};
        }
    };
    auto put = [&](int st) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int off = (r + 32 * i) * 128 + ((c ^ (r & 7)) << 4);
            *reinterpret_cast<u32x4*>(smem + st * LG_STAGE + off) = ra[st][i];
            *reinterpret_cast<u32x4*>(smem + st * LG_STAGE + LG_T * 128 + off) = rb[st][i];
        }
    };
    f32x16 acc[2][2];                 // [label tile][class tile]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    if (k0 < k1) fetch(0, k0);
    if (k0 + CK < k1) fetch(1, k0 + CK);
    auto step = [&](int st, int k) {   // stage and register set of the same parity
        put(st);
        __syncthreads();              // one barrier per step: the other stage was last read in front of the previous one
        if (k + 2 * CK < k1) fetch(st, k + 2 * CK);
        const char* sa = smem + st * LG_STAGE + (wm * 64 + l32) * 128;
        const char* sb = smem + st * LG_STAGE + LG_T * 128 + (wn * 64 + l32) * 128;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int off = ((2 * s + hf) ^ (l32 & 7)) << 4;
            const u32x4 a0 = *reinterpret_cast<const u32x4*>(sa + off), a1 = *reinterpret_cast<const u32x4*>(sa + 32 * 128 + off);
            const u32x4 b0 = *reinterpret_cast<const u32x4*>(sb + off), b1 = *reinterpret_cast<const u32x4*>(sb + 32 * 128 + off);
            mma16(acc[0][0], b0, a0, (const T*)nullptr); mma16(acc[0][1], b1, a0, (const T*)nullptr);
            mma16(acc[1][0], b0, a1, (const T*)nullptr); mma16(acc[1][1], b1, a1, (const T*)nullptr);
        }
    };
    for (int k = k0; k < k1; k += 2 * CK) {
        step(0, k);
        if (k + CK < k1) step(1, k + CK);
    }
    __syncthreads();

    // lane: label row mrow(i), register e of class tile j: class ncol(j, e)
    auto mrow = [&](int i) { return m0 + wm * 64 + i * 32 + l32; };
    auto ncol = [&](int j, int e) { return n0 + wn * 64 + j * 32 + 8 * (e >> 2) + 4 * hf + (e & 3); };

    if constexpr (EPI == LIN_STORE) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int m = mrow(i);
            if (m >= g.M) continue;
            const float sc = g.scale == 1 ? lin_row_scale(g.gout, g.gstride, g.count, g.t, g.stat[m].y, m)
                           : g.scale == 2 ? lin_row_scale(g.gout, 0, g.count, g.t, 1.f, 0) : 1.f;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const int n = ncol(j, e);
                    if (n >= g.N) continue;
                    const float v[4] = {acc[i][j][e] * sc, acc[i][j][e + 1] * sc, acc[i][j][e + 2] * sc, acc[i][j][e + 3] * sc};
                    if (g.slab) lg_store4(g.slab + ((long long)sp * g.M + m) * g.ldo + n, v, (int)g.ldo - n);
                    else        lg_store4((T*)g.out + m * g.ldo + n, v, g.N - n);
                }
        }
        return;
    }

    // z in place; classes behind the last are -inf
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int n = ncol(j, e);
            const float b = g.bias && n < g.N ? g.bias[n] : 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) acc[i][j][e] = n < g.N ? (acc[i][j][e] + b) * g.inv_t : -INFINITY;
        }

    if constexpr (EPI == LIN_LSE) {
        float2* const red = reinterpret_cast<float2*>(smem);       // [wn][128 rows]
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, acc[i][j][e]);
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float base = mx == -INFINITY ? 0.f : mx;         // every class masked by a -inf bias: the sum is 0, not NaN
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) sum += __expf(acc[i][j][e] - base);
            sum += __shfl_xor(sum, 32);
            if (hf == 0) red[wn * LG_T + wm * 64 + i * 32 + l32] = make_float2(mx, sum);
        }
        __syncthreads();
        if (tid < LG_T && m0 + tid < g.M) {
            const float2 p = red[tid], q = red[LG_T + tid];
            const float mx = fmaxf(p.x, q.x), base = mx == -INFINITY ? 0.f : mx;
            g.part[(long long)(m0 + tid) * g.ntn + tn] = make_float2(mx, p.y * __expf(p.x - base) + q.y * __expf(q.x - base));
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
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float q = __expf(acc[i][j][e] - lse);
                    acc[i][j][e] = dead || ncol(j, e) >= g.N ? 0.f : q;
                }
        }
        if (g.colsum) {
            float* const red = reinterpret_cast<float*>(smem);     // [wm][128 classes]
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float s = acc[0][j][e] * sc[0] + acc[1][j][e] * sc[1];
#pragma unroll
                    for (int d = 16; d; d >>= 1) s += __shfl_xor(s, d);
                    if (l32 == 0) red[wm * LG_T + ncol(j, e) - n0] = s;
                }
            __syncthreads();
            if (tid < LG_T && n0 + tid < g.N) g.colsum[tm * g.ldcol + n0 + tid] = red[tid] + red[LG_T + tid];
        }
#pragma unroll
        for (int pl = 0; pl < (PL ? 3 : 1); ++pl) {
            T* const dz = (T*)g.dz + (PL ? (long long)pl * g.Npad : 0);
            T* const dzt = (T*)g.dzt + (PL ? (long long)pl * g.Mpad : 0);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int m = mrow(i);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const int n = ncol(j, e);
                        const float v[4] = {acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
                        if (m < g.M && n < g.Npad) lg_store4(dz + m * g.lddz + n, v, g.Npad - n);
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            if (g.dzt && m < g.Mpad && n + x < g.N) dzt[(n + x) * g.lddzt + m] = from_f32<T>(v[x]);
                            if constexpr (PL) acc[i][j][e + x] -= to_f32(from_f32<T>(v[x]));
                        }
                    }
            }
        }
    }
}

// Tile and split of a product: the one whose modelled time is least, from the rates that the kernels reach on full chips (fp32 100, bf16 700
// and 1,300 TFLOP/s).  Both take whole rounds of the chip (256 workgroups of the large tile, 512 of the small one); the parts of a split
// reduction are written and read once more, at least 512 (bf16) or 256 (fp32) channels each.  dtype FEA_PL: K is six times the planes'.
LinTile fea_lin_tile(int dtype, long long M, long long N, long long K, bool split) {
    LinTile best{128, 1, 1e30};
    for (int tile = 128; tile <= (dtype == FEA_F32 ? 128 : 256); tile += 128) {
        const double slots = tile == 256 ? 256 : 512;
        const double rate = dtype == FEA_F32 ? 100e12 : tile == 256 ? 1300e12 : 700e12;
        const long long tiles = ((M + tile - 1) / tile) * ((N + tile - 1) / tile);
        for (int sp = 1; sp <= (split ? 32 : 1); ++sp) {
            if (sp > 1 && K / sp < (dtype == FEA_F32 ? 256 : 512)) break;
            const double rounds = (double)((tiles * sp + (long long)slots - 1) / (long long)slots);
            const double t = rounds * (2.0 * tile * tile * ((double)K / sp + 128) / (rate / slots)) + (sp > 1 ? 2.0 * sp * M * N * 4 / 4e12 + 3e-6 : 0.0);
            if (t < best.time * 0.999) best = LinTile{tile, sp, t};
        }
    }
    return best;
}

template <typename T> static void lin_launch(int epi, bool aln, const LinGemm& g, unsigned grid, hipStream_t s) {
    if (epi == LIN_LSE) {
        if (aln) hipLaunchKernelGGL((lin_gemm_kernel<T, LIN_LSE, true, false>), dim3(grid), dim3(256), 0, s, g);
        else     hipLaunchKernelGGL((lin_gemm_kernel<T, LIN_LSE, false, false>), dim3(grid), dim3(256), 0, s, g);
    } else if (epi == LIN_DZ) {
        if (aln) hipLaunchKernelGGL((lin_gemm_kernel<T, LIN_DZ, true, false>), dim3(grid), dim3(256), 0, s, g);
        else     hipLaunchKernelGGL((lin_gemm_kernel<T, LIN_DZ, false, false>), dim3(grid), dim3(256), 0, s, g);
    } else       hipLaunchKernelGGL((lin_gemm_kernel<T, LIN_STORE, true, false>), dim3(grid), dim3(256), 0, s, g);
}
int fea_lin_gemm(int epi, int dtype, int tile, LinGemm g, hipStream_t s) {
    const int epc = dtype == FEA_F32 ? 4 : 8;
    const bool aln = g.K % epc == 0 && g.lda % epc == 0 && g.ldb % epc == 0 && ((uintptr_t)g.a | (uintptr_t)g.b) % 16 == 0;
    const long long row = dtype == FEA_PL ? 3ll * g.Kp : g.K;
    FEA_CHECK(g.M > 0 && g.N > 0 && g.K > 0 && g.lda >= row && g.ldb >= row && (aln || (tile == 128 && epi != LIN_STORE && dtype != FEA_PL)), FEA_E_BADARG,
              "lin_gemm: operands of %d x %d x %d, tile %d", g.M, g.N, g.K, tile);
    FEA_CHECK(dtype != FEA_PL || (g.Kp > 0 && g.Kp % 64 == 0 && g.K == 6 * g.Kp && (epi != LIN_STORE || g.slab)), FEA_E_BADARG, "lin_gemm: planes of %d, K %d", g.Kp, g.K);
    const bool fast = dtype != FEA_F32 && aln && g.lda < (1 << 21) && g.ldb < (1 << 21);
    FEA_CHECK(fast || (tile == 128 && dtype != FEA_PL), FEA_E_UNSUPPORTED_SHAPE, "lin_gemm: tile %d, strides %lld, %lld", tile, g.lda, g.ldb);
    g.ntm = (g.M + tile - 1) / tile; g.ntn = (g.N + tile - 1) / tile;
    if (g.splits < 1) { g.splits = 1; g.kper = g.K; }
    const long long grid = (long long)g.ntm * g.ntn * g.splits;
    FEA_CHECK(grid > 0 && grid <= (1 << 23), FEA_E_UNSUPPORTED_SHAPE, "lin_gemm: %lld tiles", grid);
    if (fast)                   fea_lin_gemm256(epi, tile, dtype == FEA_PL, g, (unsigned)grid, s);
    else if (dtype == FEA_BF16) lin_launch<__bf16>(epi, aln, g, (unsigned)grid, s);
    else                        lin_launch<float>(epi, aln, g, (unsigned)grid, s);
    FEA_LAUNCH_CHECK();
    return FEA_OK;
}
