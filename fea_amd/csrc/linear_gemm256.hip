// The product of the many-class loss heads for large bf16 operands: 256 x 256 tiles, with the epilogues of linear_gemm.hip.
//
// A tile of T x T takes T T / (2 T) = T / 2 multiply-adds per operand element it reads: at 256 a CU at full matrix rate asks for
// 32 B per cycle from L2 (128: 64 B, twice what L2 gives) and for 64 KB of LDS reads per 32-channel step of 1,024 cycles.  Four waves of
// 128 x 128 read each operand twice (8 fragments of each per step and wave: half the LDS rate); eight waves of 128 x 64 would read
// 96 KB, with the fill the whole LDS rate.  So: one workgroup of 4 waves per CU, one wave per SIMD, 8 x 8 accumulators of
// v_mfma_f32_16x16x32_bf16 in the 256 accumulation registers, the rest in the other 256.
//
// Reduction in chunks of 64 channels (whole 128-byte lines), two LDS stages.  In the first half of chunk c every fourth MFMA is
// followed by one fragment read (second half of c), one LDS write of chunk c + 1 from the registers and one load of chunk c + 2 (c + 3 in
// the 128 tile, which has registers for two chunks) into the registers just freed; one barrier; in the second half the fragments of chunk c + 1 are read.  Loads are buffer loads with
// every bound in the lane's offset, so rows, classes and channels behind the end arrive as zeros without a branch.
#include "linear_loss.h"

#ifndef LB_ROT
#define LB_ROT 1
#endif


// XOR of a 128-byte row's 16-byte chunk index: conflict-free ds_read_b128 of 16 rows x 4 chunks
__device__ __forceinline__ int lb_swz(int row) { return ((row >> 1) & 3) << 1; }

__device__ __forceinline__ uint32_t lb_pack(float a, float b) {
    typedef __attribute__((ext_vector_type(2))) float f2;
    typedef __attribute__((ext_vector_type(2))) __bf16 b2;
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, b2));
}

// NT: 16-row tiles of a wave in either direction (8: 256 x 256 per workgroup, one per CU; 4: 128 x 128, two per CU)
template <int EPI, bool PL, int NT>
__global__ __launch_bounds__(256, NT == 8 ? 1 : 2) void lin_gemm256_kernel(const LinGemm g) {
    constexpr int LB_T = 32 * NT, LB_W = 16 * NT, LB_OP = LB_T * 128, LB_STAGE = 2 * LB_OP, NL = 2 * NT;
    __shared__ __attribute__((aligned(128))) char smem[2 * LB_STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave & 1, wn = wave >> 1, r16 = lane & 15, q16 = lane >> 4;
    // tiles in groups of 8 row tiles, walked along the classes: the 32 tiles that an XCD has in flight are 8 x 4
    constexpr int GM = NT;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int per = g.ntm * g.ntn, sp = id / per, it = id - sp * per;
    const int grp = it / (GM * g.ntn), gm = min(GM, g.ntm - grp * GM), in = it - grp * GM * g.ntn;
    const int tm = grp * GM + in % gm, tn = in / gm;
    const int m0 = tm * LB_T, n0 = tn * LB_T;
    const int k0 = EPI == LIN_STORE ? sp * g.kper : 0, K = max((EPI == LIN_STORE ? min(k0 + g.kper, g.K) : g.K) - k0, 0);
    const int nc = (K + 63) >> 6;

    const int kb = PL ? 0 : k0, kl = PL ? 3 * g.Kp : K;      // first channel and length of a row, as the buffers see it
    const __amdgpu_buffer_rsrc_t rsa = __builtin_amdgcn_make_buffer_rsrc((void*)((const __bf16*)g.a + m0 * g.lda + kb), 0,
        K ? (int)(((min(LB_T, g.M - m0) - 1) * g.lda + kl) * 2) : 0, 0x00020000);
    const __amdgpu_buffer_rsrc_t rsb = __builtin_amdgcn_make_buffer_rsrc((void*)((const __bf16*)g.b + n0 * g.ldb + kb), 0,
        K ? (int)(((min(LB_T, g.N - n0) - 1) * g.ldb + kl) * 2) : 0, 0x00020000);

    // staging: thread -> LDS rows r + 32 i of either operand, 16-byte chunk c.  What lies in an LDS row is chosen for the epilogue: the
    // lane that ends up with column r16 of the products holds NT consecutive labels (over its tiles i), and with tiles 2 p, 2 p + 1 of
    // the classes 8 consecutive ones: 16-byte stores of either order of dz without an exchange between lanes.
    const int r = tid >> 3, c = tid & 7;
    const int ra = (r & 15) * NT + (r >> 4), rb = ((r >> 4) & 1) * 4 + ((r >> 2) & 3) * 8 + (r & 3);
    const unsigned va = (unsigned)(ra * (int)g.lda * 2 + c * 16), vb = (unsigned)(rb * (int)g.ldb * 2 + c * 16);
    const unsigned ua = 2 * (unsigned)g.lda, sb = 64 * (unsigned)g.ldb;      // bytes of a label's row, of 32 classes' rows
    const int wofs = r * 128 + ((c ^ lb_swz(r)) << 4);
    constexpr int SETS = NT == 8 ? 1 : 2;      // chunks on the way in registers (two where there is room: a chunk is then shorter than a load)
    u32x4 st[SETS][NL];
    // the XCDs start their reduction an eighth apart (it ends where it began): in step, every workgroup of the chip would ask for the
    // same columns of its rows at a time.  Within an XCD all are in step: they share operands in its L2.
    int at = LB_ROT ? (int)(blockIdx.x & 7) * nc >> 3 : 0;
    int pair = PL ? (k0 + at * 64) / g.Kp : 0, pk = PL ? k0 + at * 64 - pair * g.Kp : 0;       // FEA_PL: the pair of planes and the channel that are loaded next
    unsigned ka = 0, kc = 0;
    bool kin = false;
    auto advance = [&](int ch) {      // byte offsets of the chunk that is loaded ch-th in a row of either operand
        kin = ch < nc && at * 64 + c * 8 < K;
        if constexpr (PL) { ka = 2u * (unsigned)(lin_plane_a(pair) * g.Kp + pk); kc = 2u * (unsigned)(lin_plane_b(pair) * g.Kp + pk); }
        else ka = kc = at * 128;
        if (++at == nc) {
            at = 0;
            if constexpr (PL) { pair = k0 / g.Kp; pk = k0 - pair * g.Kp; }
        } else if constexpr (PL) {
            pk += 64;
            if (pk >= g.Kp) { pk = 0; ++pair; }
        }
    };
    auto gload = [&](int u, int i) {
        if (i < NT) st[u][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsa, kin ? va + ka + (i / (NT / 2) * LB_W + 2 * (i % (NT / 2))) * ua : 0x7fffff00u, 0, 0));
        else        st[u][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsb, kin ? vb + kc + (i - NT) * sb : 0x7fffff00u, 0, 0));
    };
    auto lput = [&](int u, int stage, int i) { *reinterpret_cast<u32x4*>(smem + stage * LB_STAGE + (i / NT) * LB_OP + wofs + (i % NT) * 32 * 128) = st[u][i]; };

    const int fofs0 = r16 * 128 + ((q16 ^ lb_swz(r16)) << 4), fofs1 = fofs0 ^ 64;
    const int fa = wm * LB_W * 128, fb = LB_OP + wn * LB_W * 128;
    u32x4 A[2][NT], B[2][NT];
    auto frd = [&](int stage, int ks, int i) {
        const char* p = smem + stage * LB_STAGE + (ks ? fofs1 : fofs0) + (i % NT) * 16 * 128;
        if (i < NT) A[ks][i] = *reinterpret_cast<const u32x4*>(p + fa);
        else        B[ks][i - NT] = *reinterpret_cast<const u32x4*>(p + fb);
    };
    f32x4 acc[NT][NT];                // [label tile][class tile]
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto mma = [&](int ks) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, B[ks][j]), __builtin_bit_cast(bf16x8, A[ks][i]), acc[i][j], 0, 0, 0);
    };

    advance(0);
#pragma unroll
    for (int i = 0; i < NL; ++i) gload(0, i);
#pragma unroll
    for (int i = 0; i < NL; ++i) lput(0, 0, i);
#pragma unroll
    for (int u = 0; u < SETS; ++u) {
        advance(1 + u);
#pragma unroll
        for (int i = 0; i < NL; ++i) gload((1 + u) % SETS, i);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NL; ++i) frd(0, 0, i);

    // chunk ch of LDS stage s; chunk ch + 1 lies in register set u, where chunk ch + 1 + SETS follows it
    auto step = [&](int ch, int s, int u) {
        advance(ch + 1 + SETS);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NL; ++i) { frd(s, 1, i); lput(u, s ^ 1, i); gload(u, i); }
        mma(0);
#pragma unroll
        for (int i = 0; i < NL; ++i) {        // 4 MFMA (2 where NT is 4), an LDS read, an LDS write, a load
            if (NT == 8) __builtin_amdgcn_sched_group_barrier(0x008, 2, 0); else if (i & 1) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            if (NT == 8) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        // chunk ch + 1 is in LDS and nobody reads this stage's first half or the other stage any more
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NL; ++i) frd(s ^ 1, 0, i);
        mma(1);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, NT / 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
    };
    if constexpr (SETS == 1) {
        for (int ch = 0; ch < nc; ++ch) step(ch, ch & 1, 0);
    } else {
        for (int ch = 0; ch < nc; ch += 2) {
            step(ch, 0, 1);
            if (ch + 1 < nc) step(ch + 1, 1, 0);
        }
    }
    __syncthreads();

    auto mrow = [&](int i) { return m0 + wm * LB_W + r16 * NT + i; };                                    // label of tile i
    auto ncol = [&](int j) { return n0 + wn * LB_W + (j >> 1) * 32 + q16 * 8 + (j & 1) * 4; };           // first of 4 classes of tile j
    const int pcol = n0 + wn * LB_W + q16 * 8;                                                           // first of 8 classes of tiles 0, 1
    auto pairs = [&](const f32x4& x, const f32x4& y) { return u32x4{lb_pack(x[0], x[1]), lb_pack(x[2], x[3]), lb_pack(y[0], y[1]), lb_pack(y[2], y[3])}; };

    if constexpr (EPI == LIN_STORE) {
        const float common = g.scale == 2 ? lin_row_scale(g.gout, 0, g.count, g.t, 1.f, 0) : 1.f;
        const bool wide = g.slab ? g.ldo % 4 == 0 : g.N % 8 == 0 && g.ldo % 8 == 0 && (uintptr_t)g.out % 16 == 0;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int m = mrow(i);
            const float sc = g.scale == 1 ? (m < g.M ? lin_row_scale(g.gout, g.gstride, g.count, g.t, g.stat[m].y, m) : 0.f) : common;
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] *= sc;
            if (g.slab) {
                float* const o = g.slab + ((long long)sp * g.M + m) * g.ldo;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const int n = ncol(j);
                    if (wide) { if (m < g.M && n < g.N) *reinterpret_cast<f32x4*>(o + n) = acc[i][j]; }
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e) if (m < g.M && n + e < g.N) o[n + e] = acc[i][j][e];
                }
            } else {
                __bf16* const o = (__bf16*)g.out + m * g.ldo;
#pragma unroll
                for (int p = 0; p < NT / 2; ++p) {
                    if (wide) {
                        const u32x4 v = pairs(acc[i][2 * p], acc[i][2 * p + 1]);
                        if (m < g.M && pcol + 32 * p < g.N) *reinterpret_cast<u32x4*>(o + pcol + 32 * p) = v;
                    } else
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int n = ncol(2 * p + (e >> 2)) + (e & 3);
                            if (m < g.M && n < g.N) o[n] = (__bf16)acc[i][2 * p + (e >> 2)][e & 3];
                        }
                }
            }
        }
    } else {
        // z in place; classes behind the last are -inf
        const bool edge = n0 + LB_T > g.N;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int n = ncol(j) + e;
                const float b = g.bias && n < g.N ? g.bias[n] : 0.f;
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[i][j][e] = edge && n >= g.N ? -INFINITY : (acc[i][j][e] + b) * g.inv_t;
            }
    }

    if constexpr (EPI == LIN_LSE) {
        float2* const red = reinterpret_cast<float2*>(smem);       // [wn][256 labels]
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < NT; ++j) mx = fmaxf(fmaxf(mx, fmaxf(acc[i][j][0], acc[i][j][1])), fmaxf(acc[i][j][2], acc[i][j][3]));
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float base = mx == -INFINITY ? 0.f : mx;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += __expf(acc[i][j][e] - base);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (q16 == 0) red[wn * LB_T + wm * LB_W + r16 * NT + i] = make_float2(mx, sum);
        }
        __syncthreads();
        if (tid < LB_T && m0 + tid < g.M) {
            const float2 p = red[tid], q = red[LB_T + tid];
            const float mx = fmaxf(p.x, q.x), base = mx == -INFINITY ? 0.f : mx;
            g.part[(long long)(m0 + tid) * g.ntn + tn] = make_float2(mx, p.y * __expf(p.x - base) + q.y * __expf(q.x - base));
        }
    }

    if constexpr (EPI == LIN_DZ) {
        float sc[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int m = mrow(i);
            const float2 s2 = m < g.M ? g.stat[m] : make_float2(0.f, 0.f);
            const bool dead = s2.y == 0.f;
            sc[i] = dead || !g.colsum ? 0.f : lin_row_scale(g.gout, g.gstride, g.count, g.t, s2.y, m);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float q = __expf(acc[i][j][e] - s2.x);
                    acc[i][j][e] = dead || (n0 + LB_T > g.N && ncol(j) + e >= g.N) ? 0.f : q;
                }
        }
        if (g.colsum) {
            float* const red = reinterpret_cast<float*>(smem);     // [wm][256 classes]
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float s = 0.f;
#pragma unroll
                    for (int i = 0; i < NT; ++i) s += acc[i][j][e] * sc[i];
#pragma unroll
                    for (int d = 8; d; d >>= 1) s += __shfl_xor(s, d);
                    if (r16 == 0) red[wm * LB_T + ncol(j) + e - n0] = s;
                }
            __syncthreads();
            if (tid < LB_T && n0 + tid < g.N) g.colsum[tm * g.ldcol + n0 + tid] = red[tid] + red[LB_T + tid];
        }
#pragma unroll
        for (int pl = 0; pl < (PL ? 3 : 1); ++pl) {
            __bf16* const dz = (__bf16*)g.dz + (PL ? (long long)pl * g.Npad : 0);
            __bf16* const dzt = (__bf16*)g.dzt + (PL ? (long long)pl * g.Mpad : 0);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int m = mrow(i);
                __bf16* const o = dz + m * g.lddz;
#pragma unroll
                for (int p = 0; p < NT / 2; ++p) {
                    const u32x4 v = pairs(acc[i][2 * p], acc[i][2 * p + 1]);
                    if (m < g.M && pcol + 32 * p < g.Npad) *reinterpret_cast<u32x4*>(o + pcol + 32 * p) = v;
                }
            }
            if (g.dzt && mrow(0) < g.Mpad)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int n = ncol(j) + e;
                        if (n >= g.N) continue;
                        __bf16* const o = dzt + n * g.lddzt + mrow(0);
                        if constexpr (NT == 8) *reinterpret_cast<u32x4*>(o) = u32x4{lb_pack(acc[0][j][e], acc[1][j][e]), lb_pack(acc[2][j][e], acc[3][j][e]), lb_pack(acc[NT - 4][j][e], acc[NT - 3][j][e]), lb_pack(acc[NT - 2][j][e], acc[NT - 1][j][e])};
                        else                   *reinterpret_cast<u32x2*>(o) = u32x2{lb_pack(acc[0][j][e], acc[1][j][e]), lb_pack(acc[2][j][e], acc[3][j][e])};
                    }
            if constexpr (PL)
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][e] -= (float)(__bf16)acc[i][j][e];
        }
    }
}

template <bool PL, int NT> static void lb_launch(int epi, const LinGemm& g, unsigned grid, hipStream_t s) {
    if (epi == LIN_LSE)     hipLaunchKernelGGL((lin_gemm256_kernel<LIN_LSE, PL, NT>), dim3(grid), dim3(256), 0, s, g);
    else if (epi == LIN_DZ) hipLaunchKernelGGL((lin_gemm256_kernel<LIN_DZ, PL, NT>), dim3(grid), dim3(256), 0, s, g);
    else                    hipLaunchKernelGGL((lin_gemm256_kernel<LIN_STORE, PL, NT>), dim3(grid), dim3(256), 0, s, g);
}
void fea_lin_gemm256(int epi, int tile, bool planes, const LinGemm& g, unsigned grid, hipStream_t s) {
    if (tile == 256) { if (planes) lb_launch<true, 8>(epi, g, grid, s); else lb_launch<false, 8>(epi, g, grid, s); }
    else             { if (planes) lb_launch<true, 4>(epi, g, grid, s); else lb_launch<false, 4>(epi, g, grid, s); }
}
