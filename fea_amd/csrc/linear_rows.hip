// Log-sum-exp of the logits of a few label rows (up to 64) over many classes: the weight is read once, straight into the matrix
// operands, and everything else has to keep out of its way.
//
// One wave owns 16 classes over the whole reduction (v_mfma 16x16: 16 classes x 16 labels per product, NR of them); a workgroup of 4
// waves 64 classes.  The weight goes from memory to registers (a wave's 16 rows x 512 bytes in flight while the 512 bytes before
// are multiplied); the labels' hidden states, which all waves share, through LDS in the same chunks.
// Bound by the weight's bytes: 50,021 x 2,048 bf16 (205 MB) for 37 rows in 56.5 us from memory (3.6 TB/s) and 46 us (4.5 TB/s) where the
// weight is left in the 256 MB of the Infinity Cache from the call before; 32,768 x 1,024 (67 MB, there too) for one row in
// 16.6 us (4.0 TB/s), for 64 in 18.7 us.  Copies reach 5.0 TB/s.
#include "linear_loss.h"

__device__ __forceinline__ void mma16x16(f32x4& acc, const u32x4& a, const u32x4& b, const __bf16*) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
}
__device__ __forceinline__ void mma16x16(f32x4& acc, const u32x4& a, const u32x4& b, const float*) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, y.x, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, y.y, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, y.z, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, y.w, acc, 0, 0, 0);
}

template <typename T, int NR, bool ALN>
__global__ __launch_bounds__(256, NR == 4 ? 3 : 4) void lin_rows_kernel(const LinGemm g) {
    // a chunk is 256 bytes of a row; three chunks of the weight are in flight while one is multiplied.  The labels' chunk is asked for two
    // steps before it goes to LDS: loads come back in order, so waiting for one that is a step old would be waiting for the weight's
    // too.  The distance of a row in LDS puts 16 rows in 16 bank groups
    constexpr int NT = 256, CLS = 64;
    constexpr int CB = 256, LD = CB + 16, PR = CB / 16, RING = 4;
    constexpr int EPC = Elem<T>::EPC, CE = CB / (int)sizeof(T), NS = CB / 64;     // elements, products of a chunk
    __shared__ __attribute__((aligned(16))) char hs[2][16 * NR * LD];
    __shared__ float2 red[4][16 * NR];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, q16 = lane >> 4;
    const int n0 = blockIdx.x * CLS + wave * 16;
    const T* const w = (const T*)g.b + (long long)min(n0 + r16, g.N - 1) * g.ldb;
    const T* const h = (const T*)g.a;
    const int kb = blockIdx.y * g.kper, K = min(kb + g.kper, g.K);       // part of a split reduction
    u32x4 wv[RING][NS];
    auto wload = [&](int buf, int k0) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int k = k0 + (4 * s + q16) * EPC;
            wv[buf][s] = lin_load16<T, ALN>(w + k, K - k);
        }
    };
    constexpr int HP = NR * 16 * PR / NT;           // 16-byte pieces of the labels' chunk per thread
    u32x4 hv[2][HP];
    auto hload = [&](int buf, int k0) {
#pragma unroll
        for (int i = 0; i < HP; ++i) {
            const int p = tid + NT * i, row = p / PR, k = k0 + (p % PR) * EPC;
            hv[buf][i] = row < g.M ? lin_load16<T, ALN>(h + row * g.lda + k, K - k) : u32x4{0, 0, 0, 0};
        }
    };
    auto hput = [&](int buf) {
#pragma unroll
        for (int i = 0; i < HP; ++i) {
            const int p = tid + NT * i;
            *reinterpret_cast<u32x4*>(hs[buf] + (p / PR) * LD + (p % PR) * 16) = hv[buf][i];
        }
    };
    f32x4 acc[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    // The workgroups start their reduction at different chunks (it ends where it began): in step they would all ask for the same
    // columns of rows that lie a power of two apart, that is for a few of the memory channels at a time.
    const int rounds = (K - kb + RING * CE - 1) / (RING * CE), nch = rounds * RING;
    int at = (int)(3u * blockIdx.x % (unsigned)nch);
    auto chunk = [&](int ahead) { int c = at + ahead; return kb + (c >= nch ? c - nch : c) * CE; };
    hload(0, chunk(0));
    wload(0, chunk(0));
    hload(1, chunk(1));
    wload(1, chunk(1));
    wload(2, chunk(2));
    for (int r = 0; r < rounds; ++r) {
#pragma unroll
        for (int c = 0; c < RING; ++c) {      // one round of the ring, so that the buffers' indexes are constants
            hput(c & 1);
            hload(c & 1, chunk(2));
            wload((c + RING - 1) % RING, chunk(RING - 1));
            __syncthreads();                  // (also: every wave is done with the other buffer)
            if (++at == nch) at = 0;
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int i = 0; i < NR; ++i)
                    mma16x16(acc[i], wv[c][s], *reinterpret_cast<const u32x4*>(hs[c & 1] + (16 * i + r16) * LD + (4 * s + q16) * 16), (const T*)nullptr);
        }
    }
    if (g.slab) {            // split: the sums as they are, joined by lin_join_split_kernel
#pragma unroll
        for (int i = 0; i < NR; ++i)
            if (16 * i + r16 < g.M) *reinterpret_cast<f32x4*>(g.slab + ((long long)blockIdx.y * g.M + 16 * i + r16) * g.ldo + n0 + 4 * q16) = acc[i];
        return;
    }
    // the selected logits: every workgroup looks for its own classes among the entries
    __syncthreads();
    float (*const zt)[16 * NR + 1] = reinterpret_cast<float (*)[16 * NR + 1]>(&hs[0][0]);       // [classes][labels]
    // lane: label 16 i + r16, classes n0 + 4 q16 .. + 3
    float bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = g.bias && n0 + 4 * q16 + e < g.N ? g.bias[n0 + 4 * q16 + e] : 0.f;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        float z[4], mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float raw = acc[i][e] + bias[e];
            if (g.zsel) zt[wave * 16 + 4 * q16 + e][16 * i + r16] = raw * g.inv_t;
            z[e] = n0 + 4 * q16 + e < g.N ? raw * g.inv_t : -INFINITY;
            mx = fmaxf(mx, z[e]);
        }
        if (g.keep && 16 * i + r16 < g.M)
            *reinterpret_cast<f32x4*>((float*)g.keep + (16 * i + r16) * g.ldkeep + n0 + 4 * q16) = f32x4{z[0], z[1], z[2], z[3]};
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += __expf(z[e] - base);
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (q16 == 0) red[wave][16 * i + r16] = make_float2(mx, sum);
    }
    __syncthreads();
    if (g.zsel)
        for (int e = tid; e < g.M * g.sel; e += NT) {
            const long long c = g.index[e] - (long long)blockIdx.x * CLS;
            if (c >= 0 && c < CLS && (int)blockIdx.x * CLS + c < g.N) g.zsel[e] = zt[c][e / g.sel];
        }
    if (tid < 16 * NR && tid < g.M) {
        float mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) mx = fmaxf(mx, red[k][tid].x);
        const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int k = 0; k < 4; ++k) sum += red[k][tid].y * __expf(red[k][tid].x - base);
        g.part[(long long)tid * g.ntn + blockIdx.x] = make_float2(mx, sum);
    }
}

template <typename T, bool ALN> static void rows_launch(const LinGemm& g, dim3 grid, hipStream_t s) {
    if (g.M <= 16)      hipLaunchKernelGGL((lin_rows_kernel<T, 1, ALN>), grid, dim3(256), 0, s, g);
    else if (g.M <= 32) hipLaunchKernelGGL((lin_rows_kernel<T, 2, ALN>), grid, dim3(256), 0, s, g);
    else if (g.M <= 48) hipLaunchKernelGGL((lin_rows_kernel<T, 3, ALN>), grid, dim3(256), 0, s, g);
    else                hipLaunchKernelGGL((lin_rows_kernel<T, 4, ALN>), grid, dim3(256), 0, s, g);
}


// Parts of the reduction: few classes make few workgroups, and one of them reads its 64 classes no faster for that.  Below 256 of them (bf16: 128)
// about 512 in all, each with at least 8 chunks.  A loss of 30 rows x 3,840 x 3,840, one part and split: fp32 61 and 36 us, bf16 31 and
// 21.5; 64 x 2,048 x 300: 57 and 23, 23 and 17; 64 x 1,024 x 8,192 (128 workgroups): 35 and 29, 18.5 and 18; 16 x 8,192 x 16,000 (250):
// 119 and 108, 52 and 60.
int fea_lin_rows_splits(int dtype, int V, int D) {
    const int tiles = (V + 63) / 64, chunks = (D + (dtype == FEA_BF16 ? 127 : 63)) / (dtype == FEA_BF16 ? 128 : 64);
    if (tiles >= (dtype == FEA_BF16 ? 128 : 256)) return 1;
    const int want = 512 / tiles, most = chunks / 8;
    const int parts = most < 1 ? 1 : want < most ? want : most, per = (chunks + parts - 1) / parts;
    return (chunks + per - 1) / per;                            // (no part is empty)
}

// LIN_LSE of at most 64 label rows, operands of any alignment
int fea_lin_rows(int dtype, bool aligned, LinGemm g, hipStream_t s) {
    FEA_CHECK(g.M > 0 && g.M <= 64 && g.N > 0 && g.K > 0, FEA_E_BADARG, "lin_rows: %d x %d x %d", g.M, g.N, g.K);
    FEA_CHECK((g.slab != nullptr) == (g.splits > 1), FEA_E_BADARG, "lin_rows: %d parts", g.splits);
    g.ntn = (g.N + 63) / 64;
    const int unit = dtype == FEA_BF16 ? 128 : 64;             // channels of a chunk
    if (g.splits < 1) g.splits = 1;
    g.kper = ((g.K + g.splits - 1) / g.splits + unit - 1) / unit * unit;
    FEA_CHECK((long long)(g.splits - 1) * g.kper < g.K, FEA_E_BADARG, "lin_rows: %d parts of %d channels", g.splits, g.K);
    const dim3 grid((unsigned)g.ntn, (unsigned)g.splits);
    if (dtype == FEA_BF16) { if (aligned) rows_launch<__bf16, true>(g, grid, s); else rows_launch<__bf16, false>(g, grid, s); }
    else                   { if (aligned) rows_launch<float, true>(g, grid, s); else rows_launch<float, false>(g, grid, s); }
    FEA_LAUNCH_CHECK();
    return FEA_OK;
}
