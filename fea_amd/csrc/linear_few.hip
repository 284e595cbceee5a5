// Loss heads with few classes and few features over very many rows (per-pixel classes: 6 classes of 64 channels, 16.8 million pixels):
// at most 32 classes and 64 features, forward and backward each in one pass over the rows, everything between in registers.
//
// One wave takes 32 rows at a time; a row is a lane (and its partner in the other wave half) throughout.  C layout of the 32 x 32
// MFMA: lane l holds column l & 31 and rows 8 (i >> 2) + 4 (l >> 5) + (i & 3) of the result, i = 0..15.
//   logits   C1[class][row] = W . H^T       lane = row, registers = 4 classes of every 8: the softmax is in-lane sums and one exchange
//   dh       C2[d][row] = W^T . dz^T        the operand needs, per lane, the classes that its registers already hold (any order of
//                                           the reduction axis will do if both operands agree): no data moves between lanes
//   dw       C3[class][d] = dz^T . H        both operands need rows in registers.  A product with the identity turns C1's layout and
//                                           the loaded rows into that: C[row][x] = A[row][k] I[k][x] puts x in the lane and rows in
//                                           the registers; every value is multiplied by 1 and added to zeros, so nothing is rounded
// The rows are read once and dh written once: the bound is HBM (16.8 M rows of 64 bf16 channels, 6 classes: forward 0.50 ms, 4.9 TB/s;
// backward 0.86 ms, 5.3 TB/s; 2.1 M rows with 3 teacher entries: 0.11 ms, 3.4 TB/s, entries of 24 bytes a row, and 0.125 ms, 5.0 TB/s).  dz is rounded once to the storage type for the two products; it is
// unscaled there (a common factor would round the same way in every row), the row's factor meets fp32 values, or the row itself
// where every row has its own.  Partial sums of dw and db go to one slab per workgroup, joined in a fixed order.
#include "linear_loss.h"

struct LinI { static __device__ __forceinline__ int cls(int i, int hf) { return 8 * (i >> 2) + 4 * hf + (i & 3); } };

template <typename T, bool ALN>
__device__ __forceinline__ u32x4 few_load(const T* row, int d, int D) { return lin_load16<T, ALN>(row + d, D - d); }
// registers EPC s .. EPC s + EPC - 1 of a result as one operand step
template <typename T> __device__ __forceinline__ u32x4 few_pack(const float* v) {
    if constexpr (sizeof(T) == 4) { const f32x4 x = {v[0], v[1], v[2], v[3]}; return __builtin_bit_cast(u32x4, x); }
    else { const bf16x8 x = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3], (__bf16)v[4], (__bf16)v[5], (__bf16)v[6], (__bf16)v[7]}; return __builtin_bit_cast(u32x4, x); }
}
// class (or row) of element e of operand step s in this wave half, when the step is made of result registers
template <typename T> __device__ __forceinline__ int few_idx(int s, int e, int hf) { return LinI::cls(Elem<T>::EPC * s + e, hf); }

template <typename T> __device__ __forceinline__ float few_tlog(const void* p, int dt, long long e) {
    return dt == FEA_BF16 ? (float)((const __bf16*)p)[e] : ((const float*)p)[e];
}

// A row's teacher entries (forward: class and logit; backward: class and share): the first 4 are loaded together and kept, the
// others are read as they are gone through.
template <typename T> struct LinEntries {
    static constexpr int KEEP = 4;
    const LinFew& g;
    long long e0;
    long long i[KEEP];
    float v[KEEP];
    __device__ __forceinline__ float value(long long e) const { return g.tlog ? few_tlog<T>(g.tlog, g.tdt, e) : g.psel[e]; }
    __device__ __forceinline__ LinEntries(const LinFew& g_, long long row) : g(g_), e0(row * g_.K) {
        if (!g.tlog && (!g.psel || !g.gout)) return;      // cross entropy
#pragma unroll
        for (int k = 0; k < KEEP; ++k) {
            i[k] = k < g.K ? g.index[e0 + k] : -1;
            v[k] = k < g.K ? value(e0 + k) : 0.f;
        }
    }
    template <class F> __device__ __forceinline__ void each(F&& f) const {
#pragma unroll
        for (int k = 0; k < KEEP; ++k) if (k < g.K) f(k, i[k], v[k]);
        for (int k = KEEP; k < g.K; ++k) f(k, g.index[e0 + k], value(e0 + k));
    }
};

// A wave's 32 rows x NB blocks of 32 features on their way between memory, where a load or store takes whole rows (lanes along a row), and the
// operand layout, where a lane is a row: through 32 rows of LDS that only this wave uses.  Lanes along a column directly would touch 32 lines
// per load, a quarter of each.
template <typename T, int NB, bool ALN> struct LinRows {
    static constexpr int EPC = Elem<T>::EPC, CPR = NB * 32 / EPC, RPL = 64 / CPR, NK = 32 / RPL;     // 16-byte pieces of a row, rows of a load, loads
    static constexpr int LD = CPR * 16 + 16;
    char* lds;
    int row, piece;                        // of this lane in load 0
    __device__ __forceinline__ LinRows(char* p, int lane) : lds(p), row(lane / CPR), piece(lane % CPR) {}
    __device__ __forceinline__ void load(u32x4 (&v)[NK], const T* h, long long ld, long long first, long long rows, int D) const {
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            long long r = first + row + k * RPL;
            r = r < rows ? r : rows - 1;
            v[k] = few_load<T, ALN>(h + r * ld, piece * EPC, D);
        }
    }
    static __device__ __forceinline__ void fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); }
    // loaded pieces -> operand: piece 2 k + hf of row l32
    __device__ __forceinline__ void turn(const u32x4 (&v)[NK], u32x4 (&x)[NK], int l32, int hf) const {
#pragma unroll
        for (int k = 0; k < NK; ++k) *reinterpret_cast<u32x4*>(lds + (row + k * RPL) * LD + piece * 16) = v[k];
        fence();
#pragma unroll
        for (int k = 0; k < NK; ++k) x[k] = *reinterpret_cast<const u32x4*>(lds + l32 * LD + (2 * k + hf) * 16);
        fence();
    }
    // four consecutive features d .. d + 3 of row l32
    __device__ __forceinline__ void put(const f32x16& o, int q, float sc, int l32, int d) const {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(lds + l32 * LD + d * 4) = f32x4{o[4 * q] * sc, o[4 * q + 1] * sc, o[4 * q + 2] * sc, o[4 * q + 3] * sc};
        else *reinterpret_cast<bf16x4*>(lds + l32 * LD + d * 2) = bf16x4{(__bf16)(o[4 * q] * sc), (__bf16)(o[4 * q + 1] * sc), (__bf16)(o[4 * q + 2] * sc), (__bf16)(o[4 * q + 3] * sc)};
    }
    __device__ __forceinline__ void store(T* out, long long first, long long rows, int D) const {
        fence();
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const long long r = first + row + k * RPL;
            const int left = D - piece * EPC;
            const u32x4 v = *reinterpret_cast<const u32x4*>(lds + (row + k * RPL) * LD + piece * 16);
            if (r >= rows || left <= 0) continue;
            T* const o = out + r * D + piece * EPC;
            if constexpr (ALN) *reinterpret_cast<u32x4*>(o) = v;
            else {
                if (left >= EPC) __builtin_memcpy(o, &v, 16);
                else {
                    T x[EPC];
                    *reinterpret_cast<u32x4*>(x) = v;
#pragma unroll
                    for (int e = 0; e < EPC; ++e) if (e < left) o[e] = x[e];
                }
            }
        }
        fence();
    }
};

// NB blocks of 32 features, NG groups of 8 classes (4 registers)
template <typename T, int NB, int NG, bool ALN>
__global__ __launch_bounds__(256) void lin_few_fwd_kernel(const LinFew g) {
    constexpr int EPC = Elem<T>::EPC, NK = NB * 32 / (2 * EPC), NR = 4 * NG;
    const int lane = threadIdx.x & 63, l32 = lane & 31, hf = lane >> 5;
    const long long wave = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), nwaves = (long long)gridDim.x * 4;
    const long long tiles = (g.rows + 31) / 32;
    u32x4 wf[NK];
#pragma unroll
    for (int k = 0; k < NK; ++k)
        wf[k] = l32 < g.V ? few_load<T, ALN>((const T*)g.w + l32 * g.ldw, (2 * k + hf) * EPC, g.D) : u32x4{0, 0, 0, 0};
    float bias[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) bias[i] = LinI::cls(i, hf) < g.V ? (g.bias ? g.bias[LinI::cls(i, hf)] : 0.f) : -INFINITY;

    double total = 0.0;
    int counted = 0;
    __shared__ __attribute__((aligned(16))) char buf[4][32 * LinRows<T, NB, ALN>::LD];
    const LinRows<T, NB, ALN> rows(buf[threadIdx.x >> 6], lane);
    // two tiles on the way while one is worked on, their labels with them
    u32x4 nx[2][NK];
    long long nl[2];
    auto fetch = [&](int u, long long tile) {
        if (tile >= tiles) return;
        rows.load(nx[u], (const T*)g.h, g.ldh, tile * 32, g.rows, g.D);
        const long long r = tile * 32 + l32 < g.rows ? tile * 32 + l32 : g.rows - 1;
        nl[u] = g.tlog ? 0 : g.index[r];
    };
    auto body = [&](int u, long long tile) {
        u32x4 hx[NK];
        rows.turn(nx[u], hx, l32, hf);
        const long long row = tile * 32 + l32;
        const bool in = row < g.rows;
        const long long rr = in ? row : g.rows - 1;
        const long long label = nl[u];
        LinEntries<T> ent(g, rr);
        fetch(u, tile + 2 * nwaves);
        f32x16 acc;
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] = 0.f;
#pragma unroll
        for (int k = 0; k < NK; ++k) mma16(acc, wf[k], hx[k], (const T*)nullptr);
        float z[NR], mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            z[i] = LinI::cls(i, hf) < g.V ? (acc[i] + bias[i]) * g.inv_t : -INFINITY;
            mx = fmaxf(mx, z[i]);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int i = 0; i < NR; ++i) sum += __expf(z[i] - base);
        sum += __shfl_xor(sum, 32);
        float lse = logf(sum) + base, loss = 0.f;
        bool counts;
        if (!g.tlog) {
            counts = in && label != g.ignore;
            float zt = 0.f;
#pragma unroll
            for (int i = 0; i < NR; ++i) zt = LinI::cls(i, hf) == label ? z[i] : zt;
            zt += __shfl_xor(zt, 32);
            loss = lse - zt;
            loss = loss < 0.f ? 0.f : loss;
            if (label < 0 || label >= g.V) { loss = NAN; lse = NAN; }
            if (!counts) loss = 0.f;
        } else {
            float tm = -INFINITY, ts = 0.f;
            bool bad = false;
            ent.each([&](int, long long i, float a) {
                if (i >= g.V) bad = true;
                if (i >= 0) { bad |= !(a < INFINITY); tm = fmaxf(tm, a); }
            });
            counts = in && (bad || tm != -INFINITY);
            const float tb = tm == -INFINITY ? 0.f : tm;
            ent.each([&](int, long long i, float a) { if (i >= 0) ts += expf((a - tb) * g.inv_t); });
            const float lt = logf(ts);
            float pz = 0.f, pl = 0.f;                     // sum p z over the classes of this half; sum p (log p + lse)
            ent.each([&](int k, long long i, float a) {
                float p = 0.f;
                if (i >= 0 && counts) {
                    const float lp = (a - tb) * g.inv_t - lt;             // (1 / T meets the distance: the lowest value as a mask stays finite)
                    p = bad ? NAN : expf(lp);
                    if (p > 0.f) {
                        pl += p * (lp + lse);
#pragma unroll
                        for (int q = 0; q < NR; ++q) if (LinI::cls(q, hf) == i) pz += p * z[q];
                    }
                }
                if (g.psel && in && hf == 0) g.psel[rr * g.K + k] = p;
            });
            pz += __shfl_xor(pz, 32);
            loss = (pl - pz) * g.t * g.t;
            if (bad) { loss = NAN; lse = NAN; }
            if (!counts) loss = 0.f;
        }
        if (in && hf == 0) {
            if (g.stat) g.stat[row] = make_float2(counts ? lse : 0.f, counts ? 1.f : 0.f);
            if (g.loss_rows) g.loss_rows[row] = loss;
            total += (double)loss;
            counted += counts;
        }
    };
    fetch(0, wave);
    fetch(1, wave + nwaves);
    for (long long tile = wave; tile < tiles; tile += 2 * nwaves) {
        body(0, tile);
        if (tile + nwaves < tiles) body(1, tile + nwaves);
    }
    if (g.bsum) {
        __shared__ double ls[4];
        __shared__ int lc[4];
        for (int d = 32; d; d >>= 1) { total += __shfl_xor(total, d); counted += __shfl_xor(counted, d); }
        if (lane == 0) { ls[threadIdx.x >> 6] = total; lc[threadIdx.x >> 6] = counted; }
        __syncthreads();
        if (threadIdx.x == 0) { g.bsum[blockIdx.x] = (ls[0] + ls[1]) + (ls[2] + ls[3]); g.bcnt[blockIdx.x] = lc[0] + lc[1] + lc[2] + lc[3]; }
    }
}

template <typename T, int NB, int NG, bool ALN>
__global__ __launch_bounds__(256) void lin_few_bwd_kernel(const LinFew g) {
    constexpr int EPC = Elem<T>::EPC, NK = NB * 32 / (2 * EPC), NR = 4 * NG;
    constexpr int NS = (NR + EPC - 1) / EPC;              // operand steps that hold the classes
    constexpr int RS = 16 / EPC, BK = 32 / (2 * EPC);     // operand steps of 32 rows; of one block of 32 features
    const int lane = threadIdx.x & 63, l32 = lane & 31, hf = lane >> 5;
    const long long wave = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), nwaves = (long long)gridDim.x * 4;
    const long long tiles = (g.rows + 31) / 32;
    const T* const w = (const T*)g.w;
    const bool rowg = g.gstride != 0;
    u32x4 wf[NK], wt[NB][NS], idd[BK], idc[NS];
#pragma unroll
    for (int k = 0; k < NK; ++k) wf[k] = l32 < g.V ? few_load<T, ALN>(w + l32 * g.ldw, (2 * k + hf) * EPC, g.D) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        T x[EPC];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int e = 0; e < EPC; ++e) {
                const int c = few_idx<T>(s, e, hf), d = 32 * b + l32;
                x[e] = c < g.V && d < g.D ? w[c * g.ldw + d] : from_f32<T>(0.f);
            }
            wt[b][s] = *reinterpret_cast<const u32x4*>(x);
        }
#pragma unroll
        for (int e = 0; e < EPC; ++e) x[e] = from_f32<T>(few_idx<T>(s, e, hf) == l32 ? 1.f : 0.f);
        idc[s] = *reinterpret_cast<const u32x4*>(x);
    }
#pragma unroll
    for (int k = 0; k < BK; ++k) {
        T x[EPC];
#pragma unroll
        for (int e = 0; e < EPC; ++e) x[e] = from_f32<T>((2 * k + hf) * EPC + e == l32 ? 1.f : 0.f);
        idd[k] = *reinterpret_cast<const u32x4*>(x);
    }
    float bias[NR], dbs[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) { bias[i] = LinI::cls(i, hf) < g.V && g.bias ? g.bias[LinI::cls(i, hf)] : 0.f; dbs[i] = 0.f; }
    f32x16 dw[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) dw[b][e] = 0.f;

    __shared__ __attribute__((aligned(16))) char buf[4][32 * LinRows<T, NB, ALN>::LD];
    const LinRows<T, NB, ALN> rows(buf[threadIdx.x >> 6], lane);
    u32x4 nx[2][NK];
    float2 ns[2];
    long long nl[2];
    auto fetch = [&](int u, long long tile) {
        if (tile >= tiles) return;
        rows.load(nx[u], (const T*)g.h, g.ldh, tile * 32, g.rows, g.D);
        const long long r = tile * 32 + l32 < g.rows ? tile * 32 + l32 : g.rows - 1;
        ns[u] = g.stat[r];
        nl[u] = g.psel ? -1 : g.index[r];
    };
    auto body = [&](int u, long long tile) {
        u32x4 hx[NK];
        const long long row = tile * 32 + l32;
        const bool in = row < g.rows;
        const long long rr = in ? row : g.rows - 1;
        const float2 st = ns[u];
        const bool on = in && st.y != 0.f;
        const long long label = nl[u];
        LinEntries<T> ent(g, rr);
        const float sc = lin_row_scale(g.gout, g.gstride, g.count, g.t, st.y, rr);
        // a row that does not count is read as zeros: its gradients are 0 whatever it holds
        rows.turn(nx[u], hx, l32, hf);
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) hx[k][e] = on ? hx[k][e] : 0u;
        fetch(u, tile + 2 * nwaves);
        f32x16 acc;
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] = 0.f;
#pragma unroll
        for (int k = 0; k < NK; ++k) mma16(acc, wf[k], hx[k], (const T*)nullptr);
        float dz[NS * EPC];
#pragma unroll
        for (int i = 0; i < NS * EPC; ++i) {
            if (i >= NR) { dz[i] = 0.f; continue; }
            const int c = LinI::cls(i, hf);
            const float q = __expf((acc[i] + bias[i]) * g.inv_t - st.x);
            dz[i] = c == label ? q - 1.f : q;
        }
        if (g.psel)
            ent.each([&](int, long long i, float p) {
#pragma unroll
                for (int q = 0; q < NR; ++q) if (LinI::cls(q, hf) == i) dz[q] -= p;
            });
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            dz[i] = on && LinI::cls(i, hf) < g.V ? dz[i] : 0.f;
            dbs[i] += dz[i] * sc;
        }
        u32x4 dzp[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) dzp[s] = few_pack<T>(dz + EPC * s);
        if (g.dh) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                f32x16 o;
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = 0.f;
#pragma unroll
                for (int s = 0; s < NS; ++s) mma16(o, wt[b][s], dzp[s], (const T*)nullptr);
#pragma unroll
                for (int q = 0; q < 4; ++q) rows.put(o, q, sc, l32, 32 * b + 8 * q + 4 * hf);
            }
            rows.store((T*)g.dh, tile * 32, g.rows, g.D);
        }
        if (g.slab) {
            if (rowg) {                                   // every row has its own factor: it goes to the row
#pragma unroll
                for (int k = 0; k < NK; ++k) {
                    T x[EPC];
                    *reinterpret_cast<u32x4*>(x) = hx[k];
#pragma unroll
                    for (int e = 0; e < EPC; ++e) x[e] = from_f32<T>(on ? to_f32(x[e]) * sc : 0.f);
                    hx[k] = *reinterpret_cast<const u32x4*>(x);
                }
            }
            f32x16 c1;
#pragma unroll
            for (int e = 0; e < 16; ++e) c1[e] = 0.f;
#pragma unroll
            for (int s = 0; s < NS; ++s) mma16(c1, dzp[s], idc[s], (const T*)nullptr);
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = c1[e];
            u32x4 za[RS];
#pragma unroll
            for (int s = 0; s < RS; ++s) za[s] = few_pack<T>(v + EPC * s);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                f32x16 c2;
#pragma unroll
                for (int e = 0; e < 16; ++e) c2[e] = 0.f;
#pragma unroll
                for (int k = 0; k < BK; ++k) mma16(c2, hx[b * BK + k], idd[k], (const T*)nullptr);
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = c2[e];
#pragma unroll
                for (int s = 0; s < RS; ++s) mma16(dw[b], za[s], few_pack<T>(v + EPC * s), (const T*)nullptr);
            }
        }
    };
    fetch(0, wave);
    fetch(1, wave + nwaves);
    for (long long tile = wave; tile < tiles; tile += 2 * nwaves) {
        body(0, tile);
        if (tile + nwaves < tiles) body(1, tile + nwaves);
    }
    // the four waves' sums, then one slab per workgroup: [32 classes][NB * 32 features], db behind it
    __shared__ float red[4][32 * 32];
    const int wv = threadIdx.x >> 6;
    float* const slab = g.slab + (long long)blockIdx.x * g.slab_ld;
    if (g.slab) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int e = 0; e < 16; ++e) red[wv][LinI::cls(e, hf) * 32 + l32] = dw[b][e];
            __syncthreads();
            for (int i = threadIdx.x; i < 1024; i += 256) slab[(i >> 5) * (NB * 32) + 32 * b + (i & 31)] = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
            __syncthreads();
        }
    }
    if (g.dbslab) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            float s = dbs[i];
            for (int d = 16; d; d >>= 1) s += __shfl_xor(s, d);
            if (l32 == 0) red[wv][LinI::cls(i, hf)] = s;
        }
        __syncthreads();
        if (threadIdx.x < 8 * NG) g.dbslab[(long long)blockIdx.x * 32 + threadIdx.x] = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
    }
}

// dw = scale * sum of the slabs, db = sum of the db slabs: one workgroup per 4 elements of a slab's row, 64 lanes take the slabs in turn and add up in
// a fixed order
template <typename T>
__global__ __launch_bounds__(256) void lin_few_join_kernel(const LinFew g, int nslab, int ldd, T* dw, float* db) {
    __shared__ double part[4][64];
    const int x = threadIdx.x & 3, y = threadIdx.x >> 2;
    const int per = dw ? (g.D + 3) / 4 : 0;                 // workgroups of a class's row of dw; those of db behind them
    const int nw = g.V * per, c = blockIdx.x < nw ? blockIdx.x / per : -1, d = c < 0 ? (int)(blockIdx.x - nw) * 4 + x : (int)(blockIdx.x - c * per) * 4 + x;
    const bool in = c < 0 ? d < g.V : d < g.D;
    const float* p = c < 0 ? g.dbslab + d : g.slab + c * ldd + d;
    const long long step = c < 0 ? 32 : g.slab_ld;
    double s = 0.0;
    if (in)
#pragma unroll 4
        for (int k = y; k < nslab; k += 64) s += (double)p[k * step];
    part[x][y] = s;
    __syncthreads();
    for (int w = 32; w; w >>= 1) {
        if (y < w) part[x][y] += part[x][y + w];
        __syncthreads();
    }
    if (y == 0 && in) {
        s = part[x][0];
        if (c < 0) db[d] = (float)s;
        else dw[(long long)c * g.D + d] = from_f32<T>((float)s * (g.gstride ? 1.f : lin_row_scale(g.gout, 0, g.count, g.t, 1.f, 0)));
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------

// V <= 32, D <= 64, rows enough to fill the chip: below 4,096 rows the tiled product is as fast and this kernel's slab join is not
// worth it; the rule does not change with the alignment.
bool fea_lin_few(long long rows, int D, int V) { return V <= 32 && D <= 64 && rows >= 4096; }

// Workgroups, at least 4 tiles of 32 rows per wave.  Backward: two rounds of the two that a CU holds, since each leaves a slab.  Forward:
// many, so that the last round, which does not fill the chip (a CU holds three), is short: 1,024 took 576 us for 16.8 M rows, 8,192 take 499 us.
int fea_lin_few_blocks(long long rows, bool bwd) {
    const long long want = (rows + 511) / 512, most = bwd ? 1024 : 8192;
    return (int)(want < most ? want : most);
}

template <typename T, int NB, int NG> static void few_launch2(const LinFew& g, bool bwd, bool aln, unsigned grid, hipStream_t s) {
    if (bwd) {
        if (aln) hipLaunchKernelGGL((lin_few_bwd_kernel<T, NB, NG, true>), dim3(grid), dim3(256), 0, s, g);
        else     hipLaunchKernelGGL((lin_few_bwd_kernel<T, NB, NG, false>), dim3(grid), dim3(256), 0, s, g);
    } else {
        if (aln) hipLaunchKernelGGL((lin_few_fwd_kernel<T, NB, NG, true>), dim3(grid), dim3(256), 0, s, g);
        else     hipLaunchKernelGGL((lin_few_fwd_kernel<T, NB, NG, false>), dim3(grid), dim3(256), 0, s, g);
    }
}
template <typename T> static void few_launch(const LinFew& g, bool bwd, bool aln, unsigned grid, hipStream_t s) {
    const int ng = g.V <= 8 ? 1 : g.V <= 16 ? 2 : 4;
    if (g.D <= 32) {
        if (ng == 1) few_launch2<T, 1, 1>(g, bwd, aln, grid, s); else if (ng == 2) few_launch2<T, 1, 2>(g, bwd, aln, grid, s); else few_launch2<T, 1, 4>(g, bwd, aln, grid, s);
    } else {
        if (ng == 1) few_launch2<T, 2, 1>(g, bwd, aln, grid, s); else if (ng == 2) few_launch2<T, 2, 2>(g, bwd, aln, grid, s); else few_launch2<T, 2, 4>(g, bwd, aln, grid, s);
    }
}

static bool few_aligned(const LinFew& g, int dtype) {
    const int epc = dtype == FEA_BF16 ? 8 : 4;
    return g.D % epc == 0 && g.ldh % epc == 0 && g.ldw % epc == 0 && ((uintptr_t)g.h | (uintptr_t)g.w | (uintptr_t)g.dh) % 16 == 0;
}

int fea_lin_few_fwd(const LinFew& g, int dtype, hipStream_t s) {
    const unsigned grid = (unsigned)fea_lin_few_blocks(g.rows, false);
    if (dtype == FEA_BF16) few_launch<__bf16>(g, false, few_aligned(g, dtype), grid, s);
    else                   few_launch<float>(g, false, few_aligned(g, dtype), grid, s);
    FEA_LAUNCH_CHECK();
    return FEA_OK;
}

int fea_lin_few_bwd(LinFew g, int dtype, void* dw, float* db, hipStream_t s) {
    const int nslab = fea_lin_few_blocks(g.rows, true), ldd = g.D <= 32 ? 32 : 64;
    g.slab_ld = 32 * ldd;
    if (!dw) g.slab = nullptr;
    if (!db) g.dbslab = nullptr;
    if (dtype == FEA_BF16) few_launch<__bf16>(g, true, few_aligned(g, dtype), (unsigned)nslab, s);
    else                   few_launch<float>(g, true, few_aligned(g, dtype), (unsigned)nslab, s);
    FEA_LAUNCH_CHECK();
    const int n = (dw ? g.V * ((g.D + 3) / 4) : 0) + (db ? (g.V + 3) / 4 : 0);
    if (n) {
        const dim3 grid((unsigned)n);
        if (dtype == FEA_BF16) hipLaunchKernelGGL(lin_few_join_kernel<__bf16>, grid, dim3(256), 0, s, g, nslab, ldd, (__bf16*)dw, db);
        else                   hipLaunchKernelGGL(lin_few_join_kernel<float>, grid, dim3(256), 0, s, g, nslab, ldd, (float*)dw, db);
        FEA_LAUNCH_CHECK();
    }
    return FEA_OK;
}
