// Loss heads over many classes: a projection and a softmax cross entropy over its outputs, or a distillation loss against a
// teacher's top logits, forward and backward, without keeping the logits.
//
//   z_nv = (h_n . w_v + b_v) / T,  lse_n = log sum_v exp z_nv
//   cross entropy (T = 1):  l_n = lse_n - z_{n,t}                                   dz_nv = g_n (exp(z_nv - lse_n) - [v = t])
//   distillation:           l_n = T^2 sum_k p_nk (log p_nk - z_{n,i_nk} + lse_n)    dz_nv = g_n T (exp(z_nv - lse_n) - sum_{k: i_nk = v} p_nk)
//   dh = dz w, dw = dz^T h, db = sum_n dz
//
// Forward: the product with a log-sum-exp epilogue (linear_gemm.hip), the few selected logits by a gathered dot product, one
// pass that joins the column tiles of every row.  Backward, in pieces of the classes (and of the rows where there are very
// many): the product again with the softmax gradient as its epilogue, the selected entries written over it from the forward's
// fp32 values, then two products.  The workspace is bounded by the piece, not by rows x classes.
#include "linear_loss.h"
#include <limits.h>
#include <math.h>
#include <stdlib.h>

// ---- layouts ------------------------------------------------------------------------------------------------------------

// out[r][c] = in[r][c], zero for C <= c < Cpad: rows of a length that is no multiple of 16 bytes
template <typename T>
__global__ __launch_bounds__(256) void lin_pack_kernel(const T* __restrict__ in, long long ld, T* __restrict__ out, int Cpad, int C, long long total) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long r = i / Cpad;
        const int c = (int)(i - r * Cpad);
        out[i] = c < C ? in[r * ld + c] : from_f32<T>(0.f);
    }
}

// out[c][r] = in[r][c] (r < R), zero for R <= r < Rpad; rows whose gate is 0 count as zeros: what an ignored row holds (an
// infinity, a NaN) meets a zero gradient in the weight's product, and 0 x NaN must not reach the weight.  gout (nullable): rows
// times their own upstream gradient.
template <typename T>
__global__ __launch_bounds__(256) void lin_transpose_kernel(const T* __restrict__ in, long long ld, T* __restrict__ out, long long ldo,
                                                            long long R, long long Rpad, int C, const float2* __restrict__ stat,
                                                            const float* __restrict__ gout, float t) {
    __shared__ T tile[64][64 + 8 / sizeof(T)];
    const long long r0 = (long long)blockIdx.x * 64;
    const int c0 = blockIdx.y * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
#pragma unroll 4
    for (int i = y; i < 64; i += 4) {
        const long long r = r0 + i;
        T v = r < R && c0 + x < C && (!stat || stat[r].y != 0.f) ? in[r * ld + c0 + x] : from_f32<T>(0.f);
        if (gout && r < R && stat[r].y != 0.f) v = from_f32<T>(to_f32(v) * lin_row_scale(gout, 1, nullptr, t, 1.f, r));
        tile[i][x] = v;
    }
    __syncthreads();
#pragma unroll 4
    for (int i = y; i < 64; i += 4)
        if (c0 + i < C && r0 + x < Rpad) out[(long long)(c0 + i) * ldo + r0 + x] = tile[x][i];
}

// ---- forward ------------------------------------------------------------------------------------------------------------

// a . b over D elements by L lanes (a power of two), the sum in each of them
template <typename T, bool VEC>
__device__ __forceinline__ float lin_dot(const T* a, const T* b, int D, int lane, int L) {
    constexpr int EPC = Elem<T>::EPC;
    float s = 0.f;
    if constexpr (VEC) {
        for (int d = lane * EPC; d < D; d += L * EPC) {
            T x[EPC], y[EPC];
            *reinterpret_cast<u32x4*>(x) = *reinterpret_cast<const u32x4*>(a + d);
            *reinterpret_cast<u32x4*>(y) = *reinterpret_cast<const u32x4*>(b + d);
#pragma unroll
            for (int q = 0; q < EPC; ++q) s += to_f32(x[q]) * to_f32(y[q]);
        }
    } else
        for (int d = lane; d < D; d += L) s += to_f32(a[d]) * to_f32(b[d]);
    for (int d = L >> 1; d; d >>= 1) s += __shfl_xor(s, d);
    return s;
}

// zsel[n][k] = h_n . w_{index[n][k]} + b: L lanes (a power of two that covers the row in 16-byte loads, 64 at most) per entry.
// Absent entries (index < 0 or >= V) are not read.
template <typename T>
__global__ __launch_bounds__(256) void lin_select_kernel(const T* __restrict__ h, long long ldh, const T* __restrict__ w, long long ldw,
                                                         const float* __restrict__ bias, const long long* __restrict__ index, int K,
                                                         float* __restrict__ zsel, long long entries, int D, int V, int L, int vec) {
    const int lane = threadIdx.x & (L - 1), per = 256 / L;
    for (long long b0 = (long long)blockIdx.x * per; b0 < entries; b0 += (long long)gridDim.x * per) {
        const long long e = b0 + threadIdx.x / L;
        const long long i = e < entries ? index[e] : -1;
        if (i < 0 || i >= V) continue;                       // (the L lanes of an entry go together)
        const T* a = h + e / K * ldh;
        const float s = vec ? lin_dot<T, true>(a, w + i * ldw, D, lane, L) : lin_dot<T, false>(a, w + i * ldw, D, lane, L);
        if (lane == 0) zsel[e] = bias ? s + bias[i] : s;
    }
}

struct LinJoin {
    const float2* part; int ntn;          // [rows][ntn]
    float* zsel;                          // [rows][K]
    const long long* index;               // [rows][K]
    const void* tlog; int tdt;            // NULL: cross entropy (K = 1)
    long long ignore;
    float t, inv_t;
    float2* stat;                         // nullable
    float *dsel, *psel;                   // nullable, [rows][K]
    float* loss_rows;                     // nullable
    double* bsum; int* bcnt;              // nullable: sums of each block
    long long rows; int K, V, G;          // G lanes per row (power of two <= 64)
};

__device__ __forceinline__ float lin_tlog(const LinJoin& j, long long e) {
    return j.tdt == FEA_BF16 ? (float)((const __bf16*)j.tlog)[e] : ((const float*)j.tlog)[e];
}

// G lanes join the column tiles of a row and turn its selected logits into the loss and the gradient at the selected classes.
__device__ __forceinline__ void lin_join_body(const LinJoin& j, int G, int gl, long long row, bool in) {
    float loss = 0.f;
    bool counts = false;
    {
        float mx = -INFINITY, sum = 0.f;
        if (in) {
            for (int i = gl; i < j.ntn; i += G) mx = fmaxf(mx, j.part[row * j.ntn + i].x);
        }
        for (int d = G >> 1; d; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
        const float base = mx == -INFINITY ? 0.f : mx;
        if (in)
            for (int i = gl; i < j.ntn; i += G) { const float2 p = j.part[row * j.ntn + i]; sum += p.y * expf(p.x - base); }
        for (int d = G >> 1; d; d >>= 1) sum += __shfl_xor(sum, d);
        float lse = logf(sum) + base;
        const long long e0 = row * j.K;
        if (!j.tlog) {
            const long long t = in ? j.index[row] : j.ignore;
            counts = t != j.ignore;
            if (counts) {
                if (t < 0 || t >= j.V) { lse = NAN; loss = NAN; }                 // a label that names no class: loud, and not read
                else { loss = lse - j.zsel[row]; if (loss < 0.f) loss = 0.f; }    // (the two sums are rounded apart: -1e-7 is 0)
                if (gl == 0 && j.dsel) j.dsel[row] = expm1f(-loss);
            } else if (in && gl == 0 && j.dsel) j.dsel[row] = 0.f;
        } else {
            // teacher: softmax over its entries (those with a class and a logit above -inf)
            float tm = -INFINITY;
            bool bad = false;
            if (in)
                for (int k = gl; k < j.K; k += G) {
                    const long long i = j.index[e0 + k];
                    if (i >= j.V) bad = true;
                    if (i >= 0) { const float a = lin_tlog(j, e0 + k) * j.inv_t; bad |= !(a < INFINITY); tm = fmaxf(tm, a); }
                }
            for (int d = G >> 1; d; d >>= 1) { tm = fmaxf(tm, __shfl_xor(tm, d)); bad |= __shfl_xor((int)bad, d) != 0; }
            counts = in && (tm != -INFINITY || bad);
            float ts = 0.f;
            if (counts && !bad)
                for (int k = gl; k < j.K; k += G) if (j.index[e0 + k] >= 0) ts += expf(lin_tlog(j, e0 + k) * j.inv_t - tm);
            for (int d = G >> 1; d; d >>= 1) ts += __shfl_xor(ts, d);
            const float lt = logf(ts);
            if (bad) lse = NAN;
            for (int k = gl; in && k < j.K; k += G) {
                const long long i = j.index[e0 + k];
                float ds = 0.f, ps = 0.f;
                if (counts && i >= 0) {
                    if (bad) { loss = ds = ps = NAN; }
                    else {
                        const float lp = lin_tlog(j, e0 + k) * j.inv_t - tm - lt, p = expf(lp);
                        const float zq = j.zsel[e0 + k] * j.inv_t - lse;
                        if (p > 0.f) loss += p * (lp - zq);
                        ps = p;
                        if (j.dsel) {
                            float all = 0.f;              // the same class twice in a row: each entry holds the sum over both
                            for (int q = 0; q < j.K; ++q) if (j.index[e0 + q] == i) all += expf(lin_tlog(j, e0 + q) * j.inv_t - tm - lt);
                            ds = expf(zq) - all;
                        }
                    }
                }
                if (j.dsel) j.dsel[e0 + k] = ds;
                if (j.psel) j.psel[e0 + k] = ps;
            }
            for (int d = G >> 1; d; d >>= 1) loss += __shfl_xor(loss, d);
            loss = counts ? loss * j.t * j.t : 0.f;
        }
        if (in && gl == 0) {
            if (j.stat) j.stat[row] = make_float2(counts ? lse : 0.f, counts ? 1.f : 0.f);
            if (j.loss_rows) j.loss_rows[row] = loss;
        }
    }
    if (j.bsum) {
        __shared__ double ls[256];
        __shared__ int lc[256];
        ls[threadIdx.x] = gl == 0 ? (double)loss : 0.0;
        lc[threadIdx.x] = gl == 0 && counts;
        __syncthreads();
        for (int d = 128; d; d >>= 1) {
            if ((int)threadIdx.x < d) { ls[threadIdx.x] += ls[threadIdx.x + d]; lc[threadIdx.x] += lc[threadIdx.x + d]; }
            __syncthreads();
        }
        if (threadIdx.x == 0) { j.bsum[blockIdx.x] = ls[0]; j.bcnt[blockIdx.x] = lc[0]; }
    }
}

__global__ __launch_bounds__(256) void lin_join_kernel(const LinJoin j) {
    const long long row = (long long)blockIdx.x * (256 / j.G) + threadIdx.x / j.G;
    lin_join_body(j, j.G, threadIdx.x % j.G, row, row < j.rows);
}

// The same for few rows, one workgroup per row, the selected logits and the join in one launch: all waves take entries, then the
// first one joins.
template <typename T>
__global__ __launch_bounds__(256) void lin_join_rows_kernel(const LinJoin j, const T* h, long long ldh, const T* w, long long ldw, const float* bias, int D, int vec) {
    const long long row = blockIdx.x;
    for (int k = threadIdx.x >> 6; k < j.K; k += 4) {
        const long long i = j.index[row * j.K + k];
        if (i < 0 || i >= j.V) continue;
        const float s = vec ? lin_dot<T, true>(h + row * ldh, w + i * ldw, D, threadIdx.x & 63, 64) : lin_dot<T, false>(h + row * ldh, w + i * ldw, D, threadIdx.x & 63, 64);
        if ((threadIdx.x & 63) == 0) j.zsel[row * j.K + k] = bias ? s + bias[i] : s;
    }
    __threadfence_block();
    __syncthreads();
    lin_join_body(j, 64, threadIdx.x & 63, row, threadIdx.x < 64);
}

// loss[0] = sum, or sum / rows that count (0 where none does); count[0] = rows that count
__global__ __launch_bounds__(1024) void lin_total_kernel(const double* bsum, const int* bcnt, long long n, int mean, float* loss, int* count) {
    __shared__ double ls[1024];
    __shared__ long long lc[1024];
    double s = 0.0;
    long long c = 0;
    for (long long i = threadIdx.x; i < n; i += 1024) { s += bsum[i]; c += bcnt[i]; }
    ls[threadIdx.x] = s; lc[threadIdx.x] = c;
    __syncthreads();
    for (int d = 512; d; d >>= 1) {
        if ((int)threadIdx.x < d) { ls[threadIdx.x] += ls[threadIdx.x + d]; lc[threadIdx.x] += lc[threadIdx.x + d]; }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        *loss = (float)(mean ? (lc[0] ? ls[0] / (double)lc[0] : 0.0) : ls[0]);
        *count = (int)lc[0];
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------------

// dz at the selected classes of the piece [v0, v0 + N): softmax - teacher, from the forward's fp32 values.  Entries that name the
// same class hold the same value.
template <typename T>
__global__ __launch_bounds__(256) void lin_scatter_kernel(const long long* __restrict__ index, const float* __restrict__ dsel, int K,
                                                          const float2* __restrict__ stat, T* dz, long long lddz, T* dzt, long long lddzt, long long v0, int N, long long entries) {
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    if (e >= entries) return;
    const long long m = e / K, i = index[e] - v0;
    if (i < 0 || i >= N) return;
    if (stat[m].y == 0.f) return;
    const T v = from_f32<T>(dsel[e]);
    dz[m * lddz + i] = v;
    if (dzt) dzt[i * lddzt + m] = v;
}

// out = acc + slabs in split order; acc (nullable) is the fp32 sum of earlier pieces, accout where later ones follow
template <typename T>
__global__ __launch_bounds__(256) void lin_reduce_kernel(const float* __restrict__ slab, int splits, long long n, const float* acc, float* accout, T* out) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        float s = acc ? acc[i] : 0.f;
        for (int p = 0; p < splits; ++p) s += slab[p * n + i];
        if (accout) accout[i] = s;
        if (out) out[i] = from_f32<T>(s);
    }
}

// Partial bias gradient of one chunk of LIN_DB_TILES row tiles: sum over its tiles of colsum[tile][v] - sum of g * teacher share over
// its rows' entries that name v (psel NULL: share 1).  One workgroup owns 256 classes of one chunk; its waves walk the entries in
// order and the lane that owns a class adds its hits: the order is fixed.
static constexpr int LIN_DB_TILES = 16;
__global__ __launch_bounds__(256) void lin_dbias_kernel(const float* __restrict__ colsum, int tiles, long long ldcol, const long long* __restrict__ index,
                                                        const float* __restrict__ psel, int K, const float2* __restrict__ stat, const float* gout,
                                                        int gstride, const int* count, float t, long long v0, int N, long long entries,
                                                        long long chunk, double* out) {
    __shared__ double part[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b0 = blockIdx.x * 256;
    const long long ea = blockIdx.y * chunk, eb = ea + chunk < entries ? ea + chunk : entries;
    double acc[4] = {0.0, 0.0, 0.0, 0.0};             // classes b0 + lane + 64 q
    for (long long e0 = ea + wave * 64; e0 < eb; e0 += 256) {
        const long long e = e0 + lane;
        const long long i = e < eb ? index[e] - v0 - b0 : -1;
        float val = 0.f;
        bool hit = i >= 0 && i < 256 && b0 + i < N;
        if (hit) {
            const long long m = e / K;
            const float gate = stat[m].y;
            hit = gate != 0.f;
            if (hit) val = (psel ? psel[e] : 1.f) * lin_row_scale(gout, gstride, count, t, gate, m);
        }
        unsigned long long mask = __ballot(hit);
        while (mask) {
            const int l = __builtin_ctzll(mask);
            mask &= mask - 1;
            const int c = __shfl((int)i, l);
            const float v = __shfl(val, l);
            if ((c & 63) == lane) {
#pragma unroll
                for (int q = 0; q < 4; ++q) if (c >> 6 == q) acc[q] += (double)v;
            }
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) part[wave][lane + 64 * q] = acc[q];
    __syncthreads();
    const int v = b0 + threadIdx.x;
    if (v < N) {
        double s = -(part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x]);
        const int t1 = min(tiles, ((int)blockIdx.y + 1) * LIN_DB_TILES);
        for (int i = blockIdx.y * LIN_DB_TILES; i < t1; ++i) s += (double)colsum[i * ldcol + v];
        out[(long long)blockIdx.y * N + v] = s;
    }
}

// db[v] (+)= sum over the chunks, in order
__global__ __launch_bounds__(256) void lin_dbias_join_kernel(const double* __restrict__ part, int chunks, int N, float* db, int accumulate) {
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v >= N) return;
    double s = accumulate ? (double)db[v] : 0.0;
#pragma unroll 8
    for (int c = 0; c < chunks; ++c) s += part[(long long)c * N + v];
    db[v] = (float)s;
}

// ---- host ---------------------------------------------------------------------------------------------------------------

static inline long long up(long long a, long long b) { return (a + b - 1) / b * b; }

// A bump allocator over the caller's workspace; with base == NULL it only counts.
struct LinCarve {
    char* base; size_t at = 0;
    template <typename P> P* take(long long n) { P* p = reinterpret_cast<P*>(base + at); at += (size_t)up(n * (long long)sizeof(P), 256); return p; }
};

struct LinDims {
    long long rows; int D, V, K, dtype, es, epc;
    int Dp;                       // D rounded up to 16 bytes: operands with another D are copied with zeros behind it
    bool packed() const { return Dp != D; }
    bool wide;                    // row strides of 2^21 elements or more (a slice of something very wide): the 128 tile, which has 64-bit offsets
};

static LinDims lin_dims(long long rows, int D, int V, int K, int dtype) {
    LinDims d{rows, D, V, K, dtype, dtype == FEA_BF16 ? 2 : 4, dtype == FEA_BF16 ? 8 : 4, 0, false};
    d.Dp = (int)up(D, d.epc);
    return d;
}

// Forward: rows in chunks that bound the partial table to 128 MB.
struct LinFwd { long long rc; int tile, ntn, G; long long blocks; };
static LinFwd lin_fwd_plan(const LinDims& d) {
    LinFwd p;
    const long long cap = (1ll << 24) / ((d.V + 127) / 128);
    p.rc = cap < 256 ? 256 : cap / 256 * 256;
    if (p.rc > d.rows) p.rc = d.rows;
    p.tile = d.rows <= 64 ? 64 : d.wide ? 128 : fea_lin_tile(d.dtype, p.rc, d.V, d.Dp, false).tile;
    p.ntn = (d.V + p.tile - 1) / p.tile;
    p.G = 1;
    while (p.G < 64 && (p.G < p.ntn || p.G < d.K)) p.G *= 2;
    p.blocks = p.tile == 64 ? d.rows : (d.rows + 256 / p.G - 1) / (256 / p.G) + (p.rc ? d.rows / p.rc + 1 : 0);     // every chunk rounds up by itself
    return p;
}

// Backward: pieces of rc rows x vc classes.  dz and its transpose take rc x vc elements each: 2^28 at most
// (FEA_AMD_LINEAR_PIECE: tests, many pieces on small shapes).
static long long lin_piece() {
    const char* e = getenv("FEA_AMD_LINEAR_PIECE");
    const long long v = e ? atoll(e) : 0;
    return v >= 1 << 14 && v < 1 << 28 ? v : 1ll << 28;
}
struct LinBwd { long long rc; int vc, nrc, nvc, tz; LinTile th, tw; };
static LinBwd lin_bwd_plan(const LinDims& d) {
    LinBwd p;
    const long long piece = lin_piece();
    p.rc = d.rows < 32768 ? d.rows : 32768;
    if (d.V <= 1024) { const long long most = piece / up(d.V > d.D ? d.V : d.D, 256); p.rc = d.rows < most ? d.rows : most < 256 ? 256 : most / 256 * 256; }
    long long vc = piece / (p.rc > 0 ? up(p.rc, 256) : 1) / 256 * 256;
    if (vc < 256) vc = 256;
    p.vc = (int)(vc < d.V ? vc : d.V);
    p.nrc = p.rc ? (int)((d.rows + p.rc - 1) / p.rc) : 0;
    p.nvc = (d.V + p.vc - 1) / p.vc;
    p.tz = d.wide ? 128 : fea_lin_tile(d.dtype, p.rc, p.vc, d.Dp, false).tile;
    p.th = fea_lin_tile(d.dtype, p.rc, d.D, p.vc, true);
    p.tw = fea_lin_tile(d.dtype, p.vc, d.D, p.rc, true);
    return p;
}

struct LinFwdWs { void *hp, *wp; float2* part; float* zsel; double* bsum; int* bcnt; };
static size_t lin_fwd_carve(const LinDims& d, const LinFwd& p, char* base, LinFwdWs& w) {
    LinCarve c{base};
    if (fea_lin_few(d.rows, d.D, d.V)) {
        w = LinFwdWs{};
        w.bsum = c.take<double>(fea_lin_few_blocks(d.rows));
        w.bcnt = c.take<int>(fea_lin_few_blocks(d.rows));
        return c.at;
    }
    w.part = c.take<float2>(p.rc * ((d.V + (p.tile == 64 ? 63 : 127)) / (p.tile == 64 ? 64 : 128)));           // (sized for the smaller tile: row strides may ask for it)
    w.zsel = c.take<float>(d.rows * d.K);
    w.bsum = c.take<double>(p.blocks);
    w.bcnt = c.take<int>(p.blocks);
    w.hp = w.wp = nullptr;
    if (d.packed() && p.tile == 256) { w.hp = c.take<char>(p.rc * d.Dp * d.es); w.wp = c.take<char>((long long)d.V * d.Dp * d.es); }
    return c.at;
}

struct LinBwdWs { void *hp, *wp, *ht, *wt, *dz, *dzt; float *slab, *acch, *accw, *colsum; double* dbpart; };
static size_t lin_bwd_carve(const LinDims& d, const LinBwd& p, int want, char* base, LinBwdWs& w) {
    LinCarve c{base};
    const long long vp = up(p.vc, d.epc), rp = up(p.rc, d.epc);
    w = LinBwdWs{};
    if (fea_lin_few(d.rows, d.D, d.V)) {
        if (want & 2) w.slab = c.take<float>(fea_lin_few_blocks(d.rows) * 32ll * 64);
        if (want & 4) w.colsum = c.take<float>(fea_lin_few_blocks(d.rows) * 32ll);
        w.dz = c.take<char>(256);
        return c.at;
    }
    if (d.packed() && p.tz == 256) { w.hp = c.take<char>(p.rc * d.Dp * d.es); w.wp = c.take<char>((long long)p.vc * d.Dp * d.es); }
    w.dz = c.take<char>(p.rc * vp * d.es);
    if (want & 2) { w.dzt = c.take<char>(p.vc * rp * d.es); w.ht = c.take<char>(d.D * rp * d.es); }
    if (want & 1) w.wt = c.take<char>(d.D * vp * d.es);
    long long slab = 0;
    if ((want & 1) && (p.th.splits > 1 || p.nvc > 1)) slab = p.th.splits * p.rc * d.D;
    if ((want & 2) && (p.tw.splits > 1 || p.nrc > 1) && slab < (long long)p.tw.splits * p.vc * d.D) slab = (long long)p.tw.splits * p.vc * d.D;
    w.slab = c.take<float>(slab);
    if ((want & 1) && p.nvc > 1) w.acch = c.take<float>(p.rc * d.D);
    if ((want & 2) && p.nrc > 1) w.accw = c.take<float>((long long)d.V * d.D);
    if (want & 4) { const long long t = (p.rc + 127) / 128; w.colsum = c.take<float>(t * up(p.vc, 64)); w.dbpart = c.take<double>((t + LIN_DB_TILES - 1) / LIN_DB_TILES * p.vc); }
    return c.at;
}

extern "C" size_t fea_linear_loss_ws_bytes(long long rows, int D, int V, int K, int dtype, int grads) {
    if (rows <= 0 || D <= 0 || V <= 0 || K <= 0 || (dtype != FEA_F32 && dtype != FEA_BF16)) return 0;
    const LinDims d = lin_dims(rows, D, V, K, dtype);
    if (!grads) { LinFwdWs w; return lin_fwd_carve(d, lin_fwd_plan(d), nullptr, w); }
    LinBwdWs w;
    return lin_bwd_carve(d, lin_bwd_plan(d), grads, nullptr, w);
}

static int lin_pack(const LinDims& d, const void* in, long long ld, void* out, long long R, hipStream_t s) {
    const long long n = R * d.Dp;
    const unsigned grid = (unsigned)(n / 1024 < 1 ? 1 : n / 1024 > 16384 ? 16384 : n / 1024);
    if (d.dtype == FEA_BF16) hipLaunchKernelGGL(lin_pack_kernel<__bf16>, dim3(grid), dim3(256), 0, s, (const __bf16*)in, ld, (__bf16*)out, d.Dp, d.D, n);
    else                     hipLaunchKernelGGL(lin_pack_kernel<float>, dim3(grid), dim3(256), 0, s, (const float*)in, ld, (float*)out, d.Dp, d.D, n);
    FEA_LAUNCH_CHECK();
    return FEA_OK;
}

static int lin_transpose(const LinDims& d, const void* in, long long ld, void* out, long long ldo, long long R, long long Rpad, const float2* stat, const float* gout, float t, hipStream_t s) {
    const dim3 grid((unsigned)((Rpad + 63) / 64), (unsigned)((d.D + 63) / 64));
    if (d.dtype == FEA_BF16) hipLaunchKernelGGL(lin_transpose_kernel<__bf16>, grid, dim3(256), 0, s, (const __bf16*)in, ld, (__bf16*)out, ldo, R, Rpad, d.D, stat, gout, t);
    else                     hipLaunchKernelGGL(lin_transpose_kernel<float>, grid, dim3(256), 0, s, (const float*)in, ld, (float*)out, ldo, R, Rpad, d.D, stat, gout, t);
    FEA_LAUNCH_CHECK();
    return FEA_OK;
}

static int lin_reduce(const LinDims& d, const float* slab, int splits, long long n, const float* acc, float* accout, void* out, hipStream_t s) {
    const unsigned grid = (unsigned)(n / 1024 < 1 ? 1 : n / 1024 > 8192 ? 8192 : n / 1024);
    if (d.dtype == FEA_BF16) hipLaunchKernelGGL(lin_reduce_kernel<__bf16>, dim3(grid), dim3(256), 0, s, slab, splits, n, acc, accout, (__bf16*)out);
    else                     hipLaunchKernelGGL(lin_reduce_kernel<float>, dim3(grid), dim3(256), 0, s, slab, splits, n, acc, accout, (float*)out);
    FEA_LAUNCH_CHECK();
    return FEA_OK;
}

#define LIN_TRY(x) do { const int rc_ = (x); if (rc_ != FEA_OK) return rc_; } while (0)

static int lin_check(const char* who, const LinDims& d, const void* h, long long ldh, const void* w, long long ldw, const float* bias) {
    FEA_CHECK(d.dtype == FEA_F32 || d.dtype == FEA_BF16, FEA_E_BADARG, "%s: dtype %d", who, d.dtype);
    FEA_CHECK(d.rows >= 1 && d.rows <= INT_MAX / 2, FEA_E_UNSUPPORTED_SHAPE, "%s: %lld rows, 1..%d are served", who, d.rows, INT_MAX / 2);
    FEA_CHECK(d.D >= 1 && d.D <= (1 << 16), FEA_E_UNSUPPORTED_SHAPE, "%s: %d features, 1..%d are served", who, d.D, 1 << 16);
    FEA_CHECK(d.V >= 1 && d.V <= (1 << 24), FEA_E_UNSUPPORTED_SHAPE, "%s: %d classes, 1..%d are served", who, d.V, 1 << 24);
    FEA_CHECK(d.K >= 1 && d.K <= 256, FEA_E_UNSUPPORTED_SHAPE, "%s: %d teacher entries per row, 1..256 are served", who, d.K);
    FEA_CHECK(h && w, FEA_E_BADARG, "%s: null operand", who);
    FEA_CHECK(ldh >= d.D && ldw >= d.D, FEA_E_BADARG, "%s: row stride below the %d features (hidden %lld, weight %lld)", who, d.D, ldh, ldw);
    FEA_CHECK(((uintptr_t)h | (uintptr_t)w) % d.es == 0 && (uintptr_t)bias % 4 == 0, FEA_E_BADARG, "%s: misaligned operand", who);
    if (!d.packed())
        FEA_CHECK(((uintptr_t)h | (uintptr_t)w) % 16 == 0 && ldh % d.epc == 0 && ldw % d.epc == 0, FEA_E_BADARG,
                  "%s: hidden and weight need 16-byte aligned rows when the features are a multiple of %d", who, d.epc);
    return FEA_OK;
}

static int lin_forward(const char* who, LinDims d, const void* h, long long ldh, const void* w, long long ldw, const float* bias, LinJoin j,
                       float* loss, int* count, int mean, void* ws, size_t ws_bytes, hipStream_t s) {
    LIN_TRY(lin_check(who, d, h, ldh, w, ldw, bias));
    d.wide = !d.packed() && (ldh >= 1 << 21 || ldw >= 1 << 21);
    const LinFwd p = lin_fwd_plan(d);
    LinFwdWs b;
    const size_t need = lin_fwd_carve(d, p, (char*)ws, b);
    FEA_CHECK(ws && (uintptr_t)ws % 256 == 0 && ws_bytes >= need, FEA_E_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, needed (got %zu)", who, need, ws_bytes);
    FEA_CHECK(!loss == !count, FEA_E_BADARG, "%s: loss and count go together", who);
    FEA_CHECK(loss || j.loss_rows, FEA_E_BADARG, "%s: nothing to write", who);

    if (fea_lin_few(d.rows, d.D, d.V)) {
        LinFew f{};
        f.h = h; f.w = w; f.ldh = ldh; f.ldw = ldw; f.bias = bias; f.index = j.index; f.tlog = j.tlog; f.tdt = j.tdt; f.ignore = j.ignore;
        f.t = j.t; f.inv_t = j.inv_t; f.stat = j.stat; f.psel = j.psel; f.loss_rows = j.loss_rows;
        f.bsum = loss ? b.bsum : nullptr; f.bcnt = b.bcnt; f.rows = d.rows; f.D = d.D; f.V = d.V; f.K = d.K;
        LIN_TRY(fea_lin_few_fwd(f, d.dtype, s));
        if (loss) {
            hipLaunchKernelGGL(lin_total_kernel, dim3(1), dim3(1024), 0, s, (const double*)b.bsum, (const int*)b.bcnt, (long long)fea_lin_few_blocks(d.rows), mean, loss, count);
            FEA_LAUNCH_CHECK();
        }
        return FEA_OK;
    }
    const long long entries = d.rows * d.K;
    if (p.tile != 64) {
        int lanes = 1;
        while (lanes < 64 && lanes * d.epc < d.D) lanes *= 2;
        const long long blocks = (entries * lanes + 255) / 256;
        const unsigned grid = (unsigned)(blocks < 1 << 16 ? blocks : 1 << 16);
        if (d.dtype == FEA_BF16) hipLaunchKernelGGL(lin_select_kernel<__bf16>, dim3(grid), dim3(256), 0, s, (const __bf16*)h, ldh, (const __bf16*)w, ldw, bias, j.index, d.K, b.zsel, entries, d.D, d.V, lanes, d.packed() ? 0 : 1);
        else                     hipLaunchKernelGGL(lin_select_kernel<float>, dim3(grid), dim3(256), 0, s, (const float*)h, ldh, (const float*)w, ldw, bias, j.index, d.K, b.zsel, entries, d.D, d.V, lanes, d.packed() ? 0 : 1);
        FEA_LAUNCH_CHECK();
    }
    const void* wm = w;
    long long ldwm = ldw;
    const bool pack = d.packed() && p.tile == 256;       // (the other kernels take rows of any alignment)
    const int Kg = pack ? d.Dp : d.D;
    if (pack) { LIN_TRY(lin_pack(d, w, ldw, b.wp, d.V, s)); wm = b.wp; ldwm = d.Dp; }
    long long blk = 0;
    for (long long r = 0; r < d.rows; r += p.rc) {
        const long long n = d.rows - r < p.rc ? d.rows - r : p.rc;
        const void* hm = (const char*)h + r * ldh * d.es;
        long long ldhm = ldh;
        if (pack) { LIN_TRY(lin_pack(d, hm, ldh, b.hp, n, s)); hm = b.hp; ldhm = d.Dp; }
        LinGemm g{};
        g.a = hm; g.lda = ldhm; g.b = wm; g.ldb = ldwm; g.M = (int)n; g.N = d.V; g.K = Kg;
        g.bias = bias; g.inv_t = j.inv_t; g.part = b.part;
        if (p.tile == 64) LIN_TRY(fea_lin_rows(d.dtype, !d.packed(), g, s));
        else LIN_TRY(fea_lin_gemm(LIN_LSE, d.dtype, p.tile, g, s));
        LinJoin q = j;
        q.part = b.part; q.ntn = p.ntn; q.rows = n; q.K = d.K; q.V = d.V; q.G = p.G;
        q.zsel = b.zsel + r * d.K; q.index = j.index + r * d.K;
        if (q.tlog) q.tlog = (const char*)j.tlog + r * d.K * (j.tdt == FEA_BF16 ? 2 : 4);
        if (q.stat) q.stat += r;
        if (q.dsel) q.dsel += r * d.K;
        if (q.psel) q.psel += r * d.K;
        if (q.loss_rows) q.loss_rows += r;
        q.bsum = loss ? b.bsum + blk : nullptr; q.bcnt = b.bcnt + blk;
        const long long grid = p.tile == 64 ? n : (n + 256 / p.G - 1) / (256 / p.G);
        if (p.tile != 64)               hipLaunchKernelGGL(lin_join_kernel, dim3((unsigned)grid), dim3(256), 0, s, q);
        else if (d.dtype == FEA_BF16)   hipLaunchKernelGGL(lin_join_rows_kernel<__bf16>, dim3((unsigned)grid), dim3(256), 0, s, q, (const __bf16*)h, ldh, (const __bf16*)w, ldw, bias, d.D, d.packed() ? 0 : 1);
        else                            hipLaunchKernelGGL(lin_join_rows_kernel<float>, dim3((unsigned)grid), dim3(256), 0, s, q, (const float*)h, ldh, (const float*)w, ldw, bias, d.D, d.packed() ? 0 : 1);
        FEA_LAUNCH_CHECK();
        blk += grid;
    }
    if (loss) {
        hipLaunchKernelGGL(lin_total_kernel, dim3(1), dim3(1024), 0, s, (const double*)b.bsum, (const int*)b.bcnt, blk, mean, loss, count);
        FEA_LAUNCH_CHECK();
    }
    return FEA_OK;
}

extern "C" int fea_linear_ce_fwd(const void* h, long long ldh, const void* w, long long ldw, const float* bias, const long long* target,
                                 long long ignore_index, float* stat, float* dsel, float* loss_rows, float* loss, int* count, int mean,
                                 void* ws, size_t ws_bytes, long long rows, int D, int V, int dtype, void* stream) {
    FEA_CHECK(target, FEA_E_BADARG, "fea_linear_ce_fwd: null target");
    LinJoin j{};
    j.index = target; j.ignore = ignore_index; j.t = j.inv_t = 1.f;
    j.stat = (float2*)stat; j.dsel = dsel; j.loss_rows = loss_rows;
    return lin_forward("fea_linear_ce_fwd", lin_dims(rows, D, V, 1, dtype), h, ldh, w, ldw, bias, j, loss, count, mean, ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int fea_linear_kd_fwd(const void* h, long long ldh, const void* w, long long ldw, const float* bias, const void* teacher_logits,
                                 int teacher_dtype, const long long* teacher_index, int K, float temperature, float* stat, float* dsel, float* psel,
                                 float* loss_rows, float* loss, int* count, int mean, void* ws, size_t ws_bytes, long long rows, int D, int V,
                                 int dtype, void* stream) {
    FEA_CHECK(teacher_logits && teacher_index, FEA_E_BADARG, "fea_linear_kd_fwd: null teacher");
    FEA_CHECK(teacher_dtype == FEA_F32 || teacher_dtype == FEA_BF16, FEA_E_BADARG, "fea_linear_kd_fwd: teacher dtype %d", teacher_dtype);
    FEA_CHECK(temperature > 0.f && isfinite(temperature) && isfinite(1.f / temperature), FEA_E_BADARG, "fea_linear_kd_fwd: temperature %g", (double)temperature);
    LinJoin j{};
    j.index = teacher_index; j.tlog = teacher_logits; j.tdt = teacher_dtype; j.t = temperature; j.inv_t = 1.f / temperature;
    j.stat = (float2*)stat; j.dsel = dsel; j.psel = psel; j.loss_rows = loss_rows;
    return lin_forward("fea_linear_kd_fwd", lin_dims(rows, D, V, K, dtype), h, ldh, w, ldw, bias, j, loss, count, mean, ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int fea_linear_loss_bwd(const void* h, long long ldh, const void* w, long long ldw, const float* bias, const long long* index, int K,
                                   const float* stat, const float* dsel, const float* psel, const int* count, const float* gout, int gout_stride,
                                   float temperature, void* dh, void* dw, float* db, void* ws, size_t ws_bytes, long long rows, int D, int V,
                                   int dtype, void* stream) {
    const char* who = "fea_linear_loss_bwd";
    LinDims d = lin_dims(rows, D, V, K, dtype);
    hipStream_t s = (hipStream_t)stream;
    LIN_TRY(lin_check(who, d, h, ldh, w, ldw, bias));
    d.wide = !d.packed() && (ldh >= 1 << 21 || ldw >= 1 << 21);
    FEA_CHECK(index && stat && dsel && gout, FEA_E_BADARG, "%s: null operand", who);
    FEA_CHECK(gout_stride == 0 || gout_stride == 1, FEA_E_BADARG, "%s: gout_stride %d", who, gout_stride);
    FEA_CHECK(dh || dw || db, FEA_E_BADARG, "%s: no gradient asked for", who);
    FEA_CHECK(K == 1 || !db || psel, FEA_E_BADARG, "%s: the bias gradient needs psel of the forward", who);
    FEA_CHECK(temperature > 0.f && isfinite(temperature) && isfinite(1.f / temperature), FEA_E_BADARG, "%s: temperature %g", who, (double)temperature);
    const int want = (dh ? 1 : 0) | (dw ? 2 : 0) | (db ? 4 : 0);
    const LinBwd p = lin_bwd_plan(d);
    LinBwdWs b;
    const size_t need = lin_bwd_carve(d, p, want, (char*)ws, b);
    FEA_CHECK(ws && (uintptr_t)ws % 256 == 0 && ws_bytes >= need, FEA_E_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, needed (got %zu)", who, need, ws_bytes);

    if (fea_lin_few(rows, D, V)) {
        LinFew f{};
        f.h = h; f.w = w; f.ldh = ldh; f.ldw = ldw; f.bias = bias; f.index = index; f.t = temperature; f.inv_t = 1.f / temperature;
        f.stat = (float2*)stat; f.psel = (float*)psel; f.gout = gout; f.gstride = gout_stride; f.count = count;
        f.dh = dh; f.slab = b.slab; f.dbslab = b.colsum; f.rows = rows; f.D = D; f.V = V; f.K = K;
        return fea_lin_few_bwd(f, dtype, dw, db, s);
    }
    const int ck = 64;
    const bool pack = d.packed() && p.tz == 256;
    for (int ir = 0; ir < p.nrc; ++ir) {
        const long long r0 = ir * p.rc, n = rows - r0 < p.rc ? rows - r0 : p.rc, np = up(n, d.epc);
        const char* hr = (const char*)h + r0 * ldh * d.es;
        const float2* st = (const float2*)stat + r0;
        const float* go = gout + r0 * gout_stride;
        const void* hm = hr;
        long long ldhm = ldh;
        if (pack) { LIN_TRY(lin_pack(d, hr, ldh, b.hp, n, s)); hm = b.hp; ldhm = d.Dp; }
        if (dw) LIN_TRY(lin_transpose(d, hr, ldh, b.ht, np, n, np, st, gout_stride ? go : nullptr, temperature, s));
        for (int iv = 0; iv < p.nvc; ++iv) {
            const long long v0 = (long long)iv * p.vc;
            const int nv = (int)(V - v0 < p.vc ? V - v0 : p.vc), nvp = (int)up(nv, d.epc);
            const char* wr = (const char*)w + v0 * ldw * d.es;
            const void* wm = wr;
            long long ldwm = ldw;
            if (pack) { LIN_TRY(lin_pack(d, wr, ldw, b.wp, nv, s)); wm = b.wp; ldwm = d.Dp; }
            LinGemm g{};
            g.a = hm; g.lda = ldhm; g.b = wm; g.ldb = ldwm; g.M = (int)n; g.N = nv; g.K = pack ? d.Dp : D;
            g.bias = bias ? bias + v0 : nullptr; g.inv_t = 1.f / temperature; g.stat = st; g.gout = go; g.gstride = gout_stride;
            g.count = count; g.t = temperature;
            g.dz = b.dz; g.lddz = nvp; g.Npad = nvp; g.dzt = dw ? b.dzt : nullptr; g.lddzt = np; g.Mpad = (int)np;
            g.colsum = db ? b.colsum : nullptr; g.ldcol = up(p.vc, 64);
            LIN_TRY(fea_lin_gemm(LIN_DZ, dtype, p.tz, g, s));
            const long long entries = n * K;
            const long long* ix = index + r0 * K;
            const unsigned sg = (unsigned)((entries + 255) / 256);
            if (dtype == FEA_BF16) hipLaunchKernelGGL(lin_scatter_kernel<__bf16>, dim3(sg), dim3(256), 0, s, ix, dsel + r0 * K, K, st, (__bf16*)b.dz, (long long)nvp, (__bf16*)g.dzt, np, v0, nv, entries);
            else                   hipLaunchKernelGGL(lin_scatter_kernel<float>, dim3(sg), dim3(256), 0, s, ix, dsel + r0 * K, K, st, (float*)b.dz, (long long)nvp, (float*)g.dzt, np, v0, nv, entries);
            FEA_LAUNCH_CHECK();
            if (db) {
                const int tm = p.tz, tiles = (int)((n + tm - 1) / tm), chunks = (tiles + LIN_DB_TILES - 1) / LIN_DB_TILES;
                hipLaunchKernelGGL(lin_dbias_kernel, dim3((unsigned)((nv + 255) / 256), (unsigned)chunks), dim3(256), 0, s, (const float*)b.colsum, tiles, (long long)g.ldcol, ix, psel ? psel + r0 * K : nullptr, K, st, go, gout_stride, count, temperature, v0, nv, entries, (long long)LIN_DB_TILES * tm * K, b.dbpart);
                FEA_LAUNCH_CHECK();
                hipLaunchKernelGGL(lin_dbias_join_kernel, dim3((unsigned)((nv + 255) / 256)), dim3(256), 0, s, (const double*)b.dbpart, chunks, nv, db + v0, ir > 0 ? 1 : 0);
                FEA_LAUNCH_CHECK();
            }
            if (dh) {
                LIN_TRY(lin_transpose(d, wr, ldw, b.wt, nvp, nv, nvp, nullptr, nullptr, 1.f, s));
                LinGemm m{};
                m.a = b.dz; m.lda = nvp; m.b = b.wt; m.ldb = nvp; m.M = (int)n; m.N = D; m.K = nvp;
                m.scale = 1; m.stat = st; m.gout = go; m.gstride = gout_stride; m.count = count; m.t = temperature;
                void* out = (char*)dh + r0 * D * d.es;
                const bool direct = p.th.splits == 1 && p.nvc == 1;
                m.splits = p.th.splits; m.kper = (int)up((nvp + m.splits - 1) / m.splits, ck);
                if (direct) { m.out = out; m.ldo = D; } else m.slab = b.slab;
                LIN_TRY(fea_lin_gemm(LIN_STORE, dtype, p.th.tile, m, s));
                if (!direct) LIN_TRY(lin_reduce(d, b.slab, m.splits, n * D, iv > 0 ? b.acch : nullptr, iv + 1 < p.nvc ? b.acch : nullptr, iv + 1 < p.nvc ? nullptr : out, s));
            }
            if (dw) {
                LinGemm m{};
                m.a = b.dzt; m.lda = np; m.b = b.ht; m.ldb = np; m.M = nv; m.N = D; m.K = (int)np;
                m.scale = gout_stride ? 0 : 2; m.gout = go; m.count = count; m.t = temperature;
                void* out = (char*)dw + v0 * D * d.es;
                float* acc = b.accw ? b.accw + v0 * D : nullptr;
                const bool direct = p.tw.splits == 1 && p.nrc == 1;
                m.splits = p.tw.splits; m.kper = (int)up((np + m.splits - 1) / m.splits, ck);
                if (direct) { m.out = out; m.ldo = D; } else m.slab = b.slab;
                LIN_TRY(fea_lin_gemm(LIN_STORE, dtype, p.tw.tile, m, s));
                if (!direct) LIN_TRY(lin_reduce(d, b.slab, m.splits, (long long)nv * D, ir > 0 ? acc : nullptr, ir + 1 < p.nrc ? acc : nullptr, ir + 1 < p.nrc ? nullptr : out, s));
            }
        }
    }
    return FEA_OK;
}
