// Loss heads over many classes: a projection and a softmax cross entropy over its outputs, or a distillation loss against a
// teacher's top logits, forward and backward.
//
//   z_nv = (h_n . w_v + b_v) / T,  lse_n = log sum_v exp z_nv
//   cross entropy (T = 1):  l_n = lse_n - z_{n,t}                                   dz_nv = g_n (exp(z_nv - lse_n) - [v = t])
//   distillation:           l_n = T^2 sum_k p_nk (log p_nk - z_{n,i_nk} + lse_n)    dz_nv = g_n T (exp(z_nv - lse_n) - sum_{k: i_nk = v} p_nk)
//   dh = dz w, dw = dz^T h, db = sum_n dz
//
// Forward: the product with a log-sum-exp epilogue (linear_gemm256.hip, linear_gemm.hip), which also gives the few selected logits (or a
// gathered dot product does) and, where the caller has room for them, keeps all logits in 16 bits (bf16 operands, no bias gradient) or fp32; then one
// pass that joins the column tiles of every row.  Backward, in pieces of the classes (and of the rows where there are very
// many): dz from the kept logits, or by the product again with the softmax gradient as its epilogue; the selected entries from the
// forward's fp32 values; two products.  The workspace is bounded by the piece, not by rows x classes.
//
// Why keep: recomputing is a third of a training step's products (2,048 x 2,048 x 32,000 bf16: 281 us), taking dz from kept logits is one
// pass over them (51 us) and 8 % on the forward's product.  Why the labels' and teacher's entries are not taken from 16 bits: there
// softmax - share cancels.
// 2,048 x 2,048 x 32,000, us: forward's product 259, join 6, dz 51, dh 216 + 13, dw 248; 4,096 x 4,096 x 131,072, ms: 3.7, 0.02, 0.42, 3.3, 3.9.
// A whole step of the first takes 729 us, and 932 where nothing is kept.
#include "linear_loss.h"
#include <limits.h>
#include <type_traits>
#include <math.h>
#include <stdlib.h>

// ---- layouts ------------------------------------------------------------------------------------------------------------

// x as three bf16 planes (linear_loss.h): what each leaves goes to the next
__device__ __forceinline__ void lin_split3(float v, __bf16& x0, __bf16& x1, __bf16& x2) {
    x0 = (__bf16)v; v -= (float)x0;
    x1 = (__bf16)v; v -= (float)x1;
    x2 = (__bf16)v;
}

// Copies of an operand's rows [R][ld]: C elements in rows of Cpad (a multiple of 64, zero behind C); with planes (fp32 in, bf16 out) a row
// holds three of Cpad.  With stat, rows whose gate is 0 count as zeros: what an ignored row holds (an infinity, a NaN) meets a zero
// gradient in the weight's product, and 0 x NaN must not reach the weight; with gout every row is multiplied by its own
// upstream gradient (divided by count, where there is one) and rounded to the storage type once more, by half a step: hidden's elements differ
// from row to row, so these errors do not add up, while the same factor on dz's entries, all labels' close to it, would round them all
// the same way when the rows' gradients are equal (a mean taken by the caller).  Up to three operands per launch, 64 x 64 elements per workgroup.
struct LinCopy { const void* in; void* out; long long ld, ldo, R; int C, Cpad; const float2* stat; const float* gout; const int* count; float t; long long tiles; };
struct LinCopies { LinCopy j[3]; };

template <typename T, bool PL, bool ALN>
__device__ __forceinline__ void lin_copy_tile(const LinCopies& js, long long tile) {
    constexpr int EPC = Elem<T>::EPC, NV = 8 / EPC;
    int n = 0;
    while (n < 2 && tile >= js.j[n].tiles) tile -= js.j[n++].tiles;
    const LinCopy j = js.j[n];
    const int nc = j.Cpad / 64;
    const long long r0 = tile / nc * 64 + (threadIdx.x >> 3);
    const int c = (int)(tile % nc) * 64 + (threadIdx.x & 7) * 8;
    u32x4 v[2][NV];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < NV; ++q)
            v[i][q] = r0 + 32 * i < j.R ? lin_load16<T, ALN>((const T*)j.in + (r0 + 32 * i) * j.ld + c + q * EPC, j.C - c - q * EPC) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const long long r = r0 + 32 * i;
        if (r >= j.R) continue;
        T x[8];
        const bool dead = j.stat && j.stat[r].y == 0.f;
#pragma unroll
        for (int q = 0; q < NV; ++q) *reinterpret_cast<u32x4*>(x + q * EPC) = dead ? u32x4{0, 0, 0, 0} : v[i][q];
        if (j.gout) {
            const float f = lin_row_scale(j.gout, 1, j.count, j.t, 1.f, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = dead ? from_f32<T>(0.f) : from_f32<T>(to_f32(x[e]) * f);
        }
        if constexpr (PL) {
            __bf16 y[3][8];
#pragma unroll
            for (int e = 0; e < 8; ++e) lin_split3(x[e], y[0][e], y[1][e], y[2][e]);
#pragma unroll
            for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4*>((__bf16*)j.out + r * j.ldo + p * j.Cpad + c) = *reinterpret_cast<const u32x4*>(y[p]);
        } else
#pragma unroll
            for (int q = 0; q < NV; ++q) *reinterpret_cast<u32x4*>((T*)j.out + r * j.ldo + c + q * EPC) = *reinterpret_cast<const u32x4*>(x + q * EPC);
    }
}

template <typename T, bool PL, bool ALN>
__global__ __launch_bounds__(256) void lin_copy_kernel(const LinCopies js) { lin_copy_tile<T, PL, ALN>(js, blockIdx.x); }

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

// zsel[n][k] = (h_n . w_{index[n][k]} + b) / T: L lanes (a power of two that covers the row in 16-byte loads, 64 at most) per entry.
// Absent entries (index < 0 or >= V) are not read.
template <typename T>
__global__ __launch_bounds__(256) void lin_select_kernel(const T* __restrict__ h, long long ldh, const T* __restrict__ w, long long ldw,
                                                         const float* __restrict__ bias, const long long* __restrict__ index, int K,
                                                         float* __restrict__ zsel, long long entries, int D, int V, int L, int vec, float inv_t) {
    const int lane = threadIdx.x & (L - 1), per = 256 / L;
    for (long long b0 = (long long)blockIdx.x * per; b0 < entries; b0 += (long long)gridDim.x * per) {
        const long long e = b0 + threadIdx.x / L;
        const long long i = e < entries ? index[e] : -1;
        if (i < 0 || i >= V) continue;                       // (the L lanes of an entry go together)
        const T* a = h + e / K * ldh;
        const float s = vec ? lin_dot<T, true>(a, w + i * ldw, D, lane, L) : lin_dot<T, false>(a, w + i * ldw, D, lane, L);
        if (lane == 0) zsel[e] = (bias ? s + bias[i] : s) * inv_t;
    }
}

// The tiles of T columns that hold a row's selected classes (linear_loss.h), a wave per row.  Which entry comes first in a tile is left
// open: each has its own place in zsel.
__global__ __launch_bounds__(256) void lin_where_kernel(const long long* __restrict__ index, int K, long long rows, int V, int T, int ntn, uint2* __restrict__ where) {
    extern __shared__ uint32_t tab[];                    // per row: two dwords and a count for each tile
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long row = (long long)blockIdx.x * 4 + wave;
    uint32_t* const slot = tab + wave * 3 * ntn;
    int* const n = (int*)(slot + 2 * ntn);
    for (int i = lane; i < ntn; i += 64) { slot[2 * i] = slot[2 * i + 1] = ~0u; n[i] = 0; }
    __syncthreads();
    if (row < rows)
        for (int k = lane; k < K; k += 64) {
            const long long i = index[row * K + k];
            if (i < 0 || i >= V) continue;
            const int tile = (int)i / T, at = atomicAdd(n + tile, 1);
            if (at < 4) reinterpret_cast<uint16_t*>(slot + 2 * tile)[at] = (uint16_t)((int)i % T | k << 8);
        }
    __syncthreads();
    if (row < rows)
        for (int i = lane; i < ntn; i += 64) where[row * ntn + i] = n[i] > 4 ? make_uint2(0xffff0000u | LIN_MANY, ~0u) : make_uint2(slot[2 * i], slot[2 * i + 1]);
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
__device__ __forceinline__ void lin_join_body(const LinJoin& j, int G, int gl, long long row, bool in, float lse) {
    float loss = 0.f;
    bool counts = false;
    {
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
            // teacher: softmax over its entries (those with a class and a logit above -inf); lane gl holds entries gl + G q.  1 / T meets the
            // logits' distances to the largest, not the logits: a mask of the type's lowest value stays finite at T < 1
            constexpr int Q = 4;                          // K <= 256, and K <= G where G < 64
            long long ix[Q];
            float tv[Q], tm = -INFINITY, ts = 0.f;
            bool bad = false;
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                const int k = gl + G * q;
                const bool there = in && k < j.K;
                ix[q] = there ? j.index[e0 + k] : -1;
                tv[q] = there ? lin_tlog(j, e0 + k) : -INFINITY;
                if (ix[q] >= j.V) bad = true;
                if (ix[q] >= 0) { bad |= !(tv[q] < INFINITY); tm = fmaxf(tm, tv[q]); }
            }
            for (int d = G >> 1; d; d >>= 1) { tm = fmaxf(tm, __shfl_xor(tm, d)); bad |= __shfl_xor((int)bad, d) != 0; }
            counts = in && (tm != -INFINITY || bad);
            const float tb = tm == -INFINITY ? 0.f : tm;
#pragma unroll
            for (int q = 0; q < Q; ++q) { tv[q] = (tv[q] - tb) * j.inv_t; if (ix[q] >= 0) ts += expf(tv[q]); }
            for (int d = G >> 1; d; d >>= 1) ts += __shfl_xor(ts, d);
            const float lt = logf(ts);
            if (bad) lse = NAN;
            float p[Q], all[Q];
#pragma unroll
            for (int q = 0; q < Q; ++q) { p[q] = counts && ix[q] >= 0 ? expf(tv[q] - lt) : 0.f; all[q] = 0.f; }
            if (j.dsel)                                   // the same class twice in a row: each entry holds the sum over both
#pragma unroll
                for (int q = 0; q < Q; ++q)
                    for (int l = 0; l < G && l + G * q < j.K; ++l) {
                        const int other = __shfl((int)ix[q], (threadIdx.x & 63 & ~(G - 1)) + l);
                        const float share = __shfl(p[q], (threadIdx.x & 63 & ~(G - 1)) + l);
#pragma unroll
                        for (int o = 0; o < Q; ++o) all[o] += other == (int)ix[o] ? share : 0.f;
                    }
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                const int k = gl + G * q;
                if (!in || k >= j.K) continue;
                float ds = 0.f, ps = 0.f;
                if (counts && ix[q] >= 0) {
                    if (bad) { loss = ds = ps = NAN; }
                    else {
                        const float zq = j.zsel[e0 + k] - lse;
                        if (p[q] > 0.f) loss += p[q] * (tv[q] - lt - zq);
                        ds = expf(zq) - all[q];
                        ps = p[q];
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

// (max, sum) of two parts
__device__ __forceinline__ float2 lin_merge(float2 a, float2 b) {
    const float mx = fmaxf(a.x, b.x), base = mx == -INFINITY ? 0.f : mx;
    return make_float2(mx, a.y * expf(a.x - base) + b.y * expf(b.x - base));
}
__device__ __forceinline__ float2 lin_merge_lanes(float2 a, int G) {
    for (int d = G >> 1; d; d >>= 1) a = lin_merge(a, make_float2(__shfl_xor(a.x, d), __shfl_xor(a.y, d)));
    return a;
}
__device__ __forceinline__ float lin_lse_of(float2 a) { return logf(a.y) + (a.x == -INFINITY ? 0.f : a.x); }

__global__ __launch_bounds__(256) void lin_join_kernel(const LinJoin j) {
    const long long row = (long long)blockIdx.x * (256 / j.G) + threadIdx.x / j.G;
    const int gl = threadIdx.x % j.G;
    float2 a = make_float2(-INFINITY, 0.f);
    if (row < j.rows)
#pragma unroll 4
        for (int i = gl; i < j.ntn; i += j.G) a = lin_merge(a, j.part[row * j.ntn + i]);
    lin_join_body(j, j.G, gl, row, row < j.rows, lin_lse_of(lin_merge_lanes(a, j.G)));
}

// The same for few rows, one workgroup per row: all waves take tiles, then the first one joins.
__global__ __launch_bounds__(256) void lin_join_rows_kernel(const LinJoin j) {
    __shared__ float2 red[4];
    const long long row = blockIdx.x;
    float2 a = make_float2(-INFINITY, 0.f);
#pragma unroll 8
    for (int i = threadIdx.x; i < j.ntn; i += 256) a = lin_merge(a, j.part[row * j.ntn + i]);
    a = lin_merge_lanes(a, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    lin_join_body(j, 64, threadIdx.x & 63, row, threadIdx.x < 64, lin_lse_of(lin_merge(lin_merge(red[0], red[1]), lin_merge(red[2], red[3]))));
}

// A split reduction: the parts' sums make z, one workgroup per row.
struct LinParts { const float* slab; int parts; long long ld; const float* bias; float* keep; };      // keep (nullable): rows of ld
__global__ __launch_bounds__(256) void lin_join_split_kernel(const LinJoin j, const LinParts t) {
    __shared__ float2 red[4];
    const long long row = blockIdx.x, next = j.rows * t.ld;
    const float* const s = t.slab + row * t.ld;
    float2 a = make_float2(-INFINITY, 0.f);
    for (int v = 4 * threadIdx.x; v < t.ld; v += 1024) {
        f32x4 z = {0.f, 0.f, 0.f, 0.f};
        for (int p = 0; p < t.parts; p += 8) {                     // (eight on the way, added in their order)
            f32x4 x[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) x[q] = p + q < t.parts ? *reinterpret_cast<const f32x4*>(s + (p + q) * next + v) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int q = 0; q < 8; ++q) z += x[q];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = v + e < j.V ? (z[e] + (t.bias ? t.bias[v + e] : 0.f)) * j.inv_t : -INFINITY;
        if (t.keep) *reinterpret_cast<f32x4*>(t.keep + row * t.ld + v) = z;
        const float mx = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), base = mx == -INFINITY ? 0.f : mx;
        a = lin_merge(a, make_float2(mx, expf(z[0] - base) + expf(z[1] - base) + expf(z[2] - base) + expf(z[3] - base)));
    }
    for (int k = threadIdx.x; k < j.K; k += 256) {
        const long long i = j.index[row * j.K + k];
        if (i < 0 || i >= j.V) continue;
        float z = s[i];
        for (int p = 1; p < t.parts; ++p) z += s[p * next + i];
        j.zsel[row * j.K + k] = (z + (t.bias ? t.bias[i] : 0.f)) * j.inv_t;
    }
    a = lin_merge_lanes(a, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    lin_join_body(j, 64, threadIdx.x & 63, row, threadIdx.x < 64, lin_lse_of(lin_merge(lin_merge(red[0], red[1]), lin_merge(red[2], red[3]))));
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

// dz of the piece from the logits that the forward kept: exp(z - lse), 0 in rows that do not count.  Workgroup: 128 rows x 128 classes, a thread
// 8 classes of 8 rows.  Bound by memory: reads z, writes dz (4,096 x 131,072: 2.1 GB in 415 us, 5.2 TB/s).  A cross entropy's labels are set on the way, and the operands' copies for the
// products go along.
struct LinDecode {
    const void* z; long long ldz;         // at the piece's first row and class
    const float* top; long long ldtop; int shift;   // bf16: the groups' largest at the first row; a class's half tile is class >> shift
    const float2* stat; const float* gout; int gstride; const int* count; float t;
    void* dz; long long lddz; int Npad;
    float* colsum; long long ldcol;       // fp32, nullable: [tiles of 128 rows][classes] sums of row scale * softmax
    const long long* index; const float* dsel;      // nullable: one selected class per row, and dz there
    int n, nv, v0, nct;                   // rows, classes, first class, tiles of 128 columns
    unsigned blocks;                      // of this; the ones behind it copy operands
    LinCopies copies;
};
// T: what the products take; CODES: 16 bits are kept, else fp32; PL: planes
template <typename T, bool CODES, bool PL, bool ALN>
__global__ __launch_bounds__(256) void lin_decode_kernel(const LinDecode g) {
    __shared__ float ref[128], none[128], scale[128], dpick[128], red[16][128];
    __shared__ int pick[128], counts[128];
    if (blockIdx.x >= g.blocks) return lin_copy_tile<std::conditional_t<PL, float, T>, PL, ALN>(g.copies, blockIdx.x - g.blocks);
    const int id = blockIdx.x, tc = id % g.nct, tm = id / g.nct, tid = threadIdx.x;
    const int r0 = tm * 128, c = tc * 128 + (tid & 15) * 8, y = tid >> 4;
    const bool in = c < g.Npad;
    constexpr float L2E = 1.4426950408889634f;
    u32x4 z[8][CODES ? 1 : 2];
    float top[CODES ? 8 : 1];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int q = 0; q < (CODES ? 1 : 2); ++q) {
            const long long m = r0 + y + 16 * i;
            z[i][q] = in && m < g.n ? *reinterpret_cast<const u32x4*>((const char*)g.z + (m * g.ldz + c) * (CODES ? 2 : 4) + 16 * q) : u32x4{0, 0, 0, 0};
            if constexpr (CODES) top[i] = in && m < g.n ? g.top[(((g.v0 + c) >> g.shift) * g.ldtop + m) * 4 + (c >> 3 & 3)] : 0.f;
        }
    if (tid < 128) {
        const int m = r0 + tid;
        const float2 s = m < g.n ? g.stat[m] : make_float2(0.f, 0.f);
        const bool dead = s.y == 0.f;
        counts[tid] = !dead;
        none[tid] = dead || s.x > -INFINITY ? 0.f : NAN;        // exp(z - lse) where z is -inf
        ref[tid] = s.x;
        scale[tid] = dead || !g.colsum ? 0.f : lin_row_scale(g.gout, g.gstride, g.count, g.t, s.y, m);
        const long long i = g.index && !dead ? g.index[m] - g.v0 : -1;
        pick[tid] = i >= 0 && i < g.nv ? (int)i : -8;
        dpick[tid] = g.index && !dead ? g.dsel[m] : 0.f;
    }
    __syncthreads();
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int l = y + 16 * i, m = r0 + l;
        float v[8];
        const bool dead = !counts[l];
        if constexpr (CODES) {
            const float low = dead ? -INFINITY : (top[i] - ref[l]) * L2E, nil = none[l];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t u = e & 1 ? z[i][0][e >> 1] >> 16 : z[i][0][e >> 1] & 0xffffu;
                v[e] = u == 0xffffu ? nil : __builtin_amdgcn_exp2f(fmaf((float)u, -LIN_STEP * L2E, low));
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = dead ? 0.f : __expf(__builtin_bit_cast(f32x4, z[i][e >> 2])[e & 3] - ref[l]);
                sum[e] += v[e] * scale[l];
            }
        }
        if (!in || m >= g.n) continue;
        if ((unsigned)(pick[l] - c) < 8u)
#pragma unroll
            for (int e = 0; e < 8; ++e) if (pick[l] - c == e) v[e] = dpick[l];
        if constexpr (sizeof(T) == 2 && !PL) {
            __bf16 x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (__bf16)v[e];
            *reinterpret_cast<u32x4*>((__bf16*)g.dz + m * g.lddz + c) = *reinterpret_cast<const u32x4*>(x);
        } else if constexpr (PL) {
            __bf16 x[3][8];
#pragma unroll
            for (int e = 0; e < 8; ++e) lin_split3(v[e], x[0][e], x[1][e], x[2][e]);
#pragma unroll
            for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4*>((__bf16*)g.dz + m * g.lddz + (long long)p * g.Npad + c) = *reinterpret_cast<const u32x4*>(x[p]);
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) *reinterpret_cast<f32x4*>((float*)g.dz + m * g.lddz + c + 4 * q) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        }
    }
    if constexpr (!CODES) {
        if (!g.colsum) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) red[y][(tid & 15) * 8 + e] = sum[e];
        __syncthreads();
        if (tid < 128 && tc * 128 + tid < g.nv) {
            float s = 0.f;
#pragma unroll
            for (int q = 0; q < 16; ++q) s += red[q][tid];
            g.colsum[tm * g.ldcol + tc * 128 + tid] = s;
        }
    }
}

// dz at the selected classes of the piece [v0, v0 + N): softmax - teacher, from the forward's fp32 values.  Entries that name the
// same class hold the same value.  Workgroups from `blocks` on copy operands.
template <typename T, bool PL, bool ALN>
__global__ __launch_bounds__(256) void lin_scatter_kernel(const long long* __restrict__ index, const float* __restrict__ dsel, int K,
                                                          const float2* __restrict__ stat, T* dz, long long lddz, long long v0, int N, long long entries, int Npad,
                                                          unsigned blocks, const LinCopies copies) {
    if constexpr (!PL) if (blockIdx.x >= blocks) return lin_copy_tile<T, false, ALN>(copies, blockIdx.x - blocks);
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    if (e >= entries) return;
    const long long m = e / K, i = index[e] - v0;
    if (i < 0 || i >= N) return;
    if (stat[m].y == 0.f) return;
    if constexpr (PL) {
        T x[3];
        lin_split3(dsel[e], x[0], x[1], x[2]);
        for (int p = 0; p < 3; ++p) dz[m * lddz + (long long)p * Npad + i] = x[p];
    } else dz[m * lddz + i] = from_f32<T>(dsel[e]);
}

// out = acc + slabs in split order, rows of N in slabs with rows of ld = N rounded up to 4; acc (nullable, rows of ld) is the fp32 sum of
// earlier pieces, accout where later ones follow.  4 columns per thread.
template <typename T>
__global__ __launch_bounds__(256) void lin_reduce_kernel(const float* __restrict__ slab, int splits, long long M, int N, int ld, const float* acc, float* accout, T* out) {
    const long long n = M * ld, i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    f32x4 s = acc ? *reinterpret_cast<const f32x4*>(acc + i) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int p = 0; p < splits; ++p) s += *reinterpret_cast<const f32x4*>(slab + p * n + i);
    if (accout) *reinterpret_cast<f32x4*>(accout + i) = s;
    if (out) {
        const long long m = i / ld;
        const int c = (int)(i - m * ld);
        T* const o = out + m * N + c;
        if (N == ld) {
            if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(o) = s;
            else { const bf16x4 v = {(__bf16)s[0], (__bf16)s[1], (__bf16)s[2], (__bf16)s[3]}; *reinterpret_cast<bf16x4*>(o) = v; }
        } else
#pragma unroll
            for (int e = 0; e < 4; ++e) if (c + e < N) o[e] = from_f32<T>(s[e]);
    }
}

// Partial bias gradient of one chunk of LIN_DB_ROWS rows: sum over its row tiles of colsum[tile][v] - sum of g * teacher share over
// its rows' entries that name v (psel NULL: share 1).  One workgroup owns 256 classes of one chunk; its waves walk the entries in
// order and the lane that owns a class adds its hits: the order is fixed.
static constexpr int LIN_DB_ROWS = 256, LIN_DB_WAVES = 16;
__global__ __launch_bounds__(64 * LIN_DB_WAVES) void lin_dbias_kernel(const float* __restrict__ colsum, int tiles, long long ldcol, const long long* __restrict__ index,
                                                        const float* __restrict__ psel, int K, const float2* __restrict__ stat, const float* gout,
                                                        int gstride, const int* count, float t, long long v0, int N, long long entries,
                                                        int per, long long chunk, double* out) {
    __shared__ double part[LIN_DB_WAVES][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b0 = blockIdx.x * 256;
    const long long ea = blockIdx.y * chunk, eb = ea + chunk < entries ? ea + chunk : entries;
    double acc[4] = {0.0, 0.0, 0.0, 0.0};             // classes b0 + lane + 64 q
    for (long long e0 = ea + wave * 256; e0 < eb; e0 += 256 * LIN_DB_WAVES) {
        int i[4];
        float val[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {                 // (four entries of a lane at a time: their loads are in flight together)
            const long long e = e0 + 64 * u + lane;
            const long long x = e < eb ? index[e] - v0 - b0 : -1;
            const bool hit = x >= 0 && x < 256 && b0 + x < N;
            const long long m = hit ? e / K : 0;
            val[u] = hit ? (psel ? psel[e] : 1.f) * lin_row_scale(gout, gstride, count, t, stat[m].y, m) : 0.f;
            i[u] = hit ? (int)x : -1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            unsigned long long mask = __ballot(i[u] >= 0 && val[u] != 0.f);
            while (mask) {
                const int l = __builtin_ctzll(mask);
                mask &= mask - 1;
                const int c = __shfl(i[u], l);
                const float v = __shfl(val[u], l);
                if ((c & 63) == lane) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) if (c >> 6 == q) acc[q] += (double)v;
                }
            }
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) part[wave][lane + 64 * q] = acc[q];
    __syncthreads();
    const int v = b0 + threadIdx.x;
    if (threadIdx.x < 256 && v < N) {
        double s = 0.0;
#pragma unroll
        for (int w = 0; w < LIN_DB_WAVES; ++w) s -= part[w][threadIdx.x];
        const int t1 = min(tiles, ((int)blockIdx.y + 1) * per);
        for (int i = blockIdx.y * per; i < t1; ++i) s += (double)colsum[i * ldcol + v];
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
    bool odd() const { return D % epc != 0; }      // rows that are no multiple of 16 bytes
    bool straight() const { return !odd(); }       // gradients go straight to their rows (others through slabs, which have wide stores)
};

static LinDims lin_dims(long long rows, int D, int V, int K, int dtype) {
    LinDims d{rows, D, V, K, dtype, dtype == FEA_BF16 ? 2 : 4, dtype == FEA_BF16 ? 8 : 4};
    return d;
}

// The sizes that are served (lin_check says which of them a call does not keep to)
static constexpr int LIN_ROWS = INT_MAX / 2, LIN_D = 1 << 16, LIN_V = 1 << 24, LIN_K = 256;
static bool lin_served(long long rows, int D, int V, int K, int dtype) {
    return rows >= 1 && rows <= LIN_ROWS && D >= 1 && D <= LIN_D && V >= 1 && V <= LIN_V && K >= 1 && K <= LIN_K && (dtype == FEA_F32 || dtype == FEA_BF16);
}

// The form that a call's products take: the operands as they are, or fp32 as three bf16 planes where the copies pay.
struct LinForm {
    int dt, es, mul, pad;         // dtype of the products, bytes of an element, elements of a row per channel, what a row is rounded up to
    // elements of a row of k channels: an odd number of 64, so that rows do not lie a power of two apart (dz of 65,536 classes: 1 %)
    long long row(long long k) const { const long long r = up(k, pad) * mul; return r % 128 ? r : r + 64; }
    int K(long long k) const { return (int)(dt == FEA_PL ? 6 * up(k, 64) : dt == FEA_BF16 ? up(k, 64) : k); }      // reduction over k channels
};
static LinForm lin_form(int dtype, bool planes) {
    if (planes) return LinForm{FEA_PL, 2, 3, 64};
    return dtype == FEA_BF16 ? LinForm{FEA_BF16, 2, 1, 64} : LinForm{FEA_F32, 4, 1, 64};
}

// Forward: rows in chunks that bound the partial table to 128 MB.
struct LinFwd { long long rc; int tile, ntn, G; bool planes; long long blocks; int pick, parts; };   // pick: 0 selected logits by dot products, 1 out of the product, 2 with lin_where_kernel; parts: of a split reduction
static LinFwd lin_fwd_plan(const LinDims& d) {
    LinFwd p;
    const long long cap = (1ll << 24) / ((d.V + 127) / 128);
    p.rc = cap < 256 ? 256 : cap / 256 * 256;
    if (p.rc > d.rows) p.rc = d.rows;
    LinTile t = fea_lin_tile(d.dtype, p.rc, d.V, d.D, false);
    p.planes = false;
    // few tiles: the reduction is split between workgroups where that saves more than the longer join (a training step of 387 rows x 3,264 x 2,112:
    // fp32 307 and, split, 204 us, bf16 83 and 71)
    const bool split = p.rc == d.rows && d.V <= 1 << 16;
    auto product = [&](int dt, long long K) {
        const LinTile one = fea_lin_tile(dt, p.rc, d.V, K, false);
        const LinTile many = split ? fea_lin_tile(dt, p.rc, d.V, K, true) : one;
        return many.splits > 1 && many.time + 6e-6 < one.time ? many : one;
    };
    if (d.dtype == FEA_BF16) t = product(FEA_BF16, d.D);
    if (d.dtype == FEA_F32) {     // 10 bytes per element for the copies, against a third of the matrix time
        const LinTile q = product(FEA_PL, 6 * up(d.D, 64));
        if (q.time + ((double)p.rc + d.V) * d.D * 10 / 4e12 + 6e-6 < t.time) { t = q; p.planes = true; }
    }
    p.tile = t.tile;
    p.parts = t.splits;
    if (d.rows <= 64) { p.tile = 64; p.planes = false; }
    p.ntn = (d.V + p.tile - 1) / p.tile;
    // selected logits come out of the product where it can give them
    const bool tiles = p.tile != 64 && (d.dtype == FEA_BF16 || p.planes);
    if (p.tile == 64) p.parts = fea_lin_rows_splits((int)d.dtype, d.V, d.D);
    p.pick = p.parts > 1 ? 1 : p.tile == 64 ? d.rows * d.K <= 2048 : !tiles ? 0 : d.K == 1 ? 1 : d.K <= LIN_WHERE_K && p.ntn <= LIN_WHERE_T ? 2 : 0;
    p.G = 1;
    while (p.G < 64 && (p.G < (d.V + 127) / 128 || p.G < d.K)) p.G *= 2;
    p.blocks = p.tile == 64 || p.parts > 1 ? d.rows : (d.rows + 256 / p.G - 1) / (256 / p.G) + (p.rc ? d.rows / p.rc + 1 : 0);     // every chunk rounds up by itself
    return p;
}

// Backward: pieces of rc rows x vc classes.  dz takes rc x vc elements: 2^28 at most
// (FEA_AMD_LINEAR_PIECE: tests, many pieces on small shapes).
static long long lin_piece() {
    const char* e = getenv("FEA_AMD_LINEAR_PIECE");
    const long long v = e ? atoll(e) : 0;
    return v >= 1 << 14 && v < 1 << 28 ? v : 1ll << 28;
}
struct LinBwd { long long rc; int vc, nrc, nvc, tz; bool planes; LinTile th, tw; };
static LinBwd lin_bwd_plan(const LinDims& d, int want) {       // want: 1 dh, 2 dw, 4 db, 8 with the kept logits
    LinBwd p;
    const long long piece = lin_piece();
    p.rc = d.rows < 32768 ? d.rows : 32768;
    if (d.V <= 1024) { const long long most = piece / up(d.V > d.D ? d.V : d.D, 256); p.rc = d.rows < most ? d.rows : most < 256 ? 256 : most / 256 * 256; }
    long long vc = piece / (p.rc > 0 ? up(p.rc, 256) : 1) / 256 * 256;
    if (vc < 256) vc = 256;
    p.vc = (int)(vc < d.V ? vc : d.V);
    p.nrc = p.rc ? (int)((d.rows + p.rc - 1) / p.rc) : 0;
    p.nvc = (d.V + p.vc - 1) / p.vc;
    LinTile tz;
    auto tiles = [&](int dt, int mul, LinTile& z, LinTile& h, LinTile& w) {
        z = fea_lin_tile(dt, p.rc, p.vc, mul * up(d.D, 64), false);
        h = fea_lin_tile(dt, p.rc, d.D, mul * up(p.vc, 64), true);
        w = fea_lin_tile(dt, p.vc, d.D, mul * up(p.rc, 64), true);
        return (want & 8 ? 0.0 : z.time) + (want & 1 ? h.time : 0.0) + (want & 2 ? w.time : 0.0);
    };
    const double t = tiles(d.dtype, 1, tz, p.th, p.tw);
    p.planes = false;
    if (d.dtype == FEA_F32 && 3 * up(p.vc, 64) + 64 < 1 << 21) {     // (the strides that the bf16 kernels take)
        LinTile z, h, w;
        const double q = tiles(FEA_PL, 6, z, h, w);
        if (q + (((double)p.rc + p.vc) * d.D * 10 + 2.0 * p.rc * p.vc) / 4e12 + 6e-6 < t) { tz = z; p.th = h; p.tw = w; p.planes = true; }
    }
    p.tz = tz.tile;
    return p;
}

struct LinFwdWs { void *hp, *wp; float2* part; float *zsel, *slab; uint2* where; double* bsum; int* bcnt; };
static size_t lin_fwd_carve(const LinDims& d, const LinFwd& p, char* base, LinFwdWs& w) {
    LinCarve c{base};
    if (fea_lin_few(d.rows, d.D, d.V)) {
        w = LinFwdWs{};
        w.bsum = c.take<double>(fea_lin_few_blocks(d.rows, false));
        w.bcnt = c.take<int>(fea_lin_few_blocks(d.rows, false));
        return c.at;
    }
    w.part = c.take<float2>(p.rc * p.ntn);
    w.zsel = c.take<float>(d.rows * d.K);
    w.bsum = c.take<double>(p.blocks);
    w.bcnt = c.take<int>(p.blocks);
    w.hp = w.wp = nullptr;
    w.slab = p.parts > 1 ? c.take<float>(p.parts * d.rows * up(d.V, 64)) : nullptr;
    w.where = p.pick == 2 ? c.take<uint2>(p.rc * p.ntn) : nullptr;
    if (p.planes || (d.dtype == FEA_BF16 && d.odd() && p.tile != 64)) {
        const LinForm f = lin_form(d.dtype, p.planes);
        w.hp = c.take<char>(p.rc * f.row(d.D) * f.es);
        w.wp = c.take<char>(d.V * f.row(d.D) * f.es);
    }
    return c.at;
}

struct LinBwdWs { void *hp, *wp, *hg, *dz; float *slab, *acch, *accw, *colsum; double* dbpart; };
static size_t lin_bwd_carve(const LinDims& d, const LinBwd& p, int want, char* base, LinBwdWs& w) {
    LinCarve c{base};
    w = LinBwdWs{};
    if (fea_lin_few(d.rows, d.D, d.V)) {
        if (want & 2) w.slab = c.take<float>(fea_lin_few_blocks(d.rows, true) * 32ll * 64);
        if (want & 4) w.colsum = c.take<float>(fea_lin_few_blocks(d.rows, true) * 32ll);
        w.dz = c.take<char>(256);
        return c.at;
    }
    const LinForm f = lin_form(d.dtype, p.planes);
    if (p.planes || (d.dtype == FEA_BF16 && d.odd())) { w.hp = c.take<char>(p.rc * f.row(d.D) * f.es); w.wp = c.take<char>(p.vc * f.row(d.D) * f.es); }
    w.dz = c.take<char>(p.rc * f.row(p.vc) * f.es);
    if (want & 2) w.hg = c.take<char>(p.rc * f.row(d.D) * f.es);
    long long slab = 0;
    const long long ld = up(d.D, 4);
    if ((want & 1) && !(p.th.splits == 1 && p.nvc == 1 && d.straight())) slab = p.th.splits * p.rc * ld;
    if ((want & 2) && !(p.tw.splits == 1 && p.nrc == 1 && d.straight()) && slab < (long long)p.tw.splits * p.vc * ld) slab = (long long)p.tw.splits * p.vc * ld;
    w.slab = c.take<float>(slab);
    if ((want & 1) && p.nvc > 1) w.acch = c.take<float>(p.rc * ld);
    if ((want & 2) && p.nrc > 1) w.accw = c.take<float>(d.V * ld);
    if (want & 4) { const long long t = (p.rc + 127) / 128; w.colsum = c.take<float>(t * up(p.vc, 64)); w.dbpart = c.take<double>((p.rc + LIN_DB_ROWS - 1) / LIN_DB_ROWS * p.vc); }
    return c.at;
}

// Kept logits: [rows][V rounded up to 64] of 16 bits (bf16 operands) or fp32 (fp32 operands, the few rows of linear_rows.hip, split
// reductions, and where the caller asks for `wide` ones: a bias gradient is fp32), then, with 16 bits, the groups' largest.  Not for few classes, where recomputing
// reads no more.
struct LinKeep {
    bool codes;
    long long ld;
    int es;
    size_t table;                 // bytes in front of the groups' largest
    LinKeep(const LinDims& d, int wide) : codes(d.dtype == FEA_BF16 && d.rows > 64 && !wide && lin_fwd_plan(d).parts == 1), ld(up(d.V, 64)), es(codes ? 2 : 4), table((size_t)up(d.rows * ld * es, 256)) {}
};
extern "C" size_t fea_linear_loss_keep_bytes(long long rows, int D, int V, int dtype, int wide) {
    if (!lin_served(rows, D, V, 1, dtype) || fea_lin_few(rows, D, V)) return 0;
    const LinDims d = lin_dims(rows, D, V, 1, dtype);
    const LinKeep k(d, wide);
    return k.table + (k.codes ? (size_t)rows * lin_fwd_plan(d).ntn * 8 * sizeof(float) : 0);
}

extern "C" size_t fea_linear_loss_ws_bytes(long long rows, int D, int V, int K, int dtype, int grads) {
    if (!lin_served(rows, D, V, K, dtype)) return 0;
    const LinDims d = lin_dims(rows, D, V, K, dtype);
    if (!grads) { LinFwdWs w; return lin_fwd_carve(d, lin_fwd_plan(d), nullptr, w); }
    LinBwdWs w;
    return lin_bwd_carve(d, lin_bwd_plan(d, grads), grads, nullptr, w);
}

// an operand of R rows and where its copy goes (nullptr: none)
static LinCopy lin_copy_of(const LinDims& d, const LinForm& f, const void* in, long long ld, long long R, void* out) {
    LinCopy j{};
    j.in = in; j.out = out; j.ld = ld; j.ldo = f.row(d.D); j.R = R; j.C = d.D; j.Cpad = (int)up(d.D, 64);
    j.tiles = out ? (R + 63) / 64 * (j.Cpad / 64) : 0;
    return j;
}
static int lin_copy(const LinDims& d, const LinForm& f, const LinCopies& js, hipStream_t s) {
    const long long n = js.j[0].tiles + js.j[1].tiles + js.j[2].tiles;
    if (!n) return FEA_OK;
    FEA_CHECK(n < INT_MAX, FEA_E_UNSUPPORTED_SHAPE, "lin_copy: %lld tiles", n);
    const dim3 grid((unsigned)n), bl(256);
    FEA_CHECK(f.dt == FEA_PL || (f.dt == FEA_BF16 && d.odd()), FEA_E_BADARG, "lin_copy: operands that are read as they lie");
    if (f.dt == FEA_BF16) hipLaunchKernelGGL((lin_copy_kernel<__bf16, false, false>), grid, bl, 0, s, js);
    else if (d.odd())     hipLaunchKernelGGL((lin_copy_kernel<float, true, false>), grid, bl, 0, s, js);
    else                  hipLaunchKernelGGL((lin_copy_kernel<float, true, true>), grid, bl, 0, s, js);
    FEA_LAUNCH_CHECK();
    return FEA_OK;
}

static int lin_reduce(const LinDims& d, const float* slab, int splits, long long M, const float* acc, float* accout, void* out, hipStream_t s) {
    const int ld = (int)up(d.D, 4);
    const dim3 grid((unsigned)((M * ld / 4 + 255) / 256));
    if (d.dtype == FEA_BF16) hipLaunchKernelGGL(lin_reduce_kernel<__bf16>, grid, dim3(256), 0, s, slab, splits, M, d.D, ld, acc, accout, (__bf16*)out);
    else                     hipLaunchKernelGGL(lin_reduce_kernel<float>, grid, dim3(256), 0, s, slab, splits, M, d.D, ld, acc, accout, (float*)out);
    FEA_LAUNCH_CHECK();
    return FEA_OK;
}

#define LIN_TRY(x) do { const int rc_ = (x); if (rc_ != FEA_OK) return rc_; } while (0)

static int lin_check(const char* who, const LinDims& d, const void* h, long long ldh, const void* w, long long ldw, const float* bias) {
    FEA_CHECK(d.dtype == FEA_F32 || d.dtype == FEA_BF16, FEA_E_BADARG, "%s: dtype %d", who, d.dtype);
    FEA_CHECK(d.rows >= 1 && d.rows <= LIN_ROWS, FEA_E_UNSUPPORTED_SHAPE, "%s: %lld rows, 1..%d are served", who, d.rows, LIN_ROWS);
    FEA_CHECK(d.D >= 1 && d.D <= LIN_D, FEA_E_UNSUPPORTED_SHAPE, "%s: %d features, 1..%d are served", who, d.D, LIN_D);
    FEA_CHECK(d.V >= 1 && d.V <= LIN_V, FEA_E_UNSUPPORTED_SHAPE, "%s: %d classes, 1..%d are served", who, d.V, LIN_V);
    FEA_CHECK(d.K >= 1 && d.K <= LIN_K, FEA_E_UNSUPPORTED_SHAPE, "%s: %d teacher entries per row, 1..%d are served", who, d.K, LIN_K);
    FEA_CHECK(h && w, FEA_E_BADARG, "%s: null operand", who);
    FEA_CHECK(ldh >= d.D && ldw >= d.D, FEA_E_BADARG, "%s: row stride below the %d features (hidden %lld, weight %lld)", who, d.D, ldh, ldw);
    FEA_CHECK(((uintptr_t)h | (uintptr_t)w) % d.es == 0 && (uintptr_t)bias % 4 == 0, FEA_E_BADARG, "%s: misaligned operand", who);
    if (!d.odd())
        FEA_CHECK(((uintptr_t)h | (uintptr_t)w) % 16 == 0 && ldh % d.epc == 0 && ldw % d.epc == 0, FEA_E_BADARG,
                  "%s: hidden and weight need 16-byte aligned rows when the features are a multiple of %d", who, d.epc);
    if (!d.odd() && d.dtype == FEA_BF16)      // (32-bit offsets over a tile's rows)
        FEA_CHECK(ldh < 1 << 21 && ldw < 1 << 21, FEA_E_UNSUPPORTED_SHAPE, "%s: bf16 row strides below %d are served (hidden %lld, weight %lld)", who, 1 << 21, ldh, ldw);
    return FEA_OK;
}

static int lin_forward(const char* who, LinDims d, const void* h, long long ldh, const void* w, long long ldw, const float* bias, LinJoin j,
                       void* keep, int wide, float* loss, int* count, int mean, void* ws, size_t ws_bytes, hipStream_t s) {
    LIN_TRY(lin_check(who, d, h, ldh, w, ldw, bias));
    const LinFwd p = lin_fwd_plan(d);
    LinFwdWs b;
    const size_t need = lin_fwd_carve(d, p, (char*)ws, b);
    FEA_CHECK(ws && (uintptr_t)ws % 256 == 0 && ws_bytes >= need, FEA_E_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, needed (got %zu)", who, need, ws_bytes);
    FEA_CHECK(!keep || ((uintptr_t)keep % 256 == 0 && fea_linear_loss_keep_bytes(d.rows, d.D, d.V, (int)d.dtype, wide) > 0), FEA_E_BADARG, "%s: no logits are kept of these sizes, or misaligned", who);
    FEA_CHECK(!loss == !count, FEA_E_BADARG, "%s: loss and count go together", who);
    FEA_CHECK(loss || j.loss_rows, FEA_E_BADARG, "%s: nothing to write", who);

    if (fea_lin_few(d.rows, d.D, d.V)) {
        LinFew f{};
        f.h = h; f.w = w; f.ldh = ldh; f.ldw = ldw; f.bias = bias; f.index = j.index; f.tlog = j.tlog; f.tdt = j.tdt; f.ignore = j.ignore;
        f.t = j.t; f.inv_t = j.inv_t; f.stat = j.stat; f.psel = j.psel; f.loss_rows = j.loss_rows;
        f.bsum = loss ? b.bsum : nullptr; f.bcnt = b.bcnt; f.rows = d.rows; f.D = d.D; f.V = d.V; f.K = d.K;
        LIN_TRY(fea_lin_few_fwd(f, d.dtype, s));
        if (loss) {
            hipLaunchKernelGGL(lin_total_kernel, dim3(1), dim3(1024), 0, s, (const double*)b.bsum, (const int*)b.bcnt, (long long)fea_lin_few_blocks(d.rows, false), mean, loss, count);
            FEA_LAUNCH_CHECK();
        }
        return FEA_OK;
    }
    const long long entries = d.rows * d.K;
    if (!p.pick) {
        int lanes = 1;
        while (lanes < 64 && lanes * d.epc < d.D) lanes *= 2;
        const long long blocks = (entries * lanes + 255) / 256;
        const unsigned grid = (unsigned)(blocks < 1 << 16 ? blocks : 1 << 16);
        if (d.dtype == FEA_BF16) hipLaunchKernelGGL(lin_select_kernel<__bf16>, dim3(grid), dim3(256), 0, s, (const __bf16*)h, ldh, (const __bf16*)w, ldw, bias, j.index, d.K, b.zsel, entries, d.D, d.V, lanes, d.odd() ? 0 : 1, j.inv_t);
        else                     hipLaunchKernelGGL(lin_select_kernel<float>, dim3(grid), dim3(256), 0, s, (const float*)h, ldh, (const float*)w, ldw, bias, j.index, d.K, b.zsel, entries, d.D, d.V, lanes, d.odd() ? 0 : 1, j.inv_t);
        FEA_LAUNCH_CHECK();
    }
    const LinForm f = lin_form(d.dtype, p.planes);
    const bool pack = p.planes || (d.dtype == FEA_BF16 && d.odd() && p.tile != 64);       // (the others take rows of any alignment)
    long long blk = 0;
    for (long long r = 0; r < d.rows; r += p.rc) {
        const long long n = d.rows - r < p.rc ? d.rows - r : p.rc;
        const void* hr = (const char*)h + r * ldh * d.es;
        if (pack) LIN_TRY(lin_copy(d, f, LinCopies{{lin_copy_of(d, f, hr, ldh, n, b.hp), lin_copy_of(d, f, w, ldw, d.V, r ? nullptr : b.wp)}}, s));
        LinGemm g{};
        g.a = pack ? b.hp : hr; g.lda = pack ? f.row(d.D) : ldh; g.b = pack ? b.wp : w; g.ldb = pack ? f.row(d.D) : ldw;
        g.M = (int)n; g.N = d.V; g.K = pack ? f.K(d.D) : d.D; g.Kp = (int)up(d.D, 64);
        g.bias = bias; g.inv_t = j.inv_t; g.part = b.part;
        if (keep) {
            const LinKeep k(d, wide);
            g.keep = (char*)keep + r * k.ld * k.es; g.ldkeep = k.ld;
            if (k.codes) { g.ldtop = d.rows; g.top = (float*)((char*)keep + k.table) + r * 4; }
        }
        if (p.pick) { g.zsel = b.zsel + r * d.K; g.index = j.index + r * d.K; g.sel = d.K; }
        if (p.pick == 2) {
            g.where = b.where;
            hipLaunchKernelGGL(lin_where_kernel, dim3((unsigned)((n + 3) / 4)), dim3(256), 4 * 3 * p.ntn * sizeof(uint32_t), s, g.index, d.K, n, d.V, p.tile, p.ntn, b.where);
            FEA_LAUNCH_CHECK();
        }
        if (p.parts > 1) { g.zsel = nullptr; g.keep = nullptr; g.slab = b.slab; g.ldo = up(d.V, 64); g.splits = p.parts; g.kper = (int)up((g.K + p.parts - 1) / p.parts, 64); }
        if (p.tile == 64) LIN_TRY(fea_lin_rows(d.dtype, !d.odd(), g, s));
        else LIN_TRY(fea_lin_gemm(LIN_LSE, f.dt, p.tile, g, s));
        LinJoin q = j;
        q.part = b.part; q.ntn = p.ntn; q.rows = n; q.K = d.K; q.V = d.V; q.G = p.G;
        q.zsel = b.zsel + r * d.K; q.index = j.index + r * d.K;
        if (q.tlog) q.tlog = (const char*)j.tlog + r * d.K * (j.tdt == FEA_BF16 ? 2 : 4);
        if (q.stat) q.stat += r;
        if (q.dsel) q.dsel += r * d.K;
        if (q.psel) q.psel += r * d.K;
        if (q.loss_rows) q.loss_rows += r;
        q.bsum = loss ? b.bsum + blk : nullptr; q.bcnt = b.bcnt + blk;
        const long long grid = p.tile == 64 || p.parts > 1 ? n : (n + 256 / p.G - 1) / (256 / p.G);
        if (p.parts > 1)       hipLaunchKernelGGL(lin_join_split_kernel, dim3((unsigned)grid), dim3(256), 0, s, q, (LinParts{b.slab, p.parts, up(d.V, 64), bias, (float*)keep}));
        else if (p.tile == 64) hipLaunchKernelGGL(lin_join_rows_kernel, dim3((unsigned)grid), dim3(256), 0, s, q);
        else              hipLaunchKernelGGL(lin_join_kernel, dim3((unsigned)grid), dim3(256), 0, s, q);
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
                                 long long ignore_index, float* stat, float* dsel, void* keep, int wide, float* loss_rows, float* loss,
                                 int* count, int mean, void* ws, size_t ws_bytes, long long rows, int D, int V, int dtype, void* stream) {
    FEA_CHECK(target, FEA_E_BADARG, "fea_linear_ce_fwd: null target");
    LinJoin j{};
    j.index = target; j.ignore = ignore_index; j.t = j.inv_t = 1.f;
    j.stat = (float2*)stat; j.dsel = dsel; j.loss_rows = loss_rows;
    return lin_forward("fea_linear_ce_fwd", lin_dims(rows, D, V, 1, dtype), h, ldh, w, ldw, bias, j, keep, wide, loss, count, mean, ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int fea_linear_kd_fwd(const void* h, long long ldh, const void* w, long long ldw, const float* bias, const void* teacher_logits,
                                 int teacher_dtype, const long long* teacher_index, int K, float temperature, float* stat, float* dsel, float* psel,
                                 void* keep, int wide, float* loss_rows, float* loss, int* count, int mean, void* ws, size_t ws_bytes, long long rows, int D, int V,
                                 int dtype, void* stream) {
    FEA_CHECK(teacher_logits && teacher_index, FEA_E_BADARG, "fea_linear_kd_fwd: null teacher");
    FEA_CHECK(teacher_dtype == FEA_F32 || teacher_dtype == FEA_BF16, FEA_E_BADARG, "fea_linear_kd_fwd: teacher dtype %d", teacher_dtype);
    FEA_CHECK(temperature > 0.f && isfinite(temperature) && isfinite(1.f / temperature), FEA_E_BADARG, "fea_linear_kd_fwd: temperature %g", (double)temperature);
    LinJoin j{};
    j.index = teacher_index; j.tlog = teacher_logits; j.tdt = teacher_dtype; j.t = temperature; j.inv_t = 1.f / temperature;
    j.stat = (float2*)stat; j.dsel = dsel; j.psel = psel; j.loss_rows = loss_rows;
    return lin_forward("fea_linear_kd_fwd", lin_dims(rows, D, V, K, dtype), h, ldh, w, ldw, bias, j, keep, wide, loss, count, mean, ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int fea_linear_loss_bwd(const void* h, long long ldh, const void* w, long long ldw, const float* bias, const long long* index, int K,
                                   const float* stat, const float* dsel, const float* psel, const void* keep, int wide, const int* count,
                                   const float* gout, int gout_stride, float temperature, void* dh, void* dw, float* db, void* ws, size_t ws_bytes, long long rows, int D, int V,
                                   int dtype, void* stream) {
    const char* who = "fea_linear_loss_bwd";
    LinDims d = lin_dims(rows, D, V, K, dtype);
    hipStream_t s = (hipStream_t)stream;
    LIN_TRY(lin_check(who, d, h, ldh, w, ldw, bias));
    FEA_CHECK(index && stat && dsel && gout, FEA_E_BADARG, "%s: null operand", who);
    FEA_CHECK(gout_stride == 0 || gout_stride == 1, FEA_E_BADARG, "%s: gout_stride %d", who, gout_stride);
    FEA_CHECK(dh || dw || db, FEA_E_BADARG, "%s: no gradient asked for", who);
    FEA_CHECK(((uintptr_t)dh | (uintptr_t)dw) % 16 == 0 && (uintptr_t)db % 4 == 0, FEA_E_BADARG, "%s: misaligned gradient", who);
    // (few classes take the shares themselves, not their differences to the softmax)
    FEA_CHECK(K == 1 || psel || !(db || fea_lin_few(rows, D, V)), FEA_E_BADARG, "%s: %d entries per row %s need psel of the forward", who, K,
              db ? "and a bias gradient" : "over few classes");
    FEA_CHECK(temperature > 0.f && isfinite(temperature) && isfinite(1.f / temperature), FEA_E_BADARG, "%s: temperature %g", who, (double)temperature);
    FEA_CHECK(!keep || ((uintptr_t)keep % 256 == 0 && fea_linear_loss_keep_bytes(rows, D, V, dtype, wide) > 0), FEA_E_BADARG, "%s: no logits are kept of these sizes, or misaligned", who);
    const LinKeep kept(d, wide);
    FEA_CHECK(!keep || !db || !kept.codes, FEA_E_BADARG, "%s: a bias gradient needs wide kept logits", who);
    const int want = (dh ? 1 : 0) | (dw ? 2 : 0) | (db ? 4 : 0) | (keep ? 8 : 0);
    const LinBwd p = lin_bwd_plan(d, want);
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
    const LinForm f = lin_form(dtype, p.planes);
    const bool pack = p.planes || (dtype == FEA_BF16 && d.odd());
    const LinFwd kp = lin_fwd_plan(d);              // (its tiles make the kept groups)
    for (int ir = 0; ir < p.nrc; ++ir) {
        const long long r0 = ir * p.rc, n = rows - r0 < p.rc ? rows - r0 : p.rc;
        const char* hr = (const char*)h + r0 * ldh * d.es;
        const float2* st = (const float2*)stat + r0;
        const float* go = gout + r0 * gout_stride;
        for (int iv = 0; iv < p.nvc; ++iv) {
            const long long v0 = (long long)iv * p.vc;
            const int nv = (int)(V - v0 < p.vc ? V - v0 : p.vc);
            const char* wr = (const char*)w + v0 * ldw * d.es;
            // the operands' copies: packed rows, and hidden as dw takes it (gated, times each row's own upstream gradient; gated alone, it is
            // the packed one).  Hidden once for its rows, the weight's piece unless the only piece is there from the rows before
            const bool gated = dw && (!pack || gout_stride);
            LinCopies js{{lin_copy_of(d, f, hr, ldh, n, pack && iv == 0 && (!keep || (dw && !gated)) ? b.hp : nullptr), lin_copy_of(d, f, wr, ldw, nv, pack && (ir == 0 || p.nvc > 1) && (!keep || dh) ? b.wp : nullptr),
                          lin_copy_of(d, f, hr, ldh, n, gated && iv == 0 ? b.hg : nullptr)}};
            js.j[0].stat = js.j[2].stat = st;
            if (gout_stride) { js.j[2].gout = go; js.j[2].count = count; js.j[2].t = temperature; }
            if (pack && !keep) LIN_TRY(lin_copy(d, f, js, s));       // (else they go along with a kernel below)
            const void* const wk = pack ? b.wp : (const void*)wr;
            const long long ldwk = pack ? f.row(D) : ldw;
            LinGemm g{};
            g.a = pack ? b.hp : (const void*)hr; g.lda = pack ? f.row(D) : ldh; g.b = wk; g.ldb = ldwk;
            g.M = (int)n; g.N = nv; g.K = pack ? f.K(D) : D; g.Kp = (int)up(D, 64);
            g.bias = bias ? bias + v0 : nullptr; g.inv_t = 1.f / temperature; g.stat = st; g.gout = go; g.gstride = gout_stride;
            g.count = count; g.t = temperature;
            g.dz = b.dz; g.lddz = f.row(nv); g.Npad = (int)up(nv, f.pad);
            g.colsum = db ? b.colsum : nullptr; g.ldcol = up(p.vc, 64);
            if (keep) {
                LinDecode x{};
                x.z = (const char*)keep + (r0 * kept.ld + v0) * kept.es; x.ldz = kept.ld;
                x.ldtop = rows; x.top = (const float*)((const char*)keep + kept.table) + r0 * 4; x.shift = kp.tile == 256 ? 7 : 6;
                x.stat = st; x.gout = go; x.gstride = gout_stride; x.count = count; x.t = temperature;
                x.dz = b.dz; x.lddz = g.lddz; x.Npad = g.Npad; x.colsum = g.colsum; x.ldcol = g.ldcol;
                x.n = (int)n; x.nv = nv; x.v0 = (int)v0; x.nct = (nv + 127) / 128;
                if (K == 1) { x.index = index + r0; x.dsel = dsel + r0; }
                x.blocks = (unsigned)((n + 127) / 128 * x.nct); x.copies = js;
                const long long blocks = x.blocks + js.j[0].tiles + js.j[1].tiles + js.j[2].tiles;
                FEA_CHECK(blocks < INT_MAX, FEA_E_UNSUPPORTED_SHAPE, "%s: %lld tiles", who, blocks);
                const dim3 grid((unsigned)blocks), bl(256);
                auto launch = [&](auto even, auto odd) { if (d.odd()) hipLaunchKernelGGL(odd, grid, bl, 0, s, x); else hipLaunchKernelGGL(even, grid, bl, 0, s, x); };
                if (kept.codes)             launch(lin_decode_kernel<__bf16, true, false, true>, lin_decode_kernel<__bf16, true, false, false>);
                else if (dtype == FEA_BF16) launch(lin_decode_kernel<__bf16, false, false, true>, lin_decode_kernel<__bf16, false, false, false>);
                else if (p.planes)          launch(lin_decode_kernel<float, false, true, true>, lin_decode_kernel<float, false, true, false>);
                else                        launch(lin_decode_kernel<float, false, false, true>, lin_decode_kernel<float, false, false, false>);
                FEA_LAUNCH_CHECK();
            } else LIN_TRY(fea_lin_gemm(LIN_DZ, f.dt, p.tz, g, s));
            const long long entries = n * K;
            const long long* ix = index + r0 * K;
            if (!keep || K > 1) {
                const unsigned sg = (unsigned)((entries + 255) / 256);
                if (pack || keep) js = LinCopies{};
                const long long blocks = sg + js.j[0].tiles + js.j[1].tiles + js.j[2].tiles;
                FEA_CHECK(blocks < INT_MAX, FEA_E_UNSUPPORTED_SHAPE, "%s: %lld tiles", who, blocks);
                const dim3 grid((unsigned)blocks), bl(256);
                const float* ds = dsel + r0 * K;
                if (f.dt == FEA_PL)        hipLaunchKernelGGL((lin_scatter_kernel<__bf16, true, true>), grid, bl, 0, s, ix, ds, K, st, (__bf16*)b.dz, g.lddz, v0, nv, entries, g.Npad, sg, js);
                else if (f.dt == FEA_BF16) hipLaunchKernelGGL((lin_scatter_kernel<__bf16, false, true>), grid, bl, 0, s, ix, ds, K, st, (__bf16*)b.dz, g.lddz, v0, nv, entries, 0, sg, js);
                else if (d.odd())          hipLaunchKernelGGL((lin_scatter_kernel<float, false, false>), grid, bl, 0, s, ix, ds, K, st, (float*)b.dz, g.lddz, v0, nv, entries, 0, sg, js);
                else                       hipLaunchKernelGGL((lin_scatter_kernel<float, false, true>), grid, bl, 0, s, ix, ds, K, st, (float*)b.dz, g.lddz, v0, nv, entries, 0, sg, js);
                FEA_LAUNCH_CHECK();
            }
            if (db) {
                const int tm = keep ? 128 : p.tz, tiles = (int)((n + tm - 1) / tm), chunks = (int)((n + LIN_DB_ROWS - 1) / LIN_DB_ROWS);
                hipLaunchKernelGGL(lin_dbias_kernel, dim3((unsigned)((nv + 255) / 256), (unsigned)chunks), dim3(64 * LIN_DB_WAVES), 0, s, (const float*)b.colsum, tiles, (long long)g.ldcol, ix, psel ? psel + r0 * K : nullptr, K, st, go, gout_stride, count, temperature, v0, nv, entries, LIN_DB_ROWS / tm, (long long)LIN_DB_ROWS * K, b.dbpart);
                FEA_LAUNCH_CHECK();
                hipLaunchKernelGGL(lin_dbias_join_kernel, dim3((unsigned)((nv + 255) / 256)), dim3(256), 0, s, (const double*)b.dbpart, chunks, nv, db + v0, ir > 0 ? 1 : 0);
                FEA_LAUNCH_CHECK();
            }
            // out (contiguous rows of D) = dz . B or dz^T . B over k channels: straight to out, or through fp32 slabs where the reduction is
            // split or pieces before this one (acc) or behind it add to the sum
            auto product = [&](bool ta, int scale, const void* B, long long ldb, long long M, long long k, const LinTile& t, void* out, float* acc, bool first, bool last) {
                LinGemm m{};
                m.stat = st; m.gout = go; m.gstride = gout_stride; m.count = count; m.t = temperature;
                m.a = b.dz; m.lda = f.row(nv); m.ta = ta; m.b = B; m.ldb = ldb; m.scale = scale;
                m.M = (int)M; m.N = D; m.K = f.K(k); m.Kp = (int)up(k, 64); m.Kr = (int)k; m.Pa = (int)up(nv, 64); m.Pb = (int)up(D, 64);
                m.splits = t.splits; m.kper = (int)up((m.K + t.splits - 1) / t.splits, 64);
                const bool direct = t.splits == 1 && first && last && d.straight();
                m.ldo = up(D, 4);
                if (direct && f.dt != FEA_PL) m.out = out; else m.slab = direct ? (float*)out : b.slab;
                LIN_TRY(fea_lin_gemm(LIN_STORE, f.dt, t.tile, m, s));
                return direct ? FEA_OK : lin_reduce(d, b.slab, t.splits, M, first ? nullptr : acc, last ? nullptr : acc, last ? out : nullptr, s);
            };
            if (dh) LIN_TRY(product(false, 1, wk, ldwk, n, nv, p.th, (char*)dh + r0 * D * d.es, b.acch, iv == 0, iv + 1 == p.nvc));
            if (dw) LIN_TRY(product(true, gout_stride ? 0 : 2, gated ? b.hg : b.hp, f.row(D), nv, n, p.tw, (char*)dw + v0 * D * d.es, b.accw ? b.accw + v0 * up(D, 4) : nullptr, ir == 0, ir + 1 == p.nrc));
        }
    }
    return FEA_OK;
}
