// Shared between the files of the many-class loss heads: linear_loss.hip (entry points, statistics, layouts), linear_gemm256.hip (bf16 products),
// linear_gemm.hip (fp32 products, the choice of a tile), linear_rows.hip (few rows), linear_few.hip (few classes).
#pragma once
#include "common.h"

// LIN_LSE, LIN_DZ: C = A . B^T, A rows = label rows, B rows = classes, the reduction along the rows of both.
// LIN_STORE: C = A . B or A^T . B, B [K][N] with its rows along the reduction, A [M][K] or (ta) [K][M].
// Row starts are 16-byte aligned (fp32 B of LIN_STORE and both operands of the others may be odd).
enum { LIN_LSE = 0, LIN_DZ = 1, LIN_STORE = 2 };

// fp32 operands of large products as three bf16 planes: x = x0 + x1 + x2, each the rounding of what the ones before leave, so the sum holds
// all 24 bits.  A row is [plane 0 | plane 1 | plane 2], each of its length rounded up to 64 and zero behind the end.  A product runs over the
// six pairs of planes whose weight is above 2^-24 (x1 y1, x2 y0, x0 y2, x1 y0, x0 y1, x0 y0, the small ones first, all into one fp32
// sum): the bf16 matrix rate is 16 times the fp32 one, so six products still gain 2.7.  FEA_PL is the form's dtype code inside these files.
#define FEA_PL 2
__device__ __forceinline__ int lin_plane_a(int pair) { return (0x001021 >> (4 * pair & 31)) & 15; }     // (behind the last pair: any, nothing is read there)
__device__ __forceinline__ int lin_plane_b(int pair) { return (0x010201 >> (4 * pair & 31)) & 15; }

// Kept logits of a bf16 head: 16 bits each.  exp(z - lse) goes to bf16 next, which rounds it by up to 2^-8 of itself; a fixed-point z is off by
// half a step, 4.9e-4 of exp(z - lse), whatever z is.  Entries e^-64 times the largest of their
// group and less count as 0.
#define LIN_RANGE 64.f
#define LIN_STEP (LIN_RANGE / 65535.f)

// Where a row's selected classes lie: for every row and column tile up to four entries of 16 bits (column of the tile, k << 8), LIN_NONE behind
// them; LIN_MANY in the first: more than four, look through all.  At most LIN_WHERE_K entries per row, LIN_WHERE_T tiles.
#define LIN_NONE 0xffffu
#define LIN_MANY 0xfffeu
#define LIN_WHERE_K 254
#define LIN_WHERE_T 1280

struct LinGemm {
    const void *a, *b;
    long long lda, ldb;
    int M, N, K;                      // rows, columns, reduction
    int ta;                           // LIN_STORE: A is [K][M]
    int Kp, Kr, Pa, Pb;               // FEA_PL: reduction of one plane rounded up to 64 (K = 6 Kp) and as it is; planes of A / B rows that hold M / N elements
    // LIN_LSE, LIN_DZ: z = (a . b + bias) * inv_t
    const float* bias;                // [N], nullable
    float inv_t;
    float2* part;                     // LIN_LSE: [M][ntn] (max, sum of exp(z - max)) of one column tile
    void* keep; long long ldkeep;     // LIN_LSE, nullable: the logits kept for the backward, rows of ldkeep (classes rounded up to 64): fp32 z, or (bf16, with top) how far
                                      // z lies below the largest of its group, in steps of LIN_STEP (65535: LIN_RANGE and more, and classes behind the last)
    float* top; long long ldtop;      // the groups' largest, [half tile][ldtop rows][4]; a group: every fourth 8 classes of half a tile's (what a lane holds of a row)
    const float2* stat;               // LIN_DZ: [M] (log sum exp, gate)
    const float* gout; int gstride;   // upstream gradient, one value (stride 0) or one per row
    const int* count;                 // rows that count (mean), nullable
    float t;                          // temperature
    void* dz; long long lddz;         // LIN_DZ: [M][lddz]
    int Npad;                         // LIN_DZ: columns written (FEA_PL: of each plane), zero behind N
    float* colsum;                    // LIN_DZ: [tiles of A rows][N], nullable: sums of row scale * softmax over the tile's rows
    long long ldcol;
    // LIN_STORE, LIN_LSE of bf16 or FEA_PL: split over K into `splits` parts of kper: direct store to out (splits == 1, slab == NULL) or fp32 slabs (LIN_LSE: plain sums)
    void* out; long long ldo;
    float* slab;                      // [splits][M][ldo], ldo a multiple of 4 (columns behind N hold nothing)
    int scale;                        // 0: none, 1: times the row scale of C's row, 2: times the common scale (gout, count, t above)
    int splits, kper;
    int ntm, ntn;
    // LIN_LSE: selected z of the entries index[M][sel] (nullable); with bf16 or FEA_PL tiles and sel > 1 also where they are (lin_where_kernel)
    float* zsel; const long long* index; int sel;
    const uint2* where;
};

// gradient scale of a row: d loss / d (row loss) times the temperature; 0 for a row that does not count
__device__ __forceinline__ float lin_row_scale(const float* gout, int gstride, const int* count, float t, float gate, long long row) {
    float g = gout[row * gstride] * t;
    if (count) { const int c = *count; g /= (float)(c > 0 ? c : 1); }
    return gate != 0.f ? g : 0.f;
}

// 16 bytes of a row of which `left` elements remain (any sign), zeros behind them.  ALN: rows are 16-byte aligned and `left` is a multiple of
// 16 bytes.  Else the load is unaligned (one instruction all the same) or, at the end of the row, element by element.
template <typename T, bool ALN> __device__ __forceinline__ u32x4 lin_load16(const T* p, int left) {
    constexpr int EPC = Elem<T>::EPC;
    if constexpr (ALN) return left > 0 ? *reinterpret_cast<const u32x4*>(p) : u32x4{0, 0, 0, 0};
    else {
        T x[EPC];
        if (left >= EPC) __builtin_memcpy(x, p, 16);
        else
#pragma unroll
            for (int e = 0; e < EPC; ++e) x[e] = e < left ? p[e] : from_f32<T>(0.f);
        return *reinterpret_cast<const u32x4*>(x);
    }
}

// Few classes, few features, many rows (linear_few.hip)
struct LinFew {
    const void *h, *w;
    long long ldh, ldw;
    const float* bias;
    const long long* index;               // [rows][K]
    const void* tlog; int tdt;            // forward: NULL = cross entropy
    long long ignore;
    float t, inv_t;
    float2* stat;                         // forward: written (nullable); backward: read
    float* psel;                          // [rows][K] teacher shares: forward writes (nullable), backward reads (NULL: cross entropy)
    float* loss_rows;
    double* bsum; int* bcnt;              // [fea_lin_few_blocks]
    const float* gout; int gstride;
    const int* count;
    void* dh;
    float *slab, *dbslab; long long slab_ld;   // [blocks][32 * (32 or 64)], [blocks][32]
    long long rows; int D, V, K;
};
bool fea_lin_few(long long rows, int D, int V);
int fea_lin_few_blocks(long long rows, bool bwd);
int fea_lin_few_fwd(const LinFew& g, int dtype, hipStream_t s);
int fea_lin_few_bwd(LinFew g, int dtype, void* dw, float* db, hipStream_t s);

// linear_gemm.hip: which tile a product takes and into how many parts its reduction is split
struct LinTile { int tile, splits; double time; };
LinTile fea_lin_tile(int dtype, long long M, long long N, long long K, bool split);
int fea_lin_gemm(int epi, int dtype, int tile, LinGemm g, hipStream_t s);
// linear_rows.hip: LIN_LSE of up to 64 label rows; g.part [M][classes / 64], or, with g.splits > 1, sums g.slab [splits][M][ldo]
int fea_lin_rows_splits(int dtype, int V, int D);
int fea_lin_rows(int dtype, bool aligned, LinGemm g, hipStream_t s);
// linear_gemm256.hip
void fea_lin_gemm256(int epi, int tile, bool planes, const LinGemm& g, unsigned grid, hipStream_t s);
