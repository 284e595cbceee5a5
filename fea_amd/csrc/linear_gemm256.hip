// The products of the many-class loss heads on the bf16 matrix rate, 256 x 256 and 128 x 128 tiles, with the epilogues of linear_gemm.hip.
//
// A tile of T x T takes T T / (2 T) = T / 2 multiply-adds per operand element it reads: at 256 a CU at full matrix rate asks for
// 32 B per cycle from L2 (128: 64 B, twice what L2 gives) and for 64 KB of LDS reads per 32-channel step of 1,024 cycles.  Four waves of
// 128 x 128 read each operand twice (8 fragments of each per step and wave: half the LDS rate); eight waves of 128 x 64 would read
// 96 KB, with the fill the whole LDS rate.  So: one workgroup of 4 waves per CU, one wave per SIMD, 8 x 8 accumulators of
// v_mfma_f32_16x16x32_bf16 in the 256 accumulation registers, fragments and addresses in the other 256.
//
// 256 tile: chunks of 64 channels (whole 128-byte lines) go from memory to LDS without a register in between, a wave's 1,024 bytes per load, in
// a ring of five operand chunks of 32 KB (all of the CU's 160 KB): 16 loads per chunk, one per 8 MFMA, 1 to 1.5 chunks ahead; one
// barrier per chunk.  128 tile (two workgroups per CU): through registers, three chunks on the way
// (two: 20 % slower where few workgroups go through a long reduction, 150 x 4,096 x 8,000), two LDS stages.
// Loads are buffer loads with every bound in the descriptor or the lane's offset: rows, classes and channels behind the end arrive as zeros
// without a branch.
//
// Measured on 4,096 x 4,096 x 131,072 (a third of a training step each): h w^T with softmax sums and kept logits 3.7 ms (1.19 PFLOP/s;
// 3.36 without keeping), dz w 3.3 ms (1.33), dz^T h 3.9 ms (1.13); a library's plain products 2.98, 3.16 and 3.85 ms.  Bound by power:
// at 60 % of the matrix pipes' cycles the clock is down to 1.9 GHz, and a loop of nothing but these MFMA on normally distributed
// operands reaches 2.1 PFLOP/s (32 x 32 x 16 MFMA: 1.85), so what helps is less traffic and an even one: through registers and with LDS
// writes the step took 4 % longer, with the same direct loads in bursts 5 %.
#include "linear_loss.h"



// XOR of a 128-byte row's 16-byte chunk index: conflict-free ds_read_b128 of 16 rows x 4 chunks
__device__ __forceinline__ int lb_swz(int row) { return ((row >> 1) & 3) << 1; }

__device__ __forceinline__ uint32_t lb_pack(float a, float b) {
    typedef __attribute__((ext_vector_type(2))) float f2;
    typedef __attribute__((ext_vector_type(2))) __bf16 b2;
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, b2));
}

// NT: 16-row tiles of a wave in either direction (8: 256 x 256 per workgroup, one per CU; 4: 128 x 128, two per CU).
// TA, TB: the operand lies with its rows along the reduction ([k][m] / [k][n]: dz for dw, hidden and weight for dw and dh): its LDS tile is
// 64 rows of the tile's width, and fragments come out of it by the transposing read (ds_read_b64_tr_b16), two for 8 channels.
// No transposed copy of either weight, hidden or dz is ever made.
template <int EPI, bool PL, int NT, bool TA, bool TB>
__global__ __launch_bounds__(256, NT == 8 ? 1 : 2) void lin_gemm256_kernel(const LinGemm g) {
    constexpr int LB_T = 32 * NT, LB_W = 16 * NT, NL = 2 * NT;
    constexpr bool DL = NT == 8;                          // loads go to LDS by themselves
    constexpr int RB = DL ? 2 * LB_T : 2 * LB_T + 32, TOP = DL ? 64 * RB : 64 * RB + 8 * 128;     // a row along the reduction, an operand of them
    constexpr int LB_OP = TA ? TOP : LB_T * 128, LB_STAGE = LB_OP + (TB ? TOP : LB_T * 128);
    __shared__ __attribute__((aligned(128))) char smem[DL ? 5 * LB_OP : 2 * LB_STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave & 1, wn = wave >> 1, r16 = lane & 15, q16 = lane >> 4;
    // tiles in groups of 8 row tiles, walked along the classes: the 32 tiles that an XCD has in flight are 8 x 4
    constexpr int GM = NT;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int per = g.ntm * g.ntn, sp = id / per, it = id - sp * per;
    const int grp = it / (GM * g.ntn), gm = min(GM, g.ntm - grp * GM), in = it - grp * GM * g.ntn;
    const int tm = grp * GM + in % gm, tn = in / gm;
    const int m0 = tm * LB_T, n0 = tn * LB_T;
    const int k0 = EPI == LIN_DZ ? 0 : sp * g.kper, K = max((EPI == LIN_DZ ? g.K : min(k0 + g.kper, g.K)) - k0, 0);
    const int nc = (K + 63) >> 6;

    auto rsrc = [&](const __bf16* p, long long ld, int rows, int cols) {       // rows x cols of a matrix; 0 rows: nothing is read
        const int bytes = rows > 0 ? (int)(((rows - 1) * ld + cols) * 2) : 0;
        if constexpr (DL) return u32x4{(uint32_t)(uintptr_t)p, (uint32_t)((uintptr_t)p >> 32) & 0xffffu, (uint32_t)bytes, 0x00020000u};
        else return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00020000);
    };
    const int kf = PL ? 0 : k0, kl = PL ? 3 * g.Kp : K;      // first channel and length of a row along the reduction
    const __bf16 *const a = (const __bf16*)g.a, *const b = (const __bf16*)g.b;
    auto rsa = rsrc(a + m0 * g.lda + kf, g.lda, K ? min(LB_T, g.M - m0) : 0, kl);
    auto rsb = rsrc(b + n0 * g.ldb + kf, g.ldb, K ? min(LB_T, g.N - n0) : 0, kl);

    // Staging, rows along the tile: thread -> LDS rows r + 32 i, 16-byte chunk c.  Which class lies in which LDS row is chosen for the
    // epilogue: the lane that ends up with column r16 of the products holds, over tiles 2 p and 2 p + 1, 8 consecutive classes.
    const int r = tid >> 3, c = DL ? (tid & 7) ^ lb_swz(r) : tid & 7;
    const int rb = ((r >> 4) & 1) * 4 + ((r >> 2) & 3) * 8 + (r & 3);
    const int wofs = r * 128 + ((c ^ lb_swz(r)) << 4);
    // Rows along the reduction: thread -> rows tr + RPP i of the chunk's 64, 16-byte piece tc.  The 8 rows x 32 bytes that half a wave takes in
    // one transposing read have to lie in different banks.  256 tile: the 32-byte pieces of a row are XORed by fr of the row (its bits 0, 1
    // and 3), on the way in by which piece a lane loads (odd i: the row's bit 3 is set).  128 tile: a row is 32 bytes longer than its
    // data and every 8 rows have 128 more, so that tiles, steps and loads are constant offsets.
    constexpr int CPR = LB_T / 8, RPP = 256 / CPR;
    const int tr = tid / CPR, tc = DL ? (tid % CPR) ^ ((tr & 3) << 1) : tid % CPR;
    const int tofs = tr * RB + (tr >> 3) * 128 + tc * 16;
    const unsigned va = TA ? (unsigned)(tr * (int)g.lda * 2 + tc * 16) : (unsigned)(r * (int)g.lda * 2 + c * 16), va1 = DL && TA ? va + ((tc ^ 8) - tc) * 16 : va;
    const unsigned vb = TB ? (unsigned)(tr * (int)g.ldb * 2 + tc * 16) : (unsigned)(rb * (int)g.ldb * 2 + c * 16), vb1 = DL && TB ? vb + ((tc ^ 8) - tc) * 16 : vb;
    const unsigned sa = 2 * (TA ? RPP : 32) * (unsigned)g.lda, sb = 2 * (TB ? RPP : 32) * (unsigned)g.ldb;      // bytes from load i to i + 1
    constexpr int SETS = TB && !TA ? 2 : 3;           // 128 tile: chunks on the way in registers (two where a third would not fit)
    u32x4 st[DL ? 1 : SETS][DL ? 1 : NL];
    // the XCDs start their reduction an eighth apart (it ends where it began): in step, every workgroup of the chip would ask for the
    // same columns of its rows at a time.  Within an XCD all are in step: they share operands in its L2.
    // (FEA_PL: a pair of planes and a channel)
    struct Pos { int at, pair, pk; };
    const int start = (int)(blockIdx.x & 7) * nc >> 3;
    Pos pa{start, PL ? (k0 + start * 64) / g.Kp : 0, 0};
    if constexpr (PL) pa.pk = k0 + start * 64 - pa.pair * g.Kp;
    Pos pb = pa;
    unsigned ka = 0, kb = 0;
    bool ina = false, inb = false;
    const int ca = min(LB_T, (g.M - m0 + 7) & ~7), cb = min(LB_T, (g.N - n0 + 7) & ~7);        // (whole 16-byte pieces: rows are padded)
    auto next = [&](Pos& p) {
        if (++p.at == nc) {
            p.at = 0;
            if constexpr (PL) { p.pair = k0 / g.Kp; p.pk = k0 - p.pair * g.Kp; }
        } else if constexpr (PL) {
            p.pk += 64;
            if (p.pk >= g.Kp) { p.pk = 0; ++p.pair; }
        }
    };
    auto first = [&](const Pos& p) { return PL ? p.pk : k0 + p.at * 64; };
    auto advance_a = [&](int ch) {      // where A's chunk that is loaded ch-th lies (behind the last: nowhere, zeros)
        const bool live = ch < nc;
        ina = live && pa.at * 64 + c * 8 < K;
        if constexpr (TA) rsa = rsrc(a + first(pa) * g.lda + m0 + (PL ? lin_plane_a(pa.pair) * g.Pa : 0), g.lda, live ? min(64, g.Kr - first(pa)) : 0, ca);
        else ka = PL ? 2u * (unsigned)(lin_plane_a(pa.pair) * g.Kp + pa.pk) : pa.at * 128;
        next(pa);
    };
    auto advance_b = [&](int ch) {
        const bool live = ch < nc;
        inb = live && pb.at * 64 + c * 8 < K;
        if constexpr (TB) rsb = rsrc(b + first(pb) * g.ldb + n0 + (PL ? lin_plane_b(pb.pair) * g.Pb : 0), g.ldb, live ? min(64, g.Kr - first(pb)) : 0, cb);
        else kb = PL ? 2u * (unsigned)(lin_plane_b(pb.pair) * g.Kp + pb.pk) : pb.at * 128;
        next(pb);
    };
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem + wave * 1024;
    auto address = [&](int i) {        // of the lane's 16 bytes of load i (A's, then B's); 0x7fffff00: behind any end
        const int q = i % NT;
        return i < NT ? TA || ina ? (q & 1 ? va1 : va) + ka + q * sa : 0x7fffff00u : TB || inb ? (q & 1 ? vb1 : vb) + kb + q * sb : 0x7fffff00u;
    };
    auto dload = [&](int slot, int i) {     // a wave's 1,024 bytes straight to LDS: nothing lands in a register, and `landed` waits
        const uint32_t m = lds + slot * LB_OP + i % NT * 4096;
        if (i < NT) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" :: "s"(m), "v"(address(i)), "s"(rsa) : "memory", "m0");
        else        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" :: "s"(m), "v"(address(i)), "s"(rsb) : "memory", "m0");
    };
    auto gload = [&](int u, int i) {
        if constexpr (!DL) st[u][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(i < NT ? rsa : rsb, address(i), 0, 0));
    };
    auto lput = [&](int u, int stage, int i) {
        const int ofs = (i < NT ? TA : TB) ? tofs + (i % NT) * (RPP * RB + RPP / 8 * 128) : wofs + (i % NT) * 32 * 128;
        *reinterpret_cast<u32x4*>(smem + stage * LB_STAGE + (i / NT) * LB_OP + ofs) = st[u][i];
    };

    // fragments: lane -> row r16 of tile i, channels 8 q16 .. + 7 of the 32 of step ks
    const int fofs0 = r16 * 128 + ((q16 ^ lb_swz(r16)) << 4), fofs1 = fofs0 ^ 64;
    const int fofst = (8 * q16 + (r16 >> 2)) * RB + (DL ? 0 : q16 * 128) + (r16 & 3) * 8, fr = (r16 >> 2) | (q16 & 1) << 2;      // 16 lanes: 4 rows of 16 columns
    u32x4 A[2][NT], B[2][NT];
    auto frag = [&](const char* op, int w, int ks, int i, bool t) {
        if (!t) return *reinterpret_cast<const u32x4*>(op + (ks ? fofs1 : fofs0) + (w * LB_W + i * 16) * 128);
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4_t;
        const char* p = op + fofst + w * (2 * LB_W) + (DL ? (i ^ fr) * 32 + ks * (32 * RB) : i * 32 + ks * (32 * RB + 4 * 128));
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)p));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(p + 4 * RB)));
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    auto fread = [&](const char* sa_, const char* sb_, int ks, int i) {
        if (i < NT) A[ks][i] = frag(sa_, wm, ks, i, TA);
        else        B[ks][i - NT] = frag(sb_, wn, ks, i - NT, TB);
    };
    auto frd = [&](int stage, int ks, int i) { fread(smem + stage * LB_STAGE, smem + stage * LB_STAGE + LB_OP, ks, i); };
    f32x4 acc[NT][NT];                // [label tile][class tile]
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto mma = [&](int ks, int i, int j) {
        // (as inline asm where all 256 are taken: the compiler would move accumulators between the register files in every step)
        if constexpr (DL) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc[i][j]) : "v"(B[ks][j]), "v"(A[ks][i]));
        else acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, B[ks][j]), __builtin_bit_cast(bf16x8, A[ks][i]), acc[i][j], 0, 0, 0);
    };

    // LIN_LSE: the selected classes of the tile's row tid, asked for in front of the first chunk and looked at in the epilogue: where they are
    // (lin_where_kernel), or one label
    uint2 where = make_uint2(~0u, ~0u);
    if constexpr (EPI == LIN_LSE)
        if (g.zsel && tid < LB_T && m0 + tid < g.M)
            where = g.where ? g.where[(long long)(m0 + tid) * g.ntn + tn] : __builtin_bit_cast(uint2, g.index[m0 + tid]);

    if constexpr (DL) {
        // A ring of five operand chunks: A(c) in slot 2 c mod 5, B(c) in 2 c + 1 mod 5.  Half-way through chunk c its fragments are all in registers, so
        // B(c + 2) goes where A(c) was, and in the next half A(c + 3) where B(c) was.  Loads are spread evenly (one per 8 MFMA): the
        // same loads in bursts of the second half cost 3 to 5 % of the product.
        auto landed = [&](bool first) {       // everything but A's 8 loads of the chunk after the next (first: all 16 of chunk 1) is there, and read by nobody any more
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
            if (first) __builtin_amdgcn_s_waitcnt(0x4070);     // vmcnt(16) lgkmcnt(0)
            else       __builtin_amdgcn_s_waitcnt(0x0078);     // vmcnt(8) lgkmcnt(0)
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        int a0 = 0, b0 = 1, a1 = 2, b1 = 3, a2 = 4;
        advance_a(0); advance_b(0);
#pragma unroll
        for (int i = 0; i < NL; ++i) dload(i < NT ? a0 : b0, i);
        advance_a(1); advance_b(1);
#pragma unroll
        for (int i = 0; i < NL; ++i) dload(i < NT ? a1 : b1, i);
        landed(true);
        advance_a(2);
#pragma unroll
        for (int i = 0; i < NL; ++i) fread(smem + a0 * LB_OP, smem + b0 * LB_OP, 0, i < NT ? i + NT : i - NT);
        for (int ch = 0; ch < nc; ++ch) {
            // in slots of half a row of MFMAs.  First half: the second half's fragments, and A(ch + 2)
#pragma unroll
            for (int q = 0; q < NL; ++q) {
#pragma unroll
                for (int j = 0; j < NT / 2; ++j) mma(0, q / 2, (q & 1) * (NT / 2) + j);
                if (q < NT) { fread(smem + a0 * LB_OP, smem + b0 * LB_OP, 1, NT + q); fread(smem + a0 * LB_OP, smem + b0 * LB_OP, 1, q); }
                if (q & 1) dload(a2, q / 2);
                __builtin_amdgcn_sched_barrier(0);
            }
            advance_b(ch + 2);
            landed(false);
            // second half: the first fragments of chunk ch + 1 (done early: the loop's head waits for all), and B(ch + 2)
#pragma unroll
            for (int q = 0; q < NL; ++q) {
#pragma unroll
                for (int j = 0; j < NT / 2; ++j) mma(1, q / 2, (q & 1) * (NT / 2) + j);
                if (!(q & 1)) dload(a0, NT + q / 2);
                if (q < NT + 4) fread(smem + a1 * LB_OP, smem + b1 * LB_OP, 0, q < NT ? q + NT : q - NT);
                if (q >= NT && q < NT + 4) fread(smem + a1 * LB_OP, smem + b1 * LB_OP, 0, q - NT + 4);
                __builtin_amdgcn_sched_barrier(0);
            }
            advance_a(ch + 3);
            const int fa = a0, fb = b0;
            a0 = a1; b0 = b1; a1 = a2; b1 = fa; a2 = fb;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // (the loads behind the last chunk, zeros, are in LDS too)
        // (the compiler does not know that inline asm has written the accumulators that are read from here on)
        asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" ::: "memory");
    } else {
    // (in the loop's order: its waits are counted for both ways in)
    auto ahead = [&](int ch) {
        advance_a(ch); advance_b(ch);
#pragma unroll
        for (int i = 0; i < NL; ++i) { gload(ch % SETS, i); __builtin_amdgcn_sched_barrier(0); }
    };
#pragma unroll
    for (int u = 0; u < SETS; ++u) ahead(u);
#pragma unroll
    for (int i = 0; i < NL; ++i) lput(0, 0, i);
    ahead(SETS);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int f = i < NT ? i + NT : i - NT;
        if (!(TA || TB) || f < 3 || f >= NT) frd(0, 0, f);
        __builtin_amdgcn_sched_barrier(0);
    }

    // chunk ch of LDS stage s; chunk ch + 1 lies in register set u, where chunk ch + 1 + SETS follows it
    auto step = [&](int ch, int s, int u) {
        auto landed = [&]() {         // chunk ch + 1 is in LDS and nobody reads this stage or the other one's old chunk any more
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
        };
        advance_a(ch + 1 + SETS); advance_b(ch + 1 + SETS);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (TA || TB) {
            // slots: half a row of MFMAs, then a fragment of the second half (in every second slot one of this half, three tiles ahead), an
            // LDS write and a load
#pragma unroll
            for (int q = 0; q < NL; ++q) {
#pragma unroll
                for (int j = 0; j < NT / 2; ++j) mma(0, q / 2, (q & 1) * (NT / 2) + j);
                frd(s, 1, q < NT ? q + NT : q - NT);
                if (q % 2 == 0 && q / 2 + 3 < NT) frd(s, 0, q / 2 + 3);
                lput(u, s ^ 1, q);
                gload(u, q);
                __builtin_amdgcn_sched_barrier(0);
            }
            landed();
#pragma unroll
            for (int q = 0; q < NL; ++q) {
#pragma unroll
                for (int j = 0; j < NT / 2; ++j) mma(1, q / 2, (q & 1) * (NT / 2) + j);
                if (q < NT) frd(s ^ 1, 0, NT + q);
                else if (q < NT + 3) frd(s ^ 1, 0, q - NT);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            // the same by group: 2 MFMA (1 before the read in every second group), an LDS read, an LDS write, a load
#pragma unroll
            for (int q = 0; q < NL; ++q) { frd(s, 1, q); lput(u, s ^ 1, q); gload(u, q); }
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) mma(0, i, j);
#pragma unroll
            for (int q = 0; q < NL; ++q) {
                if (q & 1) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            }
            landed();
#pragma unroll
            for (int q = 0; q < NL; ++q) frd(s ^ 1, 0, q);
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) mma(1, i, j);
#pragma unroll
            for (int q = 0; q < NL; ++q) {
                __builtin_amdgcn_sched_group_barrier(0x008, NT / 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
        }
    };
    // (left in the middle, not skipped over: only so the compiler's counts of what is on the way stay exact)
    bool more = nc > 0;
    for (int ch = 0; more;)
#pragma unroll
        for (int i = 0; i < 2 * SETS; ++i) {
            step(ch, i & 1, (i + 1) % SETS);
            if (++ch >= nc) { more = false; break; }
        }
    }
    __syncthreads();

    auto mrow = [&](int i) { return m0 + wm * LB_W + i * 16 + r16; };                                    // label of tile i
    // first of the 4 classes of tile j; first of the 8 that a lane has of tiles 0 and 1: as they lie, or after an exchange between
    // neighbouring 16-lane rows
    auto ncol = [&](int j) { return n0 + wn * LB_W + (TB ? j * 16 + 4 * q16 : (j >> 1) * 32 + q16 * 8 + (j & 1) * 4); };
    const int pcol = n0 + wn * LB_W + (TB ? (q16 & 1) * 16 + (q16 >> 1) * 8 : q16 * 8);
    auto pairs = [&](const f32x4& x, const f32x4& y) {
        const u32x4 v = {lb_pack(x[0], x[1]), lb_pack(x[2], x[3]), lb_pack(y[0], y[1]), lb_pack(y[2], y[3])};
        if constexpr (!TB) return v;
        const auto r0 = __builtin_amdgcn_permlane16_swap(v[0], v[2], false, false);
        const auto r1 = __builtin_amdgcn_permlane16_swap(v[1], v[3], false, false);
        return u32x4{r0[0], r1[0], r0[1], r1[1]};
    };

    if constexpr (EPI == LIN_STORE) {
        const float common = g.scale == 2 ? lin_row_scale(g.gout, 0, g.count, g.t, 1.f, 0) : 1.f;
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
                    if (m < g.M && n < g.N) *reinterpret_cast<f32x4*>(o + n) = acc[i][j];
                }
            } else {
                __bf16* const o = (__bf16*)g.out + m * g.ldo;
#pragma unroll
                for (int p = 0; p < NT / 2; ++p) {
                    const u32x4 v = pairs(acc[i][2 * p], acc[i][2 * p + 1]);
                    if (m < g.M && pcol + 32 * p < g.N) *reinterpret_cast<u32x4*>(o + pcol + 32 * p) = v;
                }
            }
        }
    }
    if constexpr (EPI == LIN_LSE)
        if (g.slab) {            // split: the sums as they are, joined by lin_join_split_kernel
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    if (mrow(i) < g.M && ncol(j) < g.ldo) *reinterpret_cast<f32x4*>(g.slab + ((long long)sp * g.M + mrow(i)) * g.ldo + ncol(j)) = acc[i][j];
            return;
        }
    // z of a lane's 4 classes of tile j, label tile i; classes behind the last are -inf (whatever 0 times the label's row gave)
    f32x4 bias[EPI == LIN_STORE ? 1 : NT];
    if constexpr (EPI != LIN_STORE) {
        if (n0 + LB_T > g.N)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int i = 0; i < NT; ++i) acc[i][j][e] = ncol(j) + e < g.N ? acc[i][j][e] : 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) bias[j][e] = ncol(j) + e >= g.N ? -INFINITY : g.bias ? g.bias[ncol(j) + e] * g.inv_t : 0.f;
    }
    auto logits = [&](int i, int j) {
        f32x4 z;
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = fmaf(acc[i][j][e], g.inv_t, bias[j][e]);
        return z;
    };

    if constexpr (EPI == LIN_LSE) {
        // every lane's own maximum and sum of a label's 4 NT classes, joined in LDS: nothing goes across lanes on the way, and a label's kept
        // logits leave while the next one's exponentials run
        float2* const red = reinterpret_cast<float2*>(smem);       // [wn, q16][labels of the tile]
        uint2* const wanted = reinterpret_cast<uint2*>(red + 8 * LB_T);
        if (g.zsel) {
            if (!g.where) {
                const long long t = __builtin_bit_cast(long long, where);      // (~0 where the row is none: no class)
                where = make_uint2(t >= n0 && t < min(n0 + LB_T, g.N) ? 0xffff0000u | (unsigned)(t - n0) : ~0u, ~0u);
            }
            if (tid < LB_T) wanted[tid] = where;
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int m = mrow(i);
            f32x4 z[NT];
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                z[j] = logits(i, j);
                mx = fmaxf(fmaxf(mx, fmaxf(z[j][0], z[j][1])), fmaxf(z[j][2], z[j][3]));
            }
            const float base = mx == -INFINITY ? 0.f : mx;         // every class masked by a -inf bias: the sum is 0, not NaN
            if (g.keep && m < g.M) {
                if (PL || !g.top) {
                    float* const o = (float*)g.keep + m * g.ldkeep;
#pragma unroll
                    for (int j = 0; j < NT; ++j) if (ncol(j) < g.ldkeep) *reinterpret_cast<f32x4*>(o + ncol(j)) = z[j];
                } else {
                    uint16_t* const o = (uint16_t*)g.keep + m * g.ldkeep;
                    const float t = base / LIN_RANGE;
                    g.top[((n0 / LB_W + wn) * g.ldtop + m) * 4 + q16] = base;
#pragma unroll
                    for (int p = 0; p < NT / 2; ++p) {
                        u32x4 v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = z[2 * p + (e >> 1)][2 * (e & 1)], y = z[2 * p + (e >> 1)][2 * (e & 1) + 1];
                            v[e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_u16(t - x / LIN_RANGE, t - y / LIN_RANGE));
                        }
                        if (pcol + 32 * p < g.ldkeep) *reinterpret_cast<u32x4*>(o + pcol + 32 * p) = v;
                    }
                }
            }
            if (g.zsel) {
                // one lane of the chip has a selected logit: out of its 4 NT
                auto give = [&](unsigned col, int k) {
                    if (col / LB_W != (unsigned)wn || ((col >> 3) & 3) != (unsigned)q16) return;
                    const unsigned at = (col % LB_W >> 5) * 8 + (col & 7);
                    float x = z[0][0];
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) x = at == 4 * j + e ? z[j][e] : x;
                    g.zsel[(long long)m * g.sel + k] = x;
                };
                const uint2 w = wanted[wm * LB_W + i * 16 + r16];
                if ((w.x & 0xffffu) == LIN_MANY)
                    for (int k = 0; k < g.sel; ++k) {
                        const long long t = g.index[(long long)m * g.sel + k];
                        if (t >= n0 && t < min(n0 + LB_T, g.N)) give((unsigned)(t - n0), k);
                    }
                else
                    for (uint64_t h = w.x | (uint64_t)w.y << 32; (h & 0xffffu) != LIN_NONE; h = h >> 16 | (uint64_t)LIN_NONE << 48) give((unsigned)h & 255u, (int)(h >> 8) & 255);
            }
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += __expf(z[j][e] - base);
            red[(wn * 4 + q16) * LB_T + wm * LB_W + i * 16 + r16] = make_float2(mx, sum);
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
        if (tid < LB_T && m0 + tid < g.M) {
            float2 p[8];
            float mx = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) { p[w] = red[w * LB_T + tid]; mx = fmaxf(mx, p[w].x); }
            const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
            for (int w = 0; w < 8; ++w) sum += p[w].y * __expf(p[w].x - base);
            g.part[(long long)(m0 + tid) * g.ntn + tn] = make_float2(mx, sum);
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
            for (int j = 0; j < NT; ++j) {
                const f32x4 z = logits(i, j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float q = __expf(z[e] - s2.x);
                    acc[i][j][e] = dead || (n0 + LB_T > g.N && ncol(j) + e >= g.N) ? 0.f : q;
                }
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
    if (epi == LIN_LSE)     hipLaunchKernelGGL((lin_gemm256_kernel<LIN_LSE, PL, NT, false, false>), dim3(grid), dim3(256), 0, s, g);
    else if (epi == LIN_DZ) hipLaunchKernelGGL((lin_gemm256_kernel<LIN_DZ, PL, NT, false, false>), dim3(grid), dim3(256), 0, s, g);
    else if (g.ta)          hipLaunchKernelGGL((lin_gemm256_kernel<LIN_STORE, PL, NT, true, true>), dim3(grid), dim3(256), 0, s, g);
    else                    hipLaunchKernelGGL((lin_gemm256_kernel<LIN_STORE, PL, NT, false, true>), dim3(grid), dim3(256), 0, s, g);
}
void fea_lin_gemm256(int epi, int tile, bool planes, const LinGemm& g, unsigned grid, hipStream_t s) {
    if (tile == 256) { if (planes) lb_launch<true, 8>(epi, g, grid, s); else lb_launch<false, 8>(epi, g, grid, s); }
    else             { if (planes) lb_launch<true, 4>(epi, g, grid, s); else lb_launch<false, 4>(epi, g, grid, s); }
}
