// Matrix product of the block-128 format for sm_100a:
//   C[i][j] = sum_kb sa[kb][i] * sb(kb, j) * sum_{k in block kb} A[i][k] * B[j][k],   A, B E4M3, scales fp32, C bf16 or fp32.
// The scales are no powers of two and belong to 128 values of k, so the tensor core sums one block at a time (four
// tcgen05.mma.kind::f8f6f4 of K = 32 into TMEM, fp32) and registers add the blocks up: acc += (sa * sb) * partial, the scales' product
// rounded once and the fused addition once, in every form.
//
// A CTA, or a pair of CTAs on one tile (cta_group::2), holds 128 rows of X each and TN rows of Y:
//   warp 0      streams operand tiles with TMA (128-byte swizzle) into a ring of stages
//   warp 1      issues the MMAs of block kb into one of two TMEM buffers (leading CTA of a pair)
//   warp 2      brings the scales into a ring of their own with 4-byte asynchronous copies, three blocks ahead, and arrives on the
//               accumulator's barrier beside the MMAs' commit, so that the promoting warps wait once a block
//   4 .. 19     (or 4 .. 7) promote: each reads 32 lanes x 64 columns of the buffer, scales and adds them into registers while the
//               MMAs of block kb + 1 fill the other buffer, and at the end writes its part of C
// The promotion bounds the kernel: 128 x 256 values a CTA and block take 740 cycles, of which the reads of TMEM are 256, the FMAs 256 and
// the rest one probe of a barrier and the latency of the first read; the MMAs take 512.  Under the power limit the clock falls to 1.5 GHz.
// 8192^3 took 848 us with one CTA a tile and 8 promoting warps, 656 with pairs, 547 with 16 warps of 64 columns that hide one
// another's waits, 470 to 487 with the scales on the accumulator's barrier (cuBLAS in bf16 on the same device: 665 to 690 us).  These are
// launches from idle; among other work, under the power limit, it takes 550 to 565 us.
//
// X is the operand whose rows are the lanes of TMEM, Y the one whose rows are its columns: X = A, Y = B.  For few rows of A (SWAP)
// X = B: the weights fill the lanes and a tile has as many columns (a multiple of 16) as there are rows of A.
// Scales that vary by lane cost a register; scales that vary by column would have to reach every lane through shared memory, 128 bytes a
// cycle, 1024 cycles a block, where a lane has one row.  Squares (one scale per 128 columns) do not need them (ROW).  Where both vary,
// the fragment loads of TMEM give a lane 4 rows x 16 columns (FRAG): 256 cycles of shared memory, at half the rate of TMEM.  Weight
// gradients 16384 x 2048 x 7168 in 8 groups, fp32, from idle: 490 us with two rows of 32 columns a lane, 383 us so (435 us among other
// work); squares would lose (253 to 290 us).
// split > 1 (with SWAP): `split` CTAs of one cluster share a tile, each takes a part of the K blocks, sends the others their shares of the
// tile by bulk copies from shared memory to shared memory, and adds up its own in rank order: no workspace, no atomics, the same result
// in every run.  (Words one by one took 3 us read and 6 us sent for 64 rows.)  A 256 x 256 tile has four times the words to exchange:
// splitting it gained nothing (32 blocks: 18.8 us whole, 19.4 in two parts), and tiles of 128 x 64 serve the shapes that it could.
// Shapes: dense; grouped (rows of A belong to groups with their own B, sizes on the device); weight gradient (K belongs to groups);
// vectors (single tokens, a kernel of its own below).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mx8_host.cuh"
#include "mx8_ptx.cuh"

namespace mx8 {
namespace g128 {

constexpr int BK = 128;                       // bytes and elements of K per stage: one scale block
constexpr int MAX_GROUPS = 256;
constexpr int DEV_BAD_GROUPS = MX8_DEV_INPUT_GROUPS;      // device status: group sizes that do not fit the operands
constexpr int DEV_SMEM_BASE = MX8_DEV_SMEM_BASE;          // device status: dynamic shared memory does not start on a 1024-byte boundary
constexpr int EPI0 = 4;                       // the first promoting warp

// ROW: Y's scale is one number per 128 columns.  BOTH: it varies by column.
enum Scales { ROW, BOTH };

template <int CG_, int TN_, bool SWAP_, Scales SC_, bool SPLIT_>
struct Cfg {
    static constexpr int CG = CG_, TN = TN_;                  // CTAs of a tile, rows of Y
    static constexpr bool SWAP = SWAP_, SPLIT = SPLIT_;       // SPLIT: a kernel of its own, as its code takes registers from the main loop (8192^3: 487 -> 540 us)
    static constexpr Scales SC = SC_;
    static constexpr int EPI = TN / 64 * 4;                   // promoting warps of 32 rows x 64 columns: four lane quadrants for each 64 columns
    static constexpr int CW = 64;
    static constexpr bool FRAG = EPI == 16 && SC != ROW;      // values of TMEM spread over a warp as 4 rows x 16 columns of a lane
    static constexpr int THREADS = 32 * (EPI0 + EPI);
    static constexpr int ROWS = 128 * CG;                     // rows of X of a tile
    static constexpr int X_BYTES = 128 * BK, Y_BYTES = TN / CG * BK;
    static constexpr bool PART = CG == 1 && !SWAP;            // tiles with few rows of X: of 32 that have none, nothing is fetched or promoted
    static constexpr int X_BOX = PART ? 32 : 128;             // rows of X per TMA copy
    static constexpr int Y_BOX = SWAP ? 16 : TN / CG;         // rows of Y per TMA copy: with SWAP only boxes with rows are fetched
    static constexpr int STAGE = X_BYTES + Y_BYTES;
    static constexpr int STAGES = EPI == 16 ? (CG == 2 ? 6 : 4) : 3;
    static constexpr int TMEM_COLS = 2 * TN;
    static constexpr int D = 8;                               // blocks of scales in the ring
    static constexpr int XS = 128;                            // floats of a block: X's rows,
    static constexpr int SLOT = XS + (SC == ROW ? 4 : TN);    // then Y's columns (ROW: two numbers)
    static constexpr int TURN = EPI == 16 ? 1024 : 0;         // per promoting warp: where C is turned
    // where a split's shares of a tile arrive with SWAP: its columns, 128 rows each, from each of 2, 4 or 8 parts
    static constexpr int PARTS = SPLIT ? TN * 128 * 4 : 0;
    static constexpr int turn_off = STAGES * STAGE + PARTS;
    static constexpr int ring_off = turn_off + EPI * TURN;
    static constexpr int bar_off = ring_off + D * SLOT * 4;
    static constexpr int n_bars = 2 * STAGES + 5;             // full, empty; accumulator (and scales) full[2], accumulator free[2]; shares
    static constexpr int misc_off = bar_off + n_bars * 8;     // TMEM address, abort flag
    static constexpr int seg_off = misc_off + 16;             // groups: first row, first tile
    static constexpr int dynamic = seg_off + (2 * MAX_GROUPS + 2) * 4;
    static constexpr int PER_SM = EPI == 16 ? 1 : 2;
    static_assert(dynamic * PER_SM <= 232448 - 1024 * (PER_SM - 1), "shared memory budget exceeded");
    static_assert(!SPLIT || (SWAP && TN * 512 <= STAGES * STAGE), "a split sends its tile from the stage ring");
};

struct Params {
    int kblocks;                              // of K
    int tiles_x, tiles_y, group_x;            // tile grid (of one matrix), rasterisation
    int x_rows, y_rows;                       // rows of X and Y per matrix
    const float* xs;                          // scale of X's row r in block kb: xs[r + kb * xs_k], squares: xs[(r / 128) * kblocks + kb]
    long long xs_k;
    int xs_square;
    const float* ys;                          // the same for Y: squares with ROW, row blocks with BOTH
    long long ys_k;
    void* c;
    long long ldc;
    int c_f32;
    const int* group_rows;
    int groups;                               // 0: one matrix
    int wgrad;
    int rows_cap;                             // rows (wgrad: columns) of the operands that the groups divide
    int split;
    int* status;
};

struct Tile {
    int x0, x_end, x_tma;                     // first row of X of this CTA inside its matrix, one past the matrix's or group's last, first row in the tensor map
    int y0, y_end, y_tma;                     // the same for Y, y_end being the tile's
    int ncols;                                // columns of the MMA (both CTAs together)
    int k0, k1;                               // K blocks
    long long c_row;                          // first row of C of this tile's matrix
    int g;
};

// columns of an MMA: a multiple of 16 for one CTA, of 32 for a pair (16 rows of Y in each)
template <int CG>
__device__ __forceinline__ int round_cols(int n) { return (n + 16 * CG - 1) / (16 * CG) * (16 * CG); }

// seg[g] = first row of group g, seg[MAX_GROUPS + 1 + g] = first tile of group g
template <class C>
__device__ __forceinline__ Tile tile_at(int t, const Params& p, const int* seg, int pair_rank, int part) {
    Tile o;
    o.g = 0;
    o.c_row = 0;
    o.k0 = 0;
    o.k1 = p.kblocks;
    o.x0 = 0;
    o.x_end = p.x_rows;
    int first = 0, tiles_x = p.tiles_x, tiles_y = p.tiles_y, y_first = 0, y_last = p.y_rows;
    o.x_tma = o.y_tma = 0;
    if (p.groups > 0) {
        const int* firsts = seg + MAX_GROUPS + 1;
        int lo = 0, hi = p.groups - 1;                        // last group whose first tile is <= t: the one that has tile t
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (firsts[mid] <= t) lo = mid; else hi = mid - 1;
        }
        o.g = lo;
        first = firsts[lo];
        if (p.wgrad) {
            o.k0 = seg[lo] / BK;
            o.k1 = seg[lo + 1] / BK;
            o.c_row = static_cast<long long>(lo) * (C::SWAP ? p.y_rows : p.x_rows);
        } else if constexpr (C::SWAP) {
            y_first = seg[lo];
            y_last = seg[lo + 1];
            tiles_y = (y_last - y_first + C::TN - 1) / C::TN;
            o.x_tma = lo * p.x_rows;
        } else {
            o.x0 = seg[lo];
            o.x_end = seg[lo + 1];
            tiles_x = (o.x_end - o.x0 + C::ROWS - 1) / C::ROWS;
            o.y_tma = lo * p.y_rows;
        }
    }
    // groups of `group_x` tile rows, column-major inside, so that CTAs running together share panels in L2
    const int in_all = t - first, per = p.group_x * tiles_y;
    const int grp = in_all / per, in = in_all - grp * per, n = min(p.group_x, tiles_x - grp * p.group_x);
    const int ty = in / n, tx = grp * p.group_x + in - ty * n;
    o.x0 += tx * C::ROWS + pair_rank * 128;
    o.y0 = y_first + ty * C::TN;
    o.x_tma += o.x0;
    o.y_tma += o.y0;
    o.y_end = min(o.y0 + C::TN, y_last);
    o.ncols = round_cols<C::CG>(o.y_end - o.y0);
    if constexpr (C::SPLIT) {
        const int nk = o.k1 - o.k0, k0 = o.k0;
        o.k0 = k0 + nk * part / p.split;
        o.k1 = k0 + nk * (part + 1) / p.split;
    }
    return o;
}

// contiguous bytes of this CTA's shared memory to a CTA of the cluster, counted on its barrier; 16-byte aligned
__device__ __forceinline__ void bulk_send(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "r"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// 32 lanes x 16 columns
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_wait16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
// 32 lanes x 8 columns, lane l of the warp getting rows l / 4 + 8 i and columns 2 (l % 4) + {0, 1}: values 2 i and 2 i + 1
__device__ __forceinline__ void tc_ld8_frag(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(taddr) : "memory");
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr + (16u << 16)) : "memory");
}
__device__ __forceinline__ void tc_wait8(uint32_t (&r)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]) : : "memory");
}
// pairs of floats
__device__ __forceinline__ uint64_t pair(float a, float b) { return static_cast<uint64_t>(__float_as_uint(b)) << 32 | __float_as_uint(a); }
__device__ __forceinline__ float first_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float second_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
// four bytes, global -> shared, asynchronously; groups of copies complete in order
__device__ __forceinline__ void copy4(uint32_t dst, const float* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
template <int N>
__device__ __forceinline__ void set_regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void set_regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Arrive on a barrier of the pair's leading CTA.  What it orders are TMEM reads, which tcgen05.fence::before_thread_sync covers; the
// release.cluster form would also wait for the warp's outstanding global loads, once per K block (1.21 instead of 0.7 us a block).
template <int CG>
__device__ __forceinline__ void arrive_lane0(uint32_t addr, int lane) {      // predicated, so that the warp does not diverge
    if constexpr (CG == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cluster.b64 _, [%0];\n\t}" ::"r"(addr), "r"(lane) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(addr), "r"(lane) : "memory");
}

// A whole warp waits: one probe, and the bounded wait only when it fails.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const AbortCtl& ab, int code) {
    if (__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, ab, code));
}

// Arrive on `bar` of this CTA, or of both CTAs of the pair that starts at cluster rank `first`, once this thread's MMAs are complete.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar, int first) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"(static_cast<uint16_t>(3u << first)) : "memory");
    else
        tc_commit<1>(bar);
}

__device__ __forceinline__ void store_c(const Params& p, long long row, int col, float v) {
    const long long at = row * p.ldc + col;
    if (p.c_f32) static_cast<float*>(p.c)[at] = v;
    else static_cast<uint16_t*>(p.c)[at] = static_cast<uint16_t>(pack_bf16x2(v, 0.0f));
}

// C leaves through 1 KB of shared memory of a warp, 128 bytes of eight rows at a time, so that a store covers 128 consecutive bytes of a
// row (16 per lane).  (All 32 rows at once and 32 bytes of each took 3 us a tile: a store then touches 16 lines.)  The 16-byte piece k
// of row r lies in slot k ^ swizzle(r), which keeps the ways in, below, and out conflict-free: the permutation sets rows that differ by
// one apart by two slots, so that the 64-bit words of a fragment, two pieces to a row, miss each other too.
__device__ __forceinline__ int swizzle(int r) { return ((r << 1) | (r >> 2)) & 7; }
template <int ES>
__device__ __forceinline__ void emit_rows(uint32_t turn, uint8_t* c, long long pitch, bool wide, bool even, int r0, int rows, int j, int cols, int lane) {
    constexpr int PER = 128 / ES;
    if (wide && cols - j >= PER) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = i * 4 + lane / 8, piece = lane % 8;
            uint32_t w[4];
            ld_shared_v4(turn + r * 128 + ((piece ^ swizzle(r)) << 4), w[0], w[1], w[2], w[3]);
            if (r0 + r < rows) *reinterpret_cast<uint4*>(c + (r0 + r) * pitch + j * ES + piece * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
        // rows that do not start on 16-byte boundaries, or end inside: a word per lane, still consecutive
        const int left = cols - j - lane * (4 / ES);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            uint32_t w;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(turn + r * 128 + (((lane >> 2) ^ swizzle(r)) << 4) + (lane & 3) * 4));
            uint8_t* to = c + (r0 + r) * pitch + j * ES + lane * 4;
            if (r0 + r >= rows || left <= 0) continue;
            if (ES == 4 || (even && left >= 2)) {
                *reinterpret_cast<uint32_t*>(to) = w;
            } else {
                *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(w);
                if (left >= 2) *reinterpret_cast<uint16_t*>(to + 2) = static_cast<uint16_t>(w >> 16);
            }
        }
    }
}
__device__ __forceinline__ void st_shared_b32(uint32_t a, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }

// 32 rows (one a lane) x 64 columns of C
template <bool F32>
__device__ __forceinline__ void write_rows(const Params& p, const float (&acc)[64], uint32_t turn, long long row0, int rows, int col0, int cols, int lane) {
    constexpr int ES = F32 ? 4 : 2, PER = 128 / ES;
    uint8_t* c = static_cast<uint8_t*>(p.c) + (row0 * p.ldc + col0) * ES;
    const long long pitch = p.ldc * ES;
    const bool wide = ((reinterpret_cast<uintptr_t>(c) | static_cast<uintptr_t>(pitch)) & 15) == 0, even = ((reinterpret_cast<uintptr_t>(c) | static_cast<uintptr_t>(pitch)) & 3) == 0;
    const uint32_t put = turn + (lane & 7) * 128 + (swizzle(lane & 7) << 4);
    uint32_t w[F32 ? 64 : 32];                               // converted once, not by the eight lanes of every pass
#pragma unroll
    for (int i = 0; i < (F32 ? 64 : 32); ++i) w[i] = F32 ? __float_as_uint(acc[i]) : pack_bf16x2(acc[2 * i % 64], acc[(2 * i + 1) % 64]);
#pragma unroll
    for (int j = 0; j < 64; j += PER) {
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 8) {
            __syncwarp();
            if ((lane & ~7) == r0) {
#pragma unroll
                for (int k = 0; k < 8; ++k) st_shared_v4(put ^ (k << 4), w[j / (4 / ES) + 4 * k], w[j / (4 / ES) + 4 * k + 1], w[j / (4 / ES) + 4 * k + 2], w[j / (4 / ES) + 4 * k + 3]);
            }
            __syncwarp();
            emit_rows<ES>(turn, c, pitch, wide, even, r0, rows, j, cols, lane);
        }
    }
    __syncwarp();
}

__device__ __forceinline__ void put(float* to, float v) { *to = v; }
__device__ __forceinline__ void put(uint16_t* to, float v) { *to = static_cast<uint16_t>(pack_bf16x2(v, 0.0f)); }
// up to `left` of four values of a row, together where they can be
__device__ __forceinline__ void put4(float* to, const float4& v, int left) {
    if (left >= 4 && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
        *reinterpret_cast<float4*>(to) = v;
    } else {
        if (left > 0) to[0] = v.x;
        if (left > 1) to[1] = v.y;
        if (left > 2) to[2] = v.z;
        if (left > 3) to[3] = v.w;
    }
}
__device__ __forceinline__ void put4(uint16_t* to, const float4& v, int left) {
    const uint32_t a = pack_bf16x2(v.x, v.y), b = pack_bf16x2(v.z, v.w);
    if (left >= 4 && (reinterpret_cast<uintptr_t>(to) & 7) == 0) {
        *reinterpret_cast<uint2*>(to) = make_uint2(a, b);
    } else {
        if (left > 0) to[0] = static_cast<uint16_t>(a);
        if (left > 1) to[1] = static_cast<uint16_t>(a >> 16);
        if (left > 2) to[2] = static_cast<uint16_t>(b);
        if (left > 3) to[3] = static_cast<uint16_t>(b >> 16);
    }
}
// One column of C: a lane's values are its rows.  (A branch on the type and an address of its own for every value made the code so long
// that fetching it took 3 us of a single tile's 7.)
template <class T>
__device__ __forceinline__ void write_columns(T* to, long long pitch, const float (&acc)[64], int rows) {
#pragma unroll
    for (int i = 0; i < 64; ++i) {
        if (i >= rows) break;
        put(to, acc[i]);
        to += pitch;
    }
}

// 32 rows x 64 columns from a fragment: acc[8 columns of 64][row of a lane: l / 4 + 8 i]
template <bool F32>
__device__ __forceinline__ void write_rows_frag(const Params& p, const uint64_t (&acc)[8][4], uint32_t turn, long long row0, int rows, int col0, int cols, int lane) {
    constexpr int ES = F32 ? 4 : 2;
    uint8_t* c = static_cast<uint8_t*>(p.c) + (row0 * p.ldc + col0) * ES;
    const long long pitch = p.ldc * ES;
    const bool wide = ((reinterpret_cast<uintptr_t>(c) | static_cast<uintptr_t>(pitch)) & 15) == 0, even = ((reinterpret_cast<uintptr_t>(c) | static_cast<uintptr_t>(pitch)) & 3) == 0;
    const int sw = swizzle(lane >> 2) << 4;
    const uint32_t put = turn + (lane >> 2) * 128;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (8 * i >= rows) break;
#pragma unroll
        for (int half = 0; half < (F32 ? 2 : 1); ++half) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < (F32 ? 4 : 8); ++j) {
                const uint64_t v = acc[4 * half + j][i];
                if constexpr (F32) asm volatile("st.shared.b64 [%0], %1;" ::"r"(put + (((2 * j + ((lane >> 1) & 1)) << 4) ^ sw) + (lane & 1) * 8), "l"(v) : "memory");
                else st_shared_b32(put + ((j << 4) ^ sw) + (lane & 3) * 4, pack_bf16x2(first_of(v), second_of(v)));
            }
            __syncwarp();
            emit_rows<ES>(turn, c, pitch, wide, even, 8 * i, rows, half * 32, cols, lane);
        }
    }
    __syncwarp();
}

// Prefix sums of the group sizes by one warp; sizes that do not fit are cut to what the operands have, and reported.
template <class C>
__device__ __forceinline__ void group_prefix(const Params& p, int* seg, int lane) {
    int tile = 0;
    long long row = 0;
    bool bad = false;
    const int cap = p.wgrad ? p.rows_cap / BK * BK : p.rows_cap;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
        const int g = g0 + lane;
        int n = g < p.groups ? p.group_rows[g] : 0;
        if (n < 0 || (p.wgrad && n % BK) || n > cap) {
            bad = true;
            n = max(0, min(n, cap));
            if (p.wgrad) n -= n % BK;
        }
        long long end = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xFFFFFFFFu, end, o);
            if (lane >= o) end += u;
        }
        end += row;
        if (end > cap) bad = true;
        const int e = static_cast<int>(min(end, static_cast<long long>(cap))), b = static_cast<int>(min(end - n, static_cast<long long>(cap)));
        int nt = g >= p.groups ? 0 : p.wgrad ? p.tiles_x * p.tiles_y : C::SWAP ? (e - b + C::TN - 1) / C::TN * p.tiles_x : (e - b + C::ROWS - 1) / C::ROWS * p.tiles_y;
        int tt = nt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xFFFFFFFFu, tt, o);
            if (lane >= o) tt += u;
        }
        if (g < p.groups) {
            seg[g] = b;
            seg[MAX_GROUPS + 1 + g] = tile + tt - nt;
            if (g == p.groups - 1) {
                seg[p.groups] = e;
                seg[MAX_GROUPS + 1 + p.groups] = tile + tt;
            }
        }
        row = __shfl_sync(0xFFFFFFFFu, end, 31);
        tile += __shfl_sync(0xFFFFFFFFu, tt, 31);
    }
    if (__any_sync(0xFFFFFFFFu, bad) && lane == 0) atomicCAS(p.status, 0, DEV_BAD_GROUPS);
}

template <class C>
__global__ void __launch_bounds__(C::THREADS, C::PER_SM)
gemm_block128_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_y, const Params p) {
    constexpr int CG = C::CG, S = C::STAGES, D = C::D;
    // the swizzle counts from 1024-byte boundaries; with no static shared memory the dynamic part starts on one
    extern __shared__ __align__(1024) uint8_t base_ptr[];
    const uint32_t base = smem_u32(base_ptr);
    if (base & 1023u) {
        if (threadIdx.x == 0) atomicCAS(p.status, 0, DEV_SMEM_BASE);
        return;
    }
    const uint32_t full0 = base + C::bar_off, empty0 = full0 + S * 8, accfull0 = empty0 + S * 8, accfree0 = accfull0 + 16;
    const uint32_t shares = accfree0 + 16;                    // a split's shares have arrived (SWAP)
    volatile uint32_t* tmem_ptr = reinterpret_cast<volatile uint32_t*>(base_ptr + C::misc_off);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(base_ptr + C::misc_off + 8);
    float* ring = reinterpret_cast<float*>(base_ptr + C::ring_off);
    int* seg = reinterpret_cast<int*>(base_ptr + C::seg_off);
    const AbortCtl ab{abort_flag, p.status};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cluster = C::SPLIT ? CG * p.split : CG;         // CTAs that share a tile
    const int rank = cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int pair_rank = CG == 2 ? rank & 1 : 0, part = rank / CG, first_rank = rank - pair_rank;
    const int unit = blockIdx.x / cluster, units = gridDim.x / cluster;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < S; ++s) {
            mbar_init(full0 + s * 8, 1);                      // the leading CTA's arrive.expect_tx
            mbar_init(empty0 + s * 8, 1);                     // one tcgen05.commit
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(accfull0 + b * 8, 2);                   // the MMAs' commit and this CTA's scales
            mbar_init(accfree0 + b * 8, C::EPI * CG);         // promoting warps of the pair, on the leading CTA's barrier
        }
        mbar_init(shares, 1);
        fence_mbar_init();
        prefetch_tmap(&tm_x);
        prefetch_tmap(&tm_y);
    }
    if (warp == 1) {
        tmem_alloc<CG>(smem_u32(const_cast<uint32_t*>(tmem_ptr)), C::TMEM_COLS);
        tmem_relinquish<CG>();
    }
    if (warp == 2 && p.groups > 0) group_prefix<C>(p, seg, lane);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync_all();
    else if (C::SPLIT) cluster_arrive();                      // waited for before the first thing is sent
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_ptr, 0);
    const int num_tiles = p.groups > 0 ? __shfl_sync(0xFFFFFFFFu, seg[MAX_GROUPS + 1 + p.groups], 0) : p.tiles_x * p.tiles_y;

    if (warp < EPI0) {
        // with sixteen promoting warps five warpgroups run, launched with 96 registers a thread: 56 + 4 * 104 < 5 * 96
        if constexpr (C::EPI == 16) set_regs_less<56>();
        if (warp == 0) {
            // ------------------------------------------------------------ operands
            const bool leader = elect_one();
            uint32_t stage = 0, ph = 0;
            const uint32_t full_lead = CG == 2 ? map_to_cta(full0, first_rank) : full0;
            bool ok = true;
            for (int t = unit; t < num_tiles && ok; t += units) {
                const Tile ti = tile_at<C>(t, p, seg, pair_rank, part);
                const int ny = ti.ncols / CG;                 // rows of Y of this CTA
                const int x0 = __shfl_sync(0xFFFFFFFFu, ti.x_tma, 0), y0 = __shfl_sync(0xFFFFFFFFu, ti.y_tma + pair_rank * ny, 0);
                const int k0 = __shfl_sync(0xFFFFFFFFu, ti.k0, 0), k1 = __shfl_sync(0xFFFFFFFFu, ti.k1, 0);
                const int xboxes = C::PART ? __shfl_sync(0xFFFFFFFFu, min(4, (ti.x_end - ti.x0 + 31) / 32), 0) : 1;
                const int boxes = __shfl_sync(0xFFFFFFFFu, (ny + C::Y_BOX - 1) / C::Y_BOX, 0);
                for (int kb = k0; kb < k1; ++kb) {
                    if (!warp_wait(empty0 + stage * 8, ph ^ 1, ab, DEV_TIMEOUT_EMPTY)) { ok = false; break; }
                    if (leader) {
                        const uint32_t dst = base + stage * C::STAGE, bytes = xboxes * C::X_BOX * BK + boxes * C::Y_BOX * BK;
                        if (CG == 1 || pair_rank == 0) mbar_arrive_expect_tx(full0 + stage * 8, CG * bytes);
                        const uint32_t bar = full_lead + stage * 8;
                        auto load = [&](uint32_t to, const CUtensorMap* m, int y) {
                            if constexpr (CG == 2) tma_load_2d_pair(to, m, kb * BK, y, bar);
                            else tma_load_2d(to, m, kb * BK, y, bar);
                        };
#pragma unroll
                        for (int i = 0; i < 128 / C::X_BOX; ++i)
                            if (i < xboxes) load(dst + i * C::X_BOX * BK, &tm_x, x0 + i * C::X_BOX);
#pragma unroll
                        for (int i = 0; i < C::TN / CG / C::Y_BOX; ++i)
                            if (i < boxes) load(dst + C::X_BYTES + i * C::Y_BOX * BK, &tm_y, y0 + i * C::Y_BOX);
                    }
                    __syncwarp();
                    if (++stage == S) { stage = 0; ph ^= 1; }
                }
            }
        } else if (warp == 1 && pair_rank == 0) {
            // ------------------------------------------------------------ MMA
            const bool leader = elect_one();
            uint32_t stage = 0, ph = 0, it = 0;
            bool ok = true;
            for (int t = unit; t < num_tiles && ok; t += units) {
                const Tile ti = tile_at<C>(t, p, seg, pair_rank, part);
                const int n = __shfl_sync(0xFFFFFFFFu, ti.k1 - ti.k0, 0);
                const uint32_t idesc = idesc_e4m3(128 * CG, __shfl_sync(0xFFFFFFFFu, ti.ncols, 0));
                for (int i = 0; i < n; ++i, ++it) {
                    const uint32_t buf = it & 1;
                    if (!warp_wait(full0 + stage * 8, ph, ab, DEV_TIMEOUT_FULL)) { ok = false; break; }
                    if (!warp_wait(accfree0 + buf * 8, ((it >> 1) & 1) ^ 1, ab, DEV_TIMEOUT_TMEM_FREE)) { ok = false; break; }
                    tc_fence_after();
                    if (leader) {
                        const uint32_t x = desc_sw128_lo(base + stage * C::STAGE), y = desc_sw128_lo(base + stage * C::STAGE + C::X_BYTES);
                        const uint32_t d = tmem + buf * C::TN;
                        tc_mma_e4m3_lo<CG, 0>(d, x, y, idesc);
                        tc_mma_e4m3_lo<CG, 1>(d, x + 2, y + 2, idesc);
                        tc_mma_e4m3_lo<CG, 1>(d, x + 4, y + 4, idesc);
                        tc_mma_e4m3_lo<CG, 1>(d, x + 6, y + 6, idesc);
                        commit<CG>(accfull0 + buf * 8, first_rank);
                        commit<CG>(empty0 + stage * 8, first_rank);
                    }
                    __syncwarp();
                    if (++stage == S) { stage = 0; ph ^= 1; }
                }
            }
        } else if (warp == 2) {
            // ------------------------------------------------------------ scales; rows and columns beyond the tile take the last one's
            // Block m's copies go into slot m % D after block m - 5 is complete on its barrier: the promoting warps have then released
            // block m - 7 and finished block m - 8, the slot's last.  Block m - 3 is announced when its copies have landed; the wait
            // for block m - 5 has made sure that this arrival counts for the right phase of the barrier they share.
            static_assert(D == 8, "the distances above");
            constexpr int NY = C::TN / 32;
            uint32_t m = 0;
            bool ok = true;
            // block n's copies have landed
            auto announce = [&](uint32_t n) {
                __syncwarp();
                arrive_lane0<1>(accfull0 + (n & 1) * 8, lane);
            };
            auto complete = [&](uint32_t n) { return warp_wait(accfull0 + (n & 1) * 8, (n >> 1) & 1, ab, DEV_TIMEOUT_TMEM_FULL); };
            for (int t = unit; t < num_tiles && ok; t += units) {
                const Tile ti = tile_at<C>(t, p, seg, pair_rank, part);
                // offsets instead of pointers for every copy: this warp has few registers
                const int x_last = ti.x_end - 1 - lane, y_last = ti.y_end - 1 - lane;
                const float *xk = p.xs + lane, *yk = p.ys + lane;
                if (p.xs_square) xk += (static_cast<long long>(ti.g) * ((p.x_rows + 127) / 128) + min(ti.x0, p.x_rows - 1) / 128) * p.kblocks - lane;      // the tile's one number
                xk += ti.k0 * p.xs_k;
                if constexpr (C::SC == ROW) {
                    const int nb = (p.y_rows + 127) / 128;                // lane 0, 1: the number of the tile's 128 columns
                    yk += (static_cast<long long>(ti.g) * nb + min(ti.y0 / 128 + lane, nb - 1)) * p.kblocks + ti.k0 - lane;
                } else {
                    yk += ti.k0 * p.ys_k;
                }
                for (int kb = ti.k0; kb < ti.k1; ++kb, ++m) {
                    if (m >= 5 && !complete(m - 5)) { ok = false; break; }
                    const uint32_t to = smem_u32(ring + (m & (D - 1)) * C::SLOT + lane);
#pragma unroll
                    for (int i = 0; i < C::XS / 32; ++i) copy4(to + i * 128, xk + (p.xs_square ? 0 : min(ti.x0 + i * 32, x_last)));
                    if constexpr (C::SC == ROW) {
                        if (lane < 2) copy4(to + C::XS * 4, yk);
                    } else {
#pragma unroll
                        for (int i = 0; i < NY; ++i)
                            if (i * 32 < ti.ncols) copy4(to + C::XS * 4 + i * 128, yk + min(ti.y0 + i * 32, y_last));
                    }
                    copies_commit();
                    xk += p.xs_k;
                    yk += p.ys_k;
                    if (m >= 3) {
                        copies_wait<3>();
                        announce(m - 3);
                    }
                }
            }
            copies_wait<0>();
            for (uint32_t n = m < 3 ? 0 : m - 3; n < m && ok; ++n) {
                if (n >= 2 && !complete(n - 2)) break;
                announce(n);
            }
        }
    } else {
        // ------------------------------------------------------------ promotion and C
        if constexpr (C::EPI == 16) set_regs_more<104>();
        const int ew = warp - EPI0, q = warp & 3;                        // TMEM lane quadrant
        constexpr int CW = C::CW;
        const int col0 = (ew >> 2) * CW;
        const uint32_t turn = base + C::turn_off + ew * C::TURN;
        const uint32_t free_lead = CG == 2 ? map_to_cta(accfree0, first_rank) : accfree0;
        const uint32_t my_tmem = tmem + (static_cast<uint32_t>(q * 32) << 16) + col0;
        const int r = q * 32 + lane;                                     // row of this CTA's tile
        uint32_t it = 0;                                                 // blocks of this CTA so far: buffer and ring slot follow from it
        bool ok = true;
        for (int t = unit; t < num_tiles && ok; t += units) {
            int blocks, mine;                                            // columns from this warp's first on; <= 0: it only takes part in the barriers
            {
                const Tile ti = tile_at<C>(t, p, seg, pair_rank, part);
                blocks = ti.k1 - ti.k0;
                mine = !C::PART || ti.x0 + q * 32 < ti.x_end ? ti.ncols - col0 : 0;
            }
            float acc[C::FRAG ? 1 : CW];
            uint64_t frag[8][4];                                         // FRAG: pairs of columns
#pragma unroll
            for (int i = 0; i < CW; ++i) {
                if constexpr (!C::FRAG) acc[i] = 0.0f;
                else if (i < 32) frag[i / 4][i % 4] = 0;
            }
            for (; blocks > 0; --blocks, ++it) {
                const uint32_t buf = it & 1;
                if (!warp_wait(accfull0 + buf * 8, (it >> 1) & 1, ab, DEV_TIMEOUT_TMEM_FULL)) { ok = false; break; }
                tc_fence_after();
                const uint32_t src = my_tmem + buf * C::TN;
                const float* slot = ring + (it & (D - 1)) * C::SLOT;
                auto release = [&]() {                                   // the buffer's values are all in registers
                    tc_fence_before();
                    __syncwarp();
                    arrive_lane0<CG>(free_lead + buf * 8, lane);
                };
                [[maybe_unused]] uint32_t va[16], vb[16];
                if (C::PART && mine <= 0) {
                    release();
                } else if constexpr (C::SC == ROW) {
                    // 64 columns in four loads, two in flight
                    tc_ld16(src, va);
                    tc_ld16(src + 16, vb);
                    const float s = slot[r] * slot[128 + (col0 >> 7)];
                    auto add = [&](const uint32_t (&v)[16], int c) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[c + i] = fmaf(__uint_as_float(v[i]), s, acc[c + i]);
                    };
                    tc_wait16(va);
                    tc_wait16(vb);
                    add(va, 0);
                    tc_ld16(src + 32, va);
                    add(vb, 16);
                    tc_ld16(src + 48, vb);
                    tc_wait16(va);
                    tc_wait16(vb);
                    release();
                    add(va, 32);
                    add(vb, 48);
                } else if constexpr (C::FRAG) {
                    const float2* ys = reinterpret_cast<const float2*>(slot + C::XS + col0 + 2 * (lane & 3));
                    float xs[4];                                         // of this lane's four rows
#pragma unroll
                    for (int i = 0; i < 4; ++i) xs[i] = slot[q * 32 + 8 * i + (lane >> 2)];
                    // the scales' product first: it is in range, a sum times one of them may not be.  The columns' scales are read a step ahead (a
                    // step's own after its wait: weight gradients 364 -> 376 us)
                    auto add = [&](const uint32_t (&v)[8], int j, const float2& two) {
                        const uint64_t y = pair(two.x, two.y);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint64_t x = static_cast<uint64_t>(v[2 * i + 1]) << 32 | v[2 * i];
                            frag[j][i] = fma2(x, mul2(y, pair(xs[i], xs[i])), frag[j][i]);
                        }
                    };
                    uint32_t v[2][8];                                    // eight columns on their way while eight are added
                    tc_ld8_frag(src, v[0]);
                    float2 two = ys[0];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float2 now = two;
                        if (j < 7) two = ys[4 * (j + 1)];
                        tc_wait8(v[j & 1]);
                        if (j < 7) tc_ld8_frag(src + 8 * (j + 1), v[(j + 1) & 1]);
                        else release();
                        add(v[j & 1], j, now);
                    }
                } else {
                    if (mine <= 0) release();
                    const float s = slot[r];
#pragma unroll
                    for (int c = 0; c < CW; c += 16) {
                        if (c >= mine) break;
                        tc_ld16(src + c, va);
                        tc_wait16(va);
                        if (c + 16 == CW || c + 16 >= mine) release();
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const float4 y = *reinterpret_cast<const float4*>(slot + C::XS + col0 + c + i);
                            const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) acc[c + i + k] = fmaf(__uint_as_float(va[i + k]), ys[k] * s, acc[c + i + k]);
                        }
                    }
                }
            }
            if (!ok) break;
            int again = t;                                               // found anew: nothing of it has to stay in registers during the loop
            asm volatile("" : "+r"(again));
            const Tile ti = tile_at<C>(again, p, seg, pair_rank, part);
            [[maybe_unused]] const int cols = min(CW, ti.y_end - ti.y0 - col0);      // that exist
            if constexpr (C::SPLIT) {
                // this CTA's MMAs are complete (its last accumulator arrived): the stage ring is free
#pragma unroll
                for (int i = 0; i < CW; ++i)
                    if (i < cols) *reinterpret_cast<float*>(base_ptr + (i * 128 + r) * 4) = acc[i];
            } else if constexpr (C::SWAP) {
                // lanes are consecutive columns of C, registers its rows
                const long long first = (ti.c_row + ti.y0 + col0) * p.ldc + ti.x0 + r;
                if (ti.x0 + r < p.x_rows) {
                    if (p.c_f32) write_columns(static_cast<float*>(p.c) + first, p.ldc, acc, cols);
                    else write_columns(static_cast<uint16_t*>(p.c) + first, p.ldc, acc, cols);
                }
            } else {
                const int x0 = ti.x0 + q * 32, rows = min(32, ti.x_end - x0);
                if constexpr (!C::FRAG) {
                    if (p.c_f32) write_rows<true>(p, acc, turn, ti.c_row + x0, rows, ti.y0 + col0, cols, lane);
                    else write_rows<false>(p, acc, turn, ti.c_row + x0, rows, ti.y0 + col0, cols, lane);
                } else {
                    if (p.c_f32) write_rows_frag<true>(p, frag, turn, ti.c_row + x0, rows, ti.y0 + col0, cols, lane);
                    else write_rows_frag<false>(p, frag, turn, ti.c_row + x0, rows, ti.y0 + col0, cols, lane);
                }
            }
        }
    }

    if constexpr (C::SPLIT) {
        __syncwarp();
        cluster_wait();                                                  // every CTA's barriers are there
        if (unit < num_tiles) {                                          // the same in the whole cluster; with groups there may be fewer tiles
            // part j adds up columns yn j / split .. yn (j + 1) / split of the tile (rows of C): 512 bytes each, contiguous
            const Tile ti = tile_at<C>(unit, p, seg, pair_rank, part);
            const int yn = ti.y_end - ti.y0, most = (yn + p.split - 1) / p.split, first = yn * part / p.split, mine = yn * (part + 1) / p.split - first;
            fence_proxy_async_smem();                                        // the tile's words, for the copies below
            __syncthreads();
            if (threadIdx.x < p.split) {                                 // a lane for each CTA
                const int j = threadIdx.x, f = yn * j / p.split, n = yn * (j + 1) / p.split - f;
                if (j == part) mbar_arrive_expect_tx(shares, (p.split - 1) * mine * 512);
                else if (n > 0) bulk_send(map_to_cta(base + S * C::STAGE + part * most * 512, j), base + f * 512, n * 512, map_to_cta(shares, j));
            }
            __syncwarp();
            const bool got = warp_wait(shares, 0, ab, DEV_TIMEOUT_FULL);
            cluster_arrive();                                            // this CTA has its shares: what was sent to it has been read
            if (got) {
                // a warp sums a row of C, a lane four columns of it
                const float4* in = reinterpret_cast<const float4*>(base_ptr + S * C::STAGE) + lane;
                const float4* own = reinterpret_cast<const float4*>(base_ptr) + first * 32 + lane;
                const int col = ti.x0 + lane * 4, left = p.x_rows - col;
                for (int c = warp; c < mine; c += C::THREADS / 32) {
                    float4 v[8];                                         // all parts' values are on their way together
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (k < p.split) v[k] = k == part ? own[c * 32] : in[(k * most + c) * 32];
                    float4 s = v[0];
#pragma unroll
                    for (int k = 1; k < 8; ++k)
                        if (k < p.split) s = make_float4(s.x + v[k].x, s.y + v[k].y, s.z + v[k].z, s.w + v[k].w);
                    const long long to = (ti.c_row + ti.y0 + first + c) * p.ldc + col;
                    if (p.c_f32) put4(static_cast<float*>(p.c) + to, s, left);
                    else put4(static_cast<uint16_t*>(p.c) + to, s, left);
                }
            }
        } else {
            cluster_arrive();
        }
        __syncwarp();
        cluster_wait();
    }

    if (*abort_flag) {
        // a wait gave up: let copies that may still be in flight land before shared memory goes away
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
    }
    if (warp == 2) copies_wait<0>();
    __syncwarp();
    tc_fence_before();
    // nobody leaves a pair while its TMEM is written or its barriers are arrived on
    if constexpr (CG == 2) cluster_sync_all();
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<CG>(tmem, C::TMEM_COLS);
    }
}

// Single tokens: C[m][n] without tensor cores for a row or a few.  Bound by reading the weights and, for small ones, by the launch: no tensor
// map, barrier or cluster has to be set up, which costs the tiles 4 us.  A block of up to eight warps owns four rows of B, which use each
// value of A once it is decoded; a warp takes pieces of 512 k, 16 bytes a lane, which lie in one scale block; sums meet over the lanes
// and then the warps in a fixed order.  E4M3 values are exact in fp16 and fma.f32.f16 adds their exact product to a float: 1.6 instructions
// a weight for one row (decoding to floats: 2.4, 268 MB of weights in 53 instead of 44 us).  With groups a block works on one row of A
// and looks up the row's group.
constexpr int VEC_ROWS = 4;                   // rows of B of a block
constexpr int VEC_K = 512;                    // k of a warp's piece
struct VecParams {
    const uint8_t *a, *b;
    long long lda, ldb, ldsa, ldsb;
    const float *sa, *sb;
    int b_square, N, K;
    Params c;                                 // C, its pitch and type, the groups, the status word
};

// 16 bytes of a row from k on, zeros behind the row's end (whatever lies there)
__device__ __forceinline__ uint4 load16(const uint8_t* row, int k, int K) {
    if (k + 16 <= K) return __ldg(reinterpret_cast<const uint4*>(row + k));
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; i < K - k; ++i) w[i >> 2] |= static_cast<uint32_t>(row[k + i]) << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// four E4M3 bytes as halves (exact); two products of halves added to a float
__device__ __forceinline__ void e4m3x4_to_half(uint32_t v, uint32_t (&h)[2]) {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[0]) : "h"(static_cast<uint16_t>(v)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[1]) : "h"(static_cast<uint16_t>(v >> 16)));
}
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
    float d;
    asm("{\n\t.reg .f16 a0, a1, b0, b1;\n\t.reg .f32 t;\n\tmov.b32 {a0, a1}, %1;\n\tmov.b32 {b0, b1}, %2;\n\t"
        "fma.rn.f32.f16 t, a0, b0, %3;\n\tfma.rn.f32.f16 %0, a1, b1, t;\n\t}" : "=f"(d) : "r"(a), "r"(b), "f"(c));
    return d;
}

// the group that row m belongs to, -1 behind the last one; sizes that do not fit are cut as in group_prefix
__device__ __forceinline__ int group_of(const Params& p, int m, int lane, bool& bad) {
    long long row = 0;
    int mine = -1;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
        const int raw = g0 + lane < p.groups ? p.group_rows[g0 + lane] : 0, n = max(0, min(raw, p.rows_cap));
        bad |= raw != n;
        long long end = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xFFFFFFFFu, end, o);
            if (lane >= o) end += u;
        }
        end += row;
        bad |= end > p.rows_cap;
        const unsigned hit = __ballot_sync(0xFFFFFFFFu, m >= end - n && m < end);
        if (hit) mine = g0 + __ffs(hit) - 1;
        row = __shfl_sync(0xFFFFFFFFu, end, 31);
    }
    return mine;
}

template <int MT, bool GROUPED>
__global__ void __launch_bounds__(256) gemv_block128_kernel(const VecParams p) {
    __shared__ float part[8][VEC_ROWS * MT];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n0 = blockIdx.x * VEC_ROWS, m0 = blockIdx.y * MT;
    const int kblocks = (p.K + BK - 1) / BK;
    long long g = 0;
    if constexpr (GROUPED) {
        bool bad = false;
        g = group_of(p.c, m0, lane, bad);
        if (bad) atomicCAS(p.c.status, 0, DEV_BAD_GROUPS);
        if (g < 0) return;                                               // the same in the whole block
    }
    const int last = p.c.rows_cap - 1 - m0;                              // rows beyond it are it
    const uint8_t *a = p.a + m0 * p.lda, *b[VEC_ROWS];
#pragma unroll
    for (int r = 0; r < VEC_ROWS; ++r) b[r] = p.b + (g * p.N + min(n0 + r, p.N - 1)) * p.ldb;
    const float* sb = p.b_square ? p.sb + (g * ((p.N + BK - 1) / BK) + n0 / BK) * kblocks : p.sb + n0;
    float acc[VEC_ROWS][MT];
#pragma unroll
    for (int i = 0; i < VEC_ROWS * MT; ++i) acc[i / MT][i % MT] = 0.0f;
    for (int k = warp * VEC_K + lane * 16; k < p.K; k += static_cast<int>(blockDim.x) * 16) {
        uint4 w[VEC_ROWS], x[MT];
#pragma unroll
        for (int r = 0; r < VEC_ROWS; ++r) w[r] = load16(b[r], k, p.K);
#pragma unroll
        for (int m = 0; m < MT; ++m) x[m] = load16(a + min(m, last) * p.lda, k, p.K);
        const int kb = k / BK;
        float xs[MT], ws[VEC_ROWS];
#pragma unroll
        for (int m = 0; m < MT; ++m) xs[m] = p.sa[kb * p.ldsa + m0 + min(m, last)];
#pragma unroll
        for (int r = 0; r < VEC_ROWS; ++r) ws[r] = p.b_square ? (r ? ws[0] : sb[kb]) : sb[kb * p.ldsb + min(r, p.N - 1 - n0)];
        float s[VEC_ROWS][MT];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const auto word = [i](const uint4& v) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; };
            uint32_t xh[MT][2];
#pragma unroll
            for (int m = 0; m < MT; ++m) e4m3x4_to_half(word(x[m]), xh[m]);
#pragma unroll
            for (int r = 0; r < VEC_ROWS; ++r) {
                uint32_t wh[2];
                e4m3x4_to_half(word(w[r]), wh);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) s[r][m] = dot2(wh[h], xh[m][h], i || h ? s[r][m] : 0.0f);
            }
        }
#pragma unroll
        for (int r = 0; r < VEC_ROWS; ++r)
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[r][m] = fmaf(s[r][m], xs[m] * ws[r], acc[r][m]);
    }
#pragma unroll
    for (int i = 0; i < VEC_ROWS * MT; ++i) {
        float v = acc[i / MT][i % MT];
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
        if (lane == 0) part[warp][i] = v;
    }
    __syncthreads();
    const int i = threadIdx.x;
    if (i < VEC_ROWS * MT && n0 + i / MT < p.N && i % MT <= last) {
        float v = part[0][i];
        for (int w = 1; w < static_cast<int>(blockDim.x) / 32; ++w) v += part[w][i];
        store_c(p.c, m0 + i % MT, n0 + i / MT, v);
    }
}

struct Args {
    const void *A, *B;
    long long lda, ldb;
    const float *A_sc, *B_sc;
    long long ldsa, ldsb;                     // floats between K blocks of row-block scales
    int b_square;
    void* c;
    long long ldc;
    int c_f32;
    int M, N, K;
    const int* group_rows;
    int groups, wgrad;
};

static int operand_map(CUtensorMap* m, const void* base, long long rows, int K, long long ld, int box_rows) {
    const uint64_t dims[2] = {static_cast<uint64_t>(K), static_cast<uint64_t>(rows)};
    const uint64_t strides[1] = {static_cast<uint64_t>(ld)};
    const uint32_t box[2] = {BK, static_cast<uint32_t>(box_rows)};
    return make_tmap(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Tiles of grouped rows at the most: `across` for every `rows` of them, a partial one for every group, none without a row.
static long long most_tiles(long long across, int M, int rows, int groups) {
    return across * std::min<long long>(M, M / rows + groups);
}

// what the host keeps of a kernel for each device: the status word's address, once the shared memory limit is raised (two threads racing here
// find the same)
struct Vec {};                                // the kernel without tiles, among the Cfg
struct Known {
    std::atomic<int*> status;
};

template <class C>
static int known(Known*& k) {
    static Known all[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) {
        k = &all[dev & 63];
        if (k->status.load(std::memory_order_acquire)) return MX8_OK;
        int* status = device_status_ptr();
        if (!status) return MX8_ERR_CUDA;
        if constexpr (!std::is_same_v<C, Vec>) e = cudaFuncSetAttribute(gemm_block128_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::dynamic);
        if (e == cudaSuccess) {
            k->status.store(status, std::memory_order_release);
            return MX8_OK;
        }
    }
    note_cuda_error("gemm_block128 setup", cudaGetErrorString(e));
    return MX8_ERR_CUDA;
}

template <class C>
static int launch(const Args& a, int split, cudaStream_t stream) {
    CUtensorMap mx, my;
    const bool grouped = a.groups > 0 && !a.wgrad;
    int rc;
    if (C::SWAP) {
        if ((rc = operand_map(&mx, a.B, grouped ? static_cast<long long>(a.groups) * a.N : a.N, a.K, a.ldb, 128)) != MX8_OK) return rc;
        if ((rc = operand_map(&my, a.A, a.M, a.K, a.lda, C::Y_BOX)) != MX8_OK) return rc;
    } else {
        if ((rc = operand_map(&mx, a.A, a.M, a.K, a.lda, C::X_BOX)) != MX8_OK) return rc;
        if ((rc = operand_map(&my, a.B, grouped ? static_cast<long long>(a.groups) * a.N : a.N, a.K, a.ldb, C::Y_BOX)) != MX8_OK) return rc;
    }
    Known* k = nullptr;
    if ((rc = known<C>(k)) != MX8_OK) return rc;
    Params p{};
    p.kblocks = (a.K + BK - 1) / BK;
    p.x_rows = C::SWAP ? a.N : a.M;
    p.y_rows = C::SWAP ? a.M : a.N;
    p.tiles_x = (p.x_rows + C::ROWS - 1) / C::ROWS;
    p.tiles_y = (p.y_rows + C::TN - 1) / C::TN;
    p.group_x = 16;                           // 4096 rows of X walked together stay in L2 with the Y panel
    const float* bs = a.B_sc;
    p.xs = C::SWAP ? bs : a.A_sc;
    p.xs_square = C::SWAP && a.b_square;
    p.xs_k = C::SWAP ? (a.b_square ? 1 : a.ldsb) : a.ldsa;
    p.ys = C::SWAP ? a.A_sc : bs;
    p.ys_k = C::SWAP ? a.ldsa : (a.b_square ? 1 : a.ldsb);
    p.c = a.c;
    p.ldc = a.ldc;
    p.c_f32 = a.c_f32;
    p.group_rows = a.group_rows;
    p.groups = a.groups;
    p.wgrad = a.wgrad;
    p.rows_cap = a.wgrad ? a.K : a.M;
    p.split = split;
    p.status = k->status.load(std::memory_order_relaxed);
    // tiles that there can be
    long long tiles = static_cast<long long>(p.tiles_x) * p.tiles_y;
    if (a.wgrad) tiles *= a.groups;
    else if (grouped) tiles = most_tiles(C::SWAP ? p.tiles_x : p.tiles_y, a.M, C::SWAP ? C::TN : C::ROWS, a.groups);
    if (tiles > 0x7FFFFFFFll / 16) {
        note_cuda_error("gemm_block128", "more than 2^27 tiles");
        return MX8_ERR_LIMIT;
    }
    const int cluster = C::CG * split;
    long long clusters = tiles;
    const long long most = sm_count() / C::CG * C::PER_SM;
    if (!C::SPLIT && clusters > most) clusters = most;         // persistent; a split tile needs a cluster of its own
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(clusters * cluster));
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::dynamic;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm_block128_kernel<C>, mx, my, p);
    if (e != cudaSuccess) {
        note_cuda_error("gemm_block128 launch", cudaGetErrorString(e));
        return MX8_ERR_CUDA;
    }
    return MX8_OK;
}

static int launch_gemv(const Args& a, cudaStream_t st) {
    VecParams p{};
    p.a = static_cast<const uint8_t*>(a.A);
    p.b = static_cast<const uint8_t*>(a.B);
    p.lda = a.lda;
    p.ldb = a.ldb;
    p.ldsa = a.ldsa;
    p.ldsb = a.ldsb;
    p.sa = a.A_sc;
    p.sb = a.B_sc;
    p.b_square = a.b_square;
    p.N = a.N;
    p.K = a.K;
    p.c.c = a.c;
    p.c.ldc = a.ldc;
    p.c.c_f32 = a.c_f32;
    p.c.group_rows = a.group_rows;
    p.c.groups = a.groups;
    p.c.rows_cap = a.M;
    Known* k = nullptr;
    const int rc = known<Vec>(k);
    if (rc != MX8_OK) return rc;
    p.c.status = k->status.load(std::memory_order_relaxed);
    const int warps = std::min(8, (a.K + VEC_K - 1) / VEC_K);
    const int mt = a.groups > 0 || a.M == 1 ? 1 : a.M == 2 ? 2 : 4;
    const dim3 grid((a.N + VEC_ROWS - 1) / VEC_ROWS, (a.M + mt - 1) / mt);
    auto kern = a.groups > 0 ? gemv_block128_kernel<1, true>
                : mt == 1    ? gemv_block128_kernel<1, false>
                : mt == 2    ? gemv_block128_kernel<2, false>
                             : gemv_block128_kernel<4, false>;
    kern<<<grid, 32 * warps, 0, st>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        note_cuda_error("gemm_block128 launch", cudaGetErrorString(e));
        return MX8_ERR_CUDA;
    }
    return MX8_OK;
}

static int run(const Args& a, cudaStream_t st) {
    using Squares = Cfg<2, 256, false, ROW, false>;
    using Single = Cfg<1, 256, false, ROW, false>;
    using Rows = Cfg<2, 256, false, BOTH, false>;
    using Few = Cfg<1, 64, true, BOTH, false>;
    using FewSplit = Cfg<1, 64, true, BOTH, true>;
    // Tiles of 128 weights x 64 rows (`small` of them, two CTAs on a multiprocessor) for few rows, and where large tiles would leave much of
    // the device idle: they start up faster (5 against 7 us for one block of K) and more of them run at once.  Measured, us, small tiles
    // (in parts of K where they are taken) against large ones: squares 256 x 512 x 1024 (16 small tiles) 8.0 and 9.9, 512 x 1024 x 2048 (64)
    // 10.9 and 13.1, 512 x 2048 (128) by 512 7.0 and 8.4, by 4096 19.4 and 19.9, 1024 x 2048 (256) by 512 8.5 and 8.6, by 1024 11.6 and 10.3,
    // 1024 x 4096 (512) by 128 8.4 and 7.5; row blocks 1024 x 2048 x 4096 (256) 25 and 28, 1024 x 4096 x 1024 (512) 17.0 and 13.1.
    const bool grouped = a.groups > 0 && !a.wgrad;
    // Single tokens, vectors against tiles (cold caches, us): N x K = 7168 x 2048, 1 row 10.2 and 14.4, 2 rows 12.3 and 14.4, 4 rows 16.4 and 15.2;
    // 4096 x 2048, 4 rows 12.3 and 14.4, 8 rows 18.4 and 14.4; 1024 x 1024, 16 rows 8.2 and 12.3; 16384 x 16384, 1 row 61 and 68, 2 rows 68
    // and 68.  Rows of groups share no weights: 2048 x 7168, 8 rows 38.9 and 44, 16 rows 57 and 44; 1024 x 1024, 16 rows 12.3 and 15.4, 32
    // rows 16.4 and 14.4.
    const long long nk = static_cast<long long>(a.N) * a.K;
    if (!a.wgrad && (grouped ? a.M <= 8 || (a.M <= 32 && a.M * nk <= 25000000) : a.M <= 16 && (a.M - 1) * nk <= 30000000)) return launch_gemv(a, st);
    const int matrices = a.wgrad ? a.groups : 1, kb = (a.K + BK - 1) / BK / matrices;         // blocks of K, of a group on average
    const long long across = (a.N + 127ll) / 128, sms = sm_count();
    const long long small = grouped ? most_tiles(across, a.M, 64, a.groups) : across * ((a.M + 63ll) / 64) * matrices;
    if ((a.M <= 64 && a.groups == 0) || small <= sms || (small <= 2 * sms && (kb <= 4 || !a.b_square))) {
        // Parts of K, where they find multiprocessors of their own, and for a long K places beside others: 256 x 512 (16 small tiles), one part and
        // eight: 8.5 and 8.0 us by 1024, 28.9 and 12.4 by 7168; 512 x 1024 (64), one part, two and four: 8.8, 9.0, 10.1 by 1024, 19.1, 14.4, 14.3
        // by 4096, 29.6, 19.6, 18.3 by 7168.
        const long long room = kb >= 32 ? 2 * sms : sms + 16;
        const int split = kb < 8 ? 1 : small * 8 <= room ? 8 : kb < 10 ? 1 : small * 4 <= room ? 4 : small * 2 <= room ? 2 : 1;
        return split > 1 ? launch<FewSplit>(a, split, st) : launch<Few>(a, 1, st);
    }
    if (!a.b_square) return launch<Rows>(a, 1, st);
    // Groups of fewer than 1024 rows on average (of what A has room for, as the sizes are on the device): 128 rows a tile instead of the
    // 256 of a pair, as half of a pair's last tile is empty more often than not when the sizes are any; measured with such sizes alone, none
    // of them multiples of 256.  The pair reads a third less from L2.  N = 2048, K = 7168, one CTA and pairs, us: 512 rows in 32 groups 87 and
    // 132, 9001 rows 191 and 200, 16384 rows 325 and 346, 16384 rows in 8 groups 270 and 252.
    return grouped && a.M / a.groups < 1024 ? launch<Single>(a, 1, st) : launch<Squares>(a, 1, st);
}

static int check(const char* what, const Args& a, int c_dtype) {
    if (!a.A || !a.A_sc || !a.B || !a.B_sc || !a.c) return MX8_ERR_ARG;
    if (c_dtype != MX8_C_BF16 && c_dtype != MX8_C_F32) return MX8_ERR_ARG;
    if (a.groups < 0 || (a.groups > 0 && !a.group_rows)) return MX8_ERR_ARG;
    if (a.M <= 0 || a.N <= 0 || a.K <= 0 || a.lda < a.K || a.ldb < a.K || a.lda % 16 || a.ldb % 16 || a.ldsa < a.M ||
        (!a.b_square && a.ldsb < a.N) || a.ldc < a.N) {
        note_cuda_error(what, "M, N, K positive, operand pitches multiples of 16 bytes and at least a row long, scale and C pitches at least a row long");
        return MX8_ERR_SIZE;
    }
    // a tile's last coordinates lie beyond the operands' and have to fit an int too
    const int most = 0x7FFFF000;
    if (a.groups > MAX_GROUPS || a.M > most || a.K > most || std::max(a.groups, 1) * static_cast<long long>(a.N) > most) {
        note_cuda_error(what, "more than 256 groups, or more than 2^31 - 4096 rows of A, rows of B (of all groups) or columns of either");
        return MX8_ERR_LIMIT;
    }
    if (!aligned16(a.A) || !aligned16(a.B) || reinterpret_cast<uintptr_t>(a.A_sc) % 4 || reinterpret_cast<uintptr_t>(a.B_sc) % 4 ||
        reinterpret_cast<uintptr_t>(a.group_rows) % 4 || reinterpret_cast<uintptr_t>(a.c) % (c_dtype == MX8_C_F32 ? 4 : 2)) return MX8_ERR_ALIGN;
    return check_device_sm100();
}

}  // namespace g128
}  // namespace mx8

extern "C" int mx8_gemm_block128(const void* A, long long lda, const void* A_sc, long long ldsa, const void* B, long long ldb,
                                 const void* B_sc, long long ldsb, int b_square, void* C, long long ldc, int M, int N, int K,
                                 int c_dtype, const void* group_rows, int num_groups, void* stream) {
    using namespace mx8;
    const g128::Args a{A, B, lda, ldb, static_cast<const float*>(A_sc), static_cast<const float*>(B_sc), ldsa, ldsb, b_square != 0,
                       C, ldc, c_dtype == MX8_C_F32, M, N, K, static_cast<const int*>(group_rows), num_groups, 0};
    if (num_groups > 0 && !b_square) return MX8_ERR_ARG;        // experts' weights come in squares
    const int rc = g128::check("mx8_gemm_block128", a, c_dtype);
    return rc == MX8_OK ? g128::run(a, static_cast<cudaStream_t>(stream)) : rc;
}

extern "C" int mx8_gemm_block128_wgrad(const void* A_t, long long lda, const void* A_t_sc, long long ldsa, const void* B_t, long long ldb,
                                       const void* B_t_sc, long long ldsb, void* C, long long ldc, int M, int N, int rows, int c_dtype,
                                       const void* group_rows, int num_groups, void* stream) {
    using namespace mx8;
    if (num_groups <= 0) return MX8_ERR_ARG;
    const g128::Args a{A_t, B_t, lda, ldb, static_cast<const float*>(A_t_sc), static_cast<const float*>(B_t_sc), ldsa, ldsb, 0,
                       C, ldc, c_dtype == MX8_C_F32, M, N, rows, static_cast<const int*>(group_rows), num_groups, 1};
    const int rc = g128::check("mx8_gemm_block128_wgrad", a, c_dtype);
    return rc == MX8_OK ? g128::run(a, static_cast<cudaStream_t>(stream)) : rc;
}
