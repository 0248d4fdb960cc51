// Matrix product of the block-128 format for sm_100a:
//   C[i][j] = sum_kb sa[kb][i] * sb(kb, j) * sum_{k in block kb} A[i][k] * B[j][k],   A, B E4M3, scales fp32, C bf16 or fp32.
// The scales are no powers of two and belong to 128 values of k, so the tensor core sums one block at a time (four
// tcgen05.mma.kind::f8f6f4 of K = 32 into TMEM, fp32) and registers add the blocks up: acc += (sa sb) * partial, one rounding each.
//
// One CTA per tile, ten (or six) warps: warp 0 streams operand tiles with TMA (128-byte swizzle) into a ring of stages, warp 1 issues
// the MMAs of block kb into one of two TMEM buffers, the other warps read the buffer with tcgen05.ld, scale and add it into
// registers while the MMAs of block kb + 1 fill the other buffer, and at the end write C.  128 x 256 x 128 is 512 tensor cycles; the
// promotion of such a partial tile is 256 cycles of each fp32 pipe, so the two overlap when nothing stalls.
//
// X is the operand whose rows are the 128 lanes of TMEM, Y the one whose rows are its columns: X = A, Y = B for many rows of A;
// for few (SWAP) X = B, so that 128 rows of weights fill the lanes and the tokens, 16 to 64 of them, the columns.
// split > 1: a cluster of `split` CTAs shares a tile, each takes a part of the K blocks, and the partial tiles are added through
// distributed shared memory in rank order: no workspace, no atomics, the same result in every run.
// Shapes: dense; grouped (rows of A belong to groups with their own B, sizes on the device); weight gradient (K belongs to groups).
#include <atomic>

#include "mx8_host.cuh"
#include "mx8_ptx.cuh"

namespace mx8 {
namespace g128 {

constexpr int BK = 128;                       // bytes and elements of K per stage: one scale block
constexpr int MAX_GROUPS = 256;
constexpr int DEV_BAD_GROUPS = 17;            // device status: group sizes that do not fit the operands
constexpr int DEV_SMEM_BASE = 18;             // device status: dynamic shared memory does not start on a 1024-byte boundary
constexpr int RED_PITCH = 129;                // floats between columns of the tile that a split adds up

template <int TN_, bool SWAP_, bool COLVEC_>
struct Cfg {
    static constexpr int TN = TN_;
    static constexpr bool SWAP = SWAP_, COLVEC = COLVEC_;
    static constexpr int EPI = TN >= 128 ? 8 : 4;             // promoting warps
    static constexpr int CW = TN / (EPI / 4);                 // columns of a promoting warp
    static constexpr int LW = CW < 32 ? CW : 32;              // columns per tcgen05.ld
    static constexpr int X_BYTES = 128 * BK, Y_BYTES = TN * BK;
    static constexpr int STAGE = X_BYTES + Y_BYTES;
    static constexpr int STAGES = TN == 256 ? 4 : TN == 128 ? 6 : TN == 64 ? 4 : TN == 32 ? 5 : 6;
    static constexpr int THREADS = 32 * (2 + EPI);
    static constexpr int TMEM_COLS = 2 * TN < 32 ? 32 : 2 * TN;
    static constexpr int EPI_BYTES = 32 * 32 * 4;             // per warp: 32 x 32 floats of C, or its columns' scales (two buffers)
    static constexpr int epi_off = STAGES * STAGE;
    static constexpr int bar_off = epi_off + EPI * EPI_BYTES;
    static constexpr int n_bars = 2 * STAGES + 4;
    static constexpr int misc_off = bar_off + n_bars * 8;     // TMEM address, abort flag
    static constexpr int seg_off = misc_off + 16;             // groups: first row, first tile
    static constexpr int dynamic = seg_off + (2 * MAX_GROUPS + 2) * 4;
    static_assert(dynamic <= 232448, "shared memory budget exceeded");
    static_assert(TN * RED_PITCH * 4 <= STAGES * STAGE, "a split adds its tiles up in the stage ring");
    static_assert(2 * CW * 4 <= EPI_BYTES, "two buffers of column scales");
};

struct Params {
    int kblocks;                              // of K
    int tiles_x, tiles_y, group_x;            // tile grid (per group), rasterisation
    int x_rows, y_rows;                       // rows of X and Y per matrix (bounds of C)
    const float* xs;                          // scale of X's row r in block kb at xs[r_off + kb * xs_k]
    long long xs_k;
    int xs_square;                            // xs is [row blocks][kblocks]
    const float* ys;
    long long ys_k;
    int y_group;                              // rows of Y per group
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
    int x0, xn;                               // first row of X, rows that exist in this tile
    int y0, y_tma, yn;                        // first column inside C, first row of Y, columns that exist
    int k0, k1;                               // K blocks
    long long c_row;                          // first row of C of this tile's matrix
    int g;
};

__device__ __forceinline__ void tile_xy(int t, int group_x, int tiles_x, int tiles_y, int& tx, int& ty) {
    const int per = group_x * tiles_y;
    const int grp = t / per;
    const int in = t - grp * per;
    const int rows = min(group_x, tiles_x - grp * group_x);
    tx = grp * group_x + in % rows;
    ty = in / rows;
}

// seg[g] = first row of group g, seg[MAX_GROUPS + 1 + g] = first tile of group g
template <class C>
__device__ __forceinline__ Tile tile_at(int t, const Params& p, const int* seg, int rank) {
    Tile o;
    int tx, ty;
    o.g = 0;
    o.c_row = 0;
    o.k0 = 0;
    o.k1 = p.kblocks;
    int base = 0, tiles_x = p.tiles_x;
    if (p.groups > 0) {
        const int* first = seg + MAX_GROUPS + 1;
        int lo = 0, hi = p.groups - 1;                        // last group whose first tile is <= t and that has tiles
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid] <= t) lo = mid; else hi = mid - 1;
        }
        o.g = lo;
        base = first[lo];
        if (!p.wgrad) tiles_x = (first[lo + 1] - base) / p.tiles_y;
    }
    tile_xy(t - base, p.group_x, tiles_x, p.tiles_y, tx, ty);
    o.x0 = tx * 128;
    o.xn = min(128, p.x_rows - o.x0);
    o.y0 = ty * C::TN;
    o.y_tma = o.y0;
    o.yn = min(C::TN, p.y_rows - o.y0);
    if (p.groups > 0) {
        if (p.wgrad) {
            o.k0 = seg[o.g] / BK;
            o.k1 = seg[o.g + 1] / BK;
            o.c_row = static_cast<long long>(o.g) * p.x_rows;
        } else {
            o.x0 += seg[o.g];
            o.xn = min(128, seg[o.g + 1] - o.x0);
            o.y_tma += o.g * p.y_group;
        }
    }
    if (p.split > 1) {
        const int n = o.k1 - o.k0, k0 = o.k0;
        o.k0 = k0 + n * rank / p.split;
        o.k1 = k0 + n * (rank + 1) / p.split;
    }
    return o;
}

template <int N>
__device__ __forceinline__ void tc_ld(uint32_t taddr, uint32_t (&r)[N]) {
    if constexpr (N == 32) {
        tc_ld_32x32(taddr, r);
    } else {
        static_assert(N == 16, "");
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(taddr)
            : "memory");
    }
}
__device__ __forceinline__ void tc_wait(uint32_t (&r)[32]) { tc_wait_ld(r); }
__device__ __forceinline__ void tc_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// pairs of floats in 64-bit registers: one instruction for two columns
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float half_of(uint64_t v, int i) { return __uint_as_float(static_cast<uint32_t>(i ? v >> 32 : v)); }

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ void store_c(const Params& p, long long row, int col, float v) {
    const long long at = row * p.ldc + col;
    if (p.c_f32) static_cast<float*>(p.c)[at] = v;
    else static_cast<uint16_t*>(p.c)[at] = static_cast<uint16_t>(pack_bf16x2(v, 0.0f));
}

template <class C>
__global__ void __launch_bounds__(C::THREADS, C::SWAP ? 2 : 1)
gemm_block128_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_y, const Params p) {
    // the swizzle counts from 1024-byte boundaries; with no static shared memory the dynamic part starts on one
    extern __shared__ __align__(1024) uint8_t base_ptr[];
    const uint32_t base = smem_u32(base_ptr);
    if (base & 1023u) {
        if (threadIdx.x == 0) atomicCAS(p.status, 0, DEV_SMEM_BASE);
        return;
    }
    constexpr int S = C::STAGES;
    const uint32_t full0 = base + C::bar_off, empty0 = full0 + S * 8, accfull0 = empty0 + S * 8, accfree0 = accfull0 + 16;
    volatile uint32_t* tmem_ptr = reinterpret_cast<volatile uint32_t*>(base_ptr + C::misc_off);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(base_ptr + C::misc_off + 8);
    int* seg = reinterpret_cast<int*>(base_ptr + C::seg_off);
    const AbortCtl ab{abort_flag, p.status};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = p.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int unit = blockIdx.x / p.split, units = gridDim.x / p.split;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < S; ++s) {
            mbar_init(full0 + s * 8, 1);
            mbar_init(empty0 + s * 8, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(accfull0 + b * 8, 1);
            mbar_init(accfree0 + b * 8, C::EPI);
        }
        fence_mbar_init();
        prefetch_tmap(&tm_x);
        prefetch_tmap(&tm_y);
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(const_cast<uint32_t*>(tmem_ptr)), C::TMEM_COLS);
        tmem_relinquish<1>();
    }
    if (warp == 2 && p.groups > 0) {
        // prefix sums of the group sizes; sizes that do not fit are cut to what the operands have, and reported
        int row = 0, tile = 0;
        bool bad = false;
        for (int g0 = 0; g0 < p.groups; g0 += 32) {
            const int g = g0 + lane;
            int n = g < p.groups ? p.group_rows[g] : 0;
            if (n < 0 || (p.wgrad && n % BK) || n > p.rows_cap) {
                bad = true;
                n = max(0, min(n, p.rows_cap));
                if (p.wgrad) n -= n % BK;
            }
            long long r = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xFFFFFFFFu, r, o);
                if (lane >= o) r += u;
            }
            long long first = row + r - n, end = row + r;
            if (end > p.rows_cap) bad = true;
            const int cap = p.wgrad ? p.rows_cap / BK * BK : p.rows_cap;
            first = min(first, static_cast<long long>(cap));
            end = min(end, static_cast<long long>(cap));
            int nt = p.wgrad ? p.tiles_x * p.tiles_y : static_cast<int>((end - first + 127) / 128) * p.tiles_y;
            if (g >= p.groups) nt = 0;
            int tt = nt;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xFFFFFFFFu, tt, o);
                if (lane >= o) tt += u;
            }
            if (g < p.groups) {
                seg[g] = static_cast<int>(first);
                seg[MAX_GROUPS + 1 + g] = tile + tt - nt;
                if (g == p.groups - 1) {
                    seg[p.groups] = static_cast<int>(end);
                    seg[MAX_GROUPS + 1 + p.groups] = tile + tt;
                }
            }
            row = static_cast<int>(__shfl_sync(0xFFFFFFFFu, end, 31));
            tile += __shfl_sync(0xFFFFFFFFu, tt, 31);
        }
        if (__any_sync(0xFFFFFFFFu, bad) && lane == 0) atomicCAS(p.status, 0, DEV_BAD_GROUPS);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_ptr, 0);
    const int num_tiles = p.groups > 0 ? __shfl_sync(0xFFFFFFFFu, seg[MAX_GROUPS + 1 + p.groups], 0) : p.tiles_x * p.tiles_y;

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        const bool leader = elect_one();
        uint32_t stage = 0, ph = 0;
        bool ok = true;
        for (int t = unit; t < num_tiles && ok; t += units) {
            const Tile ti = tile_at<C>(t, p, seg, rank);
            const int x0 = __shfl_sync(0xFFFFFFFFu, ti.x0, 0), y0 = __shfl_sync(0xFFFFFFFFu, ti.y_tma, 0);
            const int k0 = __shfl_sync(0xFFFFFFFFu, ti.k0, 0), k1 = __shfl_sync(0xFFFFFFFFu, ti.k1, 0);
            for (int kb = k0; kb < k1; ++kb) {
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(empty0 + stage * 8, ph ^ 1, ab, DEV_TIMEOUT_EMPTY))) { ok = false; break; }
                if (leader) {
                    const uint32_t dst = base + stage * C::STAGE, bar = full0 + stage * 8;
                    mbar_arrive_expect_tx(bar, C::STAGE);
                    tma_load_2d(dst, &tm_x, kb * BK, x0, bar);
                    tma_load_2d(dst + C::X_BYTES, &tm_y, kb * BK, y0, bar);
                }
                __syncwarp();
                if (++stage == S) { stage = 0; ph ^= 1; }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA
        const bool leader = elect_one();
        constexpr uint32_t idesc = idesc_e4m3(128, C::TN);
        uint32_t stage = 0, ph = 0, it = 0;
        bool ok = true;
        for (int t = unit; t < num_tiles && ok; t += units) {
            const Tile ti = tile_at<C>(t, p, seg, rank);
            const int n = __shfl_sync(0xFFFFFFFFu, ti.k1 - ti.k0, 0);
            for (int i = 0; i < n; ++i, ++it) {
                const uint32_t buf = it & 1, use = it >> 1;
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(full0 + stage * 8, ph, ab, DEV_TIMEOUT_FULL))) { ok = false; break; }
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(accfree0 + buf * 8, (use & 1) ^ 1, ab, DEV_TIMEOUT_TMEM_FREE))) { ok = false; break; }
                tc_fence_after();
                if (leader) {
                    const uint32_t x = desc_sw128_lo(base + stage * C::STAGE), y = desc_sw128_lo(base + stage * C::STAGE + C::X_BYTES);
                    const uint32_t d = tmem + buf * C::TN;
                    tc_mma_e4m3_lo<1, 0>(d, x, y, idesc);
                    tc_mma_e4m3_lo<1, 1>(d, x + 2, y + 2, idesc);
                    tc_mma_e4m3_lo<1, 1>(d, x + 4, y + 4, idesc);
                    tc_mma_e4m3_lo<1, 1>(d, x + 6, y + 6, idesc);
                    tc_commit<1>(empty0 + stage * 8);
                    tc_commit<1>(accfull0 + buf * 8);
                }
                __syncwarp();
                if (++stage == S) { stage = 0; ph ^= 1; }
            }
        }
    } else {
        // ------------------------------------------------------------ promotion and C
        const int ew = warp - 2, q = warp & 3, half = ew >> 2;          // TMEM lane quadrant, column half
        uint8_t* stg = base_ptr + C::epi_off + ew * C::EPI_BYTES;
        float* stgf = reinterpret_cast<float*>(stg);
        const uint32_t my_tmem = tmem + (static_cast<uint32_t>(q * 32) << 16) + half * C::CW;
        const int col0 = half * C::CW;
        uint32_t it = 0;
        bool ok = true;
        for (int t = unit; t < num_tiles && ok; t += units) {
            const Tile ti = tile_at<C>(t, p, seg, rank);
            const int r = q * 32 + lane;                                 // row of the tile
            // scales of this lane's row; rows beyond the tile take the last one's
            const int xr = ti.x0 + min(r, ti.xn - 1);
            long long x_off = p.xs_square ? static_cast<long long>(xr / 128) * p.kblocks : xr;
            const float* xs = p.xs + x_off;
            const float* ys;
            int yc[C::CW / 32 > 0 ? C::CW / 32 : 1];
            if constexpr (C::COLVEC) {
                ys = p.ys;
#pragma unroll
                for (int i = 0; i < (C::CW + 31) / 32; ++i) yc[i] = ti.y0 + min(col0 + i * 32 + lane, ti.yn - 1);
            } else {
                const int nb = ti.g * ((p.y_rows + 127) / 128) + (ti.y0 + min(col0, ti.yn - 1)) / 128;
                ys = p.ys + static_cast<long long>(nb) * p.kblocks;
            }
            uint64_t acc[C::CW / 2];
#pragma unroll
            for (int i = 0; i < C::CW / 2; ++i) acc[i] = 0;
            float xn = 0.0f, yn = 0.0f, ycol[(C::CW + 31) / 32];
            auto fetch = [&](int kb) {
                xn = __ldg(xs + kb * p.xs_k);
                if constexpr (C::COLVEC) {
#pragma unroll
                    for (int i = 0; i < (C::CW + 31) / 32; ++i) ycol[i] = __ldg(ys + kb * p.ys_k + yc[i]);
                } else {
                    yn = __ldg(ys + kb);
                }
            };
            if (ti.k0 < ti.k1) fetch(ti.k0);
            for (int kb = ti.k0; kb < ti.k1; ++kb, ++it) {
                const uint32_t buf = it & 1;
                float s = xn;
                if constexpr (C::COLVEC) {
                    // two buffers: the other one may still be read by slower lanes of this warp
#pragma unroll
                    for (int i = 0; i < (C::CW + 31) / 32; ++i)
                        if (i * 32 + lane < C::CW) stgf[buf * C::CW + i * 32 + lane] = ycol[i];
                    __syncwarp();
                } else {
                    s *= yn;
                }
                if (kb + 1 < ti.k1) fetch(kb + 1);
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(accfull0 + buf * 8, (it >> 1) & 1, ab, DEV_TIMEOUT_TMEM_FULL))) { ok = false; break; }
                tc_fence_after();
                const uint64_t ss = pair(__float_as_uint(s), __float_as_uint(s));
#pragma unroll
                for (int c = 0; c < C::CW; c += C::LW) {
                    uint32_t v[C::LW];
                    tc_ld<C::LW>(my_tmem + buf * C::TN + c, v);
                    tc_wait(v);
                    if (c + C::LW == C::CW) {                            // the buffer's values are all in registers
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(accfree0 + buf * 8);
                    }
#pragma unroll
                    for (int i = 0; i < C::LW; i += 2) {
                        uint64_t part = pair(v[i], v[i + 1]);
                        if constexpr (C::COLVEC) {
                            const uint64_t cs = *reinterpret_cast<const uint64_t*>(&stgf[buf * C::CW + c + i]);
                            part = mul2(part, cs);
                        }
                        acc[(c + i) / 2] = fma2(part, ss, acc[(c + i) / 2]);
                    }
                }
            }
            if (!ok) break;
            if (p.split > 1) {
                // this CTA's MMAs are complete (its last accumulator arrived), so the stage ring is free
                float* red = reinterpret_cast<float*>(base_ptr);
#pragma unroll
                for (int i = 0; i < C::CW; ++i) red[(col0 + i) * RED_PITCH + r] = half_of(acc[i / 2], i & 1);
            } else if constexpr (C::SWAP) {
                // lanes are consecutive columns of C, registers its rows
#pragma unroll
                for (int i = 0; i < C::CW; ++i)
                    if (r < ti.xn && col0 + i < ti.yn) store_c(p, ti.y0 + col0 + i, ti.x0 + r, half_of(acc[i / 2], i & 1));
            } else {
                // 32 x 32 pieces turned through shared memory so that a store covers consecutive columns
#pragma unroll
                for (int c = 0; c < C::CW; c += 32) {
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 32; ++i) stgf[lane * 32 + (i ^ lane)] = half_of(acc[(c + i) / 2], i & 1);
                    __syncwarp();
                    const int rows = min(32, ti.xn - q * 32);
                    if (col0 + c + lane < ti.yn)
                        for (int i = 0; i < rows; ++i) store_c(p, ti.c_row + ti.x0 + q * 32 + i, ti.y0 + col0 + c + lane, stgf[i * 32 + (lane ^ i)]);
                }
                __syncwarp();
            }
        }
    }

    if (p.split > 1) {
        __syncwarp();
        cluster_sync_all();
        if (warp >= 2 && unit < num_tiles) {
            const Tile ti = tile_at<C>(unit, p, seg, rank);
            const int ew = warp - 2;
            if constexpr (C::SWAP) {
                // rank r writes its share of the tile's columns (rows of C); a lane is a row of the tile (column of C)
                const int c1 = C::TN * (rank + 1) / p.split;
                for (int c = C::TN * rank / p.split + (ew >> 2); c < min(c1, ti.yn); c += C::EPI / 4) {
                    const int r = (ew & 3) * 32 + lane;
                    const uint32_t at = base + (c * RED_PITCH + r) * 4;
                    float s = 0.0f;
                    for (int k = 0; k < p.split; ++k) s += ld_cluster(map_to_cta(at, k));
                    if (r < ti.xn) store_c(p, ti.y0 + c, ti.x0 + r, s);
                }
            } else {
                // rank r writes its share of the tile's rows; a lane is a column
                const int r1 = 128 * (rank + 1) / p.split;
                for (int r = 128 * rank / p.split + ew; r < min(r1, ti.xn); r += C::EPI) {
                    for (int c = lane; c < ti.yn; c += 32) {
                        const uint32_t at = base + (c * RED_PITCH + r) * 4;
                        float s = 0.0f;
                        for (int k = 0; k < p.split; ++k) s += ld_cluster(map_to_cta(at, k));
                        store_c(p, ti.c_row + ti.x0 + r, ti.y0 + c, s);
                    }
                }
            }
        }
        __syncwarp();
        cluster_sync_all();                                              // nobody leaves while its tile is read
    }

    if (*abort_flag) {
        // a wait gave up: let copies that may still be in flight land before shared memory goes away
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<1>(tmem, C::TMEM_COLS);
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

template <class C>
static int launch(const Args& a, int split, cudaStream_t stream) {
    CUtensorMap mx, my;
    const long long b_rows = a.groups > 0 && !a.wgrad ? static_cast<long long>(a.groups) * a.N : a.N;
    int rc;
    if (C::SWAP) {
        if ((rc = operand_map(&mx, a.B, b_rows, a.K, a.ldb, 128)) != MX8_OK) return rc;
        if ((rc = operand_map(&my, a.A, a.M, a.K, a.lda, C::TN)) != MX8_OK) return rc;
    } else {
        if ((rc = operand_map(&mx, a.A, a.M, a.K, a.lda, 128)) != MX8_OK) return rc;
        if ((rc = operand_map(&my, a.B, b_rows, a.K, a.ldb, C::TN)) != MX8_OK) return rc;
    }
    Params p{};
    p.kblocks = (a.K + BK - 1) / BK;
    p.x_rows = C::SWAP ? a.N : a.M;
    p.y_rows = C::SWAP ? a.M : a.N;
    p.tiles_x = (p.x_rows + 127) / 128;
    p.tiles_y = (p.y_rows + C::TN - 1) / C::TN;
    p.group_x = 16;                           // 16 tile rows walked together keep their X panels and the Y panel in L2
    if (C::SWAP) {
        p.xs = a.B_sc;
        p.xs_square = a.b_square;
        p.xs_k = a.b_square ? 1 : a.ldsb;
        p.ys = a.A_sc;
        p.ys_k = a.ldsa;
    } else {
        p.xs = a.A_sc;
        p.xs_k = a.ldsa;
        p.ys = a.B_sc;
        p.ys_k = a.b_square ? 1 : a.ldsb;
    }
    p.y_group = a.N;
    p.c = a.c;
    p.ldc = a.ldc;
    p.c_f32 = a.c_f32;
    p.group_rows = a.group_rows;
    p.groups = a.groups;
    p.wgrad = a.wgrad;
    p.rows_cap = a.wgrad ? a.K : a.M;
    p.split = split;
    p.status = device_status_ptr();
    if (!p.status) return MX8_ERR_CUDA;
    auto kern = gemm_block128_kernel<C>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::dynamic);
    if (e != cudaSuccess) {
        note_cuda_error("cudaFuncSetAttribute(gemm_block128)", cudaGetErrorString(e));
        return MX8_ERR_CUDA;
    }
    // tiles that there can be: with groups every one may add a partial tile row
    long long tiles = static_cast<long long>(p.tiles_x) * p.tiles_y;
    if (a.groups > 0) tiles = a.wgrad ? tiles * a.groups : static_cast<long long>(p.tiles_x + a.groups) * p.tiles_y;
    if (tiles > 0x7FFFFFFFll / 8) {
        note_cuda_error("gemm_block128", "more than 2^28 tiles");
        return MX8_ERR_LIMIT;
    }
    long long grid = tiles * split;
    const long long resident = static_cast<long long>(sm_count()) * (C::SWAP ? 2 : 1);
    if (split == 1 && grid > resident) grid = resident;        // persistent; a split tile needs a cluster of its own
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::dynamic;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = static_cast<unsigned>(split);
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kern, mx, my, p);
    if (e != cudaSuccess) {
        note_cuda_error("gemm_block128 launch", cudaGetErrorString(e));
        return MX8_ERR_CUDA;
    }
    return MX8_OK;
}

static int run(const Args& a, cudaStream_t st) {
    const int kb = (a.K + BK - 1) / BK;
    const int sms = sm_count();
    if (a.groups == 0 && a.M <= 64) {
        // few rows: weights on the TMEM lanes; the K blocks are split until two CTAs per multiprocessor are there
        const int tiles = (a.N + 127) / 128;
        int split = 2 * sms / tiles;
        split = split < 1 ? 1 : split > 8 ? 8 : split;
        if (split > kb) split = kb;
        if (a.M <= 16) return launch<Cfg<16, true, true>>(a, split, st);
        if (a.M <= 32) return launch<Cfg<32, true, true>>(a, split, st);
        return launch<Cfg<64, true, true>>(a, split, st);
    }
    const long long mt = (a.M + 127) / 128;
    const long long t256 = mt * ((a.N + 255) / 256), t128 = mt * ((a.N + 127) / 128);
    if (a.groups > 0 || t256 >= sms || a.N > 128) {
        int split = 1;
        if (a.groups == 0 && t256 * 2 <= sms) {
            split = static_cast<int>(sms / t256);
            if (split > 8) split = 8;
            if (split > kb) split = kb;
        }
        return a.b_square ? launch<Cfg<256, false, false>>(a, split, st) : launch<Cfg<256, false, true>>(a, split, st);
    }
    int split = 1;
    if (t128 * 2 <= sms) {
        split = static_cast<int>(sms / t128);
        if (split > 8) split = 8;
        if (split > kb) split = kb;
    }
    return a.b_square ? launch<Cfg<128, false, false>>(a, split, st) : launch<Cfg<128, false, true>>(a, split, st);
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
    if (a.groups > MAX_GROUPS || static_cast<long long>(a.groups) * a.N > 0x7FFFFFFFll) {
        note_cuda_error(what, "more than 256 groups, or more than 2^31 - 1 rows of B");
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
