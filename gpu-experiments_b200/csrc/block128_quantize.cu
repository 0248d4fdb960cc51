// Quantizer of the block-128 format: x [E][M][N] (bf16 or fp32) -> E4M3 bytes and one fp32 scale per block, blocks being
//   rows     1 x 128 along N (sc [E][ceil(N/128)][M], block-major so that 128 rows' scales are consecutive),
//   columns  128 x 1 along M, with the bytes transposed (fp8_t [E][N][M], sc_t [E][ceil(M/128)][N]),
//   squares  128 x 128 (sc [E][ceil(M/128)][ceil(N/128)]; the transposed form has the same scales, transposed).
// amax = largest |x| of the block, at least 2^-110; scale = amax / 448; byte = e4m3(x * 448 / amax).
// fp32 input keeps 448 / amax in two words, its rounding error in the second: the quotient is rounded once to fp32 before the rounding to
// 3 bits.  With one word a few bytes in a million land on the other side of a border.  bf16 input needs one word: against a border t
// (5 bits), 448 x and t amax are integers below 2^14 times a common power of two, so a quotient that is not on the border is at least
// 2^-14 of itself away, and the two roundings on the way are 2^-23; a quotient right on a border goes to either of its two equally near
// neighbours, as fl(x * fl(448 / amax)) falls.  (Two words there: 95 -> 104 us at 16391 x 7168 both ways.)
// A block that holds an infinity or NaN gets that as its scale and dequantizes to NaN.
//
// Bound by HBM once the instructions are few: x is read once for both orientations.  A block of 8 warps owns a 128 x 128 tile.  Half a
// warp spans a row (8 columns per lane, 16-byte loads), a lane holds 8 rows of its 8 columns, so that maxima are taken on packed
// pairs of bf16, products on pairs of fp32 (mul.f32x2), and a lane's rows are 8 consecutive bytes of the transpose.  Row maxima by four
// shuffles within the half warp, column maxima through 4 KB of shared memory; row bytes leave as 128 consecutive bytes per half warp, the
// transpose through a swizzled 16 KB tile as 16-byte pieces of 128-byte rows.  The first form (4 columns x 16 rows a lane, scalar maxima
// and products, 1700 instructions a warp) took 137 us for 16391 x 7168 gathered rows both ways, at 65 % of the issue slots;
// this one 83 us (dense rows 80 us = 5.95 TB/s, one orientation 6.2 to 6.4 TB/s, squares of fp32 6.25 TB/s).
#include "mx8_host.cuh"
#include "mx8_ptx.cuh"

namespace mx8 {
namespace q128 {

constexpr int B = 128;
constexpr int WARPS = 8;
constexpr int ROWS = B / WARPS;                    // rows per warp
constexpr uint32_t AMAX_FLOOR = (127u - 110u) << 23;   // 2^-110: 448 / amax stays finite and amax / 448 normal
constexpr int GROUP_M = 8;                         // tile rows walked together: 1 KB runs along M for the transposed bytes

struct Params {
    const void* x;
    long long ldx;
    const int* row_index;                          // source row of every output row (outside [0, src_rows): zeros), or nullptr
    int src_rows;
    int E, M, N;
    int tiles_m, tiles_n;
    uint8_t* q;
    long long ld;
    float* sc;
    uint8_t* qt;
    long long ld_t;
    float* sc_t;
    int vec_x, vec_q, vec_t;
};

__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}
// 448 / amax in two words: the rounded quotient and what is missing from it
struct Inverse {
    float hi, lo;
};
template <bool TWO>
__device__ __forceinline__ Inverse inverse_of(float amax) {
    const float hi = __fdiv_rn(448.0f, amax);
    return {hi, TWO ? fmaf(-amax, hi, 448.0f) * (hi * (1.0f / 448.0f)) : 0.0f};         // (448 - amax hi) / amax; the difference is exact
}
__device__ __forceinline__ uint64_t twice(float v) { return pair(__float_as_uint(v), __float_as_uint(v)); }
// a pair of floats times a pair of inverses (two words: rounded once but for 2^-48)
struct Inverse2 {
    uint64_t hi, lo;
};
__device__ __forceinline__ Inverse2 twice(Inverse v) { return {twice(v.hi), twice(v.lo)}; }
template <bool TWO>
__device__ __forceinline__ void mul2(uint64_t a, const Inverse2& b, float& lo, float& hi) {
    uint64_t d;
    if constexpr (!TWO) asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b.hi));
    else asm("{\n\t.reg .b64 t;\n\tmul.rn.f32x2 t, %1, %3;\n\tfma.rn.f32x2 %0, %1, %2, t;\n\t}" : "=l"(d) : "l"(a), "l"(b.hi), "l"(b.lo));
    lo = __uint_as_float(static_cast<uint32_t>(d));
    hi = __uint_as_float(static_cast<uint32_t>(d >> 32));
}
// the larger magnitude of two bf16 pairs, two floats; a NaN wins; the sign bits are arbitrary
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t max_f32(uint32_t a, uint32_t b) {
    float d;
    asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(d) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
    return __float_as_uint(d);
}

// eight consecutive elements of a row as loaded: WORDS words, and the magnitudes' maxima as MAXES words (bf16: a pair in each)
template <typename T> struct Eight;
template <> struct Eight<uint16_t> {
    static constexpr int WORDS = 4;
    uint32_t w[4];
    __device__ __forceinline__ uint64_t two(int j) const { return pair(w[j] << 16, w[j] & 0xFFFF0000u); }
    __device__ __forceinline__ void load(const uint16_t* p) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    }
    __device__ __forceinline__ void set(int i, uint16_t v) { w[i >> 1] |= static_cast<uint32_t>(v) << (16 * (i & 1)); }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max_bf16x2(a, b); }
};
template <> struct Eight<float> {
    static constexpr int WORDS = 8;
    uint32_t w[8];
    __device__ __forceinline__ uint64_t two(int j) const { return pair(w[2 * j], w[2 * j + 1]); }
    __device__ __forceinline__ void load(const float* p) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p)), u = __ldg(reinterpret_cast<const uint4*>(p) + 1);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        w[4] = u.x; w[5] = u.y; w[6] = u.z; w[7] = u.w;
    }
    __device__ __forceinline__ void set(int i, float v) { w[i] = __float_as_uint(v); }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max_f32(a, b); }
};

// magnitude of a block from its maximum's bits: sign off, the floor (an unsigned comparison keeps infinities and NaN on top)
__device__ __forceinline__ float amax_of(uint32_t bits) { return __uint_as_float(max(bits & 0x7FFFFFFFu, AMAX_FLOOR)); }
__device__ __forceinline__ uint32_t four_bytes(float a, float b, float c, float d) { return cvt_e4m3x2(a, b) | (cvt_e4m3x2(c, d) << 16); }

// SQUARE: one scale for the tile; otherwise ROW / COL say which orientations have scales of their own
template <typename T, bool ROW, bool COL, bool SQUARE>
__global__ void __launch_bounds__(32 * WARPS, sizeof(T) == 2 ? 4 : 2) quantize_block128_kernel(const Params p) {
    using E8 = Eight<T>;
    constexpr bool BF = sizeof(T) == 2;
    constexpr int W = E8::WORDS, IW = BF ? 2 : 4;
    __shared__ alignas(16) uint8_t stage[COL ? B * B : 16];
    __shared__ alignas(16) uint32_t cmax[COL && !SQUARE ? WARPS * 16 * W : WARPS];
    // inverses of the columns: those of pair j of lane l's eight at IW (16 j + l), first words, then second ones
    __shared__ alignas(16) float cinv[COL && !SQUARE ? B * IW / 2 : 4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = lane >> 4, l16 = lane & 15;
    // grid (GROUP_M * tiles_n, groups of tile rows, E): consecutive blocks walk down GROUP_M tile rows, then along N
    const int e = blockIdx.z, tn = blockIdx.x / GROUP_M, tm = blockIdx.y * GROUP_M + blockIdx.x % GROUP_M;
    if (tm >= p.tiles_m) return;
    const int m0 = tm * B + warp * ROWS + half * 8, n0 = tn * B + l16 * 8;      // this lane's first row and column

    E8 v[8];
    {
        const T* x = static_cast<const T*>(p.x) + static_cast<long long>(e) * p.M * p.ldx + n0;
        const bool whole = p.vec_x && n0 + 8 <= p.N;
        if (!p.row_index && p.vec_x && tm * B + B <= p.M && tn * B + B <= p.N) {
            x += static_cast<long long>(m0) * p.ldx;
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r].load(x + r * p.ldx);
        } else if (!p.row_index && tm * B + B <= p.M && tn * B + B <= p.N) {
            // rows off the 16-byte boundaries: element by element, all of them on their way together (4097 x 7001 bf16 both ways 37 -> 33 us;
            // aligned 16-byte windows shifted into place took 48 us where this takes 33, 3 x 1303 x 6401 fp32)
            x += static_cast<long long>(m0) * p.ldx;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
#pragma unroll
                for (int i = 0; i < W; ++i) v[r].w[i] = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[r].set(i, x[r * p.ldx + i]);
            }
        } else {
            int src = m0 + (lane & 7) < p.M ? m0 + (lane & 7) : -1;
            if (p.row_index && src >= 0) {
                src = p.row_index[src];
                if (src >= p.src_rows) src = -1;
            }
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const int s = __shfl_sync(0xFFFFFFFFu, src, r, 16);
#pragma unroll
                for (int i = 0; i < W; ++i) v[r].w[i] = 0;
                const T* row = x + s * p.ldx;
                if (s >= 0) {
                    if (whole) {
                        v[r].load(row);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (n0 + i < p.N) v[r].set(i, row[i]);
                    }
                }
            }
        }
    }

    Inverse row_inv = {0.0f, 0.0f};                // lanes r and r + 8 of a half: reciprocal scale of its row r
    Inverse tile_inv = {0.0f, 0.0f};
    if constexpr (SQUARE) {
        uint32_t a = v[0].w[0];
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (r || i) a = E8::larger(a, v[r].w[i]);
        a &= BF ? 0x7FFF7FFFu : 0x7FFFFFFFu;
        if constexpr (BF) a = max(a & 0xFFFF0000u, a << 16);
        a = __reduce_max_sync(0xFFFFFFFFu, a);
        if (lane == 0) cmax[warp] = a;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; ++w) a = max(a, cmax[w]);
        const float amax = amax_of(a);
        tile_inv = inverse_of<!BF>(amax);
        if (threadIdx.x == 0) {
            const float s = __fdiv_rn(amax, 448.0f);
            if (ROW) p.sc[(static_cast<size_t>(e) * p.tiles_m + tm) * p.tiles_n + tn] = s;
            if (COL) p.sc_t[(static_cast<size_t>(e) * p.tiles_n + tn) * p.tiles_m + tm] = s;
        }
    } else if constexpr (ROW) {
        // bf16: rows 2i and 2i + 1 share a word; then four exchanges within the half warp
        constexpr int K = BF ? 4 : 8;
        uint32_t m[K];
        if constexpr (BF) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t a = max_bf16x2(max_bf16x2(v[2 * i].w[0], v[2 * i].w[1]), max_bf16x2(v[2 * i].w[2], v[2 * i].w[3]));
                uint32_t b = max_bf16x2(max_bf16x2(v[2 * i + 1].w[0], v[2 * i + 1].w[1]), max_bf16x2(v[2 * i + 1].w[2], v[2 * i + 1].w[3]));
                m[i] = max_bf16x2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
            }
        } else {
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                m[r] = v[r].w[0];
#pragma unroll
                for (int i = 1; i < W; ++i) m[r] = max_f32(m[r], v[r].w[i]);
            }
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1)
#pragma unroll
            for (int i = 0; i < K; ++i) m[i] = E8::larger(m[i], __shfl_xor_sync(0xFFFFFFFFu, m[i], o));
        uint32_t mine = m[0];
#pragma unroll
        for (int i = 1; i < K; ++i)
            if (((lane & 7) >> (BF ? 1 : 0)) == i) mine = m[i];
        if constexpr (BF) mine = (lane & 1) ? mine & 0xFFFF0000u : mine << 16;
        const float amax = amax_of(mine);
        row_inv = inverse_of<!BF>(amax);
        if (l16 < 8 && m0 + l16 < p.M) p.sc[(static_cast<size_t>(e) * p.tiles_n + tn) * p.M + m0 + l16] = __fdiv_rn(amax, 448.0f);
    }
    if constexpr (ROW) {
        uint8_t* q = p.q + (static_cast<long long>(e) * p.M + m0) * p.ld + n0;
        const bool whole = p.vec_q && n0 + 8 <= p.N, inside = m0 + 8 <= p.M;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const Inverse2 inv = twice(SQUARE ? tile_inv : Inverse{__shfl_sync(0xFFFFFFFFu, row_inv.hi, r, 16), BF ? 0.0f : __shfl_sync(0xFFFFFFFFu, row_inv.lo, r, 16)});
            float f[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) mul2<!BF>(v[r].two(j), inv, f[2 * j], f[2 * j + 1]);
            const uint32_t lo = four_bytes(f[0], f[1], f[2], f[3]), hi = four_bytes(f[4], f[5], f[6], f[7]);
            if (inside || m0 + r < p.M) {
                if (whole) {
                    *reinterpret_cast<uint2*>(q) = make_uint2(lo, hi);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (n0 + i < p.N) q[i] = static_cast<uint8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
                }
            }
            q += p.ld;
        }
    }
    if constexpr (COL) {
        // the words are the same as before, but must not be kept in their unpacked form from the rows' products on: twice the registers
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int i = 0; i < W; ++i) asm volatile("" : "+r"(v[r].w[i]));
        if constexpr (!SQUARE) {
            uint32_t a[W];
#pragma unroll
            for (int i = 0; i < W; ++i) {
                a[i] = v[0].w[i];
#pragma unroll
                for (int r = 1; r < 8; ++r) a[i] = E8::larger(a[i], v[r].w[i]);
                a[i] = E8::larger(a[i], __shfl_xor_sync(0xFFFFFFFFu, a[i], 16));
            }
            if (half == 0) {
#pragma unroll
                for (int i = 0; i < W; i += 4) *reinterpret_cast<uint4*>(&cmax[(warp * 16 + l16) * W + i]) = make_uint4(a[i], a[i + 1], a[i + 2], a[i + 3]);
            }
            __syncthreads();
            if (threadIdx.x < B) {
                const int c = threadIdx.x;
                uint32_t m = cmax[BF ? c >> 1 : c];
#pragma unroll
                for (int w = 1; w < WARPS; ++w) m = E8::larger(m, cmax[w * 16 * W + (BF ? c >> 1 : c)]);
                if constexpr (BF) m = (c & 1) ? m & 0xFFFF0000u : m << 16;
                const float amax = amax_of(m);
                const Inverse v = inverse_of<!BF>(amax);
                float* to = &cinv[((c >> 1 & 3) * 16 + (c >> 3)) * IW + (c & 1)];
                to[0] = v.hi;
                if constexpr (!BF) to[2] = v.lo;
                if (tn * B + c < p.N) p.sc_t[(static_cast<size_t>(e) * p.tiles_m + tm) * p.N + tn * B + c] = __fdiv_rn(amax, 448.0f);
            }
            __syncthreads();
        }
        // the 8-byte piece k = 2 warp + half of column c's 128 bytes lies in slot k ^ (c / 8): sixteen lanes write sixteen different slots
        const int slot = (2 * warp + half) ^ l16;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            Inverse2 inv;
            if constexpr (SQUARE) {
                inv = twice(tile_inv);
            } else if constexpr (BF) {
                inv = {*reinterpret_cast<const uint64_t*>(&cinv[(j * 16 + l16) * IW]), 0};
            } else {
                const ulonglong2 both = *reinterpret_cast<const ulonglong2*>(&cinv[(j * 16 + l16) * IW]);
                inv = {both.x, both.y};
            }
            float f[8], g[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) mul2<!BF>(v[r].two(j), inv, f[r], g[r]);
            st_shared_v2(smem_u32(stage) + (l16 * 8 + 2 * j) * B + slot * 8, four_bytes(f[0], f[1], f[2], f[3]), four_bytes(f[4], f[5], f[6], f[7]));
            st_shared_v2(smem_u32(stage) + (l16 * 8 + 2 * j + 1) * B + slot * 8, four_bytes(g[0], g[1], g[2], g[3]), four_bytes(g[4], g[5], g[6], g[7]));
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ROWS / 4; ++k) {
            const int c = warp * ROWS + k * 4 + (lane >> 3), piece = lane & 7, g = c >> 3;
            const int n = tn * B + c, m = tm * B + piece * 16;
            if (n >= p.N || m >= p.M) continue;
            uint32_t w[4];
            ld_shared_v4(smem_u32(stage) + c * B + ((piece ^ (g >> 1)) << 4), w[0], w[1], w[2], w[3]);
            if (g & 1) {                               // the two 8-byte pieces of the 16 lie the other way round
                const uint32_t a = w[0], b = w[1];
                w[0] = w[2]; w[1] = w[3]; w[2] = a; w[3] = b;
            }
            uint8_t* dst = p.qt + (static_cast<long long>(e) * p.N + n) * p.ld_t + m;
            if (p.vec_t && m + 16 <= p.M) {
                *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (m + i < p.M) dst[i] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
            }
        }
    }
}

template <typename T, bool ROW, bool COL, bool SQUARE>
static cudaError_t launch_one(const Params& p, cudaStream_t st) {
    const dim3 grid(static_cast<unsigned>(GROUP_M * p.tiles_n), static_cast<unsigned>((p.tiles_m + GROUP_M - 1) / GROUP_M), static_cast<unsigned>(p.E));
    quantize_block128_kernel<T, ROW, COL, SQUARE><<<grid, 32 * WARPS, 0, st>>>(p);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t launch(const Params& p, bool row, bool col, bool square, cudaStream_t st) {
    if (square) return row && col ? launch_one<T, true, true, true>(p, st) : row ? launch_one<T, true, false, true>(p, st) : launch_one<T, false, true, true>(p, st);
    return row && col ? launch_one<T, true, true, false>(p, st) : row ? launch_one<T, true, false, false>(p, st) : launch_one<T, false, true, false>(p, st);
}

}  // namespace q128
}  // namespace mx8

extern "C" int mx8_quantize_block128(const void* x, int dtype, int E, int M, int N, long long ldx, const void* row_index, int src_rows,
                                     void* fp8, long long ld, void* sc, void* fp8_t, long long ld_t, void* sc_t, int square,
                                     void* stream) {
    using namespace mx8;
    const bool row = fp8 != nullptr, col = fp8_t != nullptr;
    if (!x || (!row && !col) || row != (sc != nullptr) || col != (sc_t != nullptr)) return MX8_ERR_ARG;
    if (dtype != MX8_T_BF16 && dtype != MX8_T_F32) return MX8_ERR_ARG;
    if (E <= 0 || M <= 0 || N <= 0 || ldx < N || (row && ld < N) || (col && ld_t < M) || (row_index && (E != 1 || src_rows <= 0))) {
        note_cuda_error("mx8_quantize_block128", "E, M, N positive, pitches at least a row long, row_index for one matrix with src_rows > 0");
        return MX8_ERR_SIZE;
    }
    const uintptr_t esize = dtype == MX8_T_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % esize || reinterpret_cast<uintptr_t>(sc) % 4 || reinterpret_cast<uintptr_t>(sc_t) % 4 ||
        reinterpret_cast<uintptr_t>(row_index) % 4) return MX8_ERR_ALIGN;
    const long long tiles_m = (M + 127ll) / 128, tiles_n = (N + 127ll) / 128;
    if (tiles_m > 65535ll * q128::GROUP_M || E > 65535 || N > 0x7FFFF000) {       // a tile's last column has to fit an int
        note_cuda_error("mx8_quantize_block128", "more than 65535 matrices, 67107840 rows or 2^31 - 4096 columns");
        return MX8_ERR_LIMIT;
    }
    int rc = check_device_sm100();
    if (rc != MX8_OK) return rc;
    q128::Params p{};
    p.x = x;
    p.ldx = ldx;
    p.row_index = static_cast<const int*>(row_index);
    p.src_rows = src_rows;
    p.E = E; p.M = M; p.N = N;
    p.tiles_m = static_cast<int>(tiles_m);
    p.tiles_n = static_cast<int>(tiles_n);
    p.q = static_cast<uint8_t*>(fp8);
    p.ld = ld;
    p.sc = static_cast<float*>(sc);
    p.qt = static_cast<uint8_t*>(fp8_t);
    p.ld_t = ld_t;
    p.sc_t = static_cast<float*>(sc_t);
    p.vec_x = (ldx * esize) % 16 == 0 && aligned16(x);
    p.vec_q = ld % 8 == 0 && reinterpret_cast<uintptr_t>(fp8) % 8 == 0;
    p.vec_t = ld_t % 16 == 0 && aligned16(fp8_t);
    const cudaError_t e = dtype == MX8_T_F32 ? q128::launch<float>(p, row, col, square != 0, static_cast<cudaStream_t>(stream))
                                             : q128::launch<uint16_t>(p, row, col, square != 0, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) {
        note_cuda_error("block-128 quantizer launch", cudaGetErrorString(e));
        return MX8_ERR_CUDA;
    }
    return MX8_OK;
}
