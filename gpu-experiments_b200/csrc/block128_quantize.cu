// Quantizer of the block-128 format: x [E][M][N] (bf16 or fp32) -> E4M3 bytes and one fp32 scale per block, blocks being
//   rows     1 x 128 along N (sc [E][ceil(N/128)][M], block-major so that 128 rows' scales are consecutive),
//   columns  128 x 1 along M, with the bytes transposed (fp8_t [E][N][M], sc_t [E][ceil(M/128)][N]),
//   squares  128 x 128 (sc [E][ceil(M/128)][ceil(N/128)]; the transposed form has the same scales, transposed).
// amax = largest |x| of the block, at least 2^-110; scale = amax / 448; byte = e4m3(x * (448 / amax)): one rounding of the
// reciprocal, one of the product (fp32, half a step of 2^-23 each), then the rounding to 3 bits that the format asks for.
// A block that holds an infinity or NaN gets that as its scale and dequantizes to NaN.
//
// Bound by HBM: x is read once for both orientations.  A block of 8 warps owns a 128 x 128 tile; a warp loads 16 rows into
// registers (lane = 4 columns, 16 loads in flight per lane), takes row maxima with redux.sync and column maxima through 4 KB of
// shared memory; row bytes leave as 128 consecutive bytes per warp store, transposed bytes through a swizzled 16 KB tile as 16-byte
// pieces of 128-byte rows.
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

template <typename T> struct Four;                 // four consecutive elements of a row as loaded
template <> struct Four<uint16_t> {
    uint32_t w[2];
    __device__ float get(int i) const { return __uint_as_float((i & 1) ? (w[i >> 1] & 0xFFFF0000u) : (w[i >> 1] << 16)); }
    __device__ void zero() { w[0] = w[1] = 0; }
    __device__ void load(const uint16_t* p) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
        w[0] = v.x; w[1] = v.y;
    }
    __device__ void set(int i, uint16_t v) { w[i >> 1] |= static_cast<uint32_t>(v) << (16 * (i & 1)); }
};
template <> struct Four<float> {
    uint32_t w[4];
    __device__ float get(int i) const { return __uint_as_float(w[i]); }
    __device__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }
    __device__ void load(const float* p) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    }
    __device__ void set(int i, float v) { w[i] = __float_as_uint(v); }
};

__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }   // orders |v|, NaN on top
__device__ __forceinline__ uint32_t four_bytes(float a, float b, float c, float d) { return cvt_e4m3x2(a, b) | (cvt_e4m3x2(c, d) << 16); }

// SQUARE: one scale for the tile; otherwise ROW / COL say which orientations have scales of their own
template <typename T, bool ROW, bool COL, bool SQUARE>
__global__ void __launch_bounds__(32 * WARPS, sizeof(T) == 2 ? 3 : 2) quantize_block128_kernel(const Params p) {
    __shared__ alignas(16) uint8_t stage[COL ? B * B : 16];
    __shared__ uint32_t cmax[COL && !SQUARE ? WARPS * B : WARPS];
    __shared__ alignas(16) float cinv[B];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_e = p.tiles_m * p.tiles_n;
    const int e = blockIdx.x / per_e, t = blockIdx.x - e * per_e;
    const int grp = t / (GROUP_M * p.tiles_n), in_grp = t - grp * (GROUP_M * p.tiles_n);
    const int rows_in = min(GROUP_M, p.tiles_m - grp * GROUP_M);
    const int tm = grp * GROUP_M + in_grp % rows_in, tn = in_grp / rows_in;
    const int m0 = tm * B + warp * ROWS, n0 = tn * B + lane * 4;

    Four<T> v[ROWS];
    const T* x = static_cast<const T*>(p.x) + static_cast<long long>(e) * p.M * p.ldx;
    int src = 0;
    if (lane < ROWS) {
        src = m0 + lane < p.M ? m0 + lane : -1;
        if (p.row_index && src >= 0) {
            src = p.row_index[src];
            if (src >= p.src_rows) src = -1;
        }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        v[r].zero();
        const int s = __shfl_sync(0xFFFFFFFFu, src, r);
        if (s >= 0) {
            const T* row = x + s * p.ldx + n0;
            if (p.vec_x && n0 + 4 <= p.N) {
                v[r].load(row);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n0 + i < p.N) v[r].set(i, row[i]);
            }
        }
    }

    float row_inv = 0.0f;                          // lane r < 16: reciprocal scale of row r
    float tile_inv = 0.0f;
    if constexpr (SQUARE) {
        uint32_t a = 0;
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) a = max(a, mag(v[r].get(i)));
        a = __reduce_max_sync(0xFFFFFFFFu, a);
        if (lane == 0) cmax[warp] = a;
        __syncthreads();
        a = AMAX_FLOOR;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) a = max(a, cmax[w]);
        tile_inv = __fdiv_rn(448.0f, __uint_as_float(a));
        if (threadIdx.x == 0) {
            const float s = __fdiv_rn(__uint_as_float(a), 448.0f);
            if (ROW) p.sc[(static_cast<size_t>(e) * p.tiles_m + tm) * p.tiles_n + tn] = s;
            if (COL) p.sc_t[(static_cast<size_t>(e) * p.tiles_n + tn) * p.tiles_m + tm] = s;
        }
    } else if constexpr (ROW) {
        uint32_t mine = AMAX_FLOOR;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            uint32_t a = mag(v[r].get(0));
#pragma unroll
            for (int i = 1; i < 4; ++i) a = max(a, mag(v[r].get(i)));
            a = __reduce_max_sync(0xFFFFFFFFu, a);
            if (lane == r) mine = max(mine, a);
        }
        row_inv = __fdiv_rn(448.0f, __uint_as_float(mine));
        if (lane < ROWS && m0 + lane < p.M)
            p.sc[(static_cast<size_t>(e) * p.tiles_n + tn) * p.M + m0 + lane] = __fdiv_rn(__uint_as_float(mine), 448.0f);
    }
    if constexpr (ROW) {
        uint8_t* q = p.q + (static_cast<long long>(e) * p.M + m0) * p.ld + n0;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const float inv = SQUARE ? tile_inv : __shfl_sync(0xFFFFFFFFu, row_inv, r);
            if (m0 + r >= p.M) break;
            const uint32_t b = four_bytes(v[r].get(0) * inv, v[r].get(1) * inv, v[r].get(2) * inv, v[r].get(3) * inv);
            if (p.vec_q && n0 + 4 <= p.N) {
                *reinterpret_cast<uint32_t*>(q + r * p.ld) = b;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n0 + i < p.N) q[r * p.ld + i] = static_cast<uint8_t>(b >> (8 * i));
            }
        }
    }
    if constexpr (COL) {
        float inv[4];
        if constexpr (SQUARE) {
#pragma unroll
            for (int i = 0; i < 4; ++i) inv[i] = tile_inv;
        } else {
            uint32_t a[4] = {0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = max(a[i], mag(v[r].get(i)));
            *reinterpret_cast<uint4*>(&cmax[warp * B + lane * 4]) = make_uint4(a[0], a[1], a[2], a[3]);
            __syncthreads();
            if (threadIdx.x < B) {
                uint32_t m = AMAX_FLOOR;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) m = max(m, cmax[w * B + threadIdx.x]);
                cinv[threadIdx.x] = __fdiv_rn(448.0f, __uint_as_float(m));
                const int n = tn * B + threadIdx.x;
                if (n < p.N) p.sc_t[(static_cast<size_t>(e) * p.tiles_m + tm) * p.N + n] = __fdiv_rn(__uint_as_float(m), 448.0f);
            }
            __syncthreads();
            const float4 c = *reinterpret_cast<const float4*>(&cinv[lane * 4]);
            inv[0] = c.x; inv[1] = c.y; inv[2] = c.z; inv[3] = c.w;
        }
        // column c: 16-byte piece `warp` of its 128 bytes goes to slot warp ^ ((c / 4) % 8): the eight lanes of a quarter warp
        // write, and read, eight different slots
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = four_bytes(v[4 * j].get(i) * inv[i], v[4 * j + 1].get(i) * inv[i], v[4 * j + 2].get(i) * inv[i], v[4 * j + 3].get(i) * inv[i]);
            *reinterpret_cast<uint4*>(stage + (lane * 4 + i) * B + ((warp ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ROWS / 4; ++k) {
            const int c = warp * ROWS + k * 4 + (lane >> 3), piece = lane & 7;
            const int n = tn * B + c, m = tm * B + piece * 16;
            if (n >= p.N || m >= p.M) continue;
            const uint4 w = *reinterpret_cast<const uint4*>(stage + c * B + ((piece ^ ((c >> 2) & 7)) << 4));
            uint8_t* dst = p.qt + (static_cast<long long>(e) * p.N + n) * p.ld_t + m;
            if (p.vec_t && m + 16 <= p.M) {
                *reinterpret_cast<uint4*>(dst) = w;
            } else {
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (m + i < p.M) dst[i] = static_cast<uint8_t>(ws[i >> 2] >> (8 * (i & 3)));
            }
        }
    }
}

template <typename T>
static cudaError_t launch(const Params& p, bool row, bool col, bool square, cudaStream_t st) {
    const unsigned grid = static_cast<unsigned>(p.E) * p.tiles_m * p.tiles_n;
    if (square) {
        if (row && col) quantize_block128_kernel<T, true, true, true><<<grid, 32 * WARPS, 0, st>>>(p);
        else if (row) quantize_block128_kernel<T, true, false, true><<<grid, 32 * WARPS, 0, st>>>(p);
        else quantize_block128_kernel<T, false, true, true><<<grid, 32 * WARPS, 0, st>>>(p);
    } else {
        if (row && col) quantize_block128_kernel<T, true, true, false><<<grid, 32 * WARPS, 0, st>>>(p);
        else if (row) quantize_block128_kernel<T, true, false, false><<<grid, 32 * WARPS, 0, st>>>(p);
        else quantize_block128_kernel<T, false, true, false><<<grid, 32 * WARPS, 0, st>>>(p);
    }
    return cudaGetLastError();
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
    if (tiles_m * tiles_n > 0x7FFFFFFFll / E) {
        note_cuda_error("mx8_quantize_block128", "more than 2^31 - 1 tiles of 128 x 128");
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
    p.vec_x = ldx % 4 == 0 && reinterpret_cast<uintptr_t>(x) % (4 * esize) == 0;
    p.vec_q = ld % 4 == 0 && reinterpret_cast<uintptr_t>(fp8) % 4 == 0;
    p.vec_t = ld_t % 16 == 0 && aligned16(fp8_t);
    const cudaError_t e = dtype == MX8_T_F32 ? q128::launch<float>(p, row, col, square != 0, static_cast<cudaStream_t>(stream))
                                             : q128::launch<uint16_t>(p, row, col, square != 0, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) {
        note_cuda_error("block-128 quantizer launch", cudaGetErrorString(e));
        return MX8_ERR_CUDA;
    }
    return MX8_OK;
}
