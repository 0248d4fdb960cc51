// Router of the MoE layer: softmax over the experts, top-k, per-expert counts and the balance loss, their gradient, and the
// gradient of the routing weights.
//
// forward   p = softmax(l) in fp32; S_t = the k largest logits of token t, ties to the lower expert; w = p over S_t, divided by its
//           sum when `normalize`; c_e = chosen (token, slot) pairs of expert e; P_e = sum_t p_te; V = tokens that take part;
//           L = E / (k V^2) * sum_e c_e P_e.  An expert whose logit is -inf is switched off; a token without a live expert, or with
//           its mask byte 0, takes no part (ids -1, weights 0, lse -inf).
// backward  normalised  dl = w (dw - sum_S w dw) on S;  otherwise  dl = p ([in S] dw - sum_S w dw);
//           both + p (b - sum_e b p), b_e = dL E c_e / (k V^2).
//
// One warp owns a token; lane l holds experts l*VPL .. l*VPL + VPL - 1.  The kernels are bound by instructions, not by memory (a token of
// 256 experts is 512 bytes), so the selection works on 32-bit words that hold the value's order-preserving bits, cut to 22, and the
// expert's number reversed in the other 10: all words differ, the larger word is the larger value or the lower expert, and one
// redux.sync.max finds both.  bf16 values fit in the 22 bits; for fp32 the result is checked against the full values and rows in which
// the cut bits decide (values within 2^-13 of each other) are selected again, slowly.
// Sums over tokens are made in a fixed order (registers of a warp, then warps of a block, both in 32 bits, then blocks in 64), never with
// floating-point atomics: results do not change from run to run.
#include <atomic>

#include "mx8_host.cuh"
#include "mx8_ptx.cuh"

namespace mx8 {
namespace router {

constexpr int MAX_EXPERTS = 1024;
constexpr int MAX_TOPK = 32;              // one lane per choice

struct FwdParams {
    const void* logits;
    long long ld;                         // elements between rows
    int vec;                              // rows may be read in whole-lane vectors
    int tokens, experts, topk, normalize;
    const uint8_t* mask;                  // nullptr: all tokens take part
    int* idx;
    float* weights;
    float* lse;
    int* counts;
    float* prob_sum;
    int* num_valid;
    float* loss;
    float* part_prob;                     // [blocks][experts]
    int* part_count;                      // [blocks][experts]
    int* part_valid;                      // [blocks]
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(uint16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }

// A lane's VPL consecutive logits as they lie in memory (bf16: two to a word; a single one in the low half); experts beyond the row's
// end are -inf.
template <typename T, int VPL>
struct Row {
    static constexpr int BYTES = VPL * static_cast<int>(sizeof(T));
    static constexpr int WORDS = BYTES >= 4 ? BYTES / 4 : 1;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const T* row, int lane, int experts, bool vec) {
        const int e0 = lane * VPL;
        constexpr uint32_t NONE = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
        if (BYTES >= 4 && vec) {              // VPL divides the row length: a lane is whole or empty
            const uint8_t* src = reinterpret_cast<const uint8_t*>(row + e0);
            if (e0 >= experts) {
#pragma unroll
                for (int i = 0; i < WORDS; ++i) w[i] = NONE;
            } else if constexpr (BYTES >= 16) {
#pragma unroll
                for (int i = 0; i < WORDS; i += 4) {
                    const uint4 x = __ldg(reinterpret_cast<const uint4*>(src + 4 * i));
                    w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
                }
            } else if constexpr (BYTES == 8) {
                const uint2 x = __ldg(reinterpret_cast<const uint2*>(src));
                w[0] = x.x; w[1] = x.y;
            } else {
                w[0] = __ldg(reinterpret_cast<const uint32_t*>(src));
            }
        } else {
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                if constexpr (sizeof(T) == 4) {
                    w[i] = e0 + i < experts ? __float_as_uint(row[e0 + i]) : NONE;
                } else {
                    const uint32_t v = e0 + i < experts ? static_cast<uint32_t>(row[e0 + i]) : 0xFF80u;
                    w[i / 2] = (i & 1) ? w[i / 2] | (v << 16) : v | (VPL == 1 ? 0xFF800000u : 0u);
                }
            }
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else return __uint_as_float((i & 1) ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    }
};

// Order-preserving bits of a logit: adding +0 makes -0 equal to +0 and every NaN the positive one, which lies above +inf; -inf gives
// 0x007FFFFF (bf16: 0x007F), below all that is finite: words under LIVE are switched-off experts.
constexpr uint32_t LIVE = 0x00800000u;
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k); }

// the selection's words (see above) of a lane's experts
template <typename T, int VPL>
__device__ __forceinline__ void words_of(const Row<T, VPL>& row, int lane, uint32_t (&word)[VPL]) {
    const uint32_t code = 1023u - lane * VPL;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) word[i] = (key_of(row.get(i)) & ~1023u) | (code - i);
    } else {
#pragma unroll
        for (int i = 0; i < VPL; i += 2) {
            uint32_t w;
            asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(w) : "r"(row.w[i / 2]), "r"(0u));
            w ^= ((w >> 15) & 0x00010001u) * 0x7FFFu ^ 0x80008000u;
            word[i] = (w << 16) + (code - i);
            if (i + 1 < VPL) word[i + 1] = (w & 0xFFFF0000u) + (code - i - 1);
        }
    }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// three sums over the warp at once: lanes first divide the sums among themselves, nine exchanges instead of fifteen
__device__ __forceinline__ void warp_sums(float& a, float& b, float& c, int lane) {
    const bool h = lane & 16, q = lane & 8;
    float x = h ? b : a, z = c;
    x += __shfl_xor_sync(0xFFFFFFFFu, h ? a : b, 16);                      // lanes 0 - 15: a, 16 - 31: b
    z += __shfl_xor_sync(0xFFFFFFFFu, z, 16);
    float u = q ? z : x;
    u += __shfl_xor_sync(0xFFFFFFFFu, q ? x : z, 8);                       // lanes 8 - 15 and 24 - 31: c
#pragma unroll
    for (int o = 4; o; o >>= 1) u += __shfl_xor_sync(0xFFFFFFFFu, u, o);
    a = __shfl_sync(0xFFFFFFFFu, u, 0);
    b = __shfl_sync(0xFFFFFFFFu, u, 16);
    c = __shfl_sync(0xFFFFFFFFu, u, 8);
}

// descending, by a network of compare-exchanges (19 of them for 8 words)
template <int N>
__device__ __forceinline__ void sort_words(uint32_t (&w)[N]) {
    auto cx = [&](int i, int j) {
        const uint32_t hi = max(w[i], w[j]), lo = min(w[i], w[j]);
        w[i] = hi;
        w[j] = lo;
    };
    if constexpr (N == 2) {
        cx(0, 1);
    } else if constexpr (N == 4) {
        cx(0, 1); cx(2, 3); cx(0, 2); cx(1, 3); cx(1, 2);
    } else if constexpr (N == 8) {
        cx(0, 1); cx(2, 3); cx(4, 5); cx(6, 7);
        cx(0, 2); cx(1, 3); cx(4, 6); cx(5, 7);
        cx(1, 2); cx(5, 6);
        cx(0, 4); cx(1, 5); cx(2, 6); cx(3, 7);
        cx(2, 4); cx(3, 5);
        cx(1, 2); cx(3, 4); cx(5, 6);
    }
}

// k rounds on the full keys: the largest, the lowest lane that has it, the lowest of its experts that has it; lane j gets choice j.  From the
// registers: with 512 experts two tokens in a hundred come here, and reading the row again every round took 10 us for one.
template <int VPL>
__device__ __forceinline__ int select_slowly(const Row<float, VPL>& in, int topk, int lane) {
    int my_idx = -1;
    uint32_t key[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) key[i] = key_of(in.get(i));
#pragma unroll 1
    for (int j = 0; j < topk; ++j) {
        uint32_t best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < VPL; ++i) {
            at = key[i] > best ? i : at;
            best = max(best, key[i]);
        }
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
        if (top < LIVE) break;
        const int owner = __ffs(__ballot_sync(0xFFFFFFFFu, best == top)) - 1;
#pragma unroll
        for (int i = 0; i < VPL; ++i) key[i] = lane == owner && i == at ? 0u : key[i];
        at = __shfl_sync(0xFFFFFFFFu, at, owner);
        if (lane == j) my_idx = owner * VPL + at;
    }
    return my_idx;
}

__device__ __forceinline__ float loss_of(double dot, int n, int experts, int topk) {
    return n > 0 ? static_cast<float>(dot * experts / (static_cast<double>(topk) * n * n)) : 0.0f;
}

// double sum over a block in a fixed order; the result is valid in thread 0
__device__ __forceinline__ double block_sum(double v, double* scratch) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0;
    if (threadIdx.x == 0)
        for (int w = 0; w < static_cast<int>(blockDim.x + 31) / 32; ++w) s += scratch[w];
    return s;
}

template <int VPL>
struct Shape {
    static constexpr int WARPS = VPL <= 8 ? 32 : 16;      // 64 registers a lane hold VPL = 8 logits and probability sums
};

template <typename T, int VPL>
__global__ void __launch_bounds__(Shape<VPL>::WARPS * 32) router_fwd_kernel(const FwdParams p) {
    constexpr int WARPS = Shape<VPL>::WARPS;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");        // the finishing kernel may be brought up beside this one
    extern __shared__ float smem[];
    float* warp_prob = smem;                                               // [WARPS][experts]
    int* count = reinterpret_cast<int*>(smem + WARPS * p.experts);         // [experts]
    __shared__ int valid_sum;
    __shared__ double scratch[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int e = threadIdx.x; e < p.experts; e += WARPS * 32) count[e] = 0;
    if (threadIdx.x == 0) valid_sum = 0;
    __syncthreads();
    float prob[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) prob[i] = 0.0f;
    int n_valid = 0;
    // the next token's logits are on their way while this one is worked on (a masked token's are fetched too, and dropped)
    const int step = gridDim.x * WARPS;
    int t = blockIdx.x * WARPS + warp;
    const T* row = static_cast<const T*>(p.logits) + t * p.ld;
    Row<T, VPL> next;
    uint8_t next_on = 1;
    if (t < p.tokens) {
        next.load(row, lane, p.experts, p.vec != 0);
        if (p.mask) next_on = p.mask[t];
    }
    // the logarithms of 32 tokens are taken together, a lane each: lane n % 32 holds those of the warp's n-th token
    int n = 0;
    float lse_max = 0.0f, lse_sum = 1.0f;
    auto keep_lse = [&](float mx, float sum) {
        if (lane == (n & 31)) {
            lse_max = mx;
            lse_sum = sum;
        }
        if ((++n & 31) == 0) p.lse[t - (31 - lane) * step] = lse_max + logf(lse_sum);
    };
    for (; t < p.tokens; t += step, row += step * p.ld) {
        const Row<T, VPL> in = next;
        const bool on = next_on != 0;
        if (p.tokens - t > step) {
            next.load(row + step * p.ld, lane, p.experts, p.vec != 0);
            if (p.mask) next_on = p.mask[t + step];
        }
        const size_t out = static_cast<size_t>(t) * p.topk + lane;
        // the largest logit; bf16: the first choice's word has all of it
        uint32_t word[VPL];
        words_of<T, VPL>(in, lane, word);
        uint32_t top;
        if constexpr (sizeof(T) == 4) {
            top = key_of(in.get(0));
#pragma unroll
            for (int i = 1; i < VPL; ++i) top = max(top, key_of(in.get(i)));
            top = __reduce_max_sync(0xFFFFFFFFu, top);
        }
        if constexpr (VPL <= 8) sort_words<VPL>(word);
        auto head_of = [&]() {
            uint32_t h = word[0];
            if constexpr (VPL > 8) {
#pragma unroll
                for (int i = 1; i < VPL; ++i) h = max(h, word[i]);
            }
            return h;
        };
        uint32_t best = __reduce_max_sync(0xFFFFFFFFu, head_of());
        if constexpr (sizeof(T) == 2) top = best & 0xFFFF0000u;
        if (!on || best < LIVE) {                          // masked, or every expert switched off
            if (lane < p.topk) {
                p.idx[out] = -1;
                p.weights[out] = 0.0f;
            }
            keep_lse(-INFINITY, 1.0f);
            continue;
        }
        const float mx = sizeof(T) == 4 ? value_of(top) : __uint_as_float(__float_as_uint(value_of(top)) & 0xFFFF0000u);
        float v[VPL], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            v[i] = expf(in.get(i) - mx);
            sum += v[i];
        }
        sum = warp_sum(sum);
        const float inv = __frcp_rn(sum);                  // rounded once; a weight is off by this rounding and its own (quotients rounded once: 25.0 -> 26 us at 32768 x 256)
#pragma unroll
        for (int i = 0; i < VPL; ++i) prob[i] = fmaf(v[i], inv, prob[i]);
        ++n_valid;
        int my_idx = -1;                                   // lane j: choice j
        for (int j = 0; j < p.topk; ++j) {
            if (j) best = __reduce_max_sync(0xFFFFFFFFu, head_of());
            if (best < LIVE) break;                        // fewer live experts than choices
            if (lane == j) my_idx = 1023 - static_cast<int>(best & 1023u);
            if constexpr (VPL <= 8) {
                const bool mine = word[0] == best;
#pragma unroll
                for (int i = 0; i + 1 < VPL; ++i) word[i] = mine ? word[i + 1] : word[i];
                word[VPL - 1] = mine ? 0u : word[VPL - 1];
            } else {
#pragma unroll
                for (int i = 0; i < VPL; ++i) word[i] = word[i] == best ? 0u : word[i];
            }
        }
        float my_val = my_idx >= 0 ? to_float(row[my_idx]) : 0.0f;
        if constexpr (sizeof(T) == 4) {
            // right unless the cut bits decide: the choices' full keys fall, with rising experts among equals, and as many keys of the row
            // lie above the last choice as choices do
            const uint32_t full = my_idx >= 0 ? key_of(my_val) : 0u;
            const unsigned chosen = __ballot_sync(0xFFFFFFFFu, my_idx >= 0);
            const int last = 31 - __clz(chosen);
            const uint32_t after = __shfl_down_sync(0xFFFFFFFFu, full, 1);
            const int after_idx = __shfl_down_sync(0xFFFFFFFFu, my_idx, 1);
            const bool wrong = lane < last && (full < after || (full == after && my_idx > after_idx));
            const uint32_t low = __shfl_sync(0xFFFFFFFFu, full, last);
            int above = 0;
#pragma unroll
            for (int i = 0; i < VPL; ++i) above += key_of(in.get(i)) > low;
            above = __reduce_add_sync(0xFFFFFFFFu, above);
            const int chosen_above = __popc(__ballot_sync(0xFFFFFFFFu, my_idx >= 0 && full > low));
            if (__any_sync(0xFFFFFFFFu, wrong) || above != chosen_above) {
                my_idx = select_slowly<VPL>(in, p.topk, lane);
                my_val = my_idx >= 0 ? to_float(row[my_idx]) : 0.0f;
            }
        }
        float w = my_idx >= 0 ? expf(my_val - mx) : 0.0f;
        w *= p.normalize ? __frcp_rn(warp_sum(w)) : inv;
        if (lane < p.topk) {
            p.idx[out] = my_idx;
            p.weights[out] = my_idx >= 0 ? w : 0.0f;
            if (my_idx >= 0) atomicAdd(&count[my_idx], 1);
        }
        keep_lse(mx, sum);
    }
    if (lane < (n & 31)) p.lse[t - ((n & 31) - lane) * step] = lse_max + logf(lse_sum);
#pragma unroll
    for (int i = 0; i < VPL; ++i)
        if (lane * VPL + i < p.experts) warp_prob[warp * p.experts + lane * VPL + i] = prob[i];
    if (lane == 0 && n_valid) atomicAdd(&valid_sum, n_valid);
    __syncthreads();
    const bool last = gridDim.x == 1;
    double dot = 0;
    for (int e = threadIdx.x; e < p.experts; e += WARPS * 32) {
        float s = 0.0f;
#pragma unroll 8
        for (int w = 0; w < WARPS; ++w) s += warp_prob[w * p.experts + e];
        const int c = count[e];
        if (last) {
            p.counts[e] = c;
            p.prob_sum[e] = s;
            dot += static_cast<double>(c) * s;
        } else {
            p.part_prob[static_cast<size_t>(blockIdx.x) * p.experts + e] = s;
            p.part_count[static_cast<size_t>(blockIdx.x) * p.experts + e] = c;
        }
    }
    if (last) {
        dot = block_sum(dot, scratch);
        if (threadIdx.x == 0) {
            *p.num_valid = valid_sum;
            *p.loss = loss_of(dot, valid_sum, p.experts, p.topk);
        }
    } else if (threadIdx.x == 0) {
        p.part_valid[blockIdx.x] = valid_sum;
    }
}

// Sums the blocks' partial counts and probabilities and makes the loss: one cluster of blocks, each with a share of the experts, 32
// threads on each expert.
constexpr int FINISH = 8;
__global__ void __cluster_dims__(FINISH, 1, 1) __launch_bounds__(1024) router_finish_kernel(const FwdParams p, int blocks) {
    __shared__ double sum_p[32][33];
    __shared__ int sum_c[32][33];
    __shared__ double dots[FINISH];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = blockIdx.x;
    double dot = 0;
    // rank 0's shared memory may be written once its block is known to run: every block arrives here, and waits before it stores
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    // launched while the forward kernel still runs: from here on its results are there
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int n = 0;                                              // the tokens that took part
    if (rank == 0 && warp == 0)
        for (int b = lane; b < blocks; b += 32) n += p.part_valid[b];
    for (int e0 = rank * 32; e0 < p.experts; e0 += FINISH * 32) {
        const int e = e0 + lane;                            // warps are slices of the blocks: consecutive experts in a load
        double s = 0;
        int c = 0;
        if (e < p.experts) {
#pragma unroll 4
            for (int b = warp; b < blocks; b += 32) {
                s += p.part_prob[static_cast<size_t>(b) * p.experts + e];
                c += p.part_count[static_cast<size_t>(b) * p.experts + e];
            }
        }
        sum_p[warp][lane] = s;
        sum_c[warp][lane] = c;
        __syncthreads();
        s = sum_p[lane][warp];                              // now warp = expert, lane = slice
        c = sum_c[lane][warp];
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        c = __reduce_add_sync(0xFFFFFFFFu, c);
        if (lane == 0 && e0 + warp < p.experts) {
            p.counts[e0 + warp] = c;
            p.prob_sum[e0 + warp] = static_cast<float>(s);
            dot += s * c;
        }
        __syncthreads();
    }
    if (lane == 0) sum_p[1][warp] = dot;                    // its experts' share
    __syncthreads();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp == 0) {
        dot = sum_p[1][lane];
#pragma unroll
        for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
        if (lane == 0) {
            const uint32_t to = map_to_cta(smem_u32(&dots[rank]), 0);
            asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(dot) : "memory");
        }
    }
    cluster_sync_all();
    if (rank == 0 && warp == 0) {
        n = __reduce_add_sync(0xFFFFFFFFu, n);
        if (lane == 0) {
            dot = 0;
            for (int i = 0; i < FINISH; ++i) dot += dots[i];
            *p.num_valid = n;
            *p.loss = loss_of(dot, n, p.experts, p.topk);
        }
    }
}

struct BwdParams {
    const void* logits;
    long long ld;
    int vec;
    int tokens, experts, topk, normalize;
    const int* idx;
    const float* weights;
    const float* lse;
    const int* counts;
    const int* num_valid;
    const float* d_weights;               // nullptr: zero
    const float* d_loss;                  // nullptr: zero
    void* d_logits;                       // [tokens][experts], contiguous
    int vec_out;
};

constexpr int BWD_WARPS = 8;

template <int VPL>
__host__ __device__ constexpr int bwd_blocks() { return VPL <= 8 ? 5 : VPL == 16 ? 3 : 1; }      // resident per multiprocessor

template <typename T, int VPL>
__global__ void __launch_bounds__(BWD_WARPS * 32, bwd_blocks<VPL>()) router_bwd_kernel(const BwdParams p) {
    // b of every expert; per warp: gradients at the chosen experts, zero elsewhere.  Expert lane * VPL + i lies at i * 32 + lane: no two
    // lanes of a read share a bank.
    extern __shared__ float smem[];
    auto place = [](int e) { return (e & (VPL - 1)) * 32 + e / VPL; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* bs = smem;
    float* row = smem + (warp + 1) * (32 * VPL);
    {
        const float n = static_cast<float>(*p.num_valid), g = p.d_loss ? *p.d_loss : 0.0f;
        const float f = n > 0.0f ? g * (static_cast<float>(p.experts) / (static_cast<float>(p.topk) * n)) / n : 0.0f;
        for (int e = threadIdx.x; e < 32 * VPL; e += BWD_WARPS * 32) bs[place(e)] = p.d_loss && e < p.experts ? f * static_cast<float>(p.counts[e]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) row[lane + 32 * i] = 0.0f;
    __syncthreads();
    float b[VPL];                                      // this lane's, read twice a token (before its sums were made together: 32768 x 256 13.9 -> 13.3 us, x 1024 71 -> 60 us)
#pragma unroll
    for (int i = 0; i < VPL; ++i) b[i] = bs[i * 32 + lane];
    // a token's inputs; loaded for the next token before this one's arithmetic, as nothing else hides their latency
    struct In {
        Row<T, VPL> v;
        float lse, w, dw;
        int idx;
    };
    const T* from = static_cast<const T*>(p.logits);
    auto load = [&](int t, In& in) {
        in.v.load(from + t * p.ld, lane, p.experts, p.vec != 0);
        in.lse = p.lse[t];
        in.idx = -1;
        in.w = in.dw = 0.0f;
        if (p.d_weights && lane < p.topk) {
            const size_t at = static_cast<size_t>(t) * p.topk + lane;
            in.idx = p.idx[at];
            in.w = p.weights[at];
            in.dw = p.d_weights[at];
        }
    };
    const int step = gridDim.x * BWD_WARPS;
    int t = blockIdx.x * BWD_WARPS + warp;
    In next;
    if (t < p.tokens) load(t, next);
    for (; t < p.tokens; t += step) {
        const In in = next;
        if (p.tokens - t > step) load(t + step, next);
        T* out = static_cast<T*>(p.d_logits) + static_cast<size_t>(t) * p.experts;
        float v[VPL];
        const bool on = in.lse != -INFINITY;               // a token that took no part gets zeros, whatever its logits are
        // lse is rounded, which makes all of the token's exponentials too large or too small by up to |lse| 2^-24: what counts is their
        // share of their own sum
        float dot = 0.0f, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            v[i] = on ? expf(in.v.get(i) - in.lse) : 0.0f;
            dot += v[i] * b[i];
            sum += v[i];
        }
        const int idx = in.idx >= 0 && in.idx < p.experts ? in.idx : -1;
        const float w = idx >= 0 ? in.w : 0.0f, dw = idx >= 0 ? in.dw : 0.0f, wdw = w * dw;
        float s = wdw;
        warp_sums(dot, sum, s, lane);
        const float inv = __frcp_rn(sum);
        dot *= inv;
        if (p.d_weights) {
            if (!p.normalize) dot += s;
            if (idx >= 0) row[place(idx)] = p.normalize ? w * (dw - s) : wdw;      // a token's choices are distinct
            __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) v[i] = on ? v[i] * fmaf(b[i], inv, -dot * inv) + (p.d_weights ? row[i * 32 + lane] : 0.0f) : 0.0f;
        if (p.d_weights) {
            __syncwarp();
            if (idx >= 0) row[place(idx)] = 0.0f;
            __syncwarp();
        }
        const int e0 = lane * VPL;
        constexpr int BYTES = VPL * static_cast<int>(sizeof(T));
        if (BYTES >= 4 && p.vec_out) {
            if (e0 < p.experts) {
                uint32_t o[BYTES >= 4 ? BYTES / 4 : 1];
#pragma unroll
                for (int i = 0; i < BYTES / 4; ++i) {
                    if constexpr (sizeof(T) == 4) o[i] = __float_as_uint(v[i]);
                    else o[i] = pack_bf16x2(v[(2 * i) % VPL], v[(2 * i + 1) % VPL]);
                }
                if constexpr (BYTES >= 16) {
#pragma unroll
                    for (int i = 0; i < BYTES / 4; i += 4) *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(out + e0) + 4 * i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                } else if constexpr (BYTES == 8) {
                    *reinterpret_cast<uint2*>(out + e0) = make_uint2(o[0], o[1]);
                } else if constexpr (BYTES == 4) {
                    *reinterpret_cast<uint32_t*>(out + e0) = o[0];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                if (e0 + i < p.experts) {
                    if constexpr (sizeof(T) == 4) out[e0 + i] = v[i];
                    else out[e0 + i] = static_cast<uint16_t>(pack_bf16x2(v[i], 0.0f));
                }
            }
        }
    }
}

// dw[t][j] = sum_h d_output[t][h] * combine[t*topk + j][h]: every byte of combine is used once, so the kernel is bound by reading
// it.  One block of four warps owns a token and eight of its choices: a thread holds 8 columns of d_output and has the eight rows'
// loads (16 bytes each) in flight together; fp32 sums, combined over the lanes and warps in a fixed order.
constexpr int WG_THREADS = 128;
constexpr int WG_K = 8;

template <bool VEC>
__global__ void __launch_bounds__(WG_THREADS) topk_weights_grad_kernel(const uint16_t* __restrict__ d_out, const uint16_t* __restrict__ combine,
                                                                       const int* __restrict__ idx, float* __restrict__ dw, int hidden, int topk) {
    const long long t = blockIdx.x;
    const int j0 = blockIdx.y * WG_K;
    const int nj = min(WG_K, topk - j0);
    const uint16_t* g = d_out + t * hidden;
    const uint16_t* rows = combine + (t * topk + j0) * hidden;
    float acc[WG_K];
    bool live[WG_K];
#pragma unroll
    for (int j = 0; j < WG_K; ++j) {
        acc[j] = 0.0f;
        live[j] = j < nj && (!idx || idx[t * topk + j0 + j] >= 0);         // a row that was never sent is not read
    }
    if constexpr (VEC) {
        for (int h = threadIdx.x * 8; h < hidden; h += WG_THREADS * 8) {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(g + h));
            uint4 r[WG_K];
#pragma unroll
            for (int j = 0; j < WG_K; ++j)
                if (live[j]) r[j] = __ldg(reinterpret_cast<const uint4*>(rows + static_cast<size_t>(j) * hidden + h));
            const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < WG_K; ++j) {
                if (!live[j]) continue;
                const uint32_t rw[4] = {r[j].x, r[j].y, r[j].z, r[j].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    acc[j] = fmaf(__uint_as_float(aw[i] << 16), __uint_as_float(rw[i] << 16), acc[j]);
                    acc[j] = fmaf(__uint_as_float(aw[i] & 0xFFFF0000u), __uint_as_float(rw[i] & 0xFFFF0000u), acc[j]);
                }
            }
        }
    } else {
        for (int h = threadIdx.x; h < hidden; h += WG_THREADS) {
            const float a = to_float(g[h]);
#pragma unroll
            for (int j = 0; j < WG_K; ++j)
                if (live[j]) acc[j] = fmaf(a, to_float(rows[static_cast<size_t>(j) * hidden + h]), acc[j]);
        }
    }
    __shared__ float part[WG_THREADS / 32][WG_K];
#pragma unroll
    for (int j = 0; j < WG_K; ++j) acc[j] = warp_sum(acc[j]);
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int j = 0; j < WG_K; ++j) part[threadIdx.x >> 5][j] = acc[j];
    }
    __syncthreads();
    if (threadIdx.x < nj) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < WG_THREADS / 32; ++w) s += part[w][threadIdx.x];
        dw[t * topk + j0 + threadIdx.x] = s;
    }
}

static int vpl_of(int experts) {
    int v = 1;
    while (v * 32 < experts) v *= 2;
    return v;
}

// a row can be read in one vector per lane: whole lanes, and every lane's first element on the vector's boundary
static int vec_ok(const void* base, long long ld, int experts, int vpl, int esize) {
    const int chunk = vpl * esize >= 16 ? 16 : vpl * esize;
    return chunk >= 4 && experts % vpl == 0 && reinterpret_cast<uintptr_t>(base) % chunk == 0 && (ld * esize) % chunk == 0;
}

static int grid_of(int tokens, int warps) {
    // one block per multiprocessor; up to two rounds of one block stay a single launch, which then finishes the sums itself
    const int need = (tokens + warps - 1) / warps;
    return need <= 2 ? 1 : (need < sm_count() ? need : sm_count());
}

static int warps_of(int vpl) { return vpl <= 8 ? 32 : 16; }

template <typename T, int VPL>
static cudaError_t launch_fwd(const FwdParams& p, int grid, cudaStream_t st) {
    constexpr int WARPS = Shape<VPL>::WARPS;
    const size_t smem = sizeof(float) * (WARPS + 1) * static_cast<size_t>(p.experts);
    constexpr int MOST = static_cast<int>(sizeof(float)) * (WARPS + 1) * 32 * VPL;
    auto kern = router_fwd_kernel<T, VPL>;
    if constexpr (MOST > 40 * 1024) {
        // what the kernel can need at most, not this call's own: another thread may be between its attribute and its launch
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST);
        if (e != cudaSuccess) return e;
    }
    kern<<<grid, WARPS * 32, smem, st>>>(p);
    return cudaGetLastError();
}

template <typename T, int VPL>
static cudaError_t launch_bwd(const BwdParams& p, cudaStream_t st) {
    const int need = (p.tokens + BWD_WARPS - 1) / BWD_WARPS, most = sm_count() * bwd_blocks<VPL>();
    const size_t smem = sizeof(float) * (BWD_WARPS + 1) * 32 * VPL;           // at most 36 KB
    router_bwd_kernel<T, VPL><<<need < most ? need : most, BWD_WARPS * 32, smem, st>>>(p);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t dispatch_fwd(const FwdParams& p, int vpl, int grid, cudaStream_t st) {
    switch (vpl) {
        case 1: return launch_fwd<T, 1>(p, grid, st);
        case 2: return launch_fwd<T, 2>(p, grid, st);
        case 4: return launch_fwd<T, 4>(p, grid, st);
        case 8: return launch_fwd<T, 8>(p, grid, st);
        case 16: return launch_fwd<T, 16>(p, grid, st);
        default: return launch_fwd<T, 32>(p, grid, st);
    }
}

template <typename T>
static cudaError_t dispatch_bwd(const BwdParams& p, int vpl, cudaStream_t st) {
    switch (vpl) {
        case 1: return launch_bwd<T, 1>(p, st);
        case 2: return launch_bwd<T, 2>(p, st);
        case 4: return launch_bwd<T, 4>(p, st);
        case 8: return launch_bwd<T, 8>(p, st);
        case 16: return launch_bwd<T, 16>(p, st);
        default: return launch_bwd<T, 32>(p, st);
    }
}

static bool misaligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

static int check_shape(const char* what, int dtype, long long ld, int tokens, int experts, int topk) {
    if (dtype != MX8_T_BF16 && dtype != MX8_T_F32) return MX8_ERR_ARG;
    if (tokens <= 0 || experts <= 0 || topk <= 0 || topk > experts || ld < experts) {
        note_cuda_error(what, "tokens and experts positive, 1 <= topk <= experts, row pitch >= experts");
        return MX8_ERR_SIZE;
    }
    if (experts > MAX_EXPERTS || topk > MAX_TOPK || static_cast<long long>(tokens) * topk > 0x7FFF0000ll) {
        note_cuda_error(what, "at most 1024 experts, 32 choices and 2^31 - 2^16 (token, choice) pairs");
        return MX8_ERR_LIMIT;
    }
    return MX8_OK;
}

}  // namespace router
}  // namespace mx8

extern "C" size_t mx8_router_topk_workspace_bytes(int tokens, int experts) {
    using namespace mx8;
    if (tokens <= 0 || experts <= 0 || experts > router::MAX_EXPERTS) return 0;
    const int sms = sm_count();
    const int grid = sms > 0 ? router::grid_of(tokens, router::warps_of(router::vpl_of(experts))) : 0;
    return grid > 1 ? static_cast<size_t>(grid) * (8 * static_cast<size_t>(experts) + 4) : 0;
}

extern "C" int mx8_router_topk(const void* logits, int dtype, long long ld, int tokens, int experts, int topk, int normalize,
                               const void* token_mask, void* topk_idx, void* topk_weights, void* lse, void* counts, void* prob_sum,
                               void* num_valid, void* balance_loss, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace mx8;
    if (!logits || !topk_idx || !topk_weights || !lse || !counts || !prob_sum || !num_valid || !balance_loss) return MX8_ERR_ARG;
    int rc = router::check_shape("mx8_router_topk", dtype, ld, tokens, experts, topk);
    if (rc != MX8_OK) return rc;
    const int vpl = router::vpl_of(experts);
    const int grid = router::grid_of(tokens, router::warps_of(vpl));
    const size_t need = mx8_router_topk_workspace_bytes(tokens, experts);
    if (need > 0 && (!workspace || workspace_bytes < need)) {
        note_cuda_error("mx8_router_topk", "workspace smaller than mx8_router_topk_workspace_bytes(tokens, experts)");
        return MX8_ERR_LIMIT;
    }
    if (router::misaligned(logits, dtype == MX8_T_F32 ? 4 : 2) || router::misaligned(topk_idx, 4) || router::misaligned(topk_weights, 4) ||
        router::misaligned(lse, 4) || router::misaligned(counts, 4) || router::misaligned(prob_sum, 4) || router::misaligned(num_valid, 4) ||
        router::misaligned(balance_loss, 4) || router::misaligned(workspace, 4)) return MX8_ERR_ALIGN;
    if ((rc = check_device_sm100()) != MX8_OK) return rc;
    router::FwdParams p{};
    p.logits = logits;
    p.ld = ld;
    p.vec = router::vec_ok(logits, ld, experts, vpl, dtype == MX8_T_F32 ? 4 : 2);
    p.tokens = tokens;
    p.experts = experts;
    p.topk = topk;
    p.normalize = normalize != 0;
    p.mask = static_cast<const uint8_t*>(token_mask);
    p.idx = static_cast<int*>(topk_idx);
    p.weights = static_cast<float*>(topk_weights);
    p.lse = static_cast<float*>(lse);
    p.counts = static_cast<int*>(counts);
    p.prob_sum = static_cast<float*>(prob_sum);
    p.num_valid = static_cast<int*>(num_valid);
    p.loss = static_cast<float*>(balance_loss);
    if (grid > 1) {
        p.part_prob = static_cast<float*>(workspace);
        p.part_count = reinterpret_cast<int*>(p.part_prob + static_cast<size_t>(grid) * experts);
        p.part_valid = p.part_count + static_cast<size_t>(grid) * experts;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = dtype == MX8_T_F32 ? router::dispatch_fwd<float>(p, vpl, grid, st) : router::dispatch_fwd<uint16_t>(p, vpl, grid, st);
    if (e == cudaSuccess && grid > 1) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(router::FINISH);
        cfg.blockDim = dim3(1024);
        cfg.stream = st;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, router::router_finish_kernel, p, grid);
    }
    if (e != cudaSuccess) {
        note_cuda_error("router launch", cudaGetErrorString(e));
        return MX8_ERR_CUDA;
    }
    return MX8_OK;
}

extern "C" int mx8_router_topk_bwd(const void* logits, int dtype, long long ld, int tokens, int experts, int topk, int normalize,
                                   const void* topk_idx, const void* topk_weights, const void* lse, const void* counts,
                                   const void* num_valid, const void* d_topk_weights, const void* d_balance_loss, void* d_logits,
                                   void* stream) {
    using namespace mx8;
    if (!logits || !topk_idx || !topk_weights || !lse || !counts || !num_valid || !d_logits) return MX8_ERR_ARG;
    if (!d_topk_weights && !d_balance_loss) return MX8_ERR_ARG;
    int rc = router::check_shape("mx8_router_topk_bwd", dtype, ld, tokens, experts, topk);
    if (rc != MX8_OK) return rc;
    if (router::misaligned(logits, dtype == MX8_T_F32 ? 4 : 2) || router::misaligned(d_logits, dtype == MX8_T_F32 ? 4 : 2) ||
        router::misaligned(topk_idx, 4) || router::misaligned(topk_weights, 4) || router::misaligned(lse, 4) || router::misaligned(counts, 4) ||
        router::misaligned(num_valid, 4) || router::misaligned(d_topk_weights, 4) || router::misaligned(d_balance_loss, 4)) return MX8_ERR_ALIGN;
    if ((rc = check_device_sm100()) != MX8_OK) return rc;
    const int vpl = router::vpl_of(experts), esize = dtype == MX8_T_F32 ? 4 : 2;
    router::BwdParams p{};
    p.logits = logits;
    p.ld = ld;
    p.vec = router::vec_ok(logits, ld, experts, vpl, esize);
    p.tokens = tokens;
    p.experts = experts;
    p.topk = topk;
    p.normalize = normalize != 0;
    p.idx = static_cast<const int*>(topk_idx);
    p.weights = static_cast<const float*>(topk_weights);
    p.lse = static_cast<const float*>(lse);
    p.counts = static_cast<const int*>(counts);
    p.num_valid = static_cast<const int*>(num_valid);
    p.d_weights = static_cast<const float*>(d_topk_weights);
    p.d_loss = static_cast<const float*>(d_balance_loss);
    p.d_logits = d_logits;
    p.vec_out = router::vec_ok(d_logits, experts, experts, vpl, esize);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == MX8_T_F32 ? router::dispatch_bwd<float>(p, vpl, st) : router::dispatch_bwd<uint16_t>(p, vpl, st);
    if (e != cudaSuccess) {
        note_cuda_error("router backward launch", cudaGetErrorString(e));
        return MX8_ERR_CUDA;
    }
    return MX8_OK;
}

extern "C" int mx8_moe_bwd_topk_weights(const void* d_output, const void* combine_buffer, const void* topk_idx, void* d_topk_weights,
                                        int tokens, int hidden, int topk, void* stream) {
    using namespace mx8;
    if (!d_output || !combine_buffer || !d_topk_weights) return MX8_ERR_ARG;
    if (tokens <= 0 || hidden <= 0 || topk <= 0) {
        note_cuda_error("mx8_moe_bwd_topk_weights", "tokens, hidden and topk positive");
        return MX8_ERR_SIZE;
    }
    if (router::misaligned(d_output, 2) || router::misaligned(combine_buffer, 2) || router::misaligned(topk_idx, 4) ||
        router::misaligned(d_topk_weights, 4)) return MX8_ERR_ALIGN;
    if (topk > 65535 * router::WG_K || hidden > 0x7FFFF000) {                    // a thread's next column has to fit an int
        note_cuda_error("mx8_moe_bwd_topk_weights", "more than 524280 choices per token or 2^31 - 4096 columns");
        return MX8_ERR_LIMIT;
    }
    int rc = check_device_sm100();
    if (rc != MX8_OK) return rc;
    const dim3 grid(static_cast<unsigned>(tokens), static_cast<unsigned>((topk + router::WG_K - 1) / router::WG_K));
    const auto* g = static_cast<const uint16_t*>(d_output);
    const auto* c = static_cast<const uint16_t*>(combine_buffer);
    const auto* i = static_cast<const int*>(topk_idx);
    auto* w = static_cast<float*>(d_topk_weights);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (hidden % 8 == 0 && aligned16(d_output) && aligned16(combine_buffer))
        router::topk_weights_grad_kernel<true><<<grid, router::WG_THREADS, 0, st>>>(g, c, i, w, hidden, topk);
    else
        router::topk_weights_grad_kernel<false><<<grid, router::WG_THREADS, 0, st>>>(g, c, i, w, hidden, topk);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        note_cuda_error("routing-weight gradient launch", cudaGetErrorString(e));
        return MX8_ERR_CUDA;
    }
    return MX8_OK;
}
