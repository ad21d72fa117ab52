// Router of a mixture of experts with the losses that train it, forward and backward.
//
//     p = softmax(x),  lse = log sum exp x,  experts = the k largest x (equal ones: the lower index first),
//     weights = p_j, for k > 1 divided by their sum,  counts[e] = tokens that chose e,
//     balance = E sum_e f_e P_e,  f_e = share of the kept tokens' choices that went to e,  P_e = mean of p_e over the kept tokens,
//     z = mean of lse^2 over the kept tokens.
// Backward, with f constant: dp = [chosen] d weights + g_balance E f / N [kept],
//     dx = p (dp - sum dp p) + g_z 2 lse p / N [kept].
//
// A token is handled by LANES neighbouring lanes, each with C groups of eight experts, so that a row of up to 512 experts is one
// or two 16-byte loads a lane and stays in registers; the column sums of p stay in registers over all tokens of a thread.  Every
// sum is taken in a fixed order (warp, block, then blocks in order), so results repeat bit by bit.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>
#include <stdint.h>

#include "launch.cuh"
#include "neox_b200.h"

namespace {

constexpr int THREADS = 256;
constexpr int MAX_K = 8;
constexpr unsigned ALL = 0xffffffffu;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void put(float& d, float v) { d = v; }
__device__ __forceinline__ void put(__nv_bfloat16& d, float v) { d = __float2bfloat16(v); }
__device__ __forceinline__ void put(__half& d, float v) { d = __float2half(v); }

// Eight neighbouring elements of a row as they lie in memory, -inf where the row has ended; `aligned`: rows start on 16 bytes and
// have no part of eight left over.
template <typename T> struct Eight {
    static constexpr int WORDS = sizeof(T) / 2;                 // of 16 bytes
    uint4 w[WORDS];
    __device__ __forceinline__ void load(const T* p, int left, bool aligned) {
        if (aligned && left > 0) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
            __align__(16) T t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                put(t[i], -INFINITY);
                if (i < left) t[i] = p[i];
            }
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = reinterpret_cast<const uint4*>(t)[i];
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        __align__(16) T t[8];
#pragma unroll
        for (int i = 0; i < WORDS; ++i) reinterpret_cast<uint4*>(t)[i] = w[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f(t[i]);
    }
};
template <typename T> __device__ __forceinline__ void store_8(T* p, int left, bool aligned, const float (&v)[8]) {
    if (aligned) {
        __align__(16) T t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) put(t[i], v[i]);
        const uint4* s = reinterpret_cast<const uint4*>(t);
        if (left > 0) {
            reinterpret_cast<uint4*>(p)[0] = s[0];
            if constexpr (sizeof(T) == 4) reinterpret_cast<uint4*>(p)[1] = s[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) put(p[i], v[i]);
    }
}

template <int LANES> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(ALL, v, o);
    return v;
}

// Order of the choice in one number: the bits of the value as a 32-bit float, turned so that they grow with it, -0 as 0 and NaN
// above all, then the lower index.  A 16-bit value leaves at least 13 of its 32 bits free for the index.
__device__ __forceinline__ uint32_t rising(float v) {
    float w;
    asm("add.rn.f32 %0, %1, 0f00000000;" : "=f"(w) : "f"(v));   // -0 becomes 0, NaN the one of sign 0; subnormal numbers stay
    const uint32_t u = __float_as_uint(w);
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unrisen(uint32_t t) {
    return __uint_as_float(t & 0x80000000u ? t ^ 0x80000000u : ~t);
}
template <typename T> struct Key {
    using type = uint32_t;
    static constexpr uint32_t FREE = 0x1fff;
    static __device__ __forceinline__ uint32_t of(float v, int e) { return (rising(v) & ~FREE) | (FREE - e); }
    static __device__ __forceinline__ int expert(uint32_t k) { return (int)(FREE - (k & FREE)); }
    // of a negative value the turned bits are ones where the value's are zeros
    static __device__ __forceinline__ float value(uint32_t k) { return unrisen(k & 0x80000000u ? k & ~FREE : k | FREE); }
};
template <> struct Key<float> {
    using type = unsigned long long;
    static __device__ __forceinline__ unsigned long long of(float v, int e) {
        return (unsigned long long)rising(v) << 32 | (uint32_t)(0xffff - e);
    }
    static __device__ __forceinline__ int expert(unsigned long long k) { return 0xffff - (int)(k & 0xffffu); }
    static __device__ __forceinline__ float value(unsigned long long k) { return unrisen((uint32_t)(k >> 32)); }
};

// Eight numbers in falling order: Batcher's odd-even merge of sorted halves, and the merge of a bitonic sequence.
template <typename K> __device__ __forceinline__ void order(K& a, K& b) {
    const K low = min(a, b);
    a = max(a, b);
    b = low;
}
template <typename K> __device__ __forceinline__ void sort_8(K (&v)[8]) {
    order(v[0], v[1]); order(v[2], v[3]); order(v[4], v[5]); order(v[6], v[7]);
    order(v[0], v[2]); order(v[1], v[3]); order(v[4], v[6]); order(v[5], v[7]);
    order(v[1], v[2]); order(v[5], v[6]);
    order(v[0], v[4]); order(v[1], v[5]); order(v[2], v[6]); order(v[3], v[7]);
    order(v[2], v[4]); order(v[3], v[5]);
    order(v[1], v[2]); order(v[3], v[4]); order(v[5], v[6]);
}
template <typename K> __device__ __forceinline__ void merge_8(K (&v)[8]) {
    order(v[0], v[4]); order(v[1], v[5]); order(v[2], v[6]); order(v[3], v[7]);
    order(v[0], v[2]); order(v[1], v[3]); order(v[4], v[6]); order(v[5], v[7]);
    order(v[0], v[1]); order(v[2], v[3]); order(v[4], v[5]); order(v[6], v[7]);
}

struct ForwardArgs {
    const void* x;
    long long stride;
    const uint8_t* kept;           // [tokens] or none
    float* weights;
    long long* experts;
    float4* row;                   // per token: maximum, 1 / sum, mass of the chosen, lse
    float* sums;                   // [blocks, E]: p over the kept tokens
    int* chosen;                   // [blocks, 2, E]: choices of all tokens, of the kept ones
    double* z;                     // [blocks]
    int* ticket;
    int tokens, E, k, aligned;
};

// Many tokens: one block an SM, as large as registers allow, since few threads read again what the blocks leave (32768 tokens of
// 128 experts, both kernels: 24.6 us with four blocks of 256 threads an SM, 18.3 us so).  Few: small blocks (16 tokens of 64
// experts: 6.4 against 8.1 us).
template <typename T, int C> constexpr int LARGE = sizeof(T) == 2 && C == 1 ? 1024 : 512;

// A lane sorts its eight candidates once (19 exchanges), and a choice is the largest head among the lanes: log LANES shuffles and a
// shift of the winner's list.  That, not the bytes, bounds many tokens: 32768 of 128 experts, eight choices, 12.8 us for 12 MB
// (1.8 us); with every choice a search over all candidates the two forward kernels took 33.4 us, now 16.9.
template <typename T, int LANES, int C, int THREADS>
__global__ void __launch_bounds__(THREADS) router_kernel(const ForwardArgs a) {
    constexpr int GROUPS = THREADS / LANES, WARPS = THREADS / 32, SLOTS = LANES * C * 8;
    using K = Key<T>;
    using KeyT = typename K::type;
    __shared__ int hits[2][SLOTS];
    __shared__ float cols[WARPS][SLOTS];
    __shared__ double zs[WARPS];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0;
    for (int e = threadIdx.x; e < SLOTS; e += THREADS) hits[0][e] = hits[1][e] = 0;
    __syncthreads();
    constexpr int MINE = (MAX_K + LANES - 1) / LANES;           // choices a lane writes: every LANES-th
    float col[C][8] = {};
    float z = 0.f;
    Eight<T> next[C];
    bool next_kept = false;
    auto fetch = [&](int first) {
        const int t = min(first + group, a.tokens - 1);
        const T* x = reinterpret_cast<const T*>(a.x) + (long long)t * a.stride;
#pragma unroll
        for (int c = 0; c < C; ++c) next[c].load(x + (c * LANES + lane) * 8, a.E - (c * LANES + lane) * 8, a.aligned);
        next_kept = first + group < a.tokens && (!a.kept || a.kept[t]);
    };
    // whole warps walk together: a group past the last token does the last one's work again and leaves nothing
    if (blockIdx.x * GROUPS < a.tokens) fetch(blockIdx.x * GROUPS);
    for (int first = blockIdx.x * GROUPS; first < a.tokens; first += gridDim.x * GROUPS) {
        const bool here = first + group < a.tokens, kept = next_kept;
        const int t = here ? first + group : a.tokens - 1;
        float v[C][8];
        KeyT key[C][8];
#pragma unroll
        for (int c = 0; c < C; ++c) next[c].get(v[c]);
        if (first + (int)gridDim.x * GROUPS < a.tokens) fetch(first + gridDim.x * GROUPS);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e0 = (c * LANES + lane) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) key[c][i] = e0 + i < a.E ? K::of(v[c][i], e0 + i) : 0;
            sort_8(key[c]);
        }
        if constexpr (C == 2) {                                 // the eight largest of both
#pragma unroll
            for (int i = 0; i < 8; ++i) key[0][i] = max(key[0][i], key[1][7 - i]);
            merge_8(key[0]);
        }
        KeyT mine[MINE] = {}, top = 0;
#pragma unroll
        for (int j = 0; j < MAX_K; ++j) {
            if (j >= a.k) break;
            KeyT best = key[0][0];                              // the lanes' lists are in order: only their heads compete
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) {
                const KeyT other = __shfl_xor_sync(ALL, best, o);
                best = max(best, other);
            }
            if (j == 0) top = best;
            if (j % LANES == lane) mine[j / LANES] = best;
            const bool won = key[0][0] == best;
#pragma unroll
            for (int i = 0; i + 1 < MAX_K - j; ++i) key[0][i] = won ? key[0][i + 1] : key[0][i];
        }
        const float m = fmaxf(K::value(top), -FLT_MAX);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[c][i] = __expf(v[c][i] - m);
                sum += v[c][i];
            }
        float picked[MINE], mass = 0.f;
#pragma unroll
        for (int q = 0; q < MINE; ++q) {
            picked[q] = q * LANES + lane < a.k ? __expf(K::value(mine[q]) - m) : 0.f;
            mass += picked[q];
        }
        sum = group_sum<LANES>(sum);
        mass = group_sum<LANES>(mass);
        const float inv = __frcp_rn(sum);
        if (kept)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) col[c][i] += v[c][i] * inv;
        const float norm = a.k > 1 ? __frcp_rn(mass) : inv;
#pragma unroll
        for (int q = 0; q < MINE; ++q) {
            const int j = q * LANES + lane;
            if (here && j < a.k) {
                const int e = K::expert(mine[q]);
                a.weights[(long long)t * a.k + j] = picked[q] * norm;
                a.experts[(long long)t * a.k + j] = e;
                atomicAdd(&hits[0][e], 1);
                if (kept) atomicAdd(&hits[1][e], 1);
            }
        }
        if (here && lane == 0) {
            const float lse = m + __logf(sum);
            a.row[t] = make_float4(m, inv, mass * inv, lse);
            if (kept) z += lse * lse;
        }
    }
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float s = col[c][i];
#pragma unroll
            for (int o = 16; o >= LANES; o >>= 1) s += __shfl_xor_sync(ALL, s, o);
            if ((threadIdx.x & 31) < LANES) cols[warp][(c * LANES + lane) * 8 + i] = s;
        }
    double zw = z;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) zw += __shfl_xor_sync(ALL, zw, o);
    if ((threadIdx.x & 31) == 0) zs[warp] = zw;
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += THREADS) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) s += cols[w][e];
        a.sums[(long long)blockIdx.x * a.E + e] = s;
        a.chosen[(2ll * blockIdx.x) * a.E + e] = hits[0][e];
        a.chosen[(2ll * blockIdx.x + 1) * a.E + e] = hits[1][e];
    }
    if (threadIdx.x == 0) {
        double s = 0.0;
        for (int w = 0; w < WARPS; ++w) s += zs[w];
        a.z[blockIdx.x] = s;
    }
    launch::let_successor_start();
}

struct LossArgs {
    const float* sums;
    const int* chosen;
    const double* z;
    int* ticket;
    double* part;                  // [gridDim, 2]: sum of count * column sum, sum of counts
    long long* counts;
    float* load;                   // [E + 1]: choices of the kept tokens; then 1 / kept tokens
    float* balance;
    float* z_loss;
    int blocks, E, k;
};

// Joins what the router's blocks left: 32 experts a block, 32 threads an expert, and the last block forms the losses.  Latency:
// 4 to 6 us behind the router, for 8 experts as for 128.
__global__ void __launch_bounds__(1024) router_loss_kernel(const LossArgs a) {
    __shared__ double p[32][33];
    __shared__ int n_all[32][33], n_kept[32][33];
    __shared__ double dots[32];
    __shared__ int n_sum[32];
    __shared__ int last;
    launch::wait_for_predecessor();
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, e = blockIdx.x * 32 + x;
    double s = 0.0;
    int all = 0, kept = 0;
    if (e < a.E)
#pragma unroll 5
        for (int b = y; b < a.blocks; b += 32) {
            s += a.sums[(long long)b * a.E + e];
            all += a.chosen[(2ll * b) * a.E + e];
            kept += a.chosen[(2ll * b + 1) * a.E + e];
        }
    p[x][y] = s;
    n_all[x][y] = all;
    n_kept[x][y] = kept;
    __syncthreads();
    s = p[y][x];                                                // a warp an expert now
    all = __reduce_add_sync(ALL, n_all[y][x]);
    kept = __reduce_add_sync(ALL, n_kept[y][x]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(ALL, s, o);
    const int mine = blockIdx.x * 32 + y;
    if (x == 0) {
        if (mine < a.E) {
            a.counts[mine] = all;
            a.load[mine] = (float)kept;
        }
        dots[y] = s * kept;
        n_sum[y] = kept;
    }
    __syncthreads();
    if (y == 0) {
        double dot = dots[x], n = n_sum[x];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            dot += __shfl_xor_sync(ALL, dot, o);
            n += __shfl_xor_sync(ALL, n, o);
        }
        if (x == 0) {
            a.part[2 * blockIdx.x] = dot;
            a.part[2 * blockIdx.x + 1] = n;
            __threadfence();
            last = gridDim.x == 1 || atomicAdd(a.ticket, 1) == (int)gridDim.x - 1;
            __threadfence();
        }
    }
    __syncthreads();
    if (!last || y != 0) return;
    double dot = 0.0, n = 0.0, z = 0.0;
    if (x < (int)gridDim.x) {
        dot = __ldcg(a.part + 2 * x);
        n = __ldcg(a.part + 2 * x + 1);
    }
    for (int b = x; b < a.blocks; b += 32) z += a.z[b];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        dot += __shfl_xor_sync(ALL, dot, o);
        n += __shfl_xor_sync(ALL, n, o);
        z += __shfl_xor_sync(ALL, z, o);
    }
    if (x == 0) {
        const double tokens = n / a.k;
        *a.balance = n > 0.0 ? (float)(a.E * dot / (n * tokens)) : 0.f;
        *a.z_loss = n > 0.0 ? (float)(z / tokens) : 0.f;
        a.load[a.E] = n > 0.0 ? (float)(1.0 / tokens) : 0.f;
    }
}

struct BackwardArgs {
    const void* x;
    long long stride;
    const uint8_t* kept;
    const float* weights;
    const long long* experts;
    const float4* row;
    const float* load;
    const float* g_weights;        // [tokens, k] or none
    const float* g_balance;        // or none
    const float* g_z;              // or none
    void* dx;                      // [tokens, E]
    int tokens, E, k, aligned;
};

// One pass: a token's logits give p again from its maximum and sum.  The loads' latency bounds it: 32768 tokens of 128 experts 7.6 us
// for 21 MB (3.3 us at the rate of a copy), 16384 of 512 experts 14.2 us for 36 MB (5.5 us).
template <typename T, int LANES, int C>
__global__ void __launch_bounds__(THREADS) router_grad_kernel(const BackwardArgs a) {
    constexpr int GROUPS = THREADS / LANES, MINE = (MAX_K + LANES - 1) / LANES;
    __shared__ __align__(16) float toward[GROUPS][LANES * C * 8];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const float per_token = a.load[a.E];
    // E f_e / N g = E count_e / (N k) / N g
    const float gb = a.g_balance ? *a.g_balance * (float)a.E * per_token * per_token / (float)a.k : 0.f;
    const float gz = a.g_z ? 2.f * *a.g_z * per_token : 0.f;
    float pull[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = (c * LANES + lane) * 8 + i;
            pull[c][i] = a.g_balance && e < a.E ? gb * a.load[e] : 0.f;
        }
    for (int first = blockIdx.x * GROUPS; first < a.tokens; first += gridDim.x * GROUPS) {
        const bool here = first + group < a.tokens;
        const int t = here ? first + group : a.tokens - 1;
        const T* x = reinterpret_cast<const T*>(a.x) + (long long)t * a.stride;
        const float4 r = a.row[t];
        const bool kept = !a.kept || a.kept[t];
        float p[C][8], dp[C][8];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e0 = (c * LANES + lane) * 8;
            Eight<T> raw;
            raw.load(x + e0, a.E - e0, a.aligned);
            raw.get(p[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[c][i] = __expf(p[c][i] - r.x) * r.y;
                dp[c][i] = kept ? pull[c][i] : 0.f;
            }
        }
        if (a.g_weights) {
            // a lane forms the gradient at every LANES-th choice and leaves it where the expert's lane picks it up
            const long long at = (long long)t * a.k;
            float g[MINE], dot = 0.f;
#pragma unroll
            for (int q = 0; q < MINE; ++q) {
                const int j = q * LANES + lane;
                g[q] = j < a.k ? a.g_weights[at + j] : 0.f;
                if (a.k > 1 && j < a.k) dot += g[q] * a.weights[at + j];
            }
            dot = group_sum<LANES>(dot);
            const float inv = a.k > 1 ? __frcp_rn(r.z) : 1.f;
            float4* clear = reinterpret_cast<float4*>(toward[group]);
#pragma unroll
            for (int c = 0; c < 2 * C; ++c) clear[c * LANES + lane] = make_float4(0.f, 0.f, 0.f, 0.f);
            __syncwarp();
#pragma unroll
            for (int q = 0; q < MINE; ++q) {
                const int j = q * LANES + lane;
                if (j < a.k) toward[group][(int)a.experts[at + j]] = (g[q] - dot) * inv;
            }
            __syncwarp();
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float4* from = reinterpret_cast<const float4*>(&toward[group][(c * LANES + lane) * 8]);
                const float4 lo = from[0], hi = from[1];
                const float add[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) dp[c][i] += add[i];
            }
            __syncwarp();
        }
        float inner = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) inner += dp[c][i] * p[c][i];
        inner = group_sum<LANES>(inner) - (kept ? gz * r.w : 0.f);
        if (!here) continue;
        T* dx = reinterpret_cast<T*>(a.dx) + (long long)t * a.E;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e0 = (c * LANES + lane) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) p[c][i] *= dp[c][i] - inner;
            store_8(dx + e0, a.E - e0, a.E % 8 == 0, p[c]);
        }
    }
}

int lanes_for(int E) {
    int l = 1;
    while (l < 32 && l * 8 < E) l *= 2;
    return l;
}

struct RouterPlan {
    bool large;
    int blocks;
    RouterPlan(long long tokens, int E, int dtype) {
        const int lanes = lanes_for(E);
        const long long sms = neox_sm_count(), small_groups = THREADS / lanes;
        const long long large_groups = (dtype != 1 && E <= 256 ? LARGE<__half, 1> : LARGE<__half, 2>) / lanes;
        large = (tokens + small_groups - 1) / small_groups > sms;
        const long long groups = large ? large_groups : small_groups, need = (tokens + groups - 1) / groups;
        blocks = (int)(need < 1 ? 1 : need < sms ? need : sms);
    }
};

#define FOR_TYPE(dtype, CALL)                                  \
    do {                                                       \
        if (dtype == 0) { using T = __nv_bfloat16; CALL; }     \
        else if (dtype == 1) { using T = float; CALL; }        \
        else { using T = __half; CALL; }                       \
    } while (0)

#define FOR_LANES(E, CALL)                                                     \
    do {                                                                       \
        if (E > 256) { constexpr int L = 32, C = 2; CALL; }                    \
        else if (lanes_for(E) == 32) { constexpr int L = 32, C = 1; CALL; }    \
        else if (lanes_for(E) == 16) { constexpr int L = 16, C = 1; CALL; }    \
        else if (lanes_for(E) == 8) { constexpr int L = 8, C = 1; CALL; }      \
        else if (lanes_for(E) == 4) { constexpr int L = 4, C = 1; CALL; }      \
        else if (lanes_for(E) == 2) { constexpr int L = 2, C = 1; CALL; }      \
        else { constexpr int L = 1, C = 1; CALL; }                             \
    } while (0)

bool rows_aligned(const void* p, long long stride, int E, int dtype) {
    const long long size = dtype == 1 ? 4 : 2;
    return ((uintptr_t)p & 15) == 0 && stride * size % 16 == 0 && E % 8 == 0;
}

int launched() { return cudaGetLastError() == cudaSuccess ? 0 : NEOX_ERR_LAUNCH; }

}  // namespace

extern "C" {

// Blocks whose sums the forward leaves: `scratch` holds this * (E * 12 + 8) bytes, then 16 * 17 and 16 more.
int neox_router_blocks(long long tokens, int E, int dtype) { return RouterPlan(tokens, E, dtype).blocks; }

int neox_balanced_router(const void* x, long long stride, const void* kept, int tokens, int E, int k, int dtype, float* weights,
                         long long* experts, void* row, long long* counts, float* load, float* balance, float* z_loss, void* scratch,
                         void* stream) {
    if (tokens < 0 || tokens >= 1 << 30 || E < 1 || E > 512 || k < 1 || k > MAX_K || k > E) return NEOX_ERR_SHAPE;
    const RouterPlan plan(tokens, E, dtype);
    const int blocks = plan.blocks;
    double* z = (double*)scratch;
    double* part = z + blocks;                                  // 16 blocks of 32 experts at most
    int* ticket = (int*)(part + 2 * 17);
    float* sums = (float*)(ticket + 4);
    int* chosen = (int*)(sums + (long long)blocks * E);
    const ForwardArgs f = {x, stride, (const uint8_t*)kept, weights, experts, (float4*)row, sums, chosen, z, ticket, tokens, E, k,
                           rows_aligned(x, stride, E, dtype)};
    const LossArgs l = {sums, chosen, z, ticket, part, counts, load, balance, z_loss, blocks, E, k};
    cudaStream_t st = (cudaStream_t)stream;
    if (plan.large) FOR_TYPE(dtype, FOR_LANES(E, (router_kernel<T, L, C, LARGE<T, C>><<<blocks, LARGE<T, C>, 0, st>>>(f))));
    else FOR_TYPE(dtype, FOR_LANES(E, (router_kernel<T, L, C, THREADS><<<blocks, THREADS, 0, st>>>(f))));
    if (launched() != 0) return NEOX_ERR_LAUNCH;
    return launch::overlapped(router_loss_kernel, dim3((E + 31) / 32), dim3(1024), 1, st, l);
}

int neox_balanced_router_grad(const void* x, long long stride, const void* kept, int tokens, int E, int k, int dtype,
                              const float* weights, const long long* experts, const void* row, const float* load,
                              const float* g_weights, const float* g_balance, const float* g_z, void* dx, void* stream) {
    if (tokens < 0 || tokens >= 1 << 30 || E < 1 || E > 512 || k < 1 || k > MAX_K || k > E) return NEOX_ERR_SHAPE;
    if (tokens == 0) return 0;
    const BackwardArgs b = {x, stride, (const uint8_t*)kept, weights, experts, (const float4*)row, load, g_weights, g_balance, g_z,
                            dx, tokens, E, k, rows_aligned(x, stride, E, dtype)};
    const long long groups = THREADS / lanes_for(E), need = (tokens + groups - 1) / groups, most = 8ll * neox_sm_count();
    const int blocks = (int)(need < most ? need : most);
    cudaStream_t st = (cudaStream_t)stream;
    FOR_TYPE(dtype, FOR_LANES(E, (router_grad_kernel<T, L, C><<<blocks, THREADS, 0, st>>>(b))));
    return launched();
}

}  // extern "C"
