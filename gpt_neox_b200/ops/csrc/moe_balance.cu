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

// Eight neighbouring elements of a row; `aligned`: rows start on 16 bytes and have no part of eight left over.
template <typename T> __device__ __forceinline__ void load_8(const T* p, int left, bool aligned, float (&v)[8]) {
    if (aligned) {
        __align__(16) T t[8];
        const uint4* q = reinterpret_cast<const uint4*>(p);
        uint4* d = reinterpret_cast<uint4*>(t);
        if (left > 0) {
            d[0] = __ldg(q);
            if constexpr (sizeof(T) == 4) d[1] = __ldg(q + 1);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_f(t[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = -INFINITY;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? to_f(p[i]) : -INFINITY;
    }
}
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

// Order of the choice in one number: the value's bits in an order that grows with the value, -0 as 0 and NaN above all, then
// the lower index.  Sixteen-bit values leave room for both in 32 bits.
template <typename T> struct Key {
    using type = uint32_t;
    static __device__ __forceinline__ uint32_t of(float v, int e) {
        T t;
        put(t, v);                                              // exact: v was one
        uint32_t b = *reinterpret_cast<const uint16_t*>(&t);
        if (b == 0x8000u) b = 0;
        if (v != v) b = 0x7fffu;
        b = b & 0x8000u ? 0xffffu - b : b | 0x8000u;
        return b << 16 | (uint32_t)(0xffff - e);
    }
    static __device__ __forceinline__ int expert(uint32_t k) { return 0xffff - (int)(k & 0xffffu); }
    static __device__ __forceinline__ float value(uint32_t k) {
        uint32_t b = k >> 16;
        const uint16_t s = (uint16_t)(b & 0x8000u ? b & 0x7fffu : 0xffffu - b);
        return to_f(*reinterpret_cast<const T*>(&s));
    }
};
template <> struct Key<float> {
    using type = unsigned long long;
    static __device__ __forceinline__ unsigned long long of(float v, int e) {
        uint32_t b = __float_as_uint(v);
        if (b == 0x80000000u) b = 0;
        if (v != v) b = 0x7fffffffu;
        b = b & 0x80000000u ? ~b : b | 0x80000000u;
        return (unsigned long long)b << 32 | (uint32_t)(0xffff - e);
    }
    static __device__ __forceinline__ int expert(unsigned long long k) { return 0xffff - (int)(k & 0xffffu); }
    static __device__ __forceinline__ float value(unsigned long long k) {
        const uint32_t b = (uint32_t)(k >> 32);
        return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
    }
};

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

template <typename T, int LANES, int C>
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
    float col[C][8] = {};
    double z = 0.0;
    // whole warps walk together: a group past the last token does the last one's work again and leaves nothing
    for (int first = blockIdx.x * GROUPS; first < a.tokens; first += gridDim.x * GROUPS) {
        const bool here = first + group < a.tokens;
        const int t = here ? first + group : a.tokens - 1;
        const T* x = reinterpret_cast<const T*>(a.x) + (long long)t * a.stride;
        float v[C][8];
        KeyT key[C][8];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e0 = (c * LANES + lane) * 8;
            load_8(x + e0, a.E - e0, a.aligned, v[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) key[c][i] = e0 + i < a.E ? K::of(v[c][i], e0 + i) : 0;
        }
        const bool kept = here && (!a.kept || a.kept[t]);
        KeyT picked[MAX_K];
#pragma unroll
        for (int j = 0; j < MAX_K; ++j) {
            if (j >= a.k) break;
            KeyT best = 0;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) best = key[c][i] > best ? key[c][i] : best;
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) {
                const KeyT other = __shfl_xor_sync(ALL, best, o);
                best = other > best ? other : best;
            }
            picked[j] = best;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (key[c][i] == best) key[c][i] = 0;
        }
        const float m = fmaxf(K::value(picked[0]), -FLT_MAX);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[c][i] = __expf(v[c][i] - m);
                sum += v[c][i];
            }
        sum = group_sum<LANES>(sum);
        const float inv = __frcp_rn(sum);
        if (kept)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) col[c][i] += v[c][i] * inv;
        float mass = 0.f;
#pragma unroll
        for (int j = 0; j < MAX_K; ++j)
            if (j < a.k) mass += __expf(K::value(picked[j]) - m);
        const float norm = a.k > 1 ? __frcp_rn(mass) : inv;
#pragma unroll
        for (int j = 0; j < MAX_K; ++j)
            if (here && j < a.k && j % LANES == lane) {
                const int e = K::expert(picked[j]);
                a.weights[(long long)t * a.k + j] = __expf(K::value(picked[j]) - m) * norm;
                a.experts[(long long)t * a.k + j] = e;
                atomicAdd(&hits[0][e], 1);
                if (kept) atomicAdd(&hits[1][e], 1);
            }
        if (here && lane == 0) {
            const double lse = (double)m + log((double)sum);
            a.row[t] = make_float4(m, inv, mass * inv, (float)lse);
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
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(ALL, z, o);
    if ((threadIdx.x & 31) == 0) zs[warp] = z;
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

// Joins what the router's blocks left: 32 experts a block, 32 threads an expert, and the last block forms the losses.
__global__ void __launch_bounds__(1024) router_loss_kernel(const LossArgs a) {
    __shared__ double p[32][33];
    __shared__ int n_all[32][33], n_kept[32][33];
    __shared__ int last;
    launch::wait_for_predecessor();
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, e = blockIdx.x * 32 + x;
    double s = 0.0;
    int all = 0, kept = 0;
    if (e < a.E)
        for (int b = y; b < a.blocks; b += 32) {
            s += a.sums[(long long)b * a.E + e];
            all += a.chosen[(2ll * b) * a.E + e];
            kept += a.chosen[(2ll * b + 1) * a.E + e];
        }
    p[x][y] = s;
    n_all[x][y] = all;
    n_kept[x][y] = kept;
    __syncthreads();
    if (y == 0) {
        for (int w = 1; w < 32; ++w) {
            s += p[x][w];
            all += n_all[x][w];
            kept += n_kept[x][w];
        }
        if (e < a.E) {
            a.counts[e] = all;
            a.load[e] = (float)kept;
        }
        double dot = s * kept, n = kept;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            dot += __shfl_xor_sync(ALL, dot, o);
            n += __shfl_xor_sync(ALL, n, o);
        }
        if (x == 0) {
            a.part[2 * blockIdx.x] = dot;
            a.part[2 * blockIdx.x + 1] = n;
            __threadfence();
            last = atomicAdd(a.ticket, 1) == (int)gridDim.x - 1;
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

template <typename T, int LANES, int C>
__global__ void __launch_bounds__(THREADS) router_grad_kernel(const BackwardArgs a) {
    constexpr int GROUPS = THREADS / LANES;
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
            load_8(x + e0, a.E - e0, a.aligned, p[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[c][i] = __expf(p[c][i] - r.x) * r.y;
                dp[c][i] = kept ? pull[c][i] : 0.f;
            }
        }
        if (a.g_weights) {
            const float* gw = a.g_weights + (long long)t * a.k;
            float dot = 0.f, inv = 1.f;
            if (a.k > 1) {
                const float* w = a.weights + (long long)t * a.k;
                for (int j = 0; j < a.k; ++j) dot += gw[j] * w[j];
                inv = __frcp_rn(r.z);
            }
            for (int j = 0; j < a.k; ++j) {
                const int e = (int)a.experts[(long long)t * a.k + j];
                const float g = (gw[j] - dot) * inv;
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (e == (c * LANES + lane) * 8 + i) dp[c][i] += g;
            }
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

// Blocks of the forward: four an SM keep the loads of a token's rows in flight; a block walks over several tokens once there
// are more, so that what it leaves to join stays small.
int router_blocks(long long tokens, int E) {
    const long long groups = THREADS / lanes_for(E);
    const long long need = (tokens + groups - 1) / groups, most = 4ll * neox_sm_count();
    return (int)(need < 1 ? 1 : need < most ? need : most);
}

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
int neox_router_blocks(long long tokens, int E) { return router_blocks(tokens, E); }

int neox_balanced_router(const void* x, long long stride, const void* kept, int tokens, int E, int k, int dtype, float* weights,
                         long long* experts, void* row, long long* counts, float* load, float* balance, float* z_loss, void* scratch,
                         void* stream) {
    if (tokens < 0 || E < 1 || E > 512 || k < 1 || k > MAX_K || k > E) return NEOX_ERR_SHAPE;
    const int blocks = router_blocks(tokens, E);
    double* z = (double*)scratch;
    double* part = z + blocks;                                  // 16 blocks of 32 experts at most
    int* ticket = (int*)(part + 2 * 17);
    float* sums = (float*)(ticket + 4);
    int* chosen = (int*)(sums + (long long)blocks * E);
    const ForwardArgs f = {x, stride, (const uint8_t*)kept, weights, experts, (float4*)row, sums, chosen, z, ticket, tokens, E, k,
                           rows_aligned(x, stride, E, dtype)};
    const LossArgs l = {sums, chosen, z, ticket, part, counts, load, balance, z_loss, blocks, E, k};
    cudaStream_t st = (cudaStream_t)stream;
    FOR_TYPE(dtype, FOR_LANES(E, (router_kernel<T, L, C><<<blocks, THREADS, 0, st>>>(f))));
    if (launched() != 0) return NEOX_ERR_LAUNCH;
    return launch::overlapped(router_loss_kernel, dim3((E + 31) / 32), dim3(1024), 1, st, l);
}

int neox_balanced_router_grad(const void* x, long long stride, const void* kept, int tokens, int E, int k, int dtype,
                              const float* weights, const long long* experts, const void* row, const float* load,
                              const float* g_weights, const float* g_balance, const float* g_z, void* dx, void* stream) {
    if (tokens < 0 || E < 1 || E > 512 || k < 1 || k > MAX_K || k > E) return NEOX_ERR_SHAPE;
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
