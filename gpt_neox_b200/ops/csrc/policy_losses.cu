// Losses of post-training on the logits of a language model: a preference loss over pairs of sequences and a clipped policy
// loss with a KL term, forward and backward.
//
// Rows are the tokens of a [n, s, vocab] tensor, row (i, j) at i * stride_n + j * stride_s, the vocabulary contiguous.  With
// lse(x) = max + log sum exp(x - max), the log-probability of label y is x[y] - lse(x), and every loss here is a function of
// the log-probabilities of the rows whose mask is not zero.  Its gradient is
//     dx[c] = a ([c == y] - p[c]) + b p[c] ((log p[c] - log q[c]) - KL),          p = softmax(x), q = softmax(reference),
// with one a (and, for the KL over the whole vocabulary, one b) a row.
//
// Three kernels.  `stats_kernel` streams the kept rows once and leaves (max, sum of exponentials) of every chunk of a row;
// `preference_kernel` / `policy_kernel` join them, one thread a row, in 64 bits from the sums on, and the last block to finish
// forms the loss and what the backward multiplies; `grad_kernel` streams the rows a second time and writes the gradient, zeros
// where the coefficient is zero, without reading.  The second pass over the logits cannot be saved for a preference loss: a
// pair's coefficient depends on all of its rows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>
#include <stdint.h>

#include "neox_b200.h"

namespace {

constexpr int THREADS = 256;

template <typename T> struct Elem;
template <> struct Elem<float> {
    static constexpr int PER_16 = 4;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Elem<__nv_bfloat16> {
    static constexpr int PER_16 = 8;
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16(v); }
};
template <> struct Elem<__half> {
    static constexpr int PER_16 = 8;
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half(v); }
};

__device__ __forceinline__ float2 two(uint32_t w, __nv_bfloat16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float2 two(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t pack(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T> __device__ __forceinline__ void unpack(const uint4& u, float (&v)[Elem<T>::PER_16]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (Elem<T>::PER_16 == 4) {
            v[i] = __uint_as_float(w[i]);
        } else {
            const float2 f = two(w[i], T());
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
template <typename T> __device__ __forceinline__ uint4 repack(const float (&v)[Elem<T>::PER_16]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (Elem<T>::PER_16 == 4) w[i] = __float_as_uint(v[i]);
        else w[i] = pack(v[2 * i], v[2 * i + 1], T());
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// Largest element (NaN is passed over: it shows in the sum).
template <typename T> __device__ __forceinline__ float largest(const uint4& u) {
    float v[Elem<T>::PER_16];
    unpack<T>(u, v);
    float m = v[0];
#pragma unroll
    for (int i = 1; i < Elem<T>::PER_16; ++i) m = fmaxf(m, v[i]);
    return m;
}

// Logits are read once a pass: they stay out of L1.
__device__ __forceinline__ uint4 load_16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The elements [0, count) of a row's chunk as a head up to the next 16-byte boundary, vectors and a tail.
template <typename T> struct Cut {
    int head, vectors, tail;
    __device__ __forceinline__ Cut(const T* p, int count) {
        constexpr int N = Elem<T>::PER_16;
        head = (int)(((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T));
        if (head > count) head = count;
        vectors = (count - head) / N;
        tail = count - head - vectors * N;
    }
};

struct Rows {
    const void* p;
    long long sn, ss;
    template <typename T> __device__ __forceinline__ const T* at(int i, int j) const {
        return reinterpret_cast<const T*>(p) + (long long)i * sn + (long long)j * ss;
    }
};

struct StatsArgs {
    Rows x, y;                     // policy and reference
    const long long* labels;       // [n, s]
    const float* mask;             // [n, s]
    float* part;                   // planes of [rows, splits]: max, sum (policy), max, sum (reference), sum p (x - y)
    float* target;                 // planes of [rows]: the label's logit where this share of the vocabulary has it, else 0
    int* ticket;
    long long v0;
    int rows, s, vocab, splits, chunk;
};

// A row's sums over one chunk, joined over the G threads that share it.  (m, t): maximum and sum of exponentials.
struct Sums {
    float m, t;
    __device__ __forceinline__ void join_warp() {
        const float top = warp_max(m);
        t = warp_sum(t * __expf(m - top));
        m = top;
    }
};

// G threads a chunk of a row, U 16-byte loads a thread, all of them in flight before the first is used.  A thread takes the
// maximum of what it holds and the exponentials against that, so nothing is rescaled inside the loop.
template <typename T, int G, int U>
__global__ void __launch_bounds__(THREADS) stats_kernel(const StatsArgs a) {
    constexpr int N = Elem<T>::PER_16;
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.ticket = 0;
    const unsigned item = blockIdx.x * (THREADS / G) + threadIdx.x / G;
    const int lane = threadIdx.x % G, which = blockIdx.y;
    const int row = (int)(item / (unsigned)a.splits), part = (int)(item % (unsigned)a.splits);
    if (row >= a.rows) return;
    const long long cells = (long long)a.rows * a.splits;
    float* out_m = a.part + 2 * which * cells + item;
    float* out_t = out_m + cells;
    if (a.mask[row] == 0.f) {
        if (lane == 0) {
            *out_m = -FLT_MAX;
            *out_t = 0.f;
            if (part == 0) a.target[(long long)which * a.rows + row] = 0.f;
        }
        return;
    }
    const T* x = (which ? a.y : a.x).at<T>(row / a.s, row % a.s);
    if (part == 0 && lane == G - 1) {
        const long long y = a.labels[row] - a.v0;
        a.target[(long long)which * a.rows + row] = y >= 0 && y < a.vocab ? Elem<T>::get(x[y]) : 0.f;
    }
    const int c0 = part * a.chunk, count = min(a.chunk, a.vocab - c0);
    x += c0;
    const Cut<T> cut(x, count);
    const uint4* xv = reinterpret_cast<const uint4*>(x + cut.head);
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (lane + u * G < cut.vectors) raw[u] = load_16(xv + lane + u * G);
    Sums r{-FLT_MAX, 0.f};
    float edge = -INFINITY;                                     // head and tail: at most one element a thread
    if (lane < cut.head) edge = Elem<T>::get(x[lane]);
    else if (lane - N < cut.tail && lane >= N) edge = Elem<T>::get(x[cut.head + cut.vectors * N + lane - N]);
    r.m = fmaxf(r.m, edge);
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (lane + u * G < cut.vectors) r.m = fmaxf(r.m, largest<T>(raw[u]));
    r.t = __expf(edge - r.m);
    float t1 = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (lane + u * G < cut.vectors) {
            float v[N];
            unpack<T>(raw[u], v);
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                r.t += __expf(v[i] - r.m);
                t1 += __expf(v[i + 1] - r.m);
            }
        }
    r.t += t1;
    r.join_warp();
    if constexpr (G > 32) {
        __shared__ Sums warps[THREADS / 32];
        if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = r;
        __syncthreads();
        if (threadIdx.x >= 32) return;
        r = lane < G / 32 ? warps[lane] : Sums{-FLT_MAX, 0.f};
        r.join_warp();
    }
    if (lane == 0) {
        *out_m = r.m;
        *out_t = r.t;
    }
}

// The same over policy and reference side by side, with the sum of p (x - y) that the KL over the vocabulary needs.  An entry of
// probability zero adds nothing, also where both logits are -inf.
template <typename T, int G, int U>
__global__ void __launch_bounds__(THREADS) stats_full_kernel(const StatsArgs a) {
    constexpr int N = Elem<T>::PER_16;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0;
    const unsigned item = blockIdx.x * (THREADS / G) + threadIdx.x / G;
    const int lane = threadIdx.x % G;
    const int row = (int)(item / (unsigned)a.splits), part = (int)(item % (unsigned)a.splits);
    if (row >= a.rows) return;
    const long long cells = (long long)a.rows * a.splits;
    float* out = a.part + item;
    if (a.mask[row] == 0.f) {
        if (lane == 0) {
            out[0] = out[2 * cells] = -FLT_MAX;
            out[cells] = out[3 * cells] = out[4 * cells] = 0.f;
            if (part == 0) a.target[row] = 0.f;
        }
        return;
    }
    const T* x = a.x.at<T>(row / a.s, row % a.s);
    const T* y = a.y.at<T>(row / a.s, row % a.s);
    if (part == 0 && lane == G - 1) {
        const long long l = a.labels[row] - a.v0;
        a.target[row] = l >= 0 && l < a.vocab ? Elem<T>::get(x[l]) : 0.f;
    }
    const int c0 = part * a.chunk, count = min(a.chunk, a.vocab - c0);
    x += c0;
    y += c0;
    Sums p{-FLT_MAX, 0.f}, q{-FLT_MAX, 0.f};
    float w = 0.f;
    if ((((uintptr_t)x ^ (uintptr_t)y) & 15) == 0) {
        const Cut<T> cut(x, count);
        const uint4* xv = reinterpret_cast<const uint4*>(x + cut.head);
        const uint4* yv = reinterpret_cast<const uint4*>(y + cut.head);
        uint4 xr[U], yr[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (lane + u * G < cut.vectors) {
                xr[u] = load_16(xv + lane + u * G);
                yr[u] = load_16(yv + lane + u * G);
            }
        float ex = -INFINITY, ey = -INFINITY;
        int at = -1;
        if (lane < cut.head) at = lane;
        else if (lane - N < cut.tail && lane >= N) at = cut.head + cut.vectors * N + lane - N;
        if (at >= 0) {
            ex = Elem<T>::get(x[at]);
            ey = Elem<T>::get(y[at]);
        }
        p.m = fmaxf(p.m, ex);
        q.m = fmaxf(q.m, ey);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (lane + u * G < cut.vectors) {
                p.m = fmaxf(p.m, largest<T>(xr[u]));
                q.m = fmaxf(q.m, largest<T>(yr[u]));
            }
        p.t = __expf(ex - p.m);
        q.t = __expf(ey - q.m);
        w = p.t > 0.f ? p.t * (ex - ey) : 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (lane + u * G < cut.vectors) {
                float v[N], r[N];
                unpack<T>(xr[u], v);
                unpack<T>(yr[u], r);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float e = __expf(v[i] - p.m);
                    p.t += e;
                    w += e > 0.f ? e * (v[i] - r[i]) : 0.f;
                    q.t += __expf(r[i] - q.m);
                }
            }
    } else {                                                    // rows that no common shift aligns: element by element
        for (int c = lane; c < count; c += G) {
            p.m = fmaxf(p.m, Elem<T>::get(x[c]));
            q.m = fmaxf(q.m, Elem<T>::get(y[c]));
        }
        for (int c = lane; c < count; c += G) {
            const float xe = Elem<T>::get(x[c]), ye = Elem<T>::get(y[c]), e = __expf(xe - p.m);
            p.t += e;
            w += e > 0.f ? e * (xe - ye) : 0.f;
            q.t += __expf(ye - q.m);
        }
    }
    const float own = p.m;
    p.join_warp();
    w = warp_sum(w * __expf(own - p.m));
    q.join_warp();
    if constexpr (G > 32) {
        __shared__ Sums ps[THREADS / 32], qs[THREADS / 32];
        __shared__ float ws[THREADS / 32];
        if ((threadIdx.x & 31) == 0) {
            ps[threadIdx.x >> 5] = p;
            qs[threadIdx.x >> 5] = q;
            ws[threadIdx.x >> 5] = w;
        }
        __syncthreads();
        if (threadIdx.x >= 32) return;
        p = lane < G / 32 ? ps[lane] : Sums{-FLT_MAX, 0.f};
        q = lane < G / 32 ? qs[lane] : Sums{-FLT_MAX, 0.f};
        w = lane < G / 32 ? ws[lane] : 0.f;
        const float mine = p.m;
        p.join_warp();
        w = warp_sum(w * __expf(mine - p.m));
        q.join_warp();
    }
    if (lane == 0) {
        out[0] = p.m;
        out[cells] = p.t;
        out[2 * cells] = q.m;
        out[3 * cells] = q.t;
        out[4 * cells] = w;
    }
}

// ---------------------------------------------------------------------------------------------- from rows to the loss
struct RowSums {
    const float* part;
    const float* target;
    const long long* labels;
    long long vocab;               // of all ranks: a label outside makes its row NaN
    int rows, splits;
};

// Joins a row's chunks: maximum and sum, in 64 bits.
__device__ __forceinline__ void join(const RowSums& r, int plane, int row, float& m, double& t) {
    const long long cells = (long long)r.rows * r.splits;
    const float* pm = r.part + plane * cells + (long long)row * r.splits;
    const float* pt = pm + cells;
    m = pm[0];
    for (int k = 1; k < r.splits; ++k) m = fmaxf(m, pm[k]);
    t = 0.0;
    for (int k = 0; k < r.splits; ++k) t += (double)pt[k] * (double)__expf(pm[k] - m);
}
__device__ __forceinline__ double label_logp(const RowSums& r, int which, int row, float m, double t) {
    const long long y = r.labels[row];
    if (y < 0 || y >= r.vocab) return nan("");
    return ((double)r.target[(long long)which * r.rows + row] - (double)m) - log(t);
}

// Sums of V values over the block, in a fixed order; the result is in thread 0.
template <int V> __device__ __forceinline__ void block_sum(double (&v)[V]) {
    __shared__ double red[THREADS / 32][V];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = warp_sum(v[k]);
    __syncthreads();
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < V; ++k) red[warp][k] = v[k];
    __syncthreads();
    if (threadIdx.x == 0)
#pragma unroll
        for (int k = 0; k < V; ++k)
            for (int w = 1; w < THREADS / 32; ++w) v[k] += red[w][k];
}

// True in all threads of the block that is last to come here; what the others wrote before is then visible to it.
__device__ __forceinline__ bool last_block(int* ticket) {
    __shared__ int last;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(ticket, 1) == (int)gridDim.x - 1;
    __syncthreads();
    if (last) __threadfence();
    return last;
}

struct PreferenceArgs {
    RowSums sums;
    const float* mask;
    const float* ref_logp;         // [n, s] or none
    int has_ref_logits, n, s, pieces;
    double beta, smoothing;
    float2* row;                   // per row: maximum, 1 / sum
    double* partial;               // [n * pieces, 2], then [n, 2]
    int* ticket;
    float* loss;
    float* logp;                   // [n]
    float* ref;                    // [n]
    float* coef;                   // [n]: d loss / d logp
};

// Each block joins THREADS rows of one sequence and leaves their sums; the last block adds those up in order, a warp a
// sequence, and forms, pair by pair,  z = beta ((P_c - P_r) - (R_c - R_r)),
// loss = -(1 - e) log sigma(z) - e log sigma(-z),  d loss / d P_c = -beta ((1 - e) sigma(-z) - e sigma(z)) / pairs = -d/d P_r.
__global__ void __launch_bounds__(THREADS) preference_kernel(const PreferenceArgs a) {
    const int seq = blockIdx.x / a.pieces, j = (blockIdx.x % a.pieces) * THREADS + threadIdx.x;
    double v[2] = {0.0, 0.0};
    if (j < a.s) {
        const int row = seq * a.s + j;
        const float w = a.mask[row];
        float2 keep = make_float2(0.f, 0.f);
        if (w != 0.f) {
            float m;
            double t;
            join(a.sums, 0, row, m, t);
            keep = make_float2(m, (float)(1.0 / t));
            v[0] = w * label_logp(a.sums, 0, row, m, t);
            if (a.has_ref_logits) {
                join(a.sums, 2, row, m, t);
                v[1] = w * label_logp(a.sums, 1, row, m, t);
            } else if (a.ref_logp) {
                v[1] = (double)w * a.ref_logp[row];
            }
        }
        a.row[row] = keep;
    }
    block_sum(v);
    if (threadIdx.x == 0) {
        a.partial[2 * blockIdx.x] = v[0];
        a.partial[2 * blockIdx.x + 1] = v[1];
    }
    if (!last_block(a.ticket)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    double* whole = a.partial + 2ll * gridDim.x;
    for (int i = warp; i < a.n; i += THREADS / 32) {
        double p = 0.0, r = 0.0;
        for (int k = lane; k < a.pieces; k += 32) {
            p += __ldcg(a.partial + 2ll * (i * a.pieces + k));
            r += __ldcg(a.partial + 2ll * (i * a.pieces + k) + 1);
        }
        p = warp_sum(p);
        r = warp_sum(r);
        if (lane == 0) {
            whole[2 * i] = p;
            whole[2 * i + 1] = r;
            a.logp[i] = (float)p;
            a.ref[i] = (float)r;
        }
    }
    __syncthreads();
    const int pairs = a.n / 2;
    double sum[1] = {0.0};
    for (int b = threadIdx.x; b < pairs; b += THREADS) {
        const double* c = whole + 2 * b;
        const double* r = whole + 2 * (b + pairs);
        const double z = a.beta * ((c[0] - r[0]) - (c[1] - r[1]));
        const double small = exp(-fabs(z)), soft = log1p(small);
        double loss = (1.0 - a.smoothing) * (soft + fmax(-z, 0.0));
        if (a.smoothing != 0.0) loss += a.smoothing * (soft + fmax(z, 0.0));
        sum[0] += z != z ? z : loss;
        const double up = z >= 0 ? 1.0 / (1.0 + small) : small / (1.0 + small);          // sigma(z)
        const double down = z >= 0 ? small / (1.0 + small) : 1.0 / (1.0 + small);        // sigma(-z)
        const double d = z != z ? z : -a.beta * ((1.0 - a.smoothing) * down - a.smoothing * up) / pairs;
        a.coef[b] = (float)d;
        a.coef[b + pairs] = (float)-d;
    }
    block_sum(sum);
    if (threadIdx.x == 0) *a.loss = (float)(sum[0] / pairs);
}

enum { KL_NONE = 0, KL_PLAIN, KL_ABS, KL_MSE, KL_K3, KL_FULL };

struct PolicyArgs {
    RowSums sums;
    const float* mask;
    const float* advantages;       // element (i, j) at i * adv_n + j * adv_s
    long long adv_n, adv_s;
    const float* old_logp;         // [n, s] or none: the policy itself
    const float* ref_logp;         // [n, s] or none
    int has_ref_logits, n, s, pieces, kl, by_sequence;
    double low, high, kl_beta;     // the ratio's bounds
    float2* row;                   // per row: maximum, 1 / sum
    float* slope;                  // per row: mask * d term / d logp
    float* shift;                  // per row: lse(x) - lse(y) + KL, for the KL over the vocabulary
    double* partial;               // [n * pieces, 4], then [n, 4]
    int* ticket;
    float* out;                    // loss, mean KL, share of clipped tokens
    float* logp;                   // [n, s]
    float* coef;                   // [n]: what a row's slope is multiplied by
};

// Row by row: r = exp(l - old), term = -min(r A, clip(r) A) + kl_beta KL and its slope in l; sums of mask, mask * term,
// mask * KL and mask * [clipped] by sequence, then the means.
__global__ void __launch_bounds__(THREADS) policy_kernel(const PolicyArgs a) {
    const int seq = blockIdx.x / a.pieces, j = (blockIdx.x % a.pieces) * THREADS + threadIdx.x;
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    if (j < a.s) {
        const int row = seq * a.s + j;
        const float w = a.mask[row];
        float2 keep = make_float2(0.f, 0.f);
        float slope = 0.f, shift = 0.f, logp = 0.f;
        if (w != 0.f) {
            float m;
            double t;
            join(a.sums, 0, row, m, t);
            keep = make_float2(m, (float)(1.0 / t));
            const double l = label_logp(a.sums, 0, row, m, t);
            logp = (float)l;
            const double adv = a.advantages[seq * a.adv_n + j * a.adv_s];
            const double ratio = a.old_logp ? exp(l - (double)a.old_logp[row]) : (l == l ? 1.0 : l);
            const double bounded = fmin(fmax(ratio, a.low), a.high);
            const double free = ratio * adv, held = bounded * adv;
            const bool clipped = free > held;
            double term = clipped ? -held : -free, d = clipped ? 0.0 : -free, kl = 0.0;
            if (a.kl == KL_FULL) {
                const long long cells = (long long)a.sums.rows * a.sums.splits, at = (long long)row * a.sums.splits;
                double w_sum = 0.0;
                for (int k = 0; k < a.sums.splits; ++k)
                    w_sum += (double)a.sums.part[4 * cells + at + k] * (double)__expf(a.sums.part[at + k] - m);
                float mq;
                double tq;
                join(a.sums, 2, row, mq, tq);
                const double gap = ((double)m - (double)mq) + (log(t) - log(tq));
                kl = w_sum / t - gap;
                shift = (float)(gap + kl);
            } else if (a.kl != KL_NONE) {
                double ref;
                if (a.has_ref_logits) {
                    float mq;
                    double tq;
                    join(a.sums, 2, row, mq, tq);
                    ref = label_logp(a.sums, 1, row, mq, tq);
                } else {
                    ref = a.ref_logp[row];
                }
                const double x = l - ref;
                double more;
                if (a.kl == KL_PLAIN) {
                    kl = x;
                    more = x == x ? 1.0 : x;
                } else if (a.kl == KL_ABS) {
                    kl = fabs(x);
                    more = x > 0.0 ? 1.0 : x < 0.0 ? -1.0 : x;
                } else if (a.kl == KL_MSE) {
                    kl = 0.5 * x * x;
                    more = x;
                } else {
                    const double e = expm1(-x);
                    kl = e + x;
                    more = -e;
                }
                d += a.kl_beta * more;
            }
            term += a.kl_beta * kl;
            slope = (float)(w * d);
            v[0] = w;
            v[1] = w * term;
            v[2] = w * kl;
            v[3] = clipped ? w : 0.0;
        }
        a.row[row] = keep;
        a.slope[row] = slope;
        a.logp[row] = logp;
        if (a.shift) a.shift[row] = shift;
    }
    block_sum(v);
    if (threadIdx.x == 0)
#pragma unroll
        for (int k = 0; k < 4; ++k) a.partial[4ll * blockIdx.x + k] = v[k];
    if (!last_block(a.ticket)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    double* whole = a.partial + 4ll * gridDim.x;
    for (int i = warp; i < a.n; i += THREADS / 32) {
        double p[4] = {0.0, 0.0, 0.0, 0.0};
        for (int k = lane; k < a.pieces; k += 32)
#pragma unroll
            for (int q = 0; q < 4; ++q) p[q] += __ldcg(a.partial + 4ll * (i * a.pieces + k) + q);
#pragma unroll
        for (int q = 0; q < 4; ++q) p[q] = warp_sum(p[q]);
        if (lane == 0)
#pragma unroll
            for (int q = 0; q < 4; ++q) whole[4 * i + q] = p[q];
    }
    __syncthreads();
    // mask, term, KL, clipped, sequences with a kept token, their mean terms
    double sum[6] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
    for (int i = threadIdx.x; i < a.n; i += THREADS) {
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[q] += whole[4 * i + q];
        if (whole[4 * i] > 0.0) {
            sum[4] += 1.0;
            sum[5] += whole[4 * i + 1] / whole[4 * i];
        }
    }
    block_sum(sum);
    __shared__ double total, filled;
    if (threadIdx.x == 0) {
        total = sum[0];
        filled = sum[4];
        const bool any = sum[0] != 0.0;                        // nothing kept: no loss, no gradient
        a.out[0] = !any ? 0.f : (float)(a.by_sequence ? sum[5] / sum[4] : sum[1] / sum[0]);
        a.out[1] = any ? (float)(sum[2] / sum[0]) : 0.f;
        a.out[2] = any ? (float)(sum[3] / sum[0]) : 0.f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.n; i += THREADS) {
        const double len = a.by_sequence ? whole[4 * i] * filled : total;
        a.coef[i] = len > 0.0 || (!a.by_sequence && len != 0.0) ? (float)(1.0 / len) : 0.f;
    }
}

// ---------------------------------------------------------------------------------------------- gradient
struct GradArgs {
    Rows x, y;                     // y: reference, for the KL over the vocabulary
    void* g;
    long long gn, gs;
    const long long* labels;
    const float* slope;            // per row
    const float* mask;             // per row, for b
    const float* shift;
    const float2* row;
    const float* coef;             // [n]
    const float* g_loss;           // gradient of the loss, or none
    const float* g_logp;           // [n], or none: gradient of the sequences' log-probabilities
    long long v0;
    float kl_beta;
    int rows, s, vocab, splits, chunk;
};

template <typename T, bool FULL>
__device__ __forceinline__ float grad_of(float x, float y, float m, float scale, float bscale, float shift) {
    const float e = __expf(x - m);
    if constexpr (FULL) return e > 0.f || e != e ? e * fmaf(bscale, (x - y) - shift, scale) : 0.f;
    else return e * scale;
}

template <typename T, int G, int U, bool FULL>
__global__ void __launch_bounds__(THREADS) grad_kernel(const GradArgs a) {
    constexpr int N = Elem<T>::PER_16;
    const unsigned item = blockIdx.x * (THREADS / G) + threadIdx.x / G;
    const int lane = threadIdx.x % G;
    const int row = (int)(item / (unsigned)a.splits), part = (int)(item % (unsigned)a.splits);
    if (row >= a.rows) return;
    const int i = row / a.s, j = row - i * a.s;
    const int c0 = part * a.chunk, count = min(a.chunk, a.vocab - c0);
    const T* x = a.x.at<T>(i, j) + c0;
    const T* y = FULL ? a.y.at<T>(i, j) + c0 : x;
    T* g = reinterpret_cast<T*>(a.g) + (long long)i * a.gn + (long long)j * a.gs + c0;
    float unit = a.g_loss ? *a.g_loss * a.coef[i] : 0.f;
    const float b = FULL ? unit * a.kl_beta * a.mask[row] : 0.f;
    if (a.g_logp) unit += a.g_logp[i];
    const float slope = a.slope[row];
    // a weight of zero leaves nothing, whatever it is multiplied by
    const float coef = FULL ? unit * slope : slope == 0.f ? 0.f : unit * slope;
    const Cut<T> cut(g, count);
    uint4* gv = reinterpret_cast<uint4*>(g + cut.head);
    if (FULL ? a.mask[row] == 0.f || (coef == 0.f && b == 0.f) : coef == 0.f) {
        const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (lane + u * G < cut.vectors) __stcs(gv + lane + u * G, zero);
        if (lane < cut.head) g[lane] = Elem<T>::put(0.f);
        if (lane < cut.tail) g[cut.head + cut.vectors * N + lane] = Elem<T>::put(0.f);
        return;
    }
    const float2 st = a.row[row];
    const float m = st.x, scale = -coef * st.y, bscale = b * st.y, shift = FULL ? a.shift[row] : 0.f;
    const long long label = a.labels[row] - a.v0 - c0;
    const bool together = (((uintptr_t)x ^ (uintptr_t)g) & 15) == 0 && (((uintptr_t)y ^ (uintptr_t)g) & 15) == 0;
    if (together) {
        const uint4* xv = reinterpret_cast<const uint4*>(x + cut.head);
        const uint4* yv = reinterpret_cast<const uint4*>(y + cut.head);
        uint4 xr[U], yr[FULL ? U : 1];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (lane + u * G < cut.vectors) {
                xr[u] = load_16(xv + lane + u * G);
                if constexpr (FULL) yr[u] = load_16(yv + lane + u * G);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (lane + u * G < cut.vectors) {
                float v[N], r[N];
                unpack<T>(xr[u], v);
                if constexpr (FULL) unpack<T>(yr[u], r);
                const long long d = label - cut.head - (long long)(lane + u * G) * N;
                const int hit = d >= 0 && d < N ? (int)d : -1;
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    v[k] = grad_of<T, FULL>(v[k], FULL ? r[k] : 0.f, m, scale, bscale, shift);
                    if (k == hit) v[k] += coef;
                }
                __stcs(gv + lane + u * G, repack<T>(v));
            }
        int at = -1;
        if (lane < cut.head) at = lane;
        else if (lane - N < cut.tail && lane >= N) at = cut.head + cut.vectors * N + lane - N;
        if (at >= 0) {
            float v = grad_of<T, FULL>(Elem<T>::get(x[at]), FULL ? Elem<T>::get(y[at]) : 0.f, m, scale, bscale, shift);
            if (at == label) v += coef;
            g[at] = Elem<T>::put(v);
        }
    } else {                                                    // rows that no common shift aligns: element by element
        for (int c = lane; c < count; c += G) {
            float v = grad_of<T, FULL>(Elem<T>::get(x[c]), FULL ? Elem<T>::get(y[c]) : 0.f, m, scale, bscale, shift);
            if (c == label) v += coef;
            g[c] = Elem<T>::put(v);
        }
    }
}

// Chunks of a row: what G threads with U loads each hold.  The chunks of a row are of one size, up to rounding to 8 elements.
struct Plan {
    bool warp;                     // a warp a row, else a block a chunk
    int splits, chunk;
    bool fits(long long rows, int vocab) const { return rows * splits < (1ll << 31) && (splits - 1ll) * chunk < vocab; }
};
Plan plan(int vocab, int dtype, int u) {
    const int n = dtype == 1 ? 4 : 8;
    if (vocab <= 32 * u * n) return {true, 1, vocab};
    const int most = THREADS * u * n;
    const int splits = (vocab + most - 1) / most;
    return {false, splits, ((vocab + splits - 1) / splits + 7) / 8 * 8};
}

#define FOR_TYPE(dtype, CALL)                                  \
    do {                                                       \
        if (dtype == 0) { using T = __nv_bfloat16; CALL; }     \
        else if (dtype == 1) { using T = float; CALL; }        \
        else { using T = __half; CALL; }                       \
    } while (0)

constexpr int U_ONE = 8, U_FULL = 4;

int launched() { return cudaGetLastError() == cudaSuccess ? 0 : NEOX_ERR_LAUNCH; }

}  // namespace

extern "C" {

// Chunks a row is read in: the planes that neox_vocab_stats writes are [n * s, this].
int neox_vocab_splits(int vocab, int dtype, int full) { return plan(vocab, dtype, full ? U_FULL : U_ONE).splits; }

int neox_vocab_stats(const void* x, long long xn, long long xs, const void* y, long long yn, long long ys,
                     const long long* labels, const float* mask, int n, int s, int vocab, long long v0, int dtype, int full,
                     float* part, float* target, int* ticket, void* stream) {
    if (n < 0 || s < 0 || vocab < 1 || (full && !y)) return NEOX_ERR_SHAPE;
    const Plan p = plan(vocab, dtype, full ? U_FULL : U_ONE);
    const long long rows = (long long)n * s;
    if (!p.fits(rows, vocab)) return NEOX_ERR_TOO_LARGE;
    StatsArgs a = {{x, xn, xs}, {y, yn, ys}, labels, mask, part, target, ticket, v0, (int)rows, s, vocab, p.splits, p.chunk};
    const long long per = p.warp ? THREADS / 32 : 1;
    const dim3 grid((unsigned)((rows * p.splits + per) / per), !full && y ? 2 : 1);        // one block at least: it sets the ticket
    cudaStream_t st = (cudaStream_t)stream;
    if (full) {
        if (p.warp) FOR_TYPE(dtype, (stats_full_kernel<T, 32, U_FULL><<<grid, THREADS, 0, st>>>(a)));
        else FOR_TYPE(dtype, (stats_full_kernel<T, THREADS, U_FULL><<<grid, THREADS, 0, st>>>(a)));
    } else {
        if (p.warp) FOR_TYPE(dtype, (stats_kernel<T, 32, U_ONE><<<grid, THREADS, 0, st>>>(a)));
        else FOR_TYPE(dtype, (stats_kernel<T, THREADS, U_ONE><<<grid, THREADS, 0, st>>>(a)));
    }
    return launched();
}

// Blocks that join a sequence's rows; `partial` of the two calls below holds (n * this + n) * 2 or * 4 doubles.
int neox_loss_pieces(int s) { return s > 0 ? (s + THREADS - 1) / THREADS : 1; }

int neox_preference_loss(const float* part, const float* target, int splits, const long long* labels, const float* mask,
                         const float* ref_logp, int has_ref_logits, int n, int s, long long vocab, double beta, double smoothing,
                         void* row, double* partial, int* ticket, float* loss, float* logp, float* ref, float* coef, void* stream) {
    if (n < 2 || n % 2 || s < 0) return NEOX_ERR_SHAPE;
    const int pieces = neox_loss_pieces(s);
    if ((long long)n * pieces >= (1ll << 31)) return NEOX_ERR_TOO_LARGE;
    const PreferenceArgs a = {{part, target, labels, vocab, n * s, splits}, mask, ref_logp, has_ref_logits, n, s, pieces, beta,
                              smoothing, (float2*)row, partial, ticket, loss, logp, ref, coef};
    preference_kernel<<<n * pieces, THREADS, 0, (cudaStream_t)stream>>>(a);
    return launched();
}

int neox_policy_loss(const float* part, const float* target, int splits, const long long* labels, const float* mask,
                     const float* advantages, long long adv_n, long long adv_s, const float* old_logp, const float* ref_logp,
                     int has_ref_logits, int n, int s, long long vocab, int kl, int by_sequence, double low, double high,
                     double kl_beta, void* row, float* slope, float* shift, double* partial, int* ticket, float* out, float* logp,
                     float* coef, void* stream) {
    if (n < 1 || s < 0) return NEOX_ERR_SHAPE;
    const int pieces = neox_loss_pieces(s);
    if ((long long)n * pieces >= (1ll << 31)) return NEOX_ERR_TOO_LARGE;
    const PolicyArgs a = {{part, target, labels, vocab, n * s, splits}, mask, advantages, adv_n, adv_s, old_logp, ref_logp,
                          has_ref_logits, n, s, pieces, kl, by_sequence, low, high, kl_beta, (float2*)row, slope, shift, partial,
                          ticket, out, logp, coef};
    policy_kernel<<<n * pieces, THREADS, 0, (cudaStream_t)stream>>>(a);
    return launched();
}

int neox_vocab_grad(const void* x, long long xn, long long xs, const void* y, long long yn, long long ys, void* g, long long gn,
                    long long gs, const long long* labels, const float* slope, const float* mask, const float* shift,
                    const void* row, const float* coef, const float* g_loss, const float* g_logp, float kl_beta, int n, int s,
                    int vocab, long long v0, int dtype, void* stream) {
    if (n < 0 || s < 0 || vocab < 1) return NEOX_ERR_SHAPE;
    const int full = shift != nullptr;
    const Plan p = plan(vocab, dtype, full ? U_FULL : U_ONE);
    const long long rows = (long long)n * s;
    if (rows == 0) return 0;
    if (!p.fits(rows, vocab)) return NEOX_ERR_TOO_LARGE;
    const GradArgs a = {{x, xn, xs}, {y, yn, ys}, g, gn, gs, labels, slope, mask, shift, (const float2*)row, coef, g_loss, g_logp,
                        v0, kl_beta, (int)rows, s, vocab, p.splits, p.chunk};
    const long long per = p.warp ? THREADS / 32 : 1;
    const unsigned grid = (unsigned)((rows * p.splits + per - 1) / per);
    cudaStream_t st = (cudaStream_t)stream;
    if (full) {
        if (p.warp) FOR_TYPE(dtype, (grad_kernel<T, 32, U_FULL, true><<<grid, THREADS, 0, st>>>(a)));
        else FOR_TYPE(dtype, (grad_kernel<T, THREADS, U_FULL, true><<<grid, THREADS, 0, st>>>(a)));
    } else {
        if (p.warp) FOR_TYPE(dtype, (grad_kernel<T, 32, U_ONE, false><<<grid, THREADS, 0, st>>>(a)));
        else FOR_TYPE(dtype, (grad_kernel<T, THREADS, U_ONE, false><<<grid, THREADS, 0, st>>>(a)));
    }
    return launched();
}

}  // extern "C"
