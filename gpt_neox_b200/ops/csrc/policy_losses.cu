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
// `preference_kernel` / `policy_kernel` join them, eight lanes a row, and the last block to finish forms the loss and what the
// backward multiplies; `grad_kernel` streams the rows a second time and writes the gradient, zeros
// where the coefficient is zero, without reading.  The second pass over the logits cannot be saved for a preference loss: a
// pair's coefficient depends on all of its rows.  It can be for a policy loss, whose rows need only the sum of the mask from one
// another: `policy_row_kernel`, further down, has a row in shared memory and writes its gradient with its loss.
//
// Exponentials, a lane's sums of them and gradients are in 32 bits; the lanes' sums are joined in 64, and so is everything up to the
// loss; coefficients, 1 / sum and outputs are rounded to 32.  Of a row's log-probability that leaves an error of 1e-8 to 2e-8 in half of
// the rows, and of at most some 2e-7 in those that one word outweighs (rows of 32000 to 50432 words).
//
// All of it is bound by memory traffic.  8 x 1024 tokens over 50304 bf16 words, 4506 kept, on a machine whose copies run at 6.55
// TB/s: statistics 80 us (5.7 TB/s), joining 7, gradient 190 (6.7 TB/s); loss and gradient at once 226 (5.7 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>
#include <limits.h>
#include <stdint.h>

#include "dynamic_smem.h"
#include "launch.cuh"
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
// Largest element of one and of many (NaN is passed over: it shows in the sum).
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b, __nv_bfloat16) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b, __half) {
    const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b, float) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}
template <typename T> __device__ __forceinline__ uint32_t larger(const uint4& u) {
    return larger(larger(u.x, u.y, T()), larger(u.z, u.w, T()), T());
}
template <typename T> __device__ __forceinline__ float as_max(uint32_t w) {
    if constexpr (Elem<T>::PER_16 == 4) return __uint_as_float(w);
    else {
        const float2 f = two(w, T());
        return fmaxf(f.x, f.y);
    }
}

// Two 32-bit floats in one instruction.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 parts(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 add(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 mul(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// exp(d) of the gap between two maxima, d <= 0, for the few factors that whole sums are multiplied by.  Made good are the rounding of
// the product, that of log2 e, and what ex2 is low by on average (measured: 2.2e-8 of its result for arguments above -1, 5e-8 below).
__device__ __forceinline__ float exp_of_gap(float d) {
    const float t = d * LOG2E, low = fmaf(d, LOG2E, -t) + d * 1.925963e-8f, e = exp2_fast(t);
    return d < -150.f ? 0.f : fmaf(e, fmaf(low, 0.6931472f, t < -1.f ? 5e-8f : 2.2e-8f), e);
}
__device__ __forceinline__ f32x2 tree_sum(const f32x2 (&v)[2]) { return add(v[0], v[1]); }
__device__ __forceinline__ f32x2 tree_sum(const f32x2 (&v)[4]) { return add(add(v[0], v[1]), add(v[2], v[3])); }
// exp(x + shift).  The sum first: a row's largest and lowest numbers may be as large as the type has them, and the difference of
// two 16-bit numbers near each other is exact.
__device__ __forceinline__ f32x2 exp_of(f32x2 x, f32x2 shift) {
    const float2 t = parts(mul(add(x, shift), pair(LOG2E, LOG2E)));
    return pair(exp2_fast(t.x), exp2_fast(t.y));
}
// The elements of 16 bytes as pairs.
template <typename T> __device__ __forceinline__ void pairs_of(const uint4& u, f32x2 (&v)[Elem<T>::PER_16 / 2]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (Elem<T>::PER_16 == 4) {
        v[0] = pair(__uint_as_float(w[0]), __uint_as_float(w[1]));
        v[1] = pair(__uint_as_float(w[2]), __uint_as_float(w[3]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = two(w[i], T());
            v[i] = pair(f.x, f.y);
        }
    }
}

// Logits are read once a pass: they stay out of L1.
__device__ __forceinline__ uint4 load_16(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// exp(x - m) of the elements of 16 bytes.  16-bit numbers are taken from their words by the subtraction itself (the widening is
// exact), which saves an instruction an element.
__device__ __forceinline__ f32x2 less(uint32_t w, float m, __nv_bfloat16) {
    float a, b;
    asm("{.reg .b16 x, y;\n mov.b32 {x, y}, %2;\n sub.rn.f32.bf16 %0, x, %3;\n sub.rn.f32.bf16 %1, y, %3;}"
        : "=f"(a), "=f"(b) : "r"(w), "f"(m));
    return pair(a, b);
}
__device__ __forceinline__ f32x2 less(uint32_t w, float m, __half) {
    float a, b;
    asm("{.reg .b16 x, y;\n mov.b32 {x, y}, %2;\n sub.rn.f32.f16 %0, x, %3;\n sub.rn.f32.f16 %1, y, %3;}"
        : "=f"(a), "=f"(b) : "r"(w), "f"(m));
    return pair(a, b);
}
template <typename T> __device__ __forceinline__ void exps_of(const uint4& u, float m, f32x2 (&e)[Elem<T>::PER_16 / 2]) {
    if constexpr (Elem<T>::PER_16 == 4) {
        e[0] = exp_of(pair(__uint_as_float(u.x), __uint_as_float(u.y)), pair(-m, -m));
        e[1] = exp_of(pair(__uint_as_float(u.z), __uint_as_float(u.w)), pair(-m, -m));
    } else {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = parts(mul(less(w[i], m, T()), pair(LOG2E, LOG2E)));
            e[i] = pair(exp2_fast(t.x), exp2_fast(t.y));
        }
    }
}

// Asynchronous copies of 16 bytes to shared memory, in groups: `copies_here<K>` waits until all but the last K groups of this thread
// have arrived.  Each thread reads only what it copied itself.
__device__ __forceinline__ void copy_16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_8(void* to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_sent() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int K> __device__ __forceinline__ void copies_here() { asm volatile("cp.async.wait_group %0;" ::"n"(K) : "memory"); }

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

// ---------------------------------------------------------------------------------------------- statistics of the kept rows
// One block an SM: its warps, a lane's 16-byte vectors a step, and steps in shared memory, the one being worked on among them.
template <bool FULL> struct Shape {
    static constexpr int WARPS = FULL ? 16 : 24, STAGES = FULL ? 3 : 2, VECTORS = 6;
};
constexpr int MOST_ROWS = 1024;                                 // rows a block keeps at a time
constexpr int SCAN = 8;                                         // mask words a lane has in flight

// What is left of a chunk of a row.
struct __align__(16) Part {
    double t;                      // sum of exponentials against
    float m;                       // the maximum
    float w;                       // sum of p (x - y), for the KL over the vocabulary
};

struct StatsArgs {
    Rows x, y;                     // policy and reference
    const long long* labels;       // [n, s]
    const float* mask;             // [n, s]
    Part* part;                    // [streams][rows, most]
    float* target;                 // [streams][rows]: the label's logit where this share of the vocabulary has it, else 0
    int* ticket;                   // zero for the next kernel, then the number of chunks
    long long v0;
    int rows, s, vocab;
    int streams;                   // 2: the reference's rows are further rows; 1 for the KL over the vocabulary, which reads both at once
    int chunks, most;              // of a row: as many as suit a batch that keeps everything, and the most there is room for
};

// Into how many chunks each of `rows` rows is cut, by the time of the busiest warp in steps of its loads: its chunks, each with an
// end that costs about 0.4 steps, and at the end one that is left alone, where a step takes 0.3 of what it takes among many.
__host__ __device__ __forceinline__ float cut_cost(long long rows, int vocab, int chunks, int warps, int step) {
    const float steps = (float)vocab / ((float)chunks * (float)step), each = (float)rows * (float)chunks / (float)warps;
    return fmaxf(each, 1.f) * (steps + 0.4f) + 0.3f * (ceilf(steps) + 0.4f);
}
// Elements of a chunk; the count that goes with it is at most `chunks`.
__host__ __device__ __forceinline__ int chunk_size(int vocab, int chunks) { return ((vocab + chunks - 1) / chunks + 7) / 8 * 8; }

// (m, t): maximum and sum of exponentials against it.
template <typename V> struct Sums {
    float m;
    V t;
    __device__ __forceinline__ void join_warp() {
        const float top = warp_max(m);
        t = warp_sum(t * (V)exp_of_gap(m - top));
        m = top;
    }
};

struct Kept {                      // a kept row of this block
    const void* x;
    const void* y;
    int row, stream;
};

template <bool FULL> struct StatsSmem {
    using S = Shape<FULL>;
    uint4 ring[S::STAGES][S::WARPS][S::VECTORS][32];
    Kept list[MOST_ROWS];
    int counts[S::WARPS];
    int queue[S::WARPS][4];        // chunks a warp has taken and not yet begun to sum
    int next;
};

// A warp's walk over its chunks, one step of at most 32 * U vectors at a time.
template <typename T, bool FULL> struct Walk {
    static constexpr int N = Elem<T>::PER_16, U = Shape<FULL>::VECTORS / (FULL ? 2 : 1), STEP = 32 * U;
    const T* x;
    const T* y;
    int item, entry, part;         // (kept row, chunk) of this warp: number, row in the list, chunk
    int count, vectors, head, done;
    bool apart;                    // policy and reference rows that no common shift aligns

    __device__ __forceinline__ void enter(const StatsArgs& a, const Kept* list, int first, int chunks, int chunk) {
        const int kept = item / chunks;
        part = item - kept * chunks;
        entry = kept - first;
        const int c0 = part * chunk;
        count = min(chunk, a.vocab - c0);
        x = static_cast<const T*>(list[entry].x) + c0;
        if constexpr (FULL) y = static_cast<const T*>(list[entry].y) + c0;
        const Cut<T> cut(x, count);
        head = cut.head;
        apart = FULL && (((uintptr_t)x ^ (uintptr_t)y) & 15) != 0;
        vectors = apart ? 0 : cut.vectors;
        done = 0;
    }
    __device__ __forceinline__ void request(uint4 (*slot)[32], int lane) const {
        const uint4* xv = reinterpret_cast<const uint4*>(x + head) + done + lane;
        const uint4* yv = FULL ? reinterpret_cast<const uint4*>(y + head) + done + lane : nullptr;
        const int left = vectors - done - lane;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (u * 32 < left) {
                copy_16(&slot[u][lane], xv + u * 32);
                if constexpr (FULL) copy_16(&slot[U + u][lane], yv + u * 32);
            }
    }
    __device__ __forceinline__ bool ends() const { return done + STEP >= vectors; }
};

// What a lane has of a chunk so far: the largest logit and the sums against it.
// FULL: the reference's sums too, and the sum of p (x - y).  U vectors at a time, STRIDE of them apart.
template <typename T, bool FULL, int U, int STRIDE> struct Running {
    static constexpr int N = Elem<T>::PER_16;
    float m, n;                    // policy, reference
    f32x2 t, r, w;                 // sum of exponentials (policy, reference), sum of p (x - y)

    __device__ __forceinline__ void clear() {
        m = n = -FLT_MAX;
        t = r = w = pair(0.f, 0.f);
    }
    // A new maximum: what was summed against the old one is scaled.
    __device__ __forceinline__ void raise(float px, float qx) {
        const float k = __expf(m - px);
        m = px;
        t = mul(t, pair(k, k));
        if constexpr (FULL) {
            const float kr = __expf(n - qx);
            n = qx;
            r = mul(r, pair(kr, kr));
            w = mul(w, pair(k, k));
        }
    }
    __device__ __forceinline__ void add_vectors(const uint4 (&xr)[U], const uint4 (&yr)[FULL ? U : 1], int left, bool whole) {
        uint32_t p = larger<T>(xr[0]), q = 0;
        if constexpr (FULL) q = larger<T>(yr[0]);
#pragma unroll
        for (int u = 1; u < U; ++u)
            if (whole || u * STRIDE < left) {
                p = larger(p, larger<T>(xr[u]), T());
                if constexpr (FULL) q = larger(q, larger<T>(yr[u]), T());
            }
        const float px = as_max<T>(p), qx = FULL ? as_max<T>(q) : n;
        if (px > m || qx > n) raise(fmaxf(m, px), fmaxf(n, qx));
        const f32x2 xs = pair(-m, -m), ys = pair(-n, -n), minus = pair(-1.f, -1.f);
        // a vector's sum first, then a step's: next to a word that outweighs the others they would lose their last bits one by one
        f32x2 gap = pair(0.f, 0.f), step = gap, step_r = gap;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (whole || u * STRIDE < left) {
                f32x2 e[N / 2];
                if constexpr (FULL) {
                    f32x2 v[N / 2], q2[N / 2];
                    pairs_of<T>(xr[u], v);
                    pairs_of<T>(yr[u], q2);
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) {
                        e[i] = exp_of(v[i], xs);
                        gap = fma(e[i], fma(q2[i], minus, v[i]), gap);
                        q2[i] = exp_of(q2[i], ys);
                    }
                    step_r = u == 0 ? tree_sum(q2) : add(step_r, tree_sum(q2));
                } else {
                    exps_of<T>(xr[u], m, e);
                }
                if constexpr (STRIDE == 32) {
                    step = u == 0 ? tree_sum(e) : add(step, tree_sum(e));
                } else {
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) step = u == 0 && i == 0 ? e[0] : add(step, e[i]);
                }
            }
        t = add(t, step);
        if constexpr (FULL) r = add(r, step_r);
        if constexpr (FULL) {
            const float2 g = parts(gap);
            if (g.x + g.y != g.x + g.y) {                       // 0 times infinity somewhere: what is impossible adds nothing
                float again = 0.f;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (u * STRIDE < left) {
                        float v[N], q1[N];
                        unpack<T>(xr[u], v);
                        unpack<T>(yr[u], q1);
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            const float e = __expf(v[i] - m);
                            again += e > 0.f ? e * (v[i] - q1[i]) : 0.f;
                        }
                    }
                gap = pair(again, 0.f);
            }
            w = add(w, gap);
        }
    }
    __device__ __forceinline__ void add_one(float ex, float ey) {
        raise(fmaxf(m, ex), FULL ? fmaxf(n, ey) : 0.f);
        const float e = __expf(ex - m);
        t = add(t, pair(e, 0.f));
        if constexpr (FULL) {
            w = add(w, pair(e > 0.f ? e * (ex - ey) : 0.f, 0.f));
            r = add(r, pair(__expf(ey - n), 0.f));
        }
    }
};

// One block an SM.  It counts the mask, so that every block gets the same number of chunks of kept rows (a sequence's prompt and
// padding leave whole stretches without one), and its warps take them one by one.  A lane copies its own 16-byte vectors to shared
// memory ahead of the step it works on and reads back what it copied itself, so nothing waits for another lane until a chunk ends
// in one (max, sum) that the next kernel joins.  What bounds it is memory traffic, then the issue of some 3.3 instructions an element:
// pairs of 32-bit numbers, the widening folded into the subtraction (5.5 with single additions, multiplications and conversions).
// The rows above took 106 us with a block for each chunk of a row and its loads in registers; policy and reference for the KL over
// the vocabulary 218, now 150 (6.0 TB/s).
template <typename T, bool FULL>
__global__ void __launch_bounds__(Shape<FULL>::WARPS * 32, 1) stats_kernel(const StatsArgs a) {
    using W = Walk<T, FULL>;
    constexpr int N = W::N, U = W::U, WARPS = Shape<FULL>::WARPS, STAGES = Shape<FULL>::STAGES;
    extern __shared__ __align__(16) unsigned char raw_smem[];
    StatsSmem<FULL>& sm = *reinterpret_cast<StatsSmem<FULL>*>(raw_smem);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    // each round: so many rows that this block's part fits its list
    const int round = (int)min((long long)a.rows, (long long)gridDim.x * (MOST_ROWS - 2) / a.streams);
    for (int base = 0; base < a.rows; base += round) {
        const int rows = min(round, a.rows - base);
        const int segment = ((rows + WARPS - 1) / WARPS + 31) / 32 * 32;
        const int from = base + warp * segment, to = min(base + rows, from + segment);
        int mine = 0;
        for (int r = from; r < to; r += 32 * SCAN) {
            float w[SCAN];
#pragma unroll
            for (int k = 0; k < SCAN; ++k) w[k] = r + k * 32 + lane < to ? a.mask[r + k * 32 + lane] : 0.f;
#pragma unroll
            for (int k = 0; k < SCAN; ++k) mine += __popc(__ballot_sync(0xffffffffu, w[k] != 0.f));
        }
        __syncthreads();                                        // the list of the round before is no longer read
        if (lane == 0) sm.counts[warp] = mine;
        __syncthreads();
        int before = 0, kept = 0;
        for (int w = 0; w < WARPS; ++w) {
            before += w < warp ? sm.counts[w] : 0;
            kept += sm.counts[w];
        }
        int chunks = a.chunks;
        if (round == a.rows) {                                  // all rows are known here: every block finds the same best cut
            float best = INFINITY;
            chunks = 1;
            for (int c = 1 + lane; c <= a.most; c += 32) {
                const float cost = cut_cost((long long)kept * a.streams, a.vocab, c, gridDim.x * WARPS, W::STEP * N);
                if (cost < best) {
                    best = cost;
                    chunks = c;
                }
            }
            const float least = -warp_max(-best);
            chunks = __reduce_min_sync(0xffffffffu, best == least ? chunks : INT_MAX);
        }
        const int chunk = chunk_size(a.vocab, chunks);
        chunks = (a.vocab + chunk - 1) / chunk;
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            a.ticket[0] = 0;
            a.ticket[1] = chunks;
        }
        const int items = kept * a.streams * chunks, share = items / (int)gridDim.x, more = items - share * (int)gridDim.x;
        const int lo = (int)blockIdx.x * share + min((int)blockIdx.x, more), hi = lo + share + ((int)blockIdx.x < more);
        const int first = lo / chunks, end = (hi + chunks - 1) / chunks;
        for (int k = 0; k < a.streams; ++k) {                   // the second stream's rows follow the first's
            int rank = before + k * kept;
            if (rank >= end || rank + mine <= first) continue;
            for (int r = from; r < to; r += 32 * SCAN) {
                float w[SCAN];
#pragma unroll
                for (int q = 0; q < SCAN; ++q) w[q] = r + q * 32 + lane < to ? a.mask[r + q * 32 + lane] : 0.f;
#pragma unroll
                for (int q = 0; q < SCAN; ++q) {
                    const unsigned all = __ballot_sync(0xffffffffu, w[q] != 0.f);
                    const int at = rank + __popc(all & ((1u << lane) - 1));
                    if (w[q] != 0.f && at >= first && at < end) {
                        const int row = r + q * 32 + lane, i = row / a.s, j = row - i * a.s;
                        const T* other = FULL ? a.y.template at<T>(i, j) : nullptr;
                        sm.list[at - first] = Kept{(k ? a.y : a.x).template at<T>(i, j), other, row, k};
                    }
                    rank += __popc(all);
                }
            }
        }
        if (threadIdx.x == 0) sm.next = lo + WARPS;
        __syncthreads();
        W ahead, now;                                           // the walk of the copies and that of the sums
        ahead.item = now.item = lo + warp;
        unsigned taken = 0, begun = 0;
        Running<T, FULL, U, 32> run;
        run.clear();
        if (now.item < hi) {
            ahead.enter(a, sm.list, first, chunks, chunk);
            now.enter(a, sm.list, first, chunks, chunk);
        }
        int slot = 0;
        auto request = [&](int at) {
            if (ahead.item < hi) {
                ahead.request(sm.ring[at][warp], lane);
                if (!ahead.ends()) {
                    ahead.done += W::STEP;
                } else {                                        // the next chunk of the block, whoever comes first
                    int item = 0;
                    if (lane == 0) sm.queue[warp][taken & 3] = item = atomicAdd(&sm.next, 1);
                    ahead.item = __shfl_sync(0xffffffffu, item, 0);
                    ++taken;
                    if (ahead.item < hi) ahead.enter(a, sm.list, first, chunks, chunk);
                }
            }
            copies_sent();
        };
#pragma unroll
        for (int d = 0; d < STAGES - 1; ++d) request(d);
        while (now.item < hi) {
            request(slot == 0 ? STAGES - 1 : slot - 1);         // the slot that was read last
            if (now.done == 0) {                                // head and tail of the chunk: at most one element a lane
                const int tail = now.count - now.head - now.vectors * N;
                if (FULL && now.apart) {
                    for (int c = lane; c < now.count; c += 32) run.add_one(Elem<T>::get(now.x[c]), Elem<T>::get(now.y[c]));
                } else if (now.head + tail > 0) {
                    int at = -1;
                    if (lane < now.head) at = lane;
                    else if (lane >= N && lane - N < tail) at = now.head + now.vectors * N + lane - N;
                    if (at >= 0) run.add_one(Elem<T>::get(now.x[at]), FULL ? Elem<T>::get(now.y[at]) : 0.f);
                }
            }
            copies_here<STAGES - 1>();
            const int left = now.vectors - now.done - lane;
            const uint4(*from_ring)[32] = sm.ring[slot][warp];
            uint4 xr[U], yr[FULL ? U : 1];
            if (now.vectors - now.done >= W::STEP) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    xr[u] = from_ring[u][lane];
                    if constexpr (FULL) yr[u] = from_ring[U + u][lane];
                }
                run.add_vectors(xr, yr, left, true);
            } else if (left > 0) {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (u * 32 < left) {
                        xr[u] = from_ring[u][lane];
                        if constexpr (FULL) yr[u] = from_ring[U + u][lane];
                    }
                run.add_vectors(xr, yr, left, false);
            }
            slot = slot == STAGES - 1 ? 0 : slot + 1;
            if (!now.ends()) {
                now.done += W::STEP;
                continue;
            }
            const int row = sm.list[now.entry].row, stream = sm.list[now.entry].stream;
            const long long cells = (long long)a.rows * a.most, at = (long long)row * a.most + now.part;
            Sums<double> p{run.m, (double)parts(run.t).x + (double)parts(run.t).y};
            const float own = p.m;
            p.join_warp();
            float w = 0.f;
            if constexpr (FULL) {
                Sums<double> q{run.n, (double)parts(run.r).x + (double)parts(run.r).y};
                w = warp_sum((parts(run.w).x + parts(run.w).y) * exp_of_gap(own - p.m));
                q.join_warp();
                if (lane == 0) a.part[cells + at] = Part{q.t, q.m, 0.f};
            }
            if (lane == 0) a.part[stream * cells + at] = Part{p.t, p.m, w};
            if (now.part == 0 && lane == 0) {                   // x is the row's first element here
                const long long label = a.labels[row] - a.v0;
                a.target[(long long)stream * a.rows + row] = label >= 0 && label < a.vocab ? Elem<T>::get(now.x[label]) : 0.f;
            }
            run.clear();
            __syncwarp();
            now.item = sm.queue[warp][begun++ & 3];
            if (now.item < hi) now.enter(a, sm.list, first, chunks, chunk);
        }
        copies_here<0>();
    }
    if (a.rows == 0 && blockIdx.x == 0 && threadIdx.x == 0) a.ticket[0] = a.ticket[1] = 0;
    __syncthreads();
    launch::let_successor_start();
}

// ---------------------------------------------------------------------------------------------- from rows to the loss
constexpr int LANES = 8;                                        // lanes that join a row's chunks
constexpr int ROWS = THREADS / LANES;                           // rows of a block
constexpr int NEAR = 256;                                       // sequences whose sums stay in shared memory

struct RowSums {
    const Part* part;
    const float* target;
    const long long* labels;
    const int* ticket;             // [1]: chunks of a row, where `chunks` does not say
    long long vocab;               // of all ranks: a label outside makes its row NaN
    int rows, most, chunks;
};

template <typename V> __device__ __forceinline__ V lanes_sum(V v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// A lane's first chunk of a row, asked for before it is known how many there are.
__device__ __forceinline__ Part peek(const RowSums& r, int stream, int row, bool on) {
    const int lane = threadIdx.x % LANES;
    return on && lane < r.most ? r.part[((long long)stream * r.rows + row) * r.most + lane] : Part{0.0, -FLT_MAX, 0.f};
}
// Joins a row's chunks, in 64 bits: maximum, sum and, where asked for, the sum of p (x - y).  All lanes of a warp come here, each with
// its row.
template <bool CROSS>
__device__ __forceinline__ void join(const RowSums& r, int chunks, int stream, int row, bool on, Part own, float& m, double& t, double& w) {
    const int lane = threadIdx.x % LANES;
    const Part* p = r.part + ((long long)stream * r.rows + row) * r.most;
    if (lane >= chunks) own = Part{0.0, -FLT_MAX, 0.f};
    m = own.m;
    if (on)
        for (int k = lane + LANES; k < chunks; k += LANES) m = fmaxf(m, p[k].m);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const double scale = exp_of_gap(own.m - m);
    t = own.t * scale;
    if constexpr (CROSS) w = (double)own.w * scale;
    if (on)
        for (int k = lane + LANES; k < chunks; k += LANES) {
            const Part next = p[k];
            const double factor = exp_of_gap(next.m - m);
            t += next.t * factor;
            if constexpr (CROSS) w += (double)next.w * factor;
        }
    t = lanes_sum(t);
    if constexpr (CROSS) w = lanes_sum(w);
}
// Log-probability of a label whose logit is x.
__device__ __forceinline__ double label_logp(long long vocab, long long label, float x, float m, double t) {
    return label < 0 || label >= vocab ? nan("") : ((double)x - (double)m) - log(t);
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

// Sums of every sequence's pieces, V values each, by as many neighbouring lanes as leave each four loads; `leave` gets them in one.
template <int V, typename F> __device__ __forceinline__ void sum_pieces(const double* partial, int n, int pieces, F&& leave) {
    int lanes = 1;
    while (lanes < 32 && 4 * lanes < pieces) lanes *= 2;
    const int place = threadIdx.x % lanes;
    for (int first = 0; first < n; first += THREADS / lanes) {
        const int i = first + threadIdx.x / lanes;
        double p[V] = {};
        if (i < n)
#pragma unroll 4
            for (int k = place; k < pieces; k += lanes)
#pragma unroll
                for (int q = 0; q < V; ++q) p[q] += __ldcg(partial + V * ((long long)i * pieces + k) + q);
        for (int o = lanes / 2; o > 0; o >>= 1)
#pragma unroll
            for (int q = 0; q < V; ++q) p[q] += __shfl_xor_sync(0xffffffffu, p[q], o);
        if (i < n && place == 0) leave(i, p);
    }
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

// Each block joins ROWS rows of one sequence and leaves their sums; the last block adds those up in order and forms, pair by pair,
// z = beta ((P_c - P_r) - (R_c - R_r)),
// loss = -(1 - e) log sigma(z) - e log sigma(-z),  d loss / d P_c = -beta ((1 - e) sigma(-z) - e sigma(z)) / pairs = -d/d P_r.
// Latency bounds it, a dozen trips to L2 one after another: some 7 us behind the statistics, whether of 96 rows or of 8192.
// Mask, labels and stored log-probabilities are read before the wait, here and in `policy_kernel`: whatever wrote them is done, because
// the launch in front -- the statistics, or the last of the operations that join the ranks -- is not an overlapped one and began after
// it.  Statistics launched with overlap would have to send these reads behind the wait.
__global__ void __launch_bounds__(THREADS) preference_kernel(const PreferenceArgs a) {
    const int seq = blockIdx.x / a.pieces, j = (blockIdx.x % a.pieces) * ROWS + threadIdx.x / LANES;
    const int row = seq * a.s + j;
    const float w = j < a.s ? a.mask[row] : 0.f;
    const bool on = w != 0.f;
    const long long label = on ? a.sums.labels[row] : 0;
    const float given = on && a.ref_logp ? a.ref_logp[row] : 0.f;
    launch::wait_for_predecessor();
    const Part own = peek(a.sums, 0, row, on), own_r = peek(a.sums, 1, row, on && a.has_ref_logits);
    const float x = on ? a.sums.target[row] : 0.f, y = on && a.has_ref_logits ? a.sums.target[(long long)a.sums.rows + row] : 0.f;
    const int chunks = a.sums.chunks ? a.sums.chunks : a.sums.ticket[1];
    double v[2] = {0.0, 0.0};
    float m, mr = 0.f;
    double t, tr = 0.0, none;
    join<false>(a.sums, chunks, 0, row, on, own, m, t, none);
    if (a.has_ref_logits) join<false>(a.sums, chunks, 1, row, on, own_r, mr, tr, none);
    if (j < a.s && threadIdx.x % LANES == 0) {
        a.row[row] = on ? make_float2(m, __frcp_rn((float)t)) : make_float2(0.f, 0.f);
        if (on) {
            v[0] = w * label_logp(a.sums.vocab, label, x, m, t);
            if (a.has_ref_logits) v[1] = w * label_logp(a.sums.vocab, label, y, mr, tr);
            else if (a.ref_logp) v[1] = (double)w * given;
        }
    }
    block_sum(v);
    if (threadIdx.x == 0) {
        a.partial[2ll * blockIdx.x] = v[0];
        a.partial[2ll * blockIdx.x + 1] = v[1];
    }
    if (!last_block(a.ticket)) return;
    __shared__ double near[2 * NEAR];
    double* whole = a.n <= NEAR ? near : a.partial + 2ll * gridDim.x;
    sum_pieces<2>(a.partial, a.n, a.pieces, [&](int i, const double (&p)[2]) {
        whole[2ll * i] = p[0];
        whole[2ll * i + 1] = p[1];
        a.logp[i] = (float)p[0];
        a.ref[i] = (float)p[1];
    });
    __syncthreads();
    const int pairs = a.n / 2;
    double sum[1] = {0.0};
    for (int b = threadIdx.x; b < pairs; b += THREADS) {
        const double* c = whole + 2ll * b;
        const double* r = whole + 2ll * (b + pairs);
        const double z = a.beta * ((c[0] - r[0]) - (c[1] - r[1]));
        const double small = exp(-fabs(z)), soft = log1p(small);
        double loss = (1.0 - a.smoothing) * (soft + fmax(-z, 0.0));
        if (a.smoothing != 0.0) loss += a.smoothing * (soft + fmax(z, 0.0));
        sum[0] += loss;
        const double large = 1.0 / (1.0 + small), other = small * large;                // sigma(|z|), sigma(-|z|)
        const double toward = z >= 0 ? other : large, away = z >= 0 ? large : other;    // sigma(-z), sigma(z)
        const float d = (float)(-a.beta / pairs * ((1.0 - a.smoothing) * toward - a.smoothing * away));
        a.coef[b] = d;
        a.coef[b + pairs] = -d;
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
    float* loss;
    float* kl_mean;
    float* share;                  // of clipped tokens
    float* logp;                   // [n, s]
    double* wide;                  // [n, s] or none: the same of the kept rows, not rounded
    float* coef;                   // [n]: what a row's slope is multiplied by
};

// A row's part of the policy loss: r = exp(l - old), term = -min(r A, clip(r) A) + kl_beta KL, and the term's slope in l (the KL over
// the vocabulary has its own way into the logits).
struct RowTerm {
    double term, slope, kl;
    bool clipped;
    // l: log-probability; ref: the reference's, where a KL of tokens wants it; full: the KL over the vocabulary
    __device__ __forceinline__ RowTerm(int kind, double low, double high, double kl_beta, double l, bool has_old, float old, double adv,
                                       double ref, double full) {
        const double ratio = has_old ? exp(l - (double)old) : (l == l ? 1.0 : l);
        const double free = ratio * adv, held = fmin(fmax(ratio, low), high) * adv;
        clipped = free > held;
        term = clipped ? -held : -free;
        slope = clipped ? 0.0 : -free;
        kl = 0.0;
        if (kind == KL_FULL) {
            kl = full;
        } else if (kind != KL_NONE) {
            const double gap = l - ref;
            double rise;
            if (kind == KL_PLAIN) {
                kl = gap;
                rise = gap == gap ? 1.0 : gap;
            } else if (kind == KL_ABS) {
                kl = fabs(gap);
                rise = gap > 0.0 ? 1.0 : gap < 0.0 ? -1.0 : gap;
            } else if (kind == KL_MSE) {
                kl = 0.5 * gap * gap;
                rise = gap;
            } else {
                const double e = expm1(-gap);
                kl = e + gap;
                rise = -e;
            }
            slope += kl_beta * rise;
        }
        term += kl_beta * kl;
    }
};

// Row by row the terms and their slopes; sums of mask, mask * term, mask * KL and mask * [clipped] by sequence, then the means.
__global__ void __launch_bounds__(THREADS) policy_kernel(const PolicyArgs a) {
    const int seq = blockIdx.x / a.pieces, j = (blockIdx.x % a.pieces) * ROWS + threadIdx.x / LANES;
    const int row = seq * a.s + j;
    const float w = j < a.s ? a.mask[row] : 0.f;
    const bool on = w != 0.f;
    const long long label = on ? a.sums.labels[row] : 0;
    const double adv = on ? a.advantages[seq * a.adv_n + j * a.adv_s] : 0.f;
    const float old = on && a.old_logp ? a.old_logp[row] : 0.f, given = on && a.ref_logp ? a.ref_logp[row] : 0.f;
    launch::wait_for_predecessor();
    const Part own = peek(a.sums, 0, row, on), own_q = peek(a.sums, 1, row, on && a.has_ref_logits);
    const bool two = a.has_ref_logits && a.kl != KL_FULL;
    const float x = on ? a.sums.target[row] : 0.f, y = on && two ? a.sums.target[(long long)a.sums.rows + row] : 0.f;
    const int chunks = a.sums.chunks ? a.sums.chunks : a.sums.ticket[1];
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    float m, mq = 0.f;
    double t, tq = 0.0, cross = 0.0, none;
    join<true>(a.sums, chunks, 0, row, on, own, m, t, cross);
    if (a.has_ref_logits) join<false>(a.sums, chunks, 1, row, on, own_q, mq, tq, none);
    if (j < a.s && threadIdx.x % LANES == 0) {
        float2 keep = make_float2(0.f, 0.f);
        float slope = 0.f, shift = 0.f, logp = 0.f;
        if (on) {
            keep = make_float2(m, __frcp_rn((float)t));
            const double l = label_logp(a.sums.vocab, label, x, m, t);
            logp = (float)l;
            if (a.wide) a.wide[row] = l;
            double ref = given, full = 0.0;
            if (a.kl == KL_FULL) {
                const double gap = ((double)m - (double)mq) + (log(t) - log(tq));
                full = cross / t - gap;
                shift = (float)(gap + full);
            } else if (a.has_ref_logits) {
                ref = label_logp(a.sums.vocab, label, y, mq, tq);
            }
            const RowTerm r(a.kl, a.low, a.high, a.kl_beta, l, a.old_logp != nullptr, old, adv, ref, full);
            slope = (float)(w * r.slope);
            v[0] = w;
            v[1] = w * r.term;
            v[2] = w * r.kl;
            v[3] = r.clipped ? w : 0.0;
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
    __shared__ double near[4 * NEAR];
    double* whole = a.n <= NEAR ? near : a.partial + 4ll * gridDim.x;
    sum_pieces<4>(a.partial, a.n, a.pieces, [&](int i, const double (&p)[4]) {
#pragma unroll
        for (int q = 0; q < 4; ++q) whole[4ll * i + q] = p[q];
    });
    __syncthreads();
    // mask, term, KL, clipped, sequences with a kept token, their mean terms
    double sum[6] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
    for (int i = threadIdx.x; i < a.n; i += THREADS) {
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[q] += whole[4ll * i + q];
        if (whole[4ll * i] > 0.0) {
            sum[4] += 1.0;
            sum[5] += whole[4ll * i + 1] / whole[4ll * i];
        }
    }
    block_sum(sum);
    __shared__ double total, filled;
    if (threadIdx.x == 0) {
        total = sum[0];
        filled = sum[4];
        const bool any = sum[0] != 0.0;                        // nothing kept: no loss, no gradient
        *a.loss = !any ? 0.f : (float)(a.by_sequence ? sum[5] / sum[4] : sum[1] / sum[0]);
        *a.kl_mean = any ? (float)(sum[2] / sum[0]) : 0.f;
        *a.share = any ? (float)(sum[3] / sum[0]) : 0.f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.n; i += THREADS) {
        const double len = a.by_sequence ? whole[4ll * i] * filled : total;
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
    float kl_beta, expected;       // expected: of g_loss, where the forward has written the gradient for it
    int rows, s, vocab, splits, chunk;
};

template <typename T, bool FULL>
__device__ __forceinline__ float grad_of(float x, float y, float m, float scale, float bscale, float shift) {
    const float e = __expf(x - m);
    if constexpr (FULL) return e > 0.f || e != e ? e * fmaf(bscale, (x - y) - shift, scale) : 0.f;
    else return e * scale;
}

// What the gradient of a row in shared memory is made of: dx[c] = coef [c == label] + exp(x - m) scale.
struct RowGrad {
    float m, coef, scale;
};

// exp(x - m) * scale at the elements of 16 bytes.
template <typename T> __device__ __forceinline__ uint4 grad_vector(const uint4& u, const RowGrad& r) {
    constexpr int N = Elem<T>::PER_16;
    f32x2 e[N / 2];
    exps_of<T>(u, r.m, e);
    float v[N];
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
        const float2 f = parts(mul(e[k], pair(r.scale, r.scale)));
        v[2 * k] = f.x;
        v[2 * k + 1] = f.y;
    }
    return repack<T>(v);
}

// A row's gradient by G threads: zeros; and, where no common shift aligns it with the logits, element by element.
template <typename T, int G> __device__ __forceinline__ void write_zeros(T* g, int count, int lane) {
    const Cut<T> cut(g, count);
    uint4* gv = reinterpret_cast<uint4*>(g + cut.head);
#pragma unroll 4
    for (int v = lane; v < cut.vectors; v += G) __stcs(gv + v, make_uint4(0, 0, 0, 0));
    if (lane < cut.head) g[lane] = Elem<T>::put(0.f);
    if (lane < cut.tail) g[cut.head + cut.vectors * Elem<T>::PER_16 + lane] = Elem<T>::put(0.f);
}
template <typename T, int G>
__device__ __forceinline__ void write_apart(const T* x, T* g, int count, int lane, const RowGrad& r, int label) {
    for (int c = lane; c < count; c += G) {
        float v = grad_of<T, false>(Elem<T>::get(x[c]), 0.f, r.m, r.scale, 0.f, 0.f);
        if (c == label) v += r.coef;
        g[c] = Elem<T>::put(v);
    }
}

// One chunk of a row by G threads, at most U 16-byte vectors each, all asked for before the first is used: eight of one kind of logits
// or four of both.  Rows without a gradient are written, not read.  Bound by memory traffic; for the KL over the vocabulary (1.73 GB
// in 289 us) by that and the issue of its arithmetic alike.
template <typename T, int G, int U, bool FULL> __device__ __forceinline__ void grad_chunk(const GradArgs& a, unsigned item) {
    constexpr int N = Elem<T>::PER_16;
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

template <typename T, int G, int U, bool FULL>
__global__ void __launch_bounds__(THREADS) grad_kernel(const GradArgs a) {
    grad_chunk<T, G, U, FULL>(a, blockIdx.x * (THREADS / G) + threadIdx.x / G);
}

// The same after a forward that has foreseen a gradient of the loss: nothing to do where it is that one, so few blocks look, and
// they walk over the chunks where it is another.
template <typename T, int G, int U>
__global__ void __launch_bounds__(THREADS) grad_unless_kernel(const GradArgs a, unsigned items) {
    if (*a.g_loss == a.expected) return;
    for (unsigned item = blockIdx.x * (THREADS / G) + threadIdx.x / G; item < items; item += gridDim.x * (THREADS / G))
        grad_chunk<T, G, U, false>(a, item);
}

// ---------------------------------------------------------------------------------------------- policy loss and gradient at once
// All that a row of the policy loss needs from other rows is the sum of the mask, and that is known before.  So with the gradient of
// the loss foreseen (1, or what the caller says) a block takes a row's statistics, its term and its gradient while the row is in
// shared memory: logits are read once, not twice.  The backward then only looks whether it was asked for that gradient.
// 8 x 1024 tokens over 50304 words, 4506 kept: 232 us with the mask's sums before it, against 287 for two readings; over 16384 words
// 90 against 109; 4 x 8192 over 32064 610 against 742.  What it waits for is that all threads of a block have met between sums and
// gradient.  (Leaving the row to L2 in between, four blocks an SM, 273 us: two fifths of the rows had gone when they were wanted
// again.  Rows spread over a cluster's blocks, four of them an SM: 262.  Reference logits beside the policy's in one block an SM, 384 to
// 768 threads: 404 to 437 us where the reference first and the policy once took 362, and 452 to 547 against 436 for the KL over the
// vocabulary; both rows over a cluster's blocks: 0.77 to 0.96 times as fast as two readings.)
struct AtOnceArgs {
    Rows x;
    void* g;
    long long gn, gs;
    const long long* labels;
    const float* mask;
    const float* advantages;
    long long adv_n, adv_s;
    const float* old_logp;
    const float* ref_logp;
    const double* ref_wide;        // or these: of the kept rows
    int n, s, vocab, kl, by_sequence;
    double low, high, kl_beta;
    float expected;
    float2* row;
    float* slope;
    double* parts;                 // per block: sums of mask, mask * term * coef, mask * KL, mask * [clipped]
    double* whole;                 // [n]: sums of the mask
    int* order;                    // the kept rows, then the others; behind them the number of kept ones and a ticket
    float* coef;                   // [n]
    float* loss;
    float* kl_mean;
    float* share;
    float* logp;                   // [n, s]
};

// What each sequence's slopes are multiplied by: 1 / (sum of the mask), of the whole batch or of the sequence and then shared by the
// sequences that keep something; and the order of the rows.  One block; what it does takes as long as three trips to memory or, for
// many rows, as three readings of the mask: sums, count, places.
__global__ void __launch_bounds__(1024, 1) policy_share_kernel(const AtOnceArgs a) {
    __shared__ double near[32][2];
    __shared__ int kept_by[32];
    launch::let_successor_start();
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, rows = a.n * a.s;
    int each = 1;                                                            // threads of a sequence, a power of two
    while (each < 32 && each < a.s) each *= 2;
    while (each < 1024 && each < a.s && a.n <= 512 / each) each *= 2;
    const int place = tid % each;
    double total = 0.0, filled = 0.0, w = 0.0;
    for (int first = 0; first < a.n; first += 1024 / each) {
        const int i = first + tid / each;
        w = 0.0;
        if (i < a.n)
#pragma unroll 8
            for (int j = place; j < a.s; j += each) w += a.mask[(long long)i * a.s + j];
        for (int o = min(each, 32) / 2; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
        if (each > 32) {                                                     // there is one round
            if (lane == 0) near[warp][0] = w;
            __syncthreads();
            w = 0.0;
            if (place == 0)
                for (int q = 0; q < each / 32; ++q) w += near[warp + q][0];
        }
        if (place == 0 && i < a.n) {
            a.whole[i] = w;
            total += w;
            filled += w > 0.0 ? 1.0 : 0.0;
        }
    }
    total = warp_sum(total);
    filled = warp_sum(filled);
    __syncthreads();
    if (lane == 0) {
        near[warp][0] = total;
        near[warp][1] = filled;
    }
    __syncthreads();
    total = warp_sum(near[lane][0]);                                         // in every thread, in the same order
    filled = warp_sum(near[lane][1]);
    for (int i = tid / each; i < a.n; i += 1024 / each) {                    // sums that this thread has left itself
        if (place != 0) break;
        const double len = a.by_sequence ? (a.n > 1024 / each ? a.whole[i] : w) * filled : total;
        a.coef[i] = len > 0.0 || (!a.by_sequence && len != 0.0) ? (float)(1.0 / len) : 0.f;
    }
    // the rows in a warp's part of them: kept ones counted, then placed from the front, the others behind all kept ones
    const int part = ((rows + 31) / 32 + 31) / 32 * 32, from = min(rows, warp * part), to = min(rows, from + part);
    int mine = 0;
    for (int r = from; r < to; r += 32 * SCAN) {
        float w[SCAN];
#pragma unroll
        for (int k = 0; k < SCAN; ++k) w[k] = r + k * 32 + lane < to ? a.mask[r + k * 32 + lane] : 0.f;
#pragma unroll
        for (int k = 0; k < SCAN; ++k) mine += __popc(__ballot_sync(0xffffffffu, w[k] != 0.f));
    }
    if (lane == 0) kept_by[warp] = mine;
    __syncthreads();
    int before = 0, kept = 0;
    for (int q = 0; q < 32; ++q) {
        before += q < warp ? kept_by[q] : 0;
        kept += kept_by[q];
    }
    int front = before, back = kept + from - before;
    for (int r = from; r < to; r += 32 * SCAN) {
        float w[SCAN];
#pragma unroll
        for (int k = 0; k < SCAN; ++k) w[k] = r + k * 32 + lane < to ? a.mask[r + k * 32 + lane] : 0.f;
#pragma unroll
        for (int k = 0; k < SCAN; ++k) {
            const int row = r + k * 32 + lane;
            const bool in = row < to, is = in && w[k] != 0.f;
            const unsigned all = __ballot_sync(0xffffffffu, is), none = __ballot_sync(0xffffffffu, in && !is);
            const unsigned below = (1u << lane) - 1;
            if (is) a.order[front + __popc(all & below)] = row;
            else if (in) a.order[back + __popc(none & below)] = row;
            front += __popc(all);
            back += __popc(none);
        }
    }
    if (tid == 0) {
        a.order[rows] = kept;
        a.order[rows + 1] = 0;
    }
}

constexpr int MOST_PARTS = 2048;                                // blocks of a grid

// Means from what the blocks have added up, in a fixed order.  One block; `red`: room for four numbers a warp.
template <int TPB> __device__ __forceinline__ void take_means(const AtOnceArgs& a, double (*red)[4]) {
    double v[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 2
    for (int b = threadIdx.x; b < (int)gridDim.x; b += TPB)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += __ldcg(a.parts + 4 * b + k);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = warp_sum(v[k]);
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < 4; ++k) red[warp][k] = v[k];
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = warp_sum(lane < TPB / 32 ? red[lane][k] : 0.0);
    if (lane == 0) {
        const bool any = v[0] != 0.0;
        *a.loss = any ? (float)v[1] : 0.f;
        *a.kl_mean = any ? (float)(v[2] / v[0]) : 0.f;
        *a.share = any ? (float)(v[3] / v[0]) : 0.f;
    }
}

// A block walks over its rows.  A thread copies its own vectors of a row to shared memory, takes them for the sums as they arrive, and
// when all threads have met for the row's numbers, once more for the gradient; each place that it has read the second time it fills
// with the next row's vector.  As many blocks an SM as rows fit, up to eight: while one is at its sums, another is at its gradient.
// The rows that leave nothing are written in between: while a block waits for a row, memory has time for them.
template <typename T, int TPB, int BLOCKS>
__global__ void __launch_bounds__(TPB, BLOCKS) policy_row_kernel(const AtOnceArgs a, int places) {
    constexpr int N = Elem<T>::PER_16, U = 4, TEAM = TPB / 32, PARTS = 4;
    extern __shared__ __align__(16) unsigned char raw_smem[];
    uint4* xs = reinterpret_cast<uint4*>(raw_smem);
    __shared__ Sums<double> ps[TEAM];
    __shared__ RowGrad grad;
    __shared__ int where;
    __shared__ double terms[4], sums[4];                        // of a row and of all of them
    __shared__ double wide;                                     // the row's reference in 64 bits: it comes with the logits, since a
                                                                // register for it all the way costs the statistics 4 %
    if (threadIdx.x < 4) sums[threadIdx.x] = 0.0;
    const int tid = threadIdx.x, rows = a.n * a.s;
    launch::wait_for_predecessor();
    const int kept = a.order[rows];
    const int part = (places + PARTS * TPB * U - 1) / (PARTS * TPB * U) * TPB * U;      // vectors of a part, copied as a group

    struct Place {
        const T* x;
        int row, head, vectors;
    };
    auto place = [&](int pos) {
        Place p;
        p.row = a.order[pos];
        const int i = p.row / a.s, j = p.row - i * a.s;
        p.x = a.x.at<T>(i, j);
        const Cut<T> cut(p.x, a.vocab);
        p.head = cut.head;
        p.vectors = cut.vectors;
        return p;
    };
    auto request = [&](const Place& p, int v) { copy_16(xs + v, reinterpret_cast<const uint4*>(p.x + p.head) + v); };
    auto request_wide = [&](const Place& p) {
        if (tid == 0 && a.ref_wide) copy_8(&wide, a.ref_wide + p.row);
    };
    // this block's rows: every gridDim.x-th of the kept ones and of the others
    const int grid = gridDim.x, block = blockIdx.x;
    const int mine = block < kept ? (kept - 1 - block) / grid + 1 : 0;
    const int others = block < rows - kept ? (rows - kept - 1 - block) / grid + 1 : 0;
    int written = 0;
    auto write_others = [&](int until) {
        for (; written < until; ++written) {
            const int row = a.order[kept + block + written * grid], i = row / a.s, j = row - i * a.s;
            T* g = reinterpret_cast<T*>(a.g) + (long long)i * a.gn + (long long)j * a.gs;
            write_zeros<T, TPB>(g, a.vocab, tid);
            if (tid == 0) {
                a.row[row] = make_float2(0.f, 0.f);
                a.slope[row] = 0.f;
                a.logp[row] = 0.f;
            }
        }
    };
    Place now = {};
    if (mine > 0) {
        now = place(block);
        request_wide(now);
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
            for (int v = q * part + tid; v < min((q + 1) * part, now.vectors); v += TPB) request(now, v);
            copies_sent();
        }
    }
    for (int step = 0; step < mine; ++step) {
        const int row = now.row, i = row / a.s, j = row - i * a.s;
        const T* x = now.x;
        const int tail = a.vocab - now.head - now.vectors * N;
        long long label = 0;
        float own = 0.f, old = 0.f, given = 0.f, adv = 0.f, weight = 0.f, coef_i = 0.f;
        if (tid == 0) {
            label = a.labels[row];
            weight = a.mask[row];
            old = a.old_logp ? a.old_logp[row] : 0.f;
            given = a.ref_logp ? a.ref_logp[row] : 0.f;
            adv = a.advantages[i * a.adv_n + j * a.adv_s];
            coef_i = a.coef[i];
            own = label >= 0 && label < a.vocab ? Elem<T>::get(x[label]) : 0.f;
        }
        int edge = -1;                                          // head and tail of the row: at most one element a thread
        if (tid < now.head) edge = tid;
        else if (tid - N < tail && tid >= N) edge = now.head + now.vectors * N + tid - N;
        const float ex = edge >= 0 ? Elem<T>::get(x[edge]) : 0.f;
        Running<T, false, U, TPB> run;
        run.clear();
        if (edge >= 0) run.add_one(ex, 0.f);
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
            if (q == 0) copies_here<PARTS - 1>();
            else if (q == 1) copies_here<PARTS - 2>();
            else if (q == 2) copies_here<PARTS - 3>();
            else copies_here<0>();
            const int end = min((q + 1) * part, now.vectors);
            for (int base = q * part + tid; base < end; base += U * TPB) {
                uint4 xr[U], none[1];
                if (base + (U - 1) * TPB < end) {
#pragma unroll
                    for (int u = 0; u < U; ++u) xr[u] = xs[base + u * TPB];
                    run.add_vectors(xr, none, end - base, true);
                } else {
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (base + u * TPB < end) xr[u] = xs[base + u * TPB];
                    run.add_vectors(xr, none, end - base, false);
                }
            }
        }
        const float2 halves = parts(run.t);
        Sums<double> p{run.m, (double)halves.x + (double)halves.y};
        p.join_warp();
        if (tid % 32 == 0) ps[tid / 32] = p;
        __syncthreads();
        if (tid < 32) {
            const bool is = tid < TEAM;
            const float m = warp_max(is ? ps[tid].m : -FLT_MAX);
            const double t = warp_sum(is ? ps[tid].t * (double)exp_of_gap(ps[tid].m - m) : 0.0);
            if (tid == 0) {
                const double l = label_logp(a.vocab, label, own, m, t);
                const RowTerm r(a.kl, a.low, a.high, a.kl_beta, l, a.old_logp != nullptr, old, adv, a.ref_wide ? wide : (double)given,
                                0.0);
                const float slope = (float)(weight * r.slope), inv = __frcp_rn((float)t);
                const float coef = slope == 0.f ? 0.f : a.expected * coef_i * slope;    // as in the second reading
                grad = RowGrad{m, coef, -coef * inv};
                where = (int)label;                             // one that does not fit has made everything NaN
                a.row[row] = make_float2(m, inv);
                a.slope[row] = slope;
                a.logp[row] = (float)l;
                terms[0] = weight;
                terms[1] = weight * r.term * coef_i;
                terms[2] = weight * r.kl;
                terms[3] = r.clipped ? weight : 0.0;
            }
        }
        Place next = {};
        if (step + 1 < mine) next = place(block + (step + 1) * grid);
        write_others((int)((long long)others * (step + 1) / mine));
        __syncthreads();
        const RowGrad r = grad;
        const int hot = where;
        if (tid < 4) sums[tid] += terms[tid];
        request_wide(next);
        T* g = reinterpret_cast<T*>(a.g) + (long long)i * a.gn + (long long)j * a.gs;
        if ((((uintptr_t)x ^ (uintptr_t)g) & 15) != 0) {
            write_apart<T, TPB>(x, g, a.vocab, tid, r, hot);
#pragma unroll
            for (int q = 0; q < PARTS; ++q) {
                for (int v = q * part + tid; v < min((q + 1) * part, next.vectors); v += TPB) request(next, v);
                copies_sent();
            }
        } else {
            uint4* gv = reinterpret_cast<uint4*>(g + now.head);
            const int spot = hot - now.head;
            const bool own_it = spot >= 0 && spot < now.vectors * N && spot / N % TPB == tid;
            const float xl = own_it ? Elem<T>::get(x[hot]) : 0.f;
            const uint4* nv = reinterpret_cast<const uint4*>(next.x + next.head);
            const int both = min(now.vectors, next.vectors), most = max(now.vectors, next.vectors);
#pragma unroll
            for (int q = 0; q < PARTS; ++q) {
                int v = q * part + tid;
                for (; v + (U - 1) * TPB < min((q + 1) * part, both); v += U * TPB) {
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        __stcs(gv + v + u * TPB, grad_vector<T>(xs[v + u * TPB], r));
                        copy_16(xs + v + u * TPB, nv + v + u * TPB);
                    }
                }
                for (; v < min((q + 1) * part, most); v += TPB) {
                    if (v < now.vectors) __stcs(gv + v, grad_vector<T>(xs[v], r));
                    if (v < next.vectors) request(next, v);
                }
                copies_sent();
            }
            if (own_it) g[hot] = Elem<T>::put(grad_of<T, false>(xl, 0.f, r.m, r.scale, 0.f, 0.f) + r.coef);
            if (edge >= 0) {
                float f = grad_of<T, false>(ex, 0.f, r.m, r.scale, 0.f, 0.f);
                if (edge == hot) f += r.coef;
                g[edge] = Elem<T>::put(f);
            }
        }
        now = next;
    }
    copies_here<0>();
    write_others(others);
    if (tid < 4) a.parts[4 * block + tid] = sums[tid];
    if (last_block(a.order + rows + 1)) take_means<TPB>(a, reinterpret_cast<double(*)[4]>(raw_smem));
}

// How the gradient cuts a row: G threads with U loads each, for narrow vocabularies fewer of them, so that all have something to do.
struct GradPlan {
    int threads, splits, chunk;
    GradPlan(int vocab, int dtype, int u) {
        const int n = dtype == 1 ? 4 : 8;
        threads = 32;
        while (threads < THREADS && threads * u * n < vocab) threads *= 2;
        const int most = threads * u * n;
        splits = (vocab + most - 1) / most;
        chunk = splits == 1 ? vocab : ((vocab + splits - 1) / splits + 7) / 8 * 8;
    }
    bool fits(long long rows, int vocab) const { return rows * splits < (1ll << 31) && (splits - 1ll) * chunk < vocab; }
};

// Chunks of a row that there is room for: down to a vector a lane, 64 at most; and those for a batch that keeps all its rows, where
// the kernel cannot count them.
struct StatsPlan {
    int chunks = 1, most;
    StatsPlan(long long rows, int vocab, int dtype, int full) {
        const int n = dtype == 1 ? 4 : 8, least = 32 * n, step = least * Shape<true>::VECTORS / (full ? 2 : 1);
        const int warps = (full ? Shape<true>::WARPS : Shape<false>::WARPS) * neox_sm_count();
        most = (vocab + least - 1) / least;
        const int usual = (vocab + 2 * step - 1) / (2 * step);
        if (rows > 2ll * warps && most > usual) most = usual;   // a row of its own for every warp of the machine
        if (most > 64) most = 64;
        for (int c = 1; c <= most; ++c)
            if (cut_cost(rows, vocab, c, warps, step) < cut_cost(rows, vocab, chunks, warps, step)) chunks = c;
    }
};

#define FOR_TYPE(dtype, CALL)                                  \
    do {                                                       \
        if (dtype == 0) { using T = __nv_bfloat16; CALL; }     \
        else if (dtype == 1) { using T = float; CALL; }        \
        else { using T = __half; CALL; }                       \
    } while (0)

#define FOR_THREADS(threads, CALL)                                 \
    do {                                                           \
        if (threads == 32) { constexpr int G = 32; CALL; }         \
        else if (threads == 64) { constexpr int G = 64; CALL; }    \
        else if (threads == 128) { constexpr int G = 128; CALL; }  \
        else { constexpr int G = 256; CALL; }                      \
    } while (0)

// Rows of the policy loss in shared memory: as many blocks an SM as rows fit, at most eight, or none.
struct AtOncePlan {
    int places, blocks;
    size_t bytes;
    AtOncePlan(int vocab, int dtype) {
        places = vocab / (dtype == 1 ? 4 : 8) + 1;
        bytes = places < 64 ? 1024 : (size_t)places * 16;       // and the last block's sums
        blocks = bytes <= most(8) ? 8 : bytes <= most(4) ? 4 : bytes <= most(3) ? 3 : bytes <= most(2) ? 2 : bytes <= most(1) ? 1 : 0;
    }
    // of 228 KB an SM, with 1 KB and what the kernel has besides for every block
    static constexpr size_t most(int blocks) { return (228 * 1024 / blocks - 1536) / 1024 * 1024; }
};

template <typename T, int TPB, int BLOCKS>
int rows_at_once(const AtOnceArgs& a, const AtOncePlan& p, dim3 grid, cudaStream_t st) {
    if (!allow_dynamic_smem<policy_row_kernel<T, TPB, BLOCKS>>(AtOncePlan::most(BLOCKS))) return NEOX_ERR_LAUNCH;
    return launch::overlapped_with(policy_row_kernel<T, TPB, BLOCKS>, grid, dim3(TPB), p.bytes, st, a, p.places);
}

#define LAUNCH_STATS(T, FULL)                                                                             \
    if (!allow_dynamic_smem<stats_kernel<T, FULL>>(sizeof(StatsSmem<FULL>))) return NEOX_ERR_LAUNCH;      \
    stats_kernel<T, FULL><<<blocks, Shape<FULL>::WARPS * 32, sizeof(StatsSmem<FULL>), st>>>(a)

constexpr int U_ONE = 8, U_FULL = 4;
constexpr long long MOST_TOKENS = 1ll << 30;                    // row numbers and steps past the last one stay within 32 bits

int launched() { return cudaGetLastError() == cudaSuccess ? 0 : NEOX_ERR_LAUNCH; }

// One forward or backward call.  Some forty arguments, so they come packed (the caller's side is a struct format of the same
// order: 64-bit words, doubles, ints); addresses are null where an operator has no such tensor.
struct LossCall {
    const void* x;                 // logits [n, s, vocab], element strides of the first two
    long long xn, xs;
    const void* y;                 // reference logits, or null
    long long yn, ys;
    const long long* labels;
    const float* mask;
    Part* part;                    // scratch: [streams][n * s, most]
    float* target;                 // scratch: [streams][n * s]
    int* ticket;                   // scratch: 2
    double* sums;                  // scratch: [n * pieces + n, 2 or 4]
    float2* row;                   // kept for the backward: [n * s], [n], [n * s], [n * s]
    float* coef;
    float* slope;
    float* shift;                  // the KL over the vocabulary has one
    float* loss;
    float* kl_mean;
    float* clipped;
    float* logp;                   // [n] preference, [n, s] policy
    float* ref;                    // [n]
    const float* old_logp;
    const float* ref_logp;
    const float* advantages;       // element (i, j) at i * adv_n + j * adv_s
    long long adv_n, adv_s;
    void* g;                       // backward: gradient of the logits
    long long gn, gs;
    const float* g_loss;
    const float* g_logp;
    long long v0, whole;           // first word of this share of the vocabulary; words of all shares
    void* stream;
    float* terms;                  // scratch of the policy loss with its gradient: 4 doubles a block, n doubles, n * s + 2 ints
    double* wide;                  // [n, s] or null: log-probabilities in 64 bits, left by one forward and another's reference
    double beta, smoothing, low, high;       // beta: of the preference, or the KL's weight
    double expected;               // gradient of the loss that the forward writes its gradient for
    int n, s, vocab, dtype;
    int kl, by_sequence;
    int most, chunks;              // 0 chunks: as the statistics found
    int policy, first, second;     // which loss; whether to run the statistics and what joins them
    int done;                      // forward: loss and gradient at once; backward: that was done
};

}  // namespace

extern "C" {

// Chunks of a row that the statistics have room for.
int neox_vocab_chunks(long long rows, int vocab, int dtype, int full) {
    const StatsPlan p(rows, vocab, dtype, full);
    return p.most;
}

// Blocks that join a sequence's rows.
int neox_loss_pieces(int s) { return s > 0 ? (s + ROWS - 1) / ROWS : 1; }

int neox_loss_forward(const void* packed) {
    const LossCall& c = *(const LossCall*)packed;
    const bool full = c.shift != nullptr;
    const long long rows = (long long)c.n * c.s, pieces = neox_loss_pieces(c.s);
    const int streams = !full && c.y ? 2 : 1;
    if (c.n < (c.policy ? 1 : 2) || (!c.policy && c.n % 2) || c.s < 0 || c.vocab < 1 || (full && !c.y)) return NEOX_ERR_SHAPE;
    if (rows >= MOST_TOKENS || rows * streams * c.most >= (1ll << 31) || c.n * pieces >= (1ll << 31)) return NEOX_ERR_TOO_LARGE;
    cudaStream_t st = (cudaStream_t)c.stream;
    if (c.first) {
        const StatsPlan p(rows, c.vocab, c.dtype, full);
        if (p.most != c.most) return NEOX_ERR_SHAPE;
        const StatsArgs a = {{c.x, c.xn, c.xs}, {c.y, c.yn, c.ys}, c.labels, c.mask, c.part, c.target, c.ticket, c.v0,
                             (int)rows, c.s, c.vocab, streams, p.chunks, p.most};
        const int blocks = neox_sm_count();
        if (full) FOR_TYPE(c.dtype, LAUNCH_STATS(T, true));
        else FOR_TYPE(c.dtype, LAUNCH_STATS(T, false));
        if (launched() != 0) return NEOX_ERR_LAUNCH;
    }
    if (!c.second) return 0;
    const RowSums sums = {c.part, c.target, c.labels, c.ticket, c.whole, (int)rows, c.most, c.chunks};
    const dim3 grid((unsigned)(c.n * pieces));
    if (c.policy) {
        const PolicyArgs a = {sums, c.mask, c.advantages, c.adv_n, c.adv_s, c.old_logp, c.ref_logp, c.y != nullptr, c.n, c.s,
                              (int)pieces, c.kl, c.by_sequence, c.low, c.high, c.beta, c.row, c.slope, c.shift, c.sums, c.ticket,
                              c.loss, c.kl_mean, c.clipped, c.logp, c.wide, c.coef};
        return launch::overlapped(policy_kernel, grid, dim3(THREADS), 1, st, a);
    }
    const PreferenceArgs a = {sums, c.mask, c.ref_logp, c.y != nullptr, c.n, c.s, (int)pieces, c.beta, c.smoothing, c.row, c.sums,
                              c.ticket, c.loss, c.logp, c.ref, c.coef};
    return launch::overlapped(preference_kernel, grid, dim3(THREADS), 1, st, a);
}

// Whether a row of that many words fits in shared memory.
int neox_policy_fits(int vocab, int dtype) { return AtOncePlan(vocab, dtype).blocks > 0; }

// The policy loss, without reference logits and over a whole vocabulary, together with its gradient for `expected`.
int neox_policy_at_once(const void* packed) {
    const LossCall& c = *(const LossCall*)packed;
    const long long rows = (long long)c.n * c.s;
    const AtOncePlan p(c.vocab, c.dtype);
    if (c.n < 1 || c.s < 1 || c.vocab < 1 || c.y || c.kl == KL_FULL || p.blocks == 0) return NEOX_ERR_SHAPE;
    if (rows >= MOST_TOKENS) return NEOX_ERR_TOO_LARGE;
    double* whole = (double*)c.terms + 4 * (rows < MOST_PARTS ? rows : MOST_PARTS);
    const AtOnceArgs a = {{c.x, c.xn, c.xs}, c.g, c.gn, c.gs, c.labels, c.mask, c.advantages, c.adv_n, c.adv_s, c.old_logp,
                          c.ref_logp, c.wide, c.n, c.s, c.vocab, c.kl, c.by_sequence, c.low, c.high, c.beta, (float)c.expected, c.row, c.slope,
                          (double*)c.terms, whole, (int*)(whole + c.n), c.coef, c.loss, c.kl_mean, c.clipped, c.logp};
    cudaStream_t st = (cudaStream_t)c.stream;
    policy_share_kernel<<<1, 1024, 0, st>>>(a);
    if (launched() != 0) return NEOX_ERR_LAUNCH;
    const long long fit = (long long)p.blocks * neox_sm_count(), most = fit < MOST_PARTS ? fit : MOST_PARTS;
    const dim3 grid((unsigned)(rows < most ? rows : most));
    int rc = 0;
    // threads: 32 short of what registers would hold or more, where the compiler then keeps more loads under way (4 x 8192 tokens over
    // 32064 words: 665 us with 320, 600 with 256; 8 x 1024 over 50304: 248 with 512, 241 with 384; over 100000: 501 with 768, 476 with 640)
    if (p.blocks == 8) FOR_TYPE(c.dtype, (rc = rows_at_once<T, 128, 8>(a, p, grid, st)));
    else if (p.blocks == 4) FOR_TYPE(c.dtype, (rc = rows_at_once<T, 256, 4>(a, p, grid, st)));
    else if (p.blocks == 3) FOR_TYPE(c.dtype, (rc = rows_at_once<T, 256, 3>(a, p, grid, st)));
    else if (p.blocks == 2) FOR_TYPE(c.dtype, (rc = rows_at_once<T, 384, 2>(a, p, grid, st)));
    else FOR_TYPE(c.dtype, (rc = rows_at_once<T, 640, 1>(a, p, grid, st)));
    return rc;
}

int neox_loss_backward(const void* packed) {
    const LossCall& c = *(const LossCall*)packed;
    const bool full = c.shift != nullptr;
    if (c.n < 0 || c.s < 0 || c.vocab < 1) return NEOX_ERR_SHAPE;
    const GradPlan p(c.vocab, c.dtype, full ? U_FULL : U_ONE);
    const long long rows = (long long)c.n * c.s;
    if (rows == 0) return 0;
    if (!p.fits(rows, c.vocab)) return NEOX_ERR_TOO_LARGE;
    const GradArgs a = {{c.x, c.xn, c.xs}, {c.y, c.yn, c.ys}, c.g, c.gn, c.gs, c.labels, c.slope, c.mask, c.shift, c.row, c.coef,
                        c.g_loss, c.g_logp, c.v0, (float)c.beta, (float)c.expected, (int)rows, c.s, c.vocab, p.splits,
                        p.chunk};
    const long long per = THREADS / p.threads;
    const long long items = rows * p.splits, need = (items + per - 1) / per;
    cudaStream_t st = (cudaStream_t)c.stream;
    if (c.done) {
        if (full || !c.g_loss) return NEOX_ERR_SHAPE;
        const long long few = 8ll * neox_sm_count();
        const unsigned grid = (unsigned)(need < few ? need : few);
        FOR_TYPE(c.dtype, FOR_THREADS(p.threads, (grad_unless_kernel<T, G, U_ONE><<<grid, THREADS, 0, st>>>(a, (unsigned)items))));
        return launched();
    }
    const unsigned grid = (unsigned)need;
    if (full) FOR_TYPE(c.dtype, FOR_THREADS(p.threads, (grad_kernel<T, G, U_FULL, true><<<grid, THREADS, 0, st>>>(a))));
    else FOR_TYPE(c.dtype, FOR_THREADS(p.threads, (grad_kernel<T, G, U_ONE, false><<<grid, THREADS, 0, st>>>(a))));
    return launched();
}

}  // extern "C"
