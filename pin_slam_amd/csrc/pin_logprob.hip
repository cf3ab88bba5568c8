// pin_logprob.hip -- log probabilities of given labels, with each row's entropy and its k most
// probable classes, and the gradient with respect to the logits.  Beside the reference's
// classification head (model/decoder.py:120, log_softmax and argmax).
//
// For a row z of C logits with label y:
//   m = max z,  d_j = z_j - m,  s = sum_j e^d_j,  log p_j = d_j - log s
//   log_prob = log p_y                       entropy H = log s - (sum_j e^d_j d_j) / s
// Both terms of H are >= 0 (d_j <= 0), so it loses nothing to cancellation.
//   d log_prob / d z_j = [j = y] - p_j       d H / d z_j = -p_j (log p_j + H)
// A class at -inf has p = 0 and adds nothing to any sum.  A row whose logits are all -inf has no
// distribution: log_prob -inf, entropy 0, gradient 0.  A row with a NaN or +inf logit: NaN, and -1
// for the classes.  Sums and statistics are f32 whatever the logits' type.
//
// The exponentials are taken to base 2: x_j = z_j L - fl(m L), L = log2 e, in one fma.  fl(m L)
// shifts every x_j of a row alike, and every result is a difference of such, so its rounding
// cancels.  Where m L leaves the range of f32 (rows masked by the type's lowest value throughout)
// x_j = (z_j - m) L.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "pin_slam_amd.h"

namespace {

constexpr float kInf = __builtin_huge_valf();
constexpr float kL = 1.44269504f, kLn2 = 0.693147182f;
constexpr float kFloor = -1000.f;            // 2^x is 0 well above
constexpr int kSmall = 64;                   // most classes of the kernels of one thread per row
constexpr int kSplits = 64;                  // most parts of a row

inline hipStream_t as_stream(void* s) { return (hipStream_t)s; }
inline int launch_status() { return hipGetLastError() == hipSuccess ? PIN_OK : PIN_ERR_HIP; }

// ---- types: sixteen bytes of logits as f32, and back

struct F32 {
    typedef float type;
    static constexpr int N = 4;
    static constexpr uint32_t kFill = 0xFF800000u;   // -inf in every element
    static __device__ __forceinline__ void unpack(const uint4& q, float (&o)[4]) {
        o[0] = __uint_as_float(q.x), o[1] = __uint_as_float(q.y), o[2] = __uint_as_float(q.z), o[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    static __device__ __forceinline__ float one(const float* p) { return *p; }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};

struct F16 {
    typedef _Float16 type;
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    static constexpr int N = 8;
    static constexpr uint32_t kFill = 0xFC00FC00u;
    static __device__ __forceinline__ void unpack(const uint4& q, float (&o)[8]) {
        const v8 h = __builtin_bit_cast(v8, q);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (float)h[i];
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
        v8 h;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = (_Float16)v[i];
        return __builtin_bit_cast(uint4, h);
    }
    static __device__ __forceinline__ float one(const _Float16* p) { return (float)*p; }
    static __device__ __forceinline__ void put(_Float16* p, float v) { *p = (_Float16)v; }
};

struct BF16 {
    typedef uint16_t type;
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    static constexpr int N = 8;
    static constexpr uint32_t kFill = 0xFF80FF80u;
    static __device__ __forceinline__ void unpack(const uint4& q, float (&o)[8]) {
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[2 * i] = __uint_as_float(u[i] << 16);
            o[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
        v8 h;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = (__bf16)v[i];
        return __builtin_bit_cast(uint4, h);
    }
    static __device__ __forceinline__ float one(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
    static __device__ __forceinline__ void put(uint16_t* p, float v) {
        *p = __builtin_bit_cast(uint16_t, (__bf16)v);
    }
};

// sixteen bytes at any element's address (the hardware takes unaligned vectors)
template <class T>
__device__ __forceinline__ uint4 load16(const typename T::type* p) {
    uint4 q;
    __builtin_memcpy(&q, p, 16);
    return q;
}
template <class T>
__device__ __forceinline__ void store16(typename T::type* p, const uint4& q) {
    __builtin_memcpy(p, &q, 16);
}
// the elements [0, n) of sixteen bytes, n < N; the others -inf
template <class T>
__device__ __forceinline__ uint4 load_some(const typename T::type* p, int n) {
    uint32_t u[4] = {T::kFill, T::kFill, T::kFill, T::kFill};
    if (sizeof(typename T::type) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) __builtin_memcpy(&u[i], (const char*)p + 4 * i, 4);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) {
                uint16_t h;
                __builtin_memcpy(&h, (const char*)p + 2 * i, 2);
                u[i / 2] = i & 1 ? (u[i / 2] & 0xFFFFu) | (uint32_t)h << 16 : (u[i / 2] & 0xFFFF0000u) | h;
            }
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// The registers as they are, but unknown to the compiler: what was made of them before is made
// again (two instructions an element) rather than kept beside them (a register an element).
__device__ __forceinline__ void forget(uint4& q) { asm volatile("" : "+v"(q.x), "+v"(q.y), "+v"(q.z), "+v"(q.w)); }

__device__ __forceinline__ int forget(int j) {
    asm volatile("" : "+v"(j));
    return j;
}

// ---- order: f32 values as unsigned keys in the same order, both zeros the same

__device__ __forceinline__ uint32_t order_key(float v) {
    const int32_t b = __float_as_int(v + 0.0f);
    return (uint32_t)(b < 0 ? ~b : b | (int32_t)0x80000000);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
// value and class, larger first, of equal values the lower class first; never 0
__device__ __forceinline__ uint64_t class_key(float v, uint32_t j) { return (uint64_t)order_key(v) << 32 | (uint32_t)~j; }

// ---- across the lanes of a wave

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xF, 0xF, false);
}
template <class F>
__device__ __forceinline__ uint32_t rows_of_16(uint32_t v, F f) {
    v = f(v, dpp<0xB1>(v));    // lanes ^ 1
    v = f(v, dpp<0x4E>(v));    // lanes ^ 2
    v = f(v, dpp<0x141>(v));   // the other half of 8
    return f(v, dpp<0x140>(v));   // the other half of 16
}
template <class F>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t v, F f) {
    v = rows_of_16(v, f);
    const uint32_t a = f(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
    const uint32_t b = f(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48));
    return f(a, b);
}
struct MaxF {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }
};
struct AddF {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }
};
struct MaxU {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};
__device__ __forceinline__ float wave_max(float v) { return __uint_as_float(wave_reduce(__float_as_uint(v), MaxF())); }
__device__ __forceinline__ float wave_sum(float v) { return __uint_as_float(wave_reduce(__float_as_uint(v), AddF())); }
__device__ __forceinline__ uint64_t wave_max_key(uint64_t k) {
    const uint32_t h = wave_reduce((uint32_t)(k >> 32), MaxU());
    const uint32_t l = wave_reduce((uint32_t)(k >> 32) == h ? (uint32_t)k : 0u, MaxU());
    return (uint64_t)h << 32 | l;
}

// a maximum that a NaN does not pass unseen
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// ---- a row's statistics

struct Row {
    float m, ls;   // maximum (+inf: the row has a NaN or +inf; -inf: nothing in it), log2 of the sum
    float ml;      // fl(m L), where that is finite
    bool far;      // it is not
    __device__ __forceinline__ explicit Row(float max) : m(max), ls(0.f), ml(max * kL), far(!(fabsf(max) <= 0x1p127f)) {}
    __device__ __forceinline__ bool bad() const { return m == kInf; }
    __device__ __forceinline__ bool dead() const { return m == -kInf; }
    __device__ __forceinline__ float x(float z) const { return far ? (z - m) * kL : fmaf(z, kL, -ml); }
    __device__ __forceinline__ float log_prob(float z) const {
        const float v = (x(z) - ls) * kLn2;
        // where only z L is out of range: log s is nothing beside z - m
        return bad() ? NAN : dead() ? -kInf : v == -kInf ? z - m : v;
    }
};

__device__ __forceinline__ float label_log_prob(const Row& r, float z, int64_t y, int64_t ignore, int64_t classes) {
    return y == ignore ? 0.f : y < 0 || y >= classes ? NAN : r.log_prob(z);
}
__device__ __forceinline__ float row_entropy(const Row& r, float s, float t) {
    return r.bad() ? NAN : r.dead() ? 0.f : (r.ls - t / s) * kLn2;
}

// what is written of a row
struct Out {
    float* log_prob;
    float* entropy;
    float2* stats;      // may be NULL; maximum and log2 of the sum
    float* top_lp;
    int64_t* top_idx;
};

__device__ __forceinline__ void put_top(const Out& o, const Row& r, int64_t at, uint64_t key) {
    o.top_lp[at] = r.log_prob(key_value((uint32_t)(key >> 32)));
    o.top_idx[at] = r.bad() ? -1 : (int64_t)(uint32_t)~(uint32_t)key;
}

// One part of a row, THREADS * NCH vectors of 16 bytes held in registers.
//
//   1. load; maxima of vectors, threads and of 64 groups of threads
//   2. the maximum; sum of 2^x and of 2^x x
//   3. the k-th largest of the 64 maxima is not above the k-th largest element: what is above or
//      at it, a little more than k, is collected in LDS and sorted by one wave
// At most kGt larger and kEq equal elements fit.  More equal ones (rows mostly masked, or all
// equal): the first k are found in order.  More larger ones (large values gathered in the
// classes of few threads): k times the largest below the last.
template <class T, int THREADS, int NCH, bool TOP>
__global__ void __launch_bounds__(THREADS, THREADS == 1024 ? 8 : 4)
k_label_logprob(const typename T::type* __restrict__ logits, int64_t n, int64_t classes, int64_t row_stride,
                const int64_t* __restrict__ labels, int64_t ignore, int k, int splits, int64_t part, Out out,
                float4* __restrict__ sums, uint64_t* __restrict__ keys) {
    constexpr int V = T::N, W = THREADS / 64;
    constexpr int kGt = TOP ? 4 * THREADS : 1, kEq = TOP ? 256 : 1;
    __shared__ float s_max[64];
    __shared__ float2 s_sum[W];
    __shared__ uint32_t s_kth, s_gt, s_eq, s_tot[W];
    __shared__ uint64_t s_gtk[kGt], s_eqk[kEq];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / (unsigned)splits;
    const int split = (int)(blockIdx.x - (unsigned)row * (unsigned)splits);
    const int64_t first = split * part;
    const int count = (int)(classes - first < part ? classes - first : part);   // elements of this part (may be <= 0)
    const typename T::type* z = logits + row * row_stride + first;

    uint4 q[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int j = (c * THREADS + tid) * V;
        if (j + V <= count) q[c] = load16<T>(z + j);
        else if (j < count) q[c] = load_some<T>(z + j, count - j);
        else q[c] = make_uint4(T::kFill, T::kFill, T::kFill, T::kFill);
    }
    int64_t y = 0;
    float zy = 0.f;
    if (splits == 1 && tid == 0) {
        y = labels[row];
        if (y >= 0 && y < classes) zy = T::one(z + y);
    }
    float cm[NCH], mx = -kInf;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        float v[V];
        T::unpack(q[c], v);
        cm[c] = v[0];
#pragma unroll
        for (int i = 1; i < V; ++i) cm[c] = max_nan(cm[c], v[i]);
        mx = max_nan(mx, cm[c]);
    }
    mx = mx != mx ? kInf : mx;
    // maxima of 64 groups: threads, or the lanes of 4, or of 16
    float g = mx;
    if (THREADS >= 256) {
        g = fmaxf(g, __uint_as_float(dpp<0xB1>(__float_as_uint(g))));
        g = fmaxf(g, __uint_as_float(dpp<0x4E>(__float_as_uint(g))));
    }
    if (THREADS >= 1024) {
        g = fmaxf(g, __uint_as_float(dpp<0x141>(__float_as_uint(g))));
        g = fmaxf(g, __uint_as_float(dpp<0x140>(__float_as_uint(g))));
    }
    if (THREADS > 64) {
        if (tid % (THREADS / 64) == 0) s_max[tid / (THREADS / 64)] = g;
        if (TOP && tid == 0) s_gt = 0, s_eq = 0;
        __syncthreads();
        g = s_max[lane];
    } else if (TOP && tid == 0) {
        s_gt = 0, s_eq = 0;
    }
    Row r(wave_max(g));
    if (TOP && wave == 0) {
        // the k-th largest of the groups' maxima, bit by bit
        const uint32_t key = order_key(g);
        uint32_t kth = 0;
#pragma unroll 1
        for (int b = 31; b >= 0; --b) {
            const uint32_t c = kth | 1u << b;
            if (__popcll(__ballot(key >= c)) >= k) kth = c;
        }
        if (lane == 0) s_kth = kth;
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c) forget(q[c]);
    float s = 0.f, t = 0.f;
    const auto add = [&](auto x_of) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            float v[V];
            T::unpack(q[c], v);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float x = fmaxf(x_of(v[i]), kFloor);
                const float e = __builtin_amdgcn_exp2f(x);
                s += e;
                t = fmaf(e, x, t);
            }
        }
    };
    if (!r.far) add([&](float z) { return fmaf(z, kL, -r.ml); });
    else add([&](float z) { return (z - r.m) * kL; });
    s = wave_sum(s);
    t = wave_sum(t);
    if (THREADS > 64) {
        if (lane == 0) s_sum[wave] = make_float2(s, t);
        __syncthreads();
        if (wave == 0) {
            s = t = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) s += s_sum[w].x, t += s_sum[w].y;
        }
    } else if (TOP) {
        __syncthreads();
    }
    r.ls = __builtin_amdgcn_logf(s);   // s >= 1 unless there is nothing
    if (r.dead()) r.ls = 0.f;
    const bool whole = splits == 1;
    if (tid == 0) {
        if (whole) {
            out.log_prob[row] = label_log_prob(r, zy, y, ignore, classes);
            out.entropy[row] = row_entropy(r, s, t);
            if (out.stats) out.stats[row] = make_float2(r.m, r.ls);
        } else {
            sums[blockIdx.x] = make_float4(r.m, s, t, 0.f);
        }
    }
    if (!TOP) return;
    const int64_t at = (int64_t)blockIdx.x * k;   // of the row's outputs, or of the part's keys
    const auto emit = [&](int i, uint64_t key) {
        if (whole) put_top(out, r, at + i, key);
        else keys[at + i] = key;
    };
    if (r.bad()) {
        if (tid < k) emit(tid, 0);
        return;
    }
    const float kth = key_value(s_kth);
#pragma unroll
    for (int c = 0; c < NCH; ++c) forget(q[c]);
    if (mx >= kth) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            if (cm[c] >= kth) {
                float v[V];
                T::unpack(q[c], v);
                const int j = forget((c * THREADS + tid) * V);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (v[i] > kth) {
                        const uint32_t p = atomicAdd(&s_gt, 1u);
                        if (p < kGt) s_gtk[p] = class_key(v[i], (uint32_t)(first + j + i));
                    } else if (v[i] == kth && j + i < count) {
                        const uint32_t p = atomicAdd(&s_eq, 1u);
                        if (p < kEq) s_eqk[p] = class_key(v[i], (uint32_t)(first + j + i));
                    }
                }
            }
        }
    }
    __syncthreads();
    const int gt = (int)s_gt;
    int eq = gt >= k ? 0 : (int)s_eq;
    // what is rare reads the part again
    if (gt > kGt) {
        uint64_t last = ~0ull;
        for (int i = 0; i < k; ++i) {
            uint64_t best = 0;
#pragma unroll 1
            for (int j = tid; j < count; j += THREADS) {
                const uint64_t key = class_key(T::one(z + j), (uint32_t)(first + j));
                if (key < last && key > best) best = key;
            }
            best = wave_max_key(best);
            __syncthreads();
            if (lane == 0) s_gtk[wave] = best;
            __syncthreads();
            for (int w = 0; w < W; ++w) best = s_gtk[w] > best ? s_gtk[w] : best;
            last = best;
            if (tid == 0) emit(i, best);
        }
        return;
    }
    if (eq > kEq) {
        const int need = k - gt;
        int have = 0;
        __syncthreads();
#pragma unroll 1
        for (int j0 = 0; j0 < count && have < need; j0 += THREADS) {
            const int j = j0 + tid;
            const float v = j < count ? T::one(z + j) : NAN;
            const uint64_t b = __ballot(v == kth);
            int at = have + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
            if (lane == 0) s_tot[wave] = __popcll(b);
            __syncthreads();
            for (int w = 0; w < W; ++w) {
                at += w < wave ? (int)s_tot[w] : 0;
                have += (int)s_tot[w];
            }
            if (v == kth && at < need) s_eqk[at] = class_key(v, (uint32_t)(first + j));
            __syncthreads();
        }
        eq = have < need ? have : need;
    }
    if (wave != 0) return;
    const int all = gt + eq;
    if (all <= 64) {
        const uint64_t key = lane < gt ? s_gtk[lane] : lane < all ? s_eqk[lane - gt] : 0;
        int rank = 0;
        for (int i = 0; i < all; ++i) {
            const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), i) << 32 |
                                   (uint32_t)__builtin_amdgcn_readlane((int)key, i);
            rank += other > key ? 1 : 0;
        }
        if (lane < all && rank < k) emit(rank, key);
        if (lane >= all && lane < k) emit(lane, 0);   // a part of fewer than k classes
        return;
    }
    uint64_t last = ~0ull;
    for (int i = 0; i < k; ++i) {
        uint64_t best = 0;
        for (int p = lane; p < all; p += 64) {
            const uint64_t key = p < gt ? s_gtk[p] : s_eqk[p - gt];
            if (key < last && key > best) best = key;
        }
        last = wave_max_key(best);
        if (lane == 0) emit(i, last);
    }
}

// The parts of a row joined, one wave per row, one lane per part: the sums are taken to the row's
// maximum, and the parts' sorted keys are merged.
template <class T>
__global__ void __launch_bounds__(64)
k_label_join(const typename T::type* __restrict__ logits, int64_t classes, int64_t row_stride,
             const int64_t* __restrict__ labels, int64_t ignore, int k, int splits, Out out,
             const float4* __restrict__ sums, const uint64_t* __restrict__ keys) {
    extern __shared__ uint64_t s_keys[];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    for (int i = lane; i < splits * k; i += 64) s_keys[i] = keys[row * splits * k + i];
    const int64_t y = labels[row];
    const float zy = y >= 0 && y < classes ? T::one(logits + row * row_stride + y) : 0.f;
    const float4 p = lane < splits ? sums[row * splits + lane] : make_float4(-kInf, 0.f, 0.f, 0.f);
    Row r(wave_max(p.x));
    const float x = fmaxf(r.far ? (p.x - r.m) * kL : p.x * kL - r.ml, kFloor);
    const float f = __builtin_amdgcn_exp2f(x);
    const float s = wave_sum(f * p.y), t = wave_sum(f * fmaf(p.y, x, p.z));
    r.ls = r.dead() ? 0.f : __builtin_amdgcn_logf(s);
    if (lane == 0) {
        out.log_prob[row] = label_log_prob(r, zy, y, ignore, classes);
        out.entropy[row] = row_entropy(r, s, t);
        if (out.stats) out.stats[row] = make_float2(r.m, r.ls);
    }
    if (k == 0) return;
    __syncthreads();
    int next = 0;
    uint64_t head = lane < splits ? s_keys[lane * k] : 0;
    for (int i = 0; i < k; ++i) {
        const uint64_t best = wave_max_key(head);
        if (lane == 0) put_top(out, r, row * k + i, best);
        if (head == best && lane < splits) {
            ++next;
            head = next < k ? s_keys[lane * k + next] : 0;
        }
    }
}

// Few classes: one thread per row, the workgroup's rows staged through LDS as f32 (an odd pitch:
// consecutive rows begin in different banks).
template <class T, int ROWS>
__device__ __forceinline__ void stage_rows(const typename T::type* __restrict__ logits, int64_t row0, int rows, int classes,
                                           uint32_t magic, int64_t row_stride, float* s_z) {
    const int pitch = classes | 1, all = rows * classes;
    const typename T::type* z = logits + row0 * row_stride;
    for (int e = threadIdx.x; e < all; e += ROWS) {
        const int i = (int)((uint32_t)e * magic >> 20), j = e - i * classes;
        s_z[i * pitch + j] = T::one(z + i * row_stride + j);
    }
    __syncthreads();
}

template <class T, int ROWS>
__global__ void __launch_bounds__(ROWS)
k_label_small(const typename T::type* __restrict__ logits, int64_t n, int classes, uint32_t magic, int64_t row_stride,
              const int64_t* __restrict__ labels, int64_t ignore, int k, Out out) {
    extern __shared__ float s_z[];
    const int64_t row0 = (int64_t)blockIdx.x * ROWS;
    const int rows = (int)(n - row0 < ROWS ? n - row0 : ROWS);
    stage_rows<T, ROWS>(logits, row0, rows, classes, magic, row_stride, s_z);
    if ((int)threadIdx.x >= rows) return;
    const float* z = s_z + threadIdx.x * (classes | 1);
    const int64_t row = row0 + threadIdx.x, y = labels[row];
    float m = -kInf;
    for (int j = 0; j < classes; ++j) m = max_nan(m, z[j]);
    Row r(m != m ? kInf : m);
    float s = 0.f, t = 0.f;
    for (int j = 0; j < classes; ++j) {
        const float x = fmaxf(r.x(z[j]), kFloor), e = __builtin_amdgcn_exp2f(x);
        s += e;
        t = fmaf(e, x, t);
    }
    r.ls = r.dead() ? 0.f : __builtin_amdgcn_logf(s);
    out.log_prob[row] = label_log_prob(r, y >= 0 && y < classes ? z[y] : 0.f, y, ignore, classes);
    out.entropy[row] = row_entropy(r, s, t);
    if (out.stats) out.stats[row] = make_float2(r.m, r.ls);
    float last = kInf;
    int last_j = -1;
    for (int i = 0; i < k; ++i) {   // the largest behind the last one, the first of equal ones
        float best = -kInf;
        int best_j = classes;
        for (int j = 0; j < classes; ++j) {
            const float v = z[j];
            if ((v < last || (v == last && j > last_j)) && (best_j == classes || v > best)) best = v, best_j = j;
        }
        out.top_lp[row * k + i] = r.log_prob(best);
        out.top_idx[row * k + i] = r.bad() ? -1 : best_j;
        last = best;
        last_j = best_j;
    }
}

// ---- the gradient: dz_j = -p_j (G + g_H (log p_j + H)) + the given terms

struct Grads {
    const float* lp;    // each may be NULL
    const float* ent;
    const float* top;
};

struct RowGrad {
    Row r;
    float lp, h, gh, g;   // the label's own term, H log2 e, g_H ln 2, G
    __device__ __forceinline__ RowGrad(const float2* stats, const float* entropy, const Grads& u, int64_t row, int64_t y,
                                       int64_t ignore, int64_t classes, int k)
        : r(stats[row].x) {
        r.ls = stats[row].y;
        lp = u.lp && y != ignore ? (y < 0 || y >= classes ? NAN : u.lp[row]) : 0.f;
        gh = u.ent ? u.ent[row] * kLn2 : 0.f;
        h = entropy[row] * kL;
        g = lp;
        if (u.top)
            for (int i = 0; i < k; ++i) g += u.top[row * k + i];
    }
    // without the given terms
    __device__ __forceinline__ float dz(float z) const {
        const float x = fmaxf(r.x(z) - r.ls, kFloor);
        return -__builtin_amdgcn_exp2f(x) * fmaf(gh, x + h, g);
    }
    __device__ __forceinline__ float value(float z) const { return r.dead() ? 0.f : r.bad() ? NAN : dz(z); }
};

// LANES threads per row (a part of it, gridDim.y of them), vectors of 16 bytes
template <class T, int LANES>
__global__ void __launch_bounds__(256)
k_label_bwd(const typename T::type* __restrict__ logits, int64_t n, int64_t classes, int64_t row_stride,
            const int64_t* __restrict__ labels, int64_t ignore, int k, const int64_t* __restrict__ top_idx,
            const float2* __restrict__ stats, const float* __restrict__ entropy, Grads u, int64_t part,
            typename T::type* __restrict__ out) {
    constexpr int V = T::N;
    const int lane = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const bool on = row < n;
    const int64_t first = blockIdx.y * part;
    const int64_t end = first + part < classes ? first + part : classes;
    const typename T::type* z = logits + (on ? row : 0) * row_stride;
    typename T::type* o = out + (on ? row : 0) * classes;
    const int64_t y = on ? labels[row] : ignore;
    const RowGrad d(stats, entropy, u, on ? row : 0, y, ignore, classes, k);
    const bool plain = !d.r.far && !d.r.bad() && !d.r.dead();
    if (on) {
        for (int64_t j = first + lane * V; j < end; j += LANES * V) {
            if (j + V <= end && plain) {
                float v[V];
                T::unpack(load16<T>(z + j), v);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float x = fmaxf(fmaf(v[i], kL, -d.r.ml) - d.r.ls, kFloor);
                    v[i] = -__builtin_amdgcn_exp2f(x) * fmaf(d.gh, x + d.h, d.g);
                }
                store16<T>(o + j, T::pack(v));
            } else {
                for (int64_t i = j; i < j + V && i < end; ++i) T::put(o + i, d.value(T::one(z + i)));
            }
        }
    }
    if (!u.top && !u.lp) return;
    __syncthreads();   // behind the stores of the others
    if (!on || d.r.dead()) return;
    // the given terms: the label's and the alternatives', the first of equal classes takes them all
    for (int i = lane; i <= k; i += LANES) {
        const int64_t j = i < k ? (u.top ? top_idx[row * k + i] : -1) : y == ignore ? -1 : y;
        if (j < first || j >= end) continue;
        if (i == k && u.top) {
            bool taken = false;
            for (int e = 0; e < k; ++e) taken |= top_idx[row * k + e] == j;
            if (taken) continue;
        }
        float more = i < k ? u.top[row * k + i] : d.lp;
        if (i < k && y == j) more += d.lp;
        T::put(o + j, d.value(T::one(z + j)) + more);
    }
}

template <class T, int ROWS>
__global__ void __launch_bounds__(ROWS)
k_label_bwd_small(const typename T::type* __restrict__ logits, int64_t n, int classes, uint32_t magic, int64_t row_stride,
                  const int64_t* __restrict__ labels, int64_t ignore, int k, const int64_t* __restrict__ top_idx,
                  const float2* __restrict__ stats, const float* __restrict__ entropy, Grads u,
                  typename T::type* __restrict__ out) {
    extern __shared__ float s_z[];
    const int64_t row0 = (int64_t)blockIdx.x * ROWS;
    const int rows = (int)(n - row0 < ROWS ? n - row0 : ROWS);
    stage_rows<T, ROWS>(logits, row0, rows, classes, magic, row_stride, s_z);
    const int pitch = classes | 1;
    if ((int)threadIdx.x < rows) {
        const int64_t row = row0 + threadIdx.x, y = labels[row];
        const RowGrad d(stats, entropy, u, row, y, ignore, classes, k);
        float* z = s_z + threadIdx.x * pitch;
        for (int j = 0; j < classes; ++j) z[j] = d.value(z[j]);
        if (!d.r.dead()) {
            if (y != ignore && y >= 0 && y < classes) z[y] += d.lp;
            if (u.top && !d.r.bad())
                for (int i = 0; i < k; ++i) z[top_idx[row * k + i]] += u.top[row * k + i];
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * classes; e += ROWS) {
        const int i = (int)((uint32_t)e * magic >> 20), j = e - i * classes;
        T::put(out + row0 * classes + e, s_z[i * pitch + j]);
    }
}

// ---- host

bool bad_args(const void* logits, int32_t dtype, int64_t n, int64_t classes, int64_t row_stride, const int64_t* labels,
              int32_t k) {
    if (dtype < PIN_TYPE_F32 || dtype > PIN_TYPE_BF16 || n < 0 || classes < 1 || classes > PIN_LABEL_CLASSES_MAX ||
        row_stride < 0 || k < 0 || k > PIN_LABEL_TOP_MAX || k > classes)
        return true;
    return n > 0 && (!logits || !labels || ((uintptr_t)logits & (dtype == PIN_TYPE_F32 ? 3 : 1)));
}

// How a forward is laid out: threads and vectors per thread of a workgroup, parts per row.
struct Plan {
    int threads, nch, splits;
    int64_t part;
};

constexpr int64_t kFull = 512;   // workgroups that fill the chip

Plan plan_rows(int64_t n, int64_t classes, int v) {
    Plan p{64, 1, 1, classes};
    const int64_t vecs = (classes + v - 1) / v;
    if (vecs <= 64 * 8) {
        while (64 * p.nch < vecs) p.nch *= 2;
        return p;
    }
    p.threads = vecs <= 256 * 8 ? 256 : 1024;
    p.nch = 8;
    if (p.threads == 256 && vecs <= 256 * 4) p.nch = 4;
    if (p.threads == 1024 && vecs <= 1024 * 4) p.nch = 4;
    int64_t s = (vecs + (int64_t)p.threads * p.nch - 1) / ((int64_t)p.threads * p.nch);
    if (n * s < kFull && vecs > 256 * 4) {   // few rows: smaller workgroups and more parts
        p.threads = 256;
        p.nch = 4;
        s = (vecs + 256 * 4 - 1) / (256 * 4);
        if (s > kSplits) {
            p.nch = 8;
            s = (vecs + 256 * 8 - 1) / (256 * 8);
        }
        if (s > kSplits) {
            p.threads = 1024;
            s = (vecs + 1024 * 8 - 1) / (1024 * 8);
        }
    }
    p.splits = (int)s;
    p.part = (vecs + s - 1) / s * v;
    return p;
}

inline uint32_t magic_of(int64_t classes) { return (uint32_t)((1 << 20) / classes + 1); }

struct Call {
    const void* logits;
    int64_t n, classes, row_stride;
    const int64_t* labels;
    int64_t ignore;
    int k;
    Out out;
    void* ws;
    hipStream_t st;
};

template <class T, int THREADS, int NCH>
void launch_rows(const Call& a, const Plan& p) {
    float4* sums = (float4*)a.ws;
    uint64_t* keys = (uint64_t*)(sums + (p.splits > 1 ? a.n * p.splits : 0));
    const dim3 grid((unsigned)(a.n * p.splits)), block(THREADS);
    const typename T::type* z = (const typename T::type*)a.logits;
    if (a.k > 0)
        hipLaunchKernelGGL((k_label_logprob<T, THREADS, NCH, true>), grid, block, 0, a.st, z, a.n, a.classes, a.row_stride,
                           a.labels, a.ignore, a.k, p.splits, p.part, a.out, sums, keys);
    else
        hipLaunchKernelGGL((k_label_logprob<T, THREADS, NCH, false>), grid, block, 0, a.st, z, a.n, a.classes,
                           a.row_stride, a.labels, a.ignore, a.k, p.splits, p.part, a.out, sums, keys);
    if (p.splits > 1)
        hipLaunchKernelGGL((k_label_join<T>), dim3((unsigned)a.n), dim3(64), (size_t)p.splits * a.k * 8, a.st, z, a.classes,
                           a.row_stride, a.labels, a.ignore, a.k, p.splits, a.out, sums, keys);
}

template <class T>
int run_forward(const Call& a) {
    if (a.classes <= kSmall) {
        const int rows = a.classes <= 32 ? 256 : 128;
        const int64_t blocks = (a.n + rows - 1) / rows;
        if (blocks > 0x7FFFFFFFll) return PIN_ERR_UNSUPPORTED;
        const size_t lds = (size_t)rows * (a.classes | 1) * 4;
        const typename T::type* z = (const typename T::type*)a.logits;
        if (rows == 256)
            hipLaunchKernelGGL((k_label_small<T, 256>), dim3((unsigned)blocks), dim3(256), lds, a.st, z, a.n, (int)a.classes,
                               magic_of(a.classes), a.row_stride, a.labels, a.ignore, a.k, a.out);
        else
            hipLaunchKernelGGL((k_label_small<T, 128>), dim3((unsigned)blocks), dim3(128), lds, a.st, z, a.n, (int)a.classes,
                               magic_of(a.classes), a.row_stride, a.labels, a.ignore, a.k, a.out);
        return launch_status();
    }
    const Plan p = plan_rows(a.n, a.classes, T::N);
    if (a.n * p.splits > 0x7FFFFFFFll) return PIN_ERR_UNSUPPORTED;
    if (p.splits > 1 && (!a.ws || ((uintptr_t)a.ws & 15))) return PIN_ERR_ARG;
    if (p.threads == 64) {
        if (p.nch == 1) launch_rows<T, 64, 1>(a, p);
        else if (p.nch == 2) launch_rows<T, 64, 2>(a, p);
        else if (p.nch == 4) launch_rows<T, 64, 4>(a, p);
        else launch_rows<T, 64, 8>(a, p);
    } else if (p.threads == 256) {
        if (p.nch == 4) launch_rows<T, 256, 4>(a, p);
        else launch_rows<T, 256, 8>(a, p);
    } else {
        if (p.nch == 4) launch_rows<T, 1024, 4>(a, p);
        else launch_rows<T, 1024, 8>(a, p);
    }
    return launch_status();
}

template <class T>
int run_backward(const Call& a, const int64_t* top_idx, const float2* stats, const float* entropy, const Grads& u,
                 void* d_logits) {
    typename T::type* o = (typename T::type*)d_logits;
    const typename T::type* z = (const typename T::type*)a.logits;
    if (a.classes <= kSmall) {
        const int rows = a.classes <= 32 ? 256 : 128;
        const int64_t blocks = (a.n + rows - 1) / rows;
        if (blocks > 0x7FFFFFFFll) return PIN_ERR_UNSUPPORTED;
        const size_t lds = (size_t)rows * (a.classes | 1) * 4;
        if (rows == 256)
            hipLaunchKernelGGL((k_label_bwd_small<T, 256>), dim3((unsigned)blocks), dim3(256), lds, a.st, z, a.n,
                               (int)a.classes, magic_of(a.classes), a.row_stride, a.labels, a.ignore, a.k, top_idx, stats,
                               entropy, u, o);
        else
            hipLaunchKernelGGL((k_label_bwd_small<T, 128>), dim3((unsigned)blocks), dim3(128), lds, a.st, z, a.n,
                               (int)a.classes, magic_of(a.classes), a.row_stride, a.labels, a.ignore, a.k, top_idx, stats,
                               entropy, u, o);
        return launch_status();
    }
    const int lanes = a.classes <= 16 * T::N * 4 ? 16 : a.classes <= 64 * T::N * 8 ? 64 : 256;
    int64_t part = a.classes, parts = 1;
    if (lanes == 256) {
        part = 256 * T::N * 4;
        parts = (a.classes + part - 1) / part;
    }
    const int64_t blocks = (a.n + 256 / lanes - 1) / (256 / lanes);
    if (blocks > 0x7FFFFFFFll || parts > 65535) return PIN_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)blocks, (unsigned)parts);
    if (lanes == 16)
        hipLaunchKernelGGL((k_label_bwd<T, 16>), grid, dim3(256), 0, a.st, z, a.n, a.classes, a.row_stride, a.labels,
                           a.ignore, a.k, top_idx, stats, entropy, u, part, o);
    else if (lanes == 64)
        hipLaunchKernelGGL((k_label_bwd<T, 64>), grid, dim3(256), 0, a.st, z, a.n, a.classes, a.row_stride, a.labels,
                           a.ignore, a.k, top_idx, stats, entropy, u, part, o);
    else
        hipLaunchKernelGGL((k_label_bwd<T, 256>), grid, dim3(256), 0, a.st, z, a.n, a.classes, a.row_stride, a.labels,
                           a.ignore, a.k, top_idx, stats, entropy, u, part, o);
    return launch_status();
}

}  // namespace

extern "C" {

int64_t pin_label_logprob_workspace_bytes(int64_t n, int64_t classes, int32_t dtype, int32_t top_k) {
    if (dtype < PIN_TYPE_F32 || dtype > PIN_TYPE_BF16 || n < 0 || classes < 1 || classes > PIN_LABEL_CLASSES_MAX ||
        top_k < 0 || top_k > PIN_LABEL_TOP_MAX)
        return PIN_ERR_ARG;
    if (n == 0 || classes <= kSmall) return 0;
    const Plan p = plan_rows(n, classes, dtype == PIN_TYPE_F32 ? F32::N : F16::N);
    return p.splits > 1 ? n * p.splits * (16 + 8 * (int64_t)top_k) : 0;
}

int pin_label_logprob(const void* logits, int32_t dtype, int64_t n, int64_t classes, int64_t row_stride,
                      const int64_t* labels, int64_t ignore_index, int32_t top_k, float* log_prob, float* entropy,
                      float* row_stats, float* top_log_prob, int64_t* top_index, void* workspace, void* stream) {
    if (bad_args(logits, dtype, n, classes, row_stride, labels, top_k)) return PIN_ERR_ARG;
    if (n == 0) return PIN_OK;
    if (!log_prob || !entropy || (top_k > 0 && (!top_log_prob || !top_index)) || ((uintptr_t)row_stats & 7))
        return PIN_ERR_ARG;
    const Call a{logits, n, classes, row_stride, labels, ignore_index, (int)top_k,
                 Out{log_prob, entropy, (float2*)row_stats, top_log_prob, top_index}, workspace, as_stream(stream)};
    return dtype == PIN_TYPE_F32 ? run_forward<F32>(a) : dtype == PIN_TYPE_F16 ? run_forward<F16>(a) : run_forward<BF16>(a);
}

int pin_label_logprob_bwd(const void* logits, int32_t dtype, int64_t n, int64_t classes, int64_t row_stride,
                          const int64_t* labels, int64_t ignore_index, int32_t top_k, const int64_t* top_index,
                          const float* row_stats, const float* entropy, const float* d_log_prob,
                          const float* d_entropy, const float* d_top, void* d_logits, void* stream) {
    if (bad_args(logits, dtype, n, classes, row_stride, labels, top_k)) return PIN_ERR_ARG;
    if (n == 0) return PIN_OK;
    if (!row_stats || ((uintptr_t)row_stats & 7) || !entropy || !d_logits || (d_top && top_k > 0 && !top_index) ||
        ((uintptr_t)d_logits & (dtype == PIN_TYPE_F32 ? 3 : 1)))
        return PIN_ERR_ARG;
    const Call a{logits, n, classes, row_stride, labels, ignore_index, (int)top_k, Out{}, nullptr, as_stream(stream)};
    const Grads u{d_log_prob, d_entropy, top_k > 0 ? d_top : nullptr};
    const float2* st = (const float2*)row_stats;
    return dtype == PIN_TYPE_F32   ? run_backward<F32>(a, top_index, st, entropy, u, d_logits)
           : dtype == PIN_TYPE_F16 ? run_backward<F16>(a, top_index, st, entropy, u, d_logits)
                                   : run_backward<BF16>(a, top_index, st, entropy, u, d_logits);
}

}  // extern "C"
