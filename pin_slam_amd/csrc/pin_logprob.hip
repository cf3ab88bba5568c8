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
// shifts every x_j of a row alike, by its rounding (up to 2^-25 |m L|), and every result is a
// difference of such.  The shift has to stay small, as 2^x is taken before the difference: at
// |m| = 3e9 it is 2^7, and the sum infinite or 0.  So beyond |m| = 2^20, where it is 2^-4, x_j =
// (z_j - m) L, without a shift: rows masked throughout by a large finite value, and the parts of
// rows that are, in whatever a maximum is taken of.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "pin_slam_amd.h"

namespace {

constexpr float kInf = __builtin_huge_valf();
constexpr float kL = 1.44269504f, kLn2 = 0.693147182f;
constexpr float kFloor = -1000.f;            // 2^x is 0 well above
constexpr float kNear = 0x1p20f;             // largest size of a maximum m whose fl(m L) is taken (see above)
// most classes of the kernels of one thread per row (300000 x 64 f32 with 3 alternatives: 38 us, sixteen lanes 51)
constexpr int kSmall = 64;
constexpr int kSplits = 64;                  // most parts of a row

inline hipStream_t as_stream(void* s) { return (hipStream_t)s; }
inline int launch_status() { return hipGetLastError() == hipSuccess ? PIN_OK : PIN_ERR_HIP; }

// ---- types: sixteen bytes of logits as f32, and back

struct F32 {
    typedef float type;
    static constexpr int N = 4;
    static constexpr uint32_t kFill = 0xFF800000u;   // -inf in every element
    static constexpr int kLow = 0;                   // even number of low bits that are the same in all f32 values
    static __device__ __forceinline__ void unpack(const uint4& q, float (&o)[4]) {
        o[0] = __uint_as_float(q.x), o[1] = __uint_as_float(q.y), o[2] = __uint_as_float(q.z), o[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    static __device__ __forceinline__ float one(const float* p) { return *p; }
    static __device__ __forceinline__ uint32_t bits(const float* p) { return __float_as_uint(*p); }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};

struct F16 {
    typedef _Float16 type;
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    static constexpr int N = 8;
    static constexpr uint32_t kFill = 0xFC00FC00u;
    static constexpr int kLow = 12;
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
    static __device__ __forceinline__ uint32_t bits(const _Float16* p) { return *(const uint16_t*)p; }
    static __device__ __forceinline__ void put(_Float16* p, float v) { *p = (_Float16)v; }
};

struct BF16 {
    typedef uint16_t type;
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    static constexpr int N = 8;
    static constexpr uint32_t kFill = 0xFF80FF80u;
    static constexpr int kLow = 16;
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
    static __device__ __forceinline__ uint32_t bits(const uint16_t* p) { return *p; }
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
// the elements [from, to) of sixteen bytes, from < to, the others -inf (all reads on their way at once: in
// the others' places the nearest element is read)
template <class T>
__device__ __forceinline__ uint4 load_some(const typename T::type* p, int from, int to) {
    uint32_t u[4] = {0, 0, 0, 0};
    constexpr int V = T::N, W = V / 4;   // elements, elements of 32 bits
    uint32_t e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = T::bits(p + (i < from ? from : i < to ? i : to - 1));
#pragma unroll
    for (int i = 0; i < V; ++i)
        u[i / W] |= (i < from || i >= to ? T::kFill & (0xFFFFFFFFu >> (32 - 32 / W)) : e[i]) << (i % W * 16);
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// A row as aligned vectors of 16 bytes: vector u holds the classes u V - skip and on.  Its first and
// last vector may be partly other rows'.  (Rows of an odd number of 16-bit classes, read at their own
// alignment: 66 us for 2048 x 50021 bf16; in aligned vectors 44.)
template <class T>
struct Vectors {
    const typename T::type* base;
    int skip, classes;
    int lo, hi;    // first and last vector that are the row's throughout (rows of 2 V classes or more have one)
    int count;
    __device__ __forceinline__ Vectors(const typename T::type* z, int c) : classes(c) {
        skip = (int)((uintptr_t)z & 15) / (int)sizeof(typename T::type);
        base = z - skip;
        lo = skip ? 1 : 0;
        hi = (c + skip) / T::N - 1;
        count = (c + skip + T::N - 1) / T::N;
    }
    // any vector, 0 <= u: where it is not the row's throughout, another one of the row (load() puts it right)
    __device__ __forceinline__ uint4 load_near(int u) const {
        u = u < lo ? lo : u > hi ? hi : u;
        return *(const uint4*)(base + (int64_t)u * T::N);
    }
    __device__ __forceinline__ uint4 load_edge(int u) const {
        if (u >= count) return make_uint4(T::kFill, T::kFill, T::kFill, T::kFill);
        const int to = classes + skip - u * T::N;
        return load_some<T>(base + (int64_t)u * T::N, u == 0 ? skip : 0, to < T::N ? to : T::N);
    }
    __device__ __forceinline__ bool whole(int u) const { return u >= lo && u <= hi; }
    __device__ __forceinline__ int first_class(int u) const { return u * T::N - skip; }
};

// The registers as they are, but unknown to the compiler: what was made of them before is made
// again (two instructions an element) rather than kept beside them (a register an element).
__device__ __forceinline__ void forget(uint4& q) { asm volatile("" : "+v"(q.x), "+v"(q.y), "+v"(q.z), "+v"(q.w)); }

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
struct MinU {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a < b ? a : b; }
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
    float ml;      // fl(m L), what is subtracted where m is not far
    bool far;      // (z - m) L then
    __device__ __forceinline__ explicit Row(float max) : m(max), ls(0.f), ml(max * kL), far(!(fabsf(max) <= kNear)) {}
    __device__ __forceinline__ bool bad() const { return m == kInf; }
    __device__ __forceinline__ bool dead() const { return m == -kInf; }
    __device__ __forceinline__ float x(float z) const { return far ? (z - m) * kL : fmaf(z, kL, -ml); }
    __device__ __forceinline__ float log_prob(float z) const {
        const float v = far ? fmaf(-ls, kLn2, z - m) : (x(z) - ls) * kLn2;
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
    float* stats;       // may be NULL; maximum, log2 of the sum, entropy
    float* top_lp;
    int64_t* top_idx;
};

__device__ __forceinline__ void put_row(const Out& o, const Row& r, int64_t row, float s, float t, float zy, int64_t y,
                                        int64_t ignore, int64_t classes) {
    const float h = row_entropy(r, s, t);
    o.log_prob[row] = label_log_prob(r, zy, y, ignore, classes);
    o.entropy[row] = h;
    if (o.stats) {
        o.stats[3 * row] = r.m;
        o.stats[3 * row + 1] = r.ls;
        o.stats[3 * row + 2] = h;
    }
}

__device__ __forceinline__ void put_top(const Out& o, const Row& r, int64_t at, uint64_t key) {
    o.top_lp[at] = r.log_prob(key_value((uint32_t)(key >> 32)));
    o.top_idx[at] = r.bad() ? -1 : (int64_t)(uint32_t)~(uint32_t)key;
}

// The vectors [u0, u0 + 64 W NCH) of a row up to u1, W waves, thread t's c-th being u0 + c 64 W + t, in registers.
// All are on their way before the first is looked at.
template <class T, int W, int NCH>
__device__ __forceinline__ void load_part(const Vectors<T>& z, int u0, int u1, uint4 (&q)[NCH]) {
    const int t = threadIdx.x;
#pragma unroll
    for (int c = 0; c < NCH; ++c) q[c] = z.load_near(u0 + c * 64 * W + t);
    const int last = z.hi + 1 < u1 ? z.hi + 1 : u1;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int u = u0 + c * 64 * W + t;
        if (u0 + (c + 1) * 64 * W > last || (c == 0 && u0 < z.lo)) {   // the same for all threads
            if (u >= u1) q[c] = make_uint4(T::kFill, T::kFill, T::kFill, T::kFill);
            else if (!z.whole(u)) q[c] = z.load_edge(u);
        }
    }
}

// maximum of 16 bytes of logits; NaN if one is
template <class T>
__device__ __forceinline__ float vector_max(const uint4& q) {
    if constexpr (__is_same(T, F16)) {   // two at a time
        typedef _Float16 v2 __attribute__((ext_vector_type(2)));
        const auto two = [](uint32_t u) { return __builtin_bit_cast(v2, u); };
        const v2 h = __builtin_elementwise_maximum(__builtin_elementwise_maximum(two(q.x), two(q.y)),
                                                   __builtin_elementwise_maximum(two(q.z), two(q.w)));
        return max_nan((float)h.x, (float)h.y);
    }
    float v[T::N];
    T::unpack(q, v);
    float m = v[0];
#pragma unroll
    for (int i = 1; i < T::N; ++i) m = max_nan(m, v[i]);
    return m;
}

// sums of 2^x and 2^x x
template <class T, int W, int NCH>
__device__ __forceinline__ void part_sums(const Row& r, const uint4 (&q)[NCH], int vectors, float& s, float& t) {
    s = t = 0.f;
    const auto add = [&](auto x_of) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            if (c > 0 && c * 64 * W >= vectors) break;   // the same for all threads
            float v[T::N];
            T::unpack(q[c], v);
#pragma unroll
            for (int i = 0; i < T::N; ++i) {
                const float x = fmaxf(x_of(v[i]), kFloor);
                const float e = __builtin_amdgcn_exp2f(x);
                s += e;
                t = fmaf(e, x, t);
            }
        }
    };
    if (!r.far) add([&](float z) { return fmaf(z, kL, -r.ml); });
    else add([&](float z) { return (z - r.m) * kL; });
}

// The k-th largest of the wave's keys, N in each lane, two bits at a time.  LOW: bits that are alike in all
// keys of a sign (a 16-bit type's: 0 of positive values, 1 of negative ones).
template <int LOW, int N>
__device__ __forceinline__ uint32_t kth_of_wave(const uint32_t (&key)[N], int k) {
    const auto count = [&](uint32_t c) {
        int have = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) have += __popcll(__ballot(key[i] >= c));
        return have;
    };
    uint32_t kth = 0;
#pragma unroll 1
    for (int b = 30; b >= LOW; b -= 2) {
        const uint32_t one = kth | 1u << b, two = kth | 2u << b, three = kth | 3u << b;
        const int n1 = count(one), n2 = count(two), n3 = count(three);
        kth = n3 >= k ? three : n2 >= k ? two : n1 >= k ? one : kth;
    }
    return LOW == 0 || kth & 0x80000000u ? kth : kth | ((1u << LOW) - 1);
}
template <int LOW>
__device__ __forceinline__ uint32_t kth_of_wave(uint32_t key, int k) {
    const uint32_t one[1] = {key};
    return kth_of_wave<LOW, 1>(one, k);
}

// the least value above one (a bound that v reaches if v is larger)
__device__ __forceinline__ float above(float v) { return key_value(order_key(v) + 1); }

// What reaches a bound that is not above the k-th largest, in LDS; behind it room for equal ones.
template <int MOST>
struct Candidates {
    uint64_t key[MOST + PIN_LABEL_TOP_MAX];
    uint32_t n;
    static constexpr int kMost = MOST;
    // (a lane's hits as bits first: most lanes have one or none, and a turn for each is dearer than a bit)
    template <class T>
    __device__ __forceinline__ void push_vector(const Vectors<T>& z, int u, const uint4& q, float bound) {
        constexpr int V = T::N;
        float v[V];
        T::unpack(q, v);
        const int j = z.first_class(u), lo = j < 0 ? -j : 0, room = z.classes - j, hi = room < 0 ? 0 : room < V ? room : V;
        uint32_t hits = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) hits |= v[i] >= bound ? 1u << i : 0u;
        hits &= (1u << hi) - (1u << lo);
        while (__any(hits != 0)) {
            if (hits != 0) {
                const int at = __ffs(hits) - 1;
                float w = v[0];
#pragma unroll
                for (int i = 1; i < V; ++i) w = i == at ? v[i] : w;
                const uint32_t p = atomicAdd(&n, 1u);
                if (p < MOST) key[p] = class_key(w, (uint32_t)(j + at));
                hits &= hits - 1;
            }
        }
    }
    // one wave: the k largest of `all`, in order; at least k
    template <class F>
    __device__ __forceinline__ void sort(int all, int k, F emit) const {
        const int lane = threadIdx.x & 63;
        if (all <= 64) {
            const uint64_t mine = lane < all ? key[lane] : 0;
            int rank = 0;
            for (int i = 0; i < all; ++i) {
                const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), i) << 32 |
                                       (uint32_t)__builtin_amdgcn_readlane((int)mine, i);
                rank += other > mine ? 1 : 0;
            }
            if (lane < all && rank < k) emit(rank, mine);
            return;
        }
        uint64_t last = ~0ull;
        for (int i = 0; i < k; ++i) {
            uint64_t best = 0;
            for (int p = lane; p < all; p += 64)
                if (key[p] < last && key[p] > best) best = key[p];
            last = wave_max_key(best);
            if (lane == 0) emit(i, last);
        }
    }
};

// The first `need` classes of [from, to) whose logit is `value`, put at keys[have] and on; all threads of
// the workgroup (THREADS of them), behind a barrier.  Returns how many there are now, at most `need`.
template <class T, int THREADS>
__device__ __forceinline__ int first_equal(const typename T::type* z, int from, int to, float value, int need, int have,
                                           uint64_t* keys, uint32_t* s_tot) {
    const int wave = threadIdx.x >> 6;
#pragma unroll 1
    for (int j0 = from; j0 < to && have < need; j0 += THREADS) {
        const int j = j0 + (int)threadIdx.x;
        const float v = j < to ? T::one(z + j) : NAN;
        const uint64_t b = __ballot(v == value);
        int at = have + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
        if ((threadIdx.x & 63) == 0) s_tot[wave] = __popcll(b);
        __syncthreads();
        for (int w = 0; w < THREADS / 64; ++w) {
            at += w < wave ? (int)s_tot[w] : 0;
            have += (int)s_tot[w];
        }
        if (v == value && at < need) keys[at] = class_key(v, (uint32_t)j);
        __syncthreads();
    }
    return have < need ? have : need;
}

// The k largest by k passes over the row, each the largest below the last: rows whose large logits
// are so gathered that the lists overflow.
template <class T, int THREADS, class F>
__device__ __forceinline__ void largest_by_passes(const typename T::type* z, int classes, int k, uint64_t* s_key, F emit) {
    const int wave = threadIdx.x >> 6;
    uint64_t last = ~0ull;
    for (int i = 0; i < k; ++i) {
        uint64_t best = 0;
#pragma unroll 1
        for (int j = threadIdx.x; j < classes; j += THREADS) {
            const uint64_t key = class_key(T::one(z + j), (uint32_t)j);
            if (key < last && key > best) best = key;
        }
        best = wave_max_key(best);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s_key[wave] = best;
        __syncthreads();
        for (int w = 0; w < THREADS / 64; ++w) best = s_key[w] > best ? s_key[w] : best;
        last = best;
        if (threadIdx.x == 0) emit(i, best);
    }
}

// One wave per row, 64 NCH vectors: the lanes' maxima, of which the k-th largest is not above the
// row's k-th largest logit; the sums; what is at or above that, a little more than k, sorted.
template <class T, int NCH, bool TOP>
__global__ void __launch_bounds__(64)
k_label_wave(const typename T::type* __restrict__ logits, int64_t n, int classes, int64_t row_stride,
             const int64_t* __restrict__ labels, int64_t ignore, int k, Out out) {
    __shared__ Candidates<TOP ? 256 : 1> s_c;
    __shared__ uint32_t s_tot[1];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const typename T::type* zr = logits + row * row_stride;
    const Vectors<T> z(zr, classes);
    uint4 q[NCH];
    load_part<T, 1, NCH>(z, 0, z.count, q);
    const int64_t y = labels[row];
    const float zy = y >= 0 && y < classes ? T::one(zr + y) : 0.f;
    float cm[NCH], mx = -kInf;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        cm[c] = vector_max<T>(q[c]);
        mx = max_nan(mx, cm[c]);
    }
    mx = mx != mx ? kInf : mx;
    Row r(wave_max(mx));
#pragma unroll
    for (int c = 0; c < NCH; ++c) forget(q[c]);
    float s, t;
    part_sums<T, 1, NCH>(r, q, z.count, s, t);
    s = wave_sum(s);
    t = wave_sum(t);
    r.ls = r.dead() ? 0.f : __builtin_amdgcn_logf(s);   // s >= 1 unless there is nothing
    if (lane == 0) {
        put_row(out, r, row, s, t, zy, y, ignore, classes);
        s_c.n = 0;
    }
    if (!TOP) return;
    const auto emit = [&](int i, uint64_t key) { put_top(out, r, row * k + i, key); };
    if (r.bad()) {
        if (lane < k) emit(lane, 0);
        return;
    }
    const float kth = key_value(kth_of_wave<T::kLow>(order_key(mx), k));
    __syncthreads();
#pragma unroll
    for (int c = 0; c < NCH; ++c) forget(q[c]);
    const auto collect = [&](float bound) {
#pragma unroll
        for (int c = 0; c < NCH; ++c)
            if (cm[c] >= bound) s_c.push_vector(z, c * 64 + lane, q[c], bound);
        __syncthreads();
        return (int)s_c.n;
    };
    int all = collect(kth);
    if (all > s_c.kMost) {   // many at the bound itself: those above it, and the first of the others
        __syncthreads();
        if (lane == 0) s_c.n = 0;
        __syncthreads();
        all = collect(above(kth));
        if (all > s_c.kMost) return largest_by_passes<T, 64>(zr, classes, k, s_c.key, emit);
        if (all < k) all += first_equal<T, 64>(zr, 0, classes, kth, k - all, 0, s_c.key + all, s_tot);
    }
    s_c.sort(all, k, emit);
}

// Sixteen lanes per row, 16 NCH vectors: four rows share what a wave spends on reductions.  Alternatives, few
// of them: the row's largest, then the first class that has it (looked for in the vectors whose maximum it is),
// which is marked and its vector's maximum taken again.
template <class T, int NCH, bool TOP>
__global__ void __launch_bounds__(256)
k_label_lanes(const typename T::type* __restrict__ logits, int64_t n, int classes, int64_t row_stride,
              const int64_t* __restrict__ labels, int64_t ignore, int k, Out out) {
    constexpr int V = T::N;
    const int lane = threadIdx.x & 15;
    const int64_t at = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), row = at < n ? at : n - 1;
    const bool writes = at < n && lane == 0;
    const typename T::type* zr = logits + row * row_stride;
    const Vectors<T> z(zr, classes);
    const int most = (classes + 2 * V - 2) / V;   // vectors of a row at any alignment
    uint4 q[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) q[c] = z.load_near(c * 16 + lane);
    const int64_t y = labels[row];
    const float zy = y >= 0 && y < classes ? T::one(zr + y) : 0.f;
    float cm[NCH], mx = -kInf;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int u = c * 16 + lane;
        if (!z.whole(u)) q[c] = z.load_edge(u);
        cm[c] = vector_max<T>(q[c]);
        mx = max_nan(mx, cm[c]);
    }
    mx = mx != mx ? kInf : mx;
    Row r(__uint_as_float(rows_of_16(__float_as_uint(mx), MaxF())));
#pragma unroll
    for (int c = 0; c < NCH; ++c) forget(q[c]);
    float s = 0.f, t = 0.f;
    const float off = r.far ? 0.f : r.ml, from = r.far ? r.m : 0.f;   // x = (z - from) L - off
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        if (c > 0 && c * 16 >= most) break;   // the same for all threads
        float v[V];
        T::unpack(q[c], v);
        if (__any(r.far)) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] -= from;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float x = fmaxf(fmaf(v[i], kL, -off), kFloor), e = __builtin_amdgcn_exp2f(x);
            s += e;
            t = fmaf(e, x, t);
        }
    }
    s = __uint_as_float(rows_of_16(__float_as_uint(s), AddF()));
    t = __uint_as_float(rows_of_16(__float_as_uint(t), AddF()));
    r.ls = r.dead() ? 0.f : __builtin_amdgcn_logf(s);
    if (writes) put_row(out, r, row, s, t, zy, y, ignore, classes);
    if (!TOP) return;
    uint64_t taken = 0;   // a bit per element (V NCH <= 64)
    const auto is_taken = [&](int c, int i) { return (taken >> (c * V + i) & 1) != 0; };
    for (int e = 0; e < k; ++e) {
        float best = cm[0];
#pragma unroll
        for (int c = 1; c < NCH; ++c) best = fmaxf(best, cm[c]);
        best = __uint_as_float(rows_of_16(__float_as_uint(best), MaxF()));
        int j = classes;   // my first class that has it
#pragma unroll
        for (int c = NCH - 1; c >= 0; --c) {
            if (cm[c] == best) {
                float v[V];
                T::unpack(q[c], v);
                const int j0 = z.first_class(c * 16 + lane);
#pragma unroll
                for (int i = V - 1; i >= 0; --i)
                    j = v[i] == best && !is_taken(c, i) && (unsigned)(j0 + i) < (unsigned)classes ? j0 + i : j;
            }
        }
        const int first = (int)rows_of_16((uint32_t)j, MinU());
        if (writes) {
            out.top_lp[row * k + e] = r.log_prob(best);
            out.top_idx[row * k + e] = r.bad() ? -1 : first;
        }
        if (e + 1 < k && j == first && j < classes) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int i0 = first - z.first_class(c * 16 + lane);
                if ((unsigned)i0 < (unsigned)V) {
                    taken |= 1ull << (c * V + i0);
                    float v[V];
                    T::unpack(q[c], v);
                    float m = -kInf;
#pragma unroll
                    for (int i = 0; i < V; ++i) m = fmaxf(m, is_taken(c, i) ? -kInf : v[i]);
                    cm[c] = m;
                }
            }
        }
    }
}

// A part of a long row: its maximum and sums, and for the alternatives the maxima of 64 groups of its
// vectors (four neighbouring threads' each).
template <class T, int NCH>
__global__ void __launch_bounds__(256, 8)
k_label_part(const typename T::type* __restrict__ logits, int classes, int64_t row_stride, int splits, int part,
             float4* __restrict__ sums, float* __restrict__ maxima) {
    __shared__ float s_max[4];
    __shared__ float2 s_sum[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const unsigned row = blockIdx.x / (unsigned)splits;
    const int u0 = (int)(blockIdx.x - row * (unsigned)splits) * part;
    const typename T::type* zr = logits + row * row_stride;
    const Vectors<T> z(zr, classes);
    const int u1 = u0 + part < z.count ? u0 + part : z.count;
    uint4 q[NCH];
    load_part<T, 4, NCH>(z, u0, u1, q);
    float mx = -kInf;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        if (c > 0 && u0 + c * 256 >= u1) break;
        mx = max_nan(mx, vector_max<T>(q[c]));
    }
    mx = mx != mx ? kInf : mx;
    if (maxima) {
        float g = fmaxf(mx, __uint_as_float(dpp<0xB1>(__float_as_uint(mx))));
        g = fmaxf(g, __uint_as_float(dpp<0x4E>(__float_as_uint(g))));
        if ((tid & 3) == 0) maxima[(int64_t)blockIdx.x * 64 + (tid >> 2)] = g;
    }
    mx = wave_max(mx);
    if (lane == 0) s_max[wave] = mx;
    __syncthreads();
    Row r(fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3])));
#pragma unroll
    for (int c = 0; c < NCH; ++c) forget(q[c]);
    float s, t;
    part_sums<T, 4, NCH>(r, q, u1 - u0, s, t);
    s = wave_sum(s);
    t = wave_sum(t);
    if (lane == 0) s_sum[wave] = make_float2(s, t);
    __syncthreads();
    if (tid != 0) return;
    s = (s_sum[0].x + s_sum[1].x) + (s_sum[2].x + s_sum[3].x);
    t = (s_sum[0].y + s_sum[1].y) + (s_sum[2].y + s_sum[3].y);
    sums[blockIdx.x] = make_float4(r.m, s, t, 0.f);
}

// The parts' sums taken to the row's maximum (one lane per part, every wave alike).
template <class T>
__device__ __forceinline__ Row join_sums(const float4* __restrict__ sums, const typename T::type* zr, int64_t row, int classes,
                                         const int64_t* labels, int64_t ignore, int splits, const Out& out) {
    const int lane = threadIdx.x & 63;
    const float4 p = lane < splits ? sums[row * splits + lane] : make_float4(-kInf, 0.f, 0.f, 0.f);
    const int64_t y = labels[row];
    const float zy = y >= 0 && y < classes ? T::one(zr + y) : 0.f;
    Row r(wave_max(p.x));
    // to the row's form from the one in which the part was summed: the row's own shift less the part's
    const Row q(p.x);
    const float x = fmaxf(r.far ? (q.far ? (p.x - r.m) * kL : -fmaf(r.m, kL, -q.ml)) : q.far ? fmaf(p.x, kL, -r.ml) : q.ml - r.ml,
                          kFloor);
    const float f = __builtin_amdgcn_exp2f(x);
    const float s = wave_sum(f * p.y), t = wave_sum(f * fmaf(p.y, x, p.z));
    r.ls = r.dead() ? 0.f : __builtin_amdgcn_logf(s);
    if (threadIdx.x == blockDim.x - 64) put_row(out, r, row, s, t, zy, y, ignore, classes);   // the last wave
    return r;
}

template <class T>
__global__ void __launch_bounds__(64)
k_label_join(const typename T::type* __restrict__ logits, int classes, int64_t row_stride,
             const int64_t* __restrict__ labels, int64_t ignore, int splits, Out out, const float4* __restrict__ sums) {
    join_sums<T>(sums, logits + blockIdx.x * row_stride, blockIdx.x, classes, labels, ignore, splits, out);
}

// The alternatives of a row from the maxima of its groups (64 per part of `part` vectors: group i of a part
// holds the vectors 256 c + 4 i .. 4 i + 3), and the maxima of 64 groups of groups.  The k-th largest of the
// latter bounds the k-th largest logit from below, the k-th largest of the groups' maxima above that bound
// does so closer; only the groups that reach it are read again, about k of them.
struct TopSpace {
    static constexpr int kFew = 256;
    Candidates<512> c;
    float sup[64], val[kFew];
    uint16_t list[kFew];
    uint32_t n, kth, tot[4];
    __device__ __forceinline__ void clear() { n = c.n = 0; }   // one thread, before a barrier
};

// 256 threads; m.sup and the maxima are written, with a barrier behind them.  mine: the maxima of groups
// 256 e + thread.
template <class T, int M, class F>
__device__ __forceinline__ void top_of_row(TopSpace& m, const float (&mine)[M], const float* maxima, int parts, int part,
                                           const Vectors<T>& z, const typename T::type* zr, int k, F emit) {
    constexpr int kFew = TopSpace::kFew, W = 4;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, groups = parts * 64;
    if (wave == 0) {
        const uint32_t kth = kth_of_wave<T::kLow>(order_key(m.sup[lane]), k);
        if (lane == 0) m.kth = kth;
    }
    __syncthreads();
    float kth = key_value(m.kth);
#pragma unroll
    for (int e = 0; e < M; ++e) {
        const int i = e * 256 + tid;
        if (mine[e] >= kth && i < groups) {
            const uint32_t p = atomicAdd(&m.n, 1u);
            if (p < kFew) m.val[p] = mine[e], m.list[p] = (uint16_t)i;
        }
    }
    __syncthreads();
    const int listed = (int)m.n;
    // with very many groups at the bound (rows mostly masked, or all equal) only those above it are read, and
    // the first classes at it looked for
    const bool flood = listed > kFew;
    if (listed > 2 * k && !flood) {   // a closer bound
        if (wave == 0) {
            uint32_t key[kFew / 64];
#pragma unroll
            for (int i = 0; i < kFew / 64; ++i) key[i] = i * 64 + lane < listed ? order_key(m.val[i * 64 + lane]) : 0;
            const uint32_t c = kth_of_wave<T::kLow>(key, k);
            if (lane == 0) m.kth = c;
        }
        __syncthreads();
        kth = key_value(m.kth);
    }
    // two groups at a time per wave, one vector per lane, four reads on their way
    const auto collect = [&](float bound) {
        constexpr int R = 4;
        const int per = (part + 255) / 256, some = flood ? groups : listed;
        for (int i0 = wave * 2 + (lane >> 5); i0 < some; i0 += 2 * W * R) {
            uint4 q[R];
            int at[R];
#pragma unroll
            for (int e = 0; e < R; ++e) {
                const int i = i0 + e * 2 * W, v = lane & 31;
                at[e] = -1;
                if (i < some) {
                    const int id = flood ? i : m.list[i];
                    const float top = flood ? maxima[id] : m.val[i];
                    const int in = (v >> 2) * 256 + (id & 63) * 4 + (v & 3), u = (id >> 6) * part + in;
                    if (top >= bound && (v >> 2) < per && in < part && u < z.count) at[e] = u;
                }
                q[e] = z.load_near(at[e] < 0 ? 0 : at[e]);
            }
#pragma unroll
            for (int e = 0; e < R; ++e)
                if (at[e] >= 0) m.c.push_vector(z, at[e], z.whole(at[e]) ? q[e] : z.load_edge(at[e]), bound);
        }
        __syncthreads();
        return (int)m.c.n;
    };
    bool strict = flood;
    int all = collect(strict ? above(kth) : kth);
    if (!strict && all > m.c.kMost) {
        strict = true;
        __syncthreads();
        if (tid == 0) m.c.n = 0;
        __syncthreads();
        all = collect(above(kth));
    }
    if (all > m.c.kMost) return largest_by_passes<T, 256>(zr, z.classes, k, m.c.key, emit);
    if (strict && all < k) {
        int more = 0;
        for (int p = 0; p < parts && more < k - all; ++p) {
            if (!__any(maxima[p * 64 + lane] >= kth)) continue;
            const int from = z.first_class(p * part), to = z.first_class((p + 1) * part);
            more = first_equal<T, 256>(zr, from < 0 ? 0 : from, to < z.classes ? to : z.classes, kth, k - all, more,
                                       m.c.key + all, m.tot);
        }
        all += more;
    }
    if (wave == 0) m.c.sort(all, k, emit);
}

// a thread's maximum to its four neighbours', and those of a workgroup's 64 fours to `to`
__device__ __forceinline__ void put_fours(float v, float* to) {
    v = fmaxf(v, __uint_as_float(dpp<0xB1>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(dpp<0x4E>(__float_as_uint(v))));
    if ((threadIdx.x & 3) == 0) to[threadIdx.x >> 2] = v;
}

template <class T>
__global__ void __launch_bounds__(256)
k_label_join_top(const typename T::type* __restrict__ logits, int classes, int64_t row_stride,
                 const int64_t* __restrict__ labels, int64_t ignore, int k, int splits, int part, Out out,
                 const float4* __restrict__ sums, const float* __restrict__ maxima) {
    __shared__ TopSpace s_m;
    const int64_t row = blockIdx.x;
    const typename T::type* zr = logits + row * row_stride;
    const float* mine = maxima + row * splits * 64;
    if (threadIdx.x == 0) s_m.clear();
    float g[kSplits / 4], top = -kInf;   // all on their way at once
#pragma unroll
    for (int e = 0; e < kSplits / 4; ++e) {
        const int i = e * 256 + threadIdx.x;
        g[e] = i < splits * 64 ? mine[i] : -kInf;
    }
#pragma unroll
    for (int e = 0; e < kSplits / 4; ++e) top = fmaxf(top, g[e]);
    put_fours(top, s_m.sup);
    const Row r = join_sums<T>(sums, zr, row, classes, labels, ignore, splits, out);
    const auto emit = [&](int i, uint64_t key) { put_top(out, r, row * k + i, key); };
    if (r.bad()) {
        if ((int)threadIdx.x < k) emit(threadIdx.x, 0);
        return;
    }
    __syncthreads();
    top_of_row<T>(s_m, g, mine, splits, part, Vectors<T>(zr, classes), zr, k, emit);
}

// Many long rows: a workgroup goes through a row alone, kPart vectors at a time, each thread with a running
// maximum of its own (2^x is taken to it, and what it has summed is taken to a new one), so nothing waits
// for the other threads before the row's end.
// vectors of a part (of twice as many, inputs from memory: 2048 x 50021 bf16 50 us instead of 44, 4096 x 131072 207
// instead of 190; in a training step, right behind a gradient of as many bytes, the former takes 62)
constexpr int kPart = 256 * 4;
static_assert((PIN_LABEL_CLASSES_MAX + 6) / 4 <= kSplits * 2 * kPart && (PIN_LABEL_CLASSES_MAX + 14) / 8 <= kSplits * kPart,
              "the longest row's parts");
constexpr int kRowParts = 32;      // most parts of a row here (their groups' maxima lie in LDS)

template <class T>
__global__ void __launch_bounds__(256, 8)
k_label_row(const typename T::type* __restrict__ logits, int classes, int64_t row_stride,
            const int64_t* __restrict__ labels, int64_t ignore, int k, int parts, Out out) {
    constexpr int NCH = kPart / 256;
    __shared__ TopSpace s_m;
    __shared__ float s_max[kRowParts * 64];
    __shared__ float4 s_sum[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const typename T::type* zr = logits + row * row_stride;
    const Vectors<T> z(zr, classes);
    if (tid == 0) s_m.clear();
    const int64_t y = labels[row];
    const float zy = y >= 0 && y < classes ? T::one(zr + y) : 0.f;
    // m L is taken of maxima down to -kNear only: of a thread whose classes all lie below nothing reaches the sums,
    // unless the whole row does (or lies above kNear), which is summed again
    constexpr float kLow = -kNear;
    float m = -kInf, ml = kLow * kL, s = 0.f, t = 0.f;
#pragma unroll 1
    for (int p = 0; p < parts; ++p) {
        const int u0 = p * kPart, u1 = u0 + kPart < z.count ? u0 + kPart : z.count;
        uint4 q[NCH];
        load_part<T, 4, NCH>(z, u0, u1, q);
        float mx = vector_max<T>(q[0]);
#pragma unroll
        for (int c = 1; c < NCH; ++c) mx = max_nan(mx, vector_max<T>(q[c]));
        mx = mx != mx ? kInf : mx;
        put_fours(mx, s_max + p * 64);
        if (__any(mx > m)) {
            m = fmaxf(m, mx);
            const float to = fmaxf(m, kLow) * kL, x = fmaxf(ml - to, kFloor), f = __builtin_amdgcn_exp2f(x);
            t = f * fmaf(s, x, t);
            s *= f;
            ml = to;
        }
#pragma unroll
        for (int c = 0; c < NCH; ++c) forget(q[c]);
        float ps = 0.f, pt = 0.f;   // a part's sums by themselves: the chains of a row's stay below a hundred terms
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            if (c > 0 && u0 + c * 256 >= u1) break;
            float v[T::N];
            T::unpack(q[c], v);
#pragma unroll
            for (int i = 0; i < T::N; ++i) {
                const float x = fmaxf(fmaf(v[i], kL, -ml), kFloor);
                const float e = __builtin_amdgcn_exp2f(x);
                ps += e;
                pt = fmaf(e, x, pt);
            }
        }
        s += ps;
        t += pt;
    }
    put_fours(m, s_m.sup);
    const float wm = wave_max(m);
    if (lane == 0) s_sum[wave].z = wm;
    __syncthreads();
    Row r(fmaxf(fmaxf(s_sum[0].z, s_sum[1].z), fmaxf(s_sum[2].z, s_sum[3].z)));
    if (r.far && !r.bad() && !r.dead()) {
        s = t = 0.f;
#pragma unroll 1
        for (int p = 0; p < parts; ++p) {
            const int u0 = p * kPart, u1 = u0 + kPart < z.count ? u0 + kPart : z.count;
            uint4 q[NCH];
            load_part<T, 4, NCH>(z, u0, u1, q);
            float ps, pt;
            part_sums<T, 4, NCH>(r, q, u1 - u0, ps, pt);
            s += ps;
            t += pt;
        }
    } else {
        const float x = fmaxf(ml - r.ml, kFloor), f = __builtin_amdgcn_exp2f(x);
        t = f * fmaf(s, x, t);
        s *= f;
    }
    s = wave_sum(s);
    t = wave_sum(t);
    if (lane == 0) s_sum[wave].x = s, s_sum[wave].y = t;
    __syncthreads();
    s = (s_sum[0].x + s_sum[1].x) + (s_sum[2].x + s_sum[3].x);
    t = (s_sum[0].y + s_sum[1].y) + (s_sum[2].y + s_sum[3].y);
    r.ls = r.dead() ? 0.f : __builtin_amdgcn_logf(s);
    if (tid == 192) put_row(out, r, row, s, t, zy, y, ignore, classes);   // (the first wave has more to do)
    if (k == 0) return;
    const auto emit = [&](int i, uint64_t key) { put_top(out, r, row * k + i, key); };
    if (r.bad()) {
        if (tid < k) emit(tid, 0);
        return;
    }
    float g[kRowParts / 4];
#pragma unroll
    for (int e = 0; e < kRowParts / 4; ++e) g[e] = e * 4 < parts ? s_max[e * 256 + tid] : -kInf;   // (parts * 64 of them written)
    top_of_row<T>(s_m, g, s_max, parts, kPart, z, zr, k, emit);
}

// Few classes: one thread per row, the workgroup's rows staged through LDS as f32 (an odd pitch:
// consecutive rows begin in different banks).  Rows without gaps are read as vectors, eight on their way
// per thread (1M x 20 f32 with 3 alternatives: element by element 65 us, in vectors and with the row in
// registers 30).
template <class T, int ROWS>
__device__ __forceinline__ void stage_rows(const typename T::type* __restrict__ logits, int64_t row0, int rows, int classes,
                                           uint32_t magic, int64_t row_stride, float* s_z) {
    constexpr int V = T::N, B = 8;
    const int pad = 1 - (classes & 1), all = rows * classes;
    const typename T::type* z = logits + row0 * row_stride;
    const auto at = [&](int e) { return e + (int)(__umul24((uint32_t)e, magic) >> 20) * pad; };   // e: row classes + class
    if (row_stride == classes && ((uintptr_t)z & 15) == 0) {
        const int vecs = all / V;
        for (int u0 = threadIdx.x; u0 < vecs; u0 += ROWS * B) {
            uint4 q[B];
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const int u = u0 + i * ROWS;
                q[i] = *(const uint4*)(z + (u < vecs ? u : u0) * V);
            }
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const int u = u0 + i * ROWS;
                if (u < vecs) {
                    float v[V];
                    T::unpack(q[i], v);
#pragma unroll
                    for (int j = 0; j < V; ++j) s_z[at(u * V + j)] = v[j];
                }
            }
        }
        const int e = vecs * V + (int)threadIdx.x;
        if (e < all) s_z[at(e)] = T::one(z + e);
    } else {
        for (int e = threadIdx.x; e < all; e += ROWS) {
            const int i = (int)(__umul24((uint32_t)e, magic) >> 20);
            s_z[e + i * pad] = T::one(z + i * row_stride + (e - i * classes));
        }
    }
    __syncthreads();
}

template <class T, int ROWS, int MOST>
__global__ void __launch_bounds__(ROWS)
k_label_small(const typename T::type* __restrict__ logits, int64_t n, int classes, uint32_t magic, int64_t row_stride,
              const int64_t* __restrict__ labels, int64_t ignore, int k, Out out) {
    extern __shared__ float s_z[];
    const int64_t row0 = (int64_t)blockIdx.x * ROWS;
    const int rows = (int)(n - row0 < ROWS ? n - row0 : ROWS);
    const int64_t row = row0 + threadIdx.x, y = (int)threadIdx.x < rows ? labels[row] : 0;
    stage_rows<T, ROWS>(logits, row0, rows, classes, magic, row_stride, s_z);
    if ((int)threadIdx.x >= rows) return;
    const float* zr = s_z + threadIdx.x * (classes | 1);
    // the row in registers, four classes at a time; what is behind it is NaN: neither exponentiated (kFloor is
    // the larger) nor taken for the largest
    float z[MOST], m = -kInf;
#pragma unroll
    for (int c = 0; c < MOST; c += 4)
        if (c < classes) {   // the same for all threads, as below
#pragma unroll
            for (int j = c; j < c + 4; ++j) {
                const float v = zr[j < classes ? j : c];
                m = max_nan(m, v);
                z[j] = j < classes ? v : NAN;
            }
        }
    Row r(m != m ? kInf : m);
    float s = 0.f, t = 0.f;
    const auto add = [&](auto x_of) {
#pragma unroll
        for (int c = 0; c < MOST; c += 4)
            if (c < classes) {
#pragma unroll
                for (int j = c; j < c + 4; ++j) {
                    const float x = fmaxf(x_of(z[j]), kFloor), e = __builtin_amdgcn_exp2f(x);
                    s += e;
                    t = fmaf(e, x, t);
                }
            }
    };
    if (!r.far) add([&](float v) { return fmaf(v, kL, -r.ml); });
    else add([&](float v) { return (v - r.m) * kL; });
    r.ls = r.dead() ? 0.f : __builtin_amdgcn_logf(s);
    put_row(out, r, row, s, t, y >= 0 && y < classes ? zr[y] : 0.f, y, ignore, classes);
    if (r.bad()) {
        for (int i = 0; i < k; ++i) put_top(out, r, row * k + i, 0);
        return;
    }
    // k times the largest, then the first that equals it; what was taken is NaN
    float best = m;
    for (int i = 0; i < k; ++i) {
        int at = 0;
#pragma unroll
        for (int c = MOST - 4; c >= 0; c -= 4)
            if (c < classes) {
#pragma unroll
                for (int j = c + 3; j >= c; --j) at = z[j] == best ? j : at;
            }
        out.top_lp[row * k + i] = r.log_prob(best);
        out.top_idx[row * k + i] = at;
        if (i + 1 == k) break;
        best = -kInf;
#pragma unroll
        for (int c = 0; c < MOST; c += 4)
            if (c < classes) {
#pragma unroll
                for (int j = c; j < c + 4; ++j) {
                    z[j] = j == at ? NAN : z[j];
                    best = fmaxf(best, z[j]);
                }
            }
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
    // top: the sum of the alternatives' upstream gradients
    __device__ __forceinline__ RowGrad(const float* stats, const Grads& u, int64_t row, int64_t y, int64_t ignore,
                                       int64_t classes, float top)
        : r(stats[3 * row]) {
        r.ls = stats[3 * row + 1];
        lp = u.lp && y != ignore ? (y < 0 || y >= classes ? NAN : u.lp[row]) : 0.f;
        gh = u.ent ? u.ent[row] * kLn2 : 0.f;
        h = stats[3 * row + 2] * kL;
        g = lp + top;
    }
    // without the given terms
    __device__ __forceinline__ float dz(float z) const {
        const float x = fmaxf(r.x(z) - r.ls, kFloor);
        return -__builtin_amdgcn_exp2f(x) * fmaf(gh, x + h, g);
    }
    __device__ __forceinline__ float value(float z) const { return r.dead() ? 0.f : r.bad() ? NAN : dz(z); }
};

template <int LANES>
__device__ __forceinline__ float sum_of(float v) {   // over a row's lanes, of more than 64 over the wave's
    return LANES == 16 ? __uint_as_float(rows_of_16(__float_as_uint(v), AddF())) : wave_sum(v);
}

// LANES threads per row, or per part of it (gridDim.y of them).  The vectors are the gradient's, aligned; the
// logits' may lie otherwise.
template <class T, int LANES>
__global__ void __launch_bounds__(256)
k_label_bwd(const typename T::type* __restrict__ logits, int64_t n, int classes, int64_t row_stride,
            const int64_t* __restrict__ labels, int64_t ignore, int k, const int64_t* __restrict__ top_idx,
            const float* __restrict__ stats, Grads u, int part, typename T::type* __restrict__ out) {
    constexpr int V = T::N, B = 4;
    const int lane = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const bool on = row < n;
    const typename T::type* z = logits + (on ? row : 0) * row_stride;
    typename T::type* o = out + (on ? row : 0) * classes;
    const Vectors<T> w(o, classes);
    const int u0 = blockIdx.y * part, u1 = u0 + part < w.count ? u0 + part : w.count;
    const int64_t y = on ? labels[row] : ignore;
    // the given terms, one lane each (k < LANES): the alternatives', behind them the label's, which an
    // alternative of the same class takes along
    const int g = (int)(threadIdx.x & 63) % LANES;
    const bool top = u.top && on && g < k;
    const int64_t pj = top ? top_idx[row * k + g] : g == k && u.lp && y != ignore ? y : -1;
    const bool given = pj >= 0 && pj < classes;
    const float pz = given ? T::one(z + pj) : 0.f;
    float more = top ? u.top[row * k + g] : 0.f;
    const RowGrad d(stats, u, on ? row : 0, y, ignore, classes, u.top ? sum_of<LANES>(more) : 0.f);
    const bool plain = !d.r.bad() && !d.r.dead(), some_far = __any(d.r.far);
    const float off = d.r.far ? 0.f : d.r.ml, from = d.r.far ? d.r.m : 0.f;   // x = (z - from) L - off
    if (on) {
        for (int v0 = u0 + lane; v0 < u1; v0 += LANES * B) {
            uint4 q[B];
#pragma unroll
            for (int c = 0; c < B; ++c) {
                int v = v0 + c * LANES;
                v = v < w.lo ? w.lo : v > w.hi ? w.hi : v;
                q[c] = load16<T>(z + w.first_class(v));
            }
#pragma unroll
            for (int c = 0; c < B; ++c) {
                const int v = v0 + c * LANES, j = w.first_class(v);
                if (v >= u1) break;
                if (w.whole(v) && plain) {
                    float f[V];
                    T::unpack(q[c], f);
                    if (some_far) {
#pragma unroll
                        for (int i = 0; i < V; ++i) f[i] -= from;
                    }
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float x = fmaxf(fmaf(f[i], kL, -off) - d.r.ls, kFloor);
                        f[i] = -__builtin_amdgcn_exp2f(x) * fmaf(d.gh, x + d.h, d.g);
                    }
                    *(uint4*)(o + j) = T::pack(f);
                } else {
                    for (int i = j < 0 ? 0 : j; i < j + V && i < classes; ++i) T::put(o + i, d.value(T::one(z + i)));
                }
            }
        }
    }
    if (!u.top && !u.lp) return;
    const bool same = top && pj == y;
    uint64_t any = __ballot(same);
    if (LANES == 16) any = any >> (threadIdx.x & 48) & 0xFFFF;
    if (same || g == k) more += d.lp;
    __syncthreads();   // behind the stores of the others
    if (LANES > 64 && threadIdx.x >= 64) return;
    const int u_of = (int)((pj + w.skip) / V);
    if (given && !(g == k && any) && u_of >= u0 && u_of < u1 && !d.r.dead()) T::put(o + pj, d.value(pz) + more);
}

template <class T, int ROWS>
__global__ void __launch_bounds__(ROWS)
k_label_bwd_small(const typename T::type* __restrict__ logits, int64_t n, int classes, uint32_t magic, int64_t row_stride,
                  const int64_t* __restrict__ labels, int64_t ignore, int k, const int64_t* __restrict__ top_idx,
                  const float* __restrict__ stats, Grads u,
                  typename T::type* __restrict__ out) {
    extern __shared__ float s_z[];
    const int64_t row0 = (int64_t)blockIdx.x * ROWS;
    const int rows = (int)(n - row0 < ROWS ? n - row0 : ROWS);
    stage_rows<T, ROWS>(logits, row0, rows, classes, magic, row_stride, s_z);
    const int pitch = classes | 1;
    if ((int)threadIdx.x < rows) {
        const int64_t row = row0 + threadIdx.x, y = labels[row];
        float top = 0.f;
        if (u.top)
            for (int i = 0; i < k; ++i) top += u.top[row * k + i];
        const RowGrad d(stats, u, row, y, ignore, classes, top);
        float* z = s_z + threadIdx.x * pitch;
        if (!d.r.far && !d.r.bad() && !d.r.dead()) {
#pragma unroll 4
            for (int j = 0; j < classes; ++j) {
                const float x = fmaxf(fmaf(z[j], kL, -d.r.ml) - d.r.ls, kFloor);
                z[j] = -__builtin_amdgcn_exp2f(x) * fmaf(d.gh, x + d.h, d.g);
            }
        } else {
            for (int j = 0; j < classes; ++j) z[j] = d.value(z[j]);
        }
        if (!d.r.dead()) {
            if (y != ignore && y >= 0 && y < classes) z[y] += d.lp;
            if (u.top && !d.r.bad())
                for (int i = 0; i < k; ++i) z[top_idx[row * k + i]] += u.top[row * k + i];
        }
    }
    __syncthreads();
    constexpr int V = T::N;
    const int all = rows * classes, pad = pitch - classes;
    const auto at = [&](int e) { return e + (int)(__umul24((uint32_t)e, magic) >> 20) * pad; };
    typename T::type* o = out + row0 * classes;
    const int vecs = ((uintptr_t)o & 15) == 0 ? all / V : 0;
    for (int v = threadIdx.x; v < vecs; v += ROWS) {
        float f[V];
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = s_z[at(v * V + i)];
        *(uint4*)(o + v * V) = T::pack(f);
    }
    for (int e = vecs * V + threadIdx.x; e < all; e += ROWS) T::put(o + e, s_z[at(e)]);
}

// ---- host

bool bad_args(const void* logits, int32_t dtype, int64_t n, int64_t classes, int64_t row_stride, const int64_t* labels,
              int32_t k) {
    if (dtype < PIN_TYPE_F32 || dtype > PIN_TYPE_BF16 || n < 0 || classes < 1 || classes > PIN_LABEL_CLASSES_MAX ||
        row_stride < 0 || k < 0 || k > PIN_LABEL_TOP_MAX || k > classes)
        return true;
    return n > 0 && (!logits || !labels || ((uintptr_t)logits & (dtype == PIN_TYPE_F32 ? 3 : 1)));
}

// How a forward of more than kSmall classes is laid out.
struct Plan {
    int nch;       // one wave per row, nch vectors per lane; 0: parts of `part` vectors, `splits` of them
    int splits, part;
    int alone;     // a workgroup goes through a row alone, this many parts
    int lanes;     // sixteen lanes per row, this many vectors each
};

// Sixteen lanes per row look at their elements once per alternative, a wave per row at a few more than k in
// all, after a longer preparation.  200000 x 128 bf16 with 3 alternatives: 47 us and 121; 16384 x 1003 f16
// with 8: 50 and 24.  A wave whose lanes with elements are hardly more than k finds no bound by them: 200000 x
// 128 with 20: 191 and 485.  With few rows it is the longest row that counts: 64 x 1003 with 8: 23 us and 6.
constexpr int64_t kManyRows = 4096;
constexpr int64_t kFull = 1024;    // workgroups that fill the chip
constexpr int64_t kBatch = 1 << 23;  // rows of one launch
constexpr int64_t kGrid = (1 << 24) - 1;  // workgroups of 256 threads of one launch: it has fewer than 2^32 threads
static_assert(kBatch <= kGrid && kGrid / kSplits >= kFull, "a batch of split rows is many");
// ... when each has a workgroup to itself, or its rows are short: 256 x 50021 bf16 with 20 alternatives 16.8 us
// (in parts, joined, 21.9), 1 x 32768 with 5 8.0 (9.0), but 1 x 131072 with 20 19.6 (12.5).
constexpr int64_t kRows = 256;
constexpr int64_t kShort = 6;

Plan plan_rows(int64_t n, int64_t classes, int v, int k) {
    const int64_t vecs = (classes + 2 * v - 2) / v;   // at any alignment
    Plan p{1, 1, (int)vecs, 0, 0};
    if (vecs <= 16 * 8) {
        int nch = 1;
        while (16 * nch < vecs) nch *= 2;
        const int looks = k * nch * v;   // elements a lane looks at for all alternatives
        if (looks <= (n < kManyRows ? 32 : 160) || (vecs <= 2 * k && n >= kManyRows)) {
            p.lanes = nch;
            return p;
        }
    }
    if (vecs <= 64 * 8) {
        while (64 * p.nch < vecs) p.nch *= 2;
        return p;
    }
    p.nch = 0;
    const int64_t parts = (vecs + kPart - 1) / kPart;
    if (parts <= kRowParts && (n >= kRows || parts <= kShort)) {
        p.part = kPart;
        p.alone = (int)parts;
        return p;
    }
    // no more parts than it takes, but with few rows enough to fill the chip, of two vectors per thread or more
    int64_t s = (vecs + kPart - 1) / kPart;
    if (s > kSplits) s = (vecs + 2 * kPart - 1) / (2 * kPart);
    int64_t more = (kFull + n - 1) / n;
    if (more > (vecs + 511) / 512) more = (vecs + 511) / 512;
    if (more > kSplits) more = kSplits;
    p.splits = (int)(s > more ? s : more);
    p.part = (int)((vecs + p.splits - 1) / p.splits);
    return p;
}

// Rows of one launch, and so rows whose parts lie in the workspace at a time.
inline int64_t batch_of(const Plan& p) { return p.splits > 1 ? kGrid / p.splits : kBatch; }

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

template <class T, int NCH>
void launch_wave(const Call& a) {
    const typename T::type* z = (const typename T::type*)a.logits;
    if (a.k > 0)
        hipLaunchKernelGGL((k_label_wave<T, NCH, true>), dim3((unsigned)a.n), dim3(64), 0, a.st, z, a.n, (int)a.classes,
                           a.row_stride, a.labels, a.ignore, a.k, a.out);
    else
        hipLaunchKernelGGL((k_label_wave<T, NCH, false>), dim3((unsigned)a.n), dim3(64), 0, a.st, z, a.n, (int)a.classes,
                           a.row_stride, a.labels, a.ignore, a.k, a.out);
}

template <class T, int NCH>
void launch_lanes(const Call& a) {
    const typename T::type* z = (const typename T::type*)a.logits;
    const dim3 grid((unsigned)((a.n + 15) / 16));
    if (a.k > 0)
        hipLaunchKernelGGL((k_label_lanes<T, NCH, true>), grid, dim3(256), 0, a.st, z, a.n, (int)a.classes, a.row_stride,
                           a.labels, a.ignore, a.k, a.out);
    else
        hipLaunchKernelGGL((k_label_lanes<T, NCH, false>), grid, dim3(256), 0, a.st, z, a.n, (int)a.classes, a.row_stride,
                           a.labels, a.ignore, a.k, a.out);
}

template <class T>
int forward_rows(const Call& a, const Plan& p) {
    if (a.classes <= kSmall) {
        const int rows = a.classes <= 32 ? 256 : 128;
        const int64_t blocks = (a.n + rows - 1) / rows;
        const size_t lds = (size_t)rows * (a.classes | 1) * 4;
        const typename T::type* z = (const typename T::type*)a.logits;
        const auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(rows), lds, a.st, z, a.n, (int)a.classes,
                               magic_of(a.classes), a.row_stride, a.labels, a.ignore, a.k, a.out);
        };
        if (a.classes <= 8) go(k_label_small<T, 256, 8>);
        else if (a.classes <= 16) go(k_label_small<T, 256, 16>);
        else if (a.classes <= 32) go(k_label_small<T, 256, 32>);
        else go(k_label_small<T, 128, 64>);
        return launch_status();
    }
    if (p.lanes > 0) {
        if (p.lanes == 1) launch_lanes<T, 1>(a);
        else if (p.lanes == 2) launch_lanes<T, 2>(a);
        else if (p.lanes == 4) launch_lanes<T, 4>(a);
        else launch_lanes<T, 8>(a);
        return launch_status();
    }
    if (p.nch > 0) {
        if (p.nch == 1) launch_wave<T, 1>(a);
        else if (p.nch == 2) launch_wave<T, 2>(a);
        else if (p.nch == 4) launch_wave<T, 4>(a);
        else launch_wave<T, 8>(a);
        return launch_status();
    }
    const typename T::type* z = (const typename T::type*)a.logits;
    if (p.alone > 0) {
        hipLaunchKernelGGL((k_label_row<T>), dim3((unsigned)a.n), dim3(256), 0, a.st, z, (int)a.classes, a.row_stride,
                           a.labels, a.ignore, a.k, p.alone, a.out);
        return launch_status();
    }
    if (!a.ws || ((uintptr_t)a.ws & 15)) return PIN_ERR_ARG;
    float4* sums = (float4*)a.ws;
    float* maxima = a.k > 0 ? (float*)(sums + a.n * p.splits) : nullptr;
    const dim3 grid((unsigned)(a.n * p.splits)), rows((unsigned)a.n);
    const auto parts = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, a.st, z, (int)a.classes, a.row_stride, p.splits, p.part, sums, maxima);
    };
    if constexpr (T::N == F32::N) {   // (the longest rows of 16-bit classes fit kSplits parts of kPart)
        if (p.part > kPart) parts(k_label_part<T, 8>);
        else parts(k_label_part<T, 4>);
    } else {
        parts(k_label_part<T, 4>);
    }
    if (a.k > 0)
        hipLaunchKernelGGL((k_label_join_top<T>), rows, dim3(256), 0, a.st, z, (int)a.classes, a.row_stride, a.labels,
                           a.ignore, a.k, p.splits, p.part, a.out, sums, maxima);
    else
        hipLaunchKernelGGL((k_label_join<T>), rows, dim3(64), 0, a.st, z, (int)a.classes, a.row_stride, a.labels, a.ignore,
                           p.splits, a.out, sums);
    return launch_status();
}

// Rows in batches; the batches of split rows take turns in the workspace, which the stream's order allows.
template <class T>
int run_forward(const Call& a) {
    const Plan p = plan_rows(a.n, a.classes, T::N, a.k);
    const int64_t batch = batch_of(p);
    for (int64_t row = 0; row < a.n; row += batch) {
        Call b = a;
        b.n = a.n - row < batch ? a.n - row : batch;
        b.logits = (const typename T::type*)a.logits + row * a.row_stride;
        b.labels += row;
        b.out.log_prob += row;
        b.out.entropy += row;
        if (a.out.stats) b.out.stats += 3 * row;
        if (a.k > 0) b.out.top_lp += row * a.k, b.out.top_idx += row * a.k;
        const int rc = forward_rows<T>(b, p);
        if (rc != PIN_OK) return rc;
    }
    return PIN_OK;
}

template <class T>
int backward_rows(const Call& a, const int64_t* top_idx, const float* stats, const Grads& u, void* d_logits) {
    typename T::type* o = (typename T::type*)d_logits;
    const typename T::type* z = (const typename T::type*)a.logits;
    if (a.classes <= kSmall) {
        const int rows = a.classes <= 32 ? 256 : 128;
        const int64_t blocks = (a.n + rows - 1) / rows;
        const size_t lds = (size_t)rows * (a.classes | 1) * 4;
        if (rows == 256)
            hipLaunchKernelGGL((k_label_bwd_small<T, 256>), dim3((unsigned)blocks), dim3(256), lds, a.st, z, a.n,
                               (int)a.classes, magic_of(a.classes), a.row_stride, a.labels, a.ignore, a.k, top_idx, stats,
                               u, o);
        else
            hipLaunchKernelGGL((k_label_bwd_small<T, 128>), dim3((unsigned)blocks), dim3(128), lds, a.st, z, a.n,
                               (int)a.classes, magic_of(a.classes), a.row_stride, a.labels, a.ignore, a.k, top_idx, stats,
                               u, o);
        return launch_status();
    }
    // sixteen lanes per row (and one more than k): 16384 x 1003 f16 with 8 alternatives 18 us, 64 lanes 22;
    // 64 lanes up to 64 * 8 vectors: 16384 x 3000 bf16 45 us, a workgroup 49
    const int lanes = a.classes <= 16 * T::N * 8 && a.k < 16 ? 16 : a.classes <= 64 * T::N * 8 ? 64 : 256;
    const int64_t vecs = (a.classes + 2 * T::N - 2) / T::N;
    const int part = lanes == 256 ? 256 * 4 : (int)vecs;
    const int64_t parts = (vecs + part - 1) / part;
    const int64_t blocks = (a.n + 256 / lanes - 1) / (256 / lanes);
    if (parts > 65535) return PIN_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)blocks, (unsigned)parts);
    if (lanes == 16)
        hipLaunchKernelGGL((k_label_bwd<T, 16>), grid, dim3(256), 0, a.st, z, a.n, (int)a.classes, a.row_stride, a.labels,
                           a.ignore, a.k, top_idx, stats, u, part, o);
    else if (lanes == 64)
        hipLaunchKernelGGL((k_label_bwd<T, 64>), grid, dim3(256), 0, a.st, z, a.n, (int)a.classes, a.row_stride, a.labels,
                           a.ignore, a.k, top_idx, stats, u, part, o);
    else
        hipLaunchKernelGGL((k_label_bwd<T, 256>), grid, dim3(256), 0, a.st, z, a.n, (int)a.classes, a.row_stride, a.labels,
                           a.ignore, a.k, top_idx, stats, u, part, o);
    return launch_status();
}

template <class T>
int run_backward(const Call& a, const int64_t* top_idx, const float* stats, const Grads& u, void* d_logits) {
    for (int64_t row = 0; row < a.n; row += kBatch) {
        Call b = a;
        b.n = a.n - row < kBatch ? a.n - row : kBatch;
        b.logits = (const typename T::type*)a.logits + row * a.row_stride;
        b.labels += row;
        const Grads v{u.lp ? u.lp + row : nullptr, u.ent ? u.ent + row : nullptr, u.top ? u.top + row * a.k : nullptr};
        const int rc = backward_rows<T>(b, top_idx ? top_idx + row * a.k : nullptr, stats + 3 * row, v,
                                        (typename T::type*)d_logits + row * a.classes);
        if (rc != PIN_OK) return rc;
    }
    return PIN_OK;
}

}  // namespace

extern "C" {

int64_t pin_label_logprob_workspace_bytes(int64_t n, int64_t classes, int32_t dtype, int32_t top_k) {
    if (dtype < PIN_TYPE_F32 || dtype > PIN_TYPE_BF16 || n < 0 || classes < 1 || classes > PIN_LABEL_CLASSES_MAX ||
        top_k < 0 || top_k > PIN_LABEL_TOP_MAX)
        return PIN_ERR_ARG;
    if (n == 0 || classes <= kSmall) return 0;
    const Plan p = plan_rows(n, classes, dtype == PIN_TYPE_F32 ? F32::N : F16::N, top_k);
    const int64_t rows = n < batch_of(p) ? n : batch_of(p);
    return p.lanes > 0 || p.nch > 0 || p.alone > 0 ? 0 : rows * p.splits * (16 + (top_k > 0 ? 256 : 0));
}

int pin_label_logprob(const void* logits, int32_t dtype, int64_t n, int64_t classes, int64_t row_stride,
                      const int64_t* labels, int64_t ignore_index, int32_t top_k, float* log_prob, float* entropy,
                      float* row_stats, float* top_log_prob, int64_t* top_index, void* workspace, void* stream) {
    if (bad_args(logits, dtype, n, classes, row_stride, labels, top_k)) return PIN_ERR_ARG;
    if (n == 0) return PIN_OK;
    if (!log_prob || !entropy || (top_k > 0 && (!top_log_prob || !top_index)))
        return PIN_ERR_ARG;
    const Call a{logits, n, classes, row_stride, labels, ignore_index, (int)top_k,
                 Out{log_prob, entropy, row_stats, top_log_prob, top_index}, workspace, as_stream(stream)};
    return dtype == PIN_TYPE_F32 ? run_forward<F32>(a) : dtype == PIN_TYPE_F16 ? run_forward<F16>(a) : run_forward<BF16>(a);
}

int pin_label_logprob_bwd(const void* logits, int32_t dtype, int64_t n, int64_t classes, int64_t row_stride,
                          const int64_t* labels, int64_t ignore_index, int32_t top_k, const int64_t* top_index,
                          const float* row_stats, const float* d_log_prob, const float* d_entropy, const float* d_top,
                          void* d_logits, void* stream) {
    if (bad_args(logits, dtype, n, classes, row_stride, labels, top_k)) return PIN_ERR_ARG;
    if (n == 0) return PIN_OK;
    if (!row_stats || !d_logits || (d_top && top_k > 0 && !top_index) ||
        ((uintptr_t)d_logits & (dtype == PIN_TYPE_F32 ? 3 : 1)))
        return PIN_ERR_ARG;
    const Call a{logits, n, classes, row_stride, labels, ignore_index, (int)top_k, Out{}, nullptr, as_stream(stream)};
    const Grads u{d_log_prob, d_entropy, top_k > 0 ? d_top : nullptr};
    return dtype == PIN_TYPE_F32   ? run_backward<F32>(a, top_index, row_stats, u, d_logits)
           : dtype == PIN_TYPE_F16 ? run_backward<F16>(a, top_index, row_stats, u, d_logits)
                                   : run_backward<BF16>(a, top_index, row_stats, u, d_logits);
}

}  // extern "C"
