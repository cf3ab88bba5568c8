// pin_adamw.hip -- AdamW over many tensors at once, the two moments held in 32 bits or in 8.
// Beside the mapping loop's Adam kernels (pin_train.hip), which step f32 features and one decoder.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// State lies in flat arrays in which each tensor begins at a multiple of 256 elements.
//
// Moments in 8 bits.  256 consecutive elements of an array share a power of two per moment, the
// exponent E of the block's largest finite value.
//   first moment   sign, 4 bits of exponent, 3 of mantissa: the bit pattern of an e4m3 float whose
//                  value 2^7 stands for 2^E (down to 2^(E-16) with gradual underflow); 0x7F = NaN
//   second moment  5 bits of exponent e, 3 of mantissa f: (1 + f/8) 2^(e - 30 + E); 0 = zero,
//                  0xFF = NaN.  A positive second moment is never stored as zero: it divides.
// Moving averages change by (1 - b) of a difference per step, far less than half a code: rounding
// to nearest would hold them where they are.  So a value between two codes goes to the upper one
// with the probability of its place between them, decided by 17 bits that a hash makes of the
// element's place and the step: its expectation is kept, the same call gives the same bits, and
// no element depends on another.  Averages are formed in 64 bits from the decoded values, so
// neither the codes nor their exponents depend on a rounding of the arithmetic.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <math.h>
#include <stdint.h>

#include "pin_slam_amd.h"

namespace {

constexpr int kBlock = 256;
constexpr int kGroup = PIN_ADAMW_BLOCK;       // elements that share their exponents
constexpr int kChunk = 1024;                  // elements of one workgroup
constexpr int64_t kChunks = 0xFFFFFFFFll / kBlock;   // workgroups of one launch: it has fewer than 2^32 threads
constexpr int kTensors = 112;                 // tensors of one launch (its table is a kernel argument)
static_assert(kTensors <= 128, "the table is searched by two ballots");
constexpr uint32_t kMix1 = 0x9E3779B1u, kMix2 = 0x6A09E667u, kMix3 = 0xBB67AE85u;   // fractional bits of the
                                                                                    // golden ratio, sqrt 2, sqrt 3
constexpr int kLeast = -900;                  // least exponent of a block

struct AdamwTable {
    void* p[kTensors];
    const void* g[kTensors];
    int64_t n[kTensors];
    uint32_t block0[kTensors];   // first 256-element block of the state
    uint32_t chunk0[kTensors];   // first workgroup
    int count;
};

struct AdamwScalars {
    double b1, b2, c1, c2;       // betas, 1 - betas
    float decay, step_size, bc2_sqrt;
    uint32_t key;
};
static_assert(sizeof(AdamwScalars) <= PIN_ADAMW_SCALARS_BYTES, "");

__host__ __device__ inline uint32_t mix32(uint32_t x) {
    x ^= x >> 16;
    x *= kMix1;
    x ^= x >> 15;
    x *= kMix2;
    return x ^ (x >> 16);
}

__host__ __device__ inline AdamwScalars adamw_scalars(double lr, double b1, double b2, double wd, int64_t step,
                                                      uint32_t salt) {
    AdamwScalars a;
    a.b1 = b1;
    a.b2 = b2;
    a.c1 = 1.0 - b1;
    a.c2 = 1.0 - b2;
    a.decay = (float)(1.0 - lr * wd);
    a.step_size = (float)(lr / (1.0 - pow(b1, (double)step)));
    a.bc2_sqrt = (float)sqrt(1.0 - pow(b2, (double)step));
    a.key = mix32(salt + (uint32_t)step * kMix2);
    return a;
}

__global__ void k_adamw_scalars(int64_t* __restrict__ step, const float* __restrict__ lr_dev, double lr, double b1,
                                double b2, double wd, uint32_t salt, AdamwScalars* __restrict__ out) {
    const int64_t t = *step + 1;
    *step = t;
    *out = adamw_scalars(lr_dev ? (double)*lr_dev : lr, b1, b2, wd, t, salt);
}

inline hipStream_t as_stream(void* s) { return (hipStream_t)s; }
inline int launch_status() { return hipGetLastError() == hipSuccess ? PIN_OK : PIN_ERR_HIP; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half(v); }
__device__ __forceinline__ void from_f32(float v, __hip_bfloat16& o) { o = __float2bfloat16(v); }

// four consecutive elements in one access, or (where they are not all there, or not aligned) one by one;
// which of the two is the same for the wave
template <class T>
struct alignas(4 * sizeof(T)) Four {
    T v[4];
};
template <class T>
__device__ __forceinline__ bool aligned4(const T* p) {
    return ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0;
}
template <class T>
__device__ __forceinline__ void load4(const T* __restrict__ p, int64_t i, int64_t n, bool whole, float (&o)[4]) {
    if (whole) {
        const Four<T> f = *(const Four<T>*)(p + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = to_f32(f.v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = i + k < n ? to_f32(p[i + k]) : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void store4(T* __restrict__ p, int64_t i, int64_t n, bool whole, const float (&v)[4]) {
    if (whole) {
        Four<T> f;
#pragma unroll
        for (int k = 0; k < 4; ++k) from_f32(v[k], f.v[k]);
        *(Four<T>*)(p + i) = f;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) from_f32(v[k], p[i + k]);
    }
}

// the tensor of a workgroup: the last whose first workgroup is not behind it
__device__ __forceinline__ int find_tensor(const AdamwTable& t, uint32_t chunk) {
    const int lane = threadIdx.x & 63;
    const uint32_t a = lane < t.count ? t.chunk0[lane] : ~0u;
    const uint32_t b = lane + 64 < t.count ? t.chunk0[lane + 64] : ~0u;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(a <= chunk)) + __popcll(__ballot(b <= chunk)) - 1);
}

__device__ __forceinline__ int wave_of() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

__device__ __forceinline__ float adamw_update(float p, float m, float v, float eps, const AdamwScalars& a) {
    p = p * a.decay;
    return p - a.step_size * (m / (sqrtf(v) / a.bc2_sqrt + eps));
}

template <class T, bool MASTER>
__global__ void __launch_bounds__(kBlock)
k_adamw32(AdamwTable t, float* __restrict__ m_, float* __restrict__ v_, float* __restrict__ w_, float eps,
          AdamwScalars host, const AdamwScalars* __restrict__ dev) {
    const AdamwScalars a = dev ? *dev : host;
    const int k = find_tensor(t, blockIdx.x);
    const int64_t n = t.n[k];
    const int64_t i0 = (int64_t)(blockIdx.x - t.chunk0[k]) * kChunk + wave_of() * kGroup, i = i0 + (threadIdx.x & 63) * 4;
    if (i >= n) return;
    const int64_t s = (int64_t)t.block0[k] * kGroup + i;   // 16-byte aligned, padded to whole blocks
    const T* gp = (const T*)t.g[k];
    T* pp = (T*)t.p[k];
    const bool all = i0 + kGroup <= n;
    float p[4], g[4];
    load4(gp, i, n, all && aligned4(gp), g);
    if (MASTER) load4(w_ + (s - i), i, n, all, p);
    else load4((const T*)pp, i, n, all && aligned4(pp), p);
    float4 m4 = *(float4*)(m_ + s), v4 = *(float4*)(v_ + s);
    float m[4] = {m4.x, m4.y, m4.z, m4.w}, v[4] = {v4.x, v4.y, v4.z, v4.w};
    const float b1 = (float)a.b1, b2 = (float)a.b2, c1 = (float)a.c1, c2 = (float)a.c2;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        m[j] = m[j] * b1 + g[j] * c1;
        v[j] = v[j] * b2 + (c2 * g[j]) * g[j];   // in this order: g^2 itself may be out of range
        p[j] = adamw_update(p[j], m[j], v[j], eps, a);
    }
    *(float4*)(m_ + s) = make_float4(m[0], m[1], m[2], m[3]);
    *(float4*)(v_ + s) = make_float4(v[0], v[1], v[2], v[3]);
    if (MASTER) store4(w_ + (s - i), i, n, all, p);
    store4(pp, i, n, all && aligned4(pp), p);
}

__device__ __forceinline__ double pow2(int e) { return __longlong_as_double((long long)(e + 1023) << 52); }

// the decoded values without their blocks' powers of two: first moment * 2^(7 - E), second * 2^-E
__device__ __forceinline__ void decode_m(uint32_t c, float (&o)[4]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    o[0] = a.x;
    o[1] = a.y;
    o[2] = b.x;
    o[3] = b.y;
}
__device__ __forceinline__ float decode_v(uint32_t c) {
    const float x = __uint_as_float((c + ((127 - 30) << 3)) << 20);
    return c == 0 ? 0.f : c == 0xFF ? __uint_as_float(0x7FC00000u) : x;
}

__device__ __forceinline__ uint32_t hi32(double x) { return (uint32_t)((uint64_t)__double_as_longlong(x) >> 32); }

template <int CTRL>
__device__ __forceinline__ int max_of_lanes(int v) {
    const int b = __builtin_amdgcn_update_dpp(v, v, CTRL, 0xF, 0xF, false);
    return b > v ? b : v;
}
// the largest of the wave's values
__device__ __forceinline__ int wave_max(int v) {
    v = max_of_lanes<0xB1>(v);    // lanes ^ 1
    v = max_of_lanes<0x4E>(v);    // lanes ^ 2
    v = max_of_lanes<0x141>(v);   // the other half of 8
    v = max_of_lanes<0x140>(v);   // the other half of 16
    const int a = max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
    return max(a, max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// exponent of the largest finite of a block's values, four per lane
__device__ __forceinline__ int block_exponent(const double (&x)[4]) {
    int h = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int a = (int)(hi32(x[j]) & 0x7FFFFFFF);
        h = a < 0x7FF00000 && a > h ? a : h;
    }
    const int e = (wave_max(h) >> 20) - 1023;
    return e < kLeast ? kLeast : e;
}

__device__ __forceinline__ uint32_t encode_m(double x, int e, uint32_t dither) {
    const uint32_t h = hi32(x), a = h & 0x7FFFFFFF;
    int c = (int)((a + dither) >> 17) - ((e + 1023 - 14) << 3);
    if ((int)a < (e - 13 + 1023) << 20) c = (int)(fabs(x) * pow2(16 - e) + (double)dither * 0x1p-17);
    return a >= 0x7FF00000u ? 0x7F : (uint32_t)c | (h >> 31 << 7);
}
__device__ __forceinline__ uint32_t encode_v(double x, int e, uint32_t dither) {
    const uint32_t h = hi32(x);
    int c = (int)((h + dither) >> 17) - ((e + 1023 - 30) << 3);
    c = x > 0.0 ? (c < 1 ? 1 : c) : 0;
    return h >= 0x7FF00000u ? 0xFF : (uint32_t)c;
}

// One wave per block of 256 elements, four per lane.  The parameter's step is taken in f32 from the new
// averages before they are coded, numerator and denominator over a power of two: that of the block's largest
// square root or of eps, whichever is larger, so that the denominator is at most a few units whatever the
// size of the gradients and however far the second moment has decayed.  What the hardware's square root and
// reciprocal (one unit in the last place each) need is normal numbers.  Elements for which that does not give
// them (a second moment far below its block's largest with hardly any eps beside it, a first moment that is
// beyond f32 over the power of two) take the step in 64 bits.
template <class T, bool MASTER>
__global__ void __launch_bounds__(kBlock)
k_adamw8(AdamwTable t, uint32_t* __restrict__ m_, uint32_t* __restrict__ v_, short2* __restrict__ e_,
         float* __restrict__ w_, float eps, AdamwScalars host, const AdamwScalars* __restrict__ dev) {
    const AdamwScalars a = dev ? *dev : host;
    const int k = find_tensor(t, blockIdx.x);
    const int64_t n = t.n[k];
    const int64_t i0 = (int64_t)(blockIdx.x - t.chunk0[k]) * kChunk + wave_of() * kGroup;
    if (i0 >= n) return;
    const int lane = threadIdx.x & 63;
    const int64_t b = (int64_t)t.block0[k] + i0 / kGroup;
    const int64_t i = i0 + lane * 4, s = b * kGroup + lane * 4;
    const T* gp = (const T*)t.g[k];
    T* pp = (T*)t.p[k];
    const bool all = i0 + kGroup <= n, pa = all && aligned4(pp);
    float p[4], g[4], cm[4];
    load4(gp, i, n, all && aligned4(gp), g);
    if (MASTER) load4(w_ + (s - i), i, n, all, p);
    else load4((const T*)pp, i, n, pa, p);
    const uint32_t um = m_[s / 4], uv = v_[s / 4];
    const short2 e = e_[b];
    decode_m(um, cm);
    const double sm = pow2(e.x - 7) * a.b1, sv = pow2(e.y) * a.b2;
    double m[4], v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const double d = (double)g[j];
        m[j] = (double)cm[j] * sm + d * a.c1;
        v[j] = (double)decode_v((uv >> 8 * j) & 0xFF) * sv + d * d * a.c2;
    }
    const int em = block_exponent(m), ev = block_exponent(v), ee = ((__float_as_int(eps) >> 23) & 0xFF) - 127;
    const int half = ev >> 1 > ee ? ev >> 1 : ee;   // (ee of 0 is -127)
    const double down = pow2(-half), down2 = pow2(-2 * half);
    const float inv = 1.f / a.bc2_sqrt, eps_down = (float)((double)eps * down);
    float d[4], vs[4], ms[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        vs[j] = (float)(v[j] * down2);
        ms[j] = (float)(m[j] * down);
        d[j] = ms[j] * __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_sqrtf(vs[j]), inv, eps_down));
    }
    // Beside this much of eps, what f32 cannot hold of a second moment (2^-126 and less) adds nothing.
    if (eps_down < inv * 0x1p-36f || em - half > 125) {   // the same for the wave
        // a first moment of zero asks for no more than a denominator that is not
        const float still = eps_down >= 0x1p-100f ? 0.f : 0x1p-100f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (!(vs[j] >= (m[j] == 0.0 ? still : 0x1p-100f) && fabsf(ms[j]) <= 0x1p126f))
                d[j] = (float)(m[j] / (sqrt(v[j]) * (double)inv + (double)eps));
    }
    uint32_t om = 0, ov = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        p[j] = p[j] * a.decay - a.step_size * d[j];
        const uint32_t h = mix32(a.key + ((uint32_t)s + j) * kMix3);
        om |= encode_m(m[j], em, h & 0x1FFFF) << 8 * j;
        ov |= encode_v(v[j], ev, h >> 15) << 8 * j;
    }
    m_[s / 4] = om;
    v_[s / 4] = ov;
    if (lane == 0) e_[b] = make_short2((short)em, (short)ev);
    if (MASTER) store4(w_ + (s - i), i, n, all, p);
    store4(pp, i, n, pa, p);
}

__global__ void __launch_bounds__(kBlock)
k_adamw_moments(const uint32_t* __restrict__ m_, const uint32_t* __restrict__ v_, const short2* __restrict__ e_,
                int64_t quads, float4* __restrict__ om, float4* __restrict__ ov) {
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i >= quads) return;
    const short2 e = e_[i / (kGroup / 4)];
    const double sm = pow2(e.x - 7), sv = pow2(e.y);
    float c[4], m[4], v[4];
    decode_m(m_[i], c);
    const uint32_t uv = v_[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        m[j] = (float)((double)c[j] * sm);
        v[j] = (float)((double)decode_v((uv >> 8 * j) & 0xFF) * sv);
    }
    om[i] = make_float4(m[0], m[1], m[2], m[3]);
    ov[i] = make_float4(v[0], v[1], v[2], v[3]);
}

template <class T>
void launch_adamw(const AdamwTable& t, uint32_t chunks, int bits, void* m, void* v, int16_t* e, float* w, float eps,
                  const AdamwScalars& a, const AdamwScalars* dev, hipStream_t st) {
    const dim3 grid(chunks), block(kBlock);
    if (bits == 32 && w)
        hipLaunchKernelGGL((k_adamw32<T, true>), grid, block, 0, st, t, (float*)m, (float*)v, w, eps, a, dev);
    else if (bits == 32)
        hipLaunchKernelGGL((k_adamw32<T, false>), grid, block, 0, st, t, (float*)m, (float*)v, w, eps, a, dev);
    else if (w)
        hipLaunchKernelGGL((k_adamw8<T, true>), grid, block, 0, st, t, (uint32_t*)m, (uint32_t*)v, (short2*)e, w, eps, a,
                           dev);
    else
        hipLaunchKernelGGL((k_adamw8<T, false>), grid, block, 0, st, t, (uint32_t*)m, (uint32_t*)v, (short2*)e, w, eps, a,
                           dev);
}

bool good_rates(double lr, double b1, double b2, double wd) {
    return lr >= 0.0 && isfinite(lr) && b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0 && wd >= 0.0 && isfinite(wd);
}

}  // namespace

extern "C" {

int pin_adamw_scalars(int64_t* step, const float* lr_device, double lr, double beta1, double beta2,
                      double weight_decay, uint32_t salt, void* scalars, void* stream) {
    if (!step || !scalars || ((uintptr_t)scalars & 7) || !good_rates(lr_device ? 0.0 : lr, beta1, beta2, weight_decay))
        return PIN_ERR_ARG;
    hipLaunchKernelGGL(k_adamw_scalars, dim3(1), dim3(1), 0, as_stream(stream), step, lr_device, lr, beta1, beta2,
                       weight_decay, salt, (AdamwScalars*)scalars);
    return launch_status();
}

int pin_adamw_step(void* const* params, const void* const* grads, const int64_t* sizes, const int64_t* offsets,
                   int32_t count, int32_t dtype, int32_t state_bits, void* exp_avg, void* exp_avg_sq,
                   int16_t* exponents, float* master, int64_t state_elements, double lr, double beta1, double beta2,
                   double eps, double weight_decay, int64_t step, uint32_t salt, const void* scalars, void* stream) {
    if (count < 0 || (count > 0 && (!params || !grads || !sizes || !offsets || !exp_avg || !exp_avg_sq)) ||
        dtype < PIN_TYPE_F32 || dtype > PIN_TYPE_BF16 || (state_bits != 8 && state_bits != 32) ||
        (count > 0 && state_bits == 8 && !exponents) || !(eps >= 0.0) || ((uintptr_t)scalars & 7) ||
        (!scalars && (step < 1 || !good_rates(lr, beta1, beta2, weight_decay))))
        return PIN_ERR_ARG;
    if (((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq | (uintptr_t)master) & 15 || ((uintptr_t)exponents & 3))
        return PIN_ERR_ARG;
    if (state_elements < 0 || state_elements % kGroup || state_elements / kGroup > 0xFFFFFFFFll) return PIN_ERR_ARG;
    const uintptr_t odd = dtype == PIN_TYPE_F32 ? 3 : 1;
    int64_t behind = 0;   // every tensor's blocks lie behind the last one's: no two share a block
    for (int32_t k = 0; k < count; ++k) {
        if (sizes[k] < 0 || offsets[k] < behind || offsets[k] % kGroup || sizes[k] > state_elements - offsets[k])
            return PIN_ERR_ARG;
        if (sizes[k] > 0 && (!params[k] || !grads[k] || (((uintptr_t)params[k] | (uintptr_t)grads[k]) & odd)))
            return PIN_ERR_ARG;
        behind = offsets[k] + (sizes[k] + kGroup - 1) / kGroup * kGroup;
    }
    const AdamwScalars a = scalars ? AdamwScalars{} : adamw_scalars(lr, beta1, beta2, weight_decay, step, salt);
    AdamwTable t;
    t.count = 0;
    int64_t chunks = 0;
    for (int32_t k = 0; k <= count; ++k) {
        const int64_t more = k < count ? (sizes[k] + kChunk - 1) / kChunk : 0;
        if (more > kChunks) return PIN_ERR_UNSUPPORTED;
        if (t.count > 0 && (k == count || t.count == kTensors || chunks + more > kChunks)) {
            if (dtype == PIN_TYPE_F32)
                launch_adamw<float>(t, (uint32_t)chunks, state_bits, exp_avg, exp_avg_sq, exponents, master, (float)eps, a,
                                    (const AdamwScalars*)scalars, as_stream(stream));
            else if (dtype == PIN_TYPE_F16)
                launch_adamw<__half>(t, (uint32_t)chunks, state_bits, exp_avg, exp_avg_sq, exponents, master, (float)eps, a,
                                     (const AdamwScalars*)scalars, as_stream(stream));
            else
                launch_adamw<__hip_bfloat16>(t, (uint32_t)chunks, state_bits, exp_avg, exp_avg_sq, exponents, master,
                                             (float)eps, a, (const AdamwScalars*)scalars, as_stream(stream));
            const int rc = launch_status();
            if (rc != PIN_OK) return rc;
            t.count = 0;
            chunks = 0;
        }
        if (more == 0) continue;
        t.p[t.count] = params[k];
        t.g[t.count] = grads[k];
        t.n[t.count] = sizes[k];
        t.block0[t.count] = (uint32_t)(offsets[k] / kGroup);
        t.chunk0[t.count] = (uint32_t)chunks;
        ++t.count;
        chunks += more;
    }
    return PIN_OK;
}

int pin_adamw_moments(const void* exp_avg, const void* exp_avg_sq, const int16_t* exponents, int64_t n, float* m,
                      float* v, void* stream) {
    if (n < 0 || n % kGroup) return PIN_ERR_ARG;
    if (n == 0) return PIN_OK;
    if (!exp_avg || !exp_avg_sq || !exponents || !m || !v) return PIN_ERR_ARG;
    if (((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq | (uintptr_t)exponents) & 3 || ((uintptr_t)m | (uintptr_t)v) & 15)
        return PIN_ERR_ARG;
    const int64_t blocks = (n / 4 + kBlock - 1) / kBlock;
    if (blocks > kChunks) return PIN_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(k_adamw_moments, dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream),
                       (const uint32_t*)exp_avg, (const uint32_t*)exp_avg_sq, (const short2*)exponents, n / 4, (float4*)m,
                       (float4*)v);
    return launch_status();
}

}  // extern "C"
