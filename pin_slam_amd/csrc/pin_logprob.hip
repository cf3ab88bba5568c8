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
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <math.h>
#include <stdint.h>

#include "pin_slam_amd.h"

namespace {

constexpr int kBlock = 256;
constexpr float kInf = __builtin_huge_valf();

inline hipStream_t as_stream(void* s) { return (hipStream_t)s; }
inline int launch_status() { return hipGetLastError() == hipSuccess ? PIN_OK : PIN_ERR_HIP; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half(v); }
__device__ __forceinline__ void from_f32(float v, __hip_bfloat16& o) { o = __float2bfloat16(v); }

// a f32 value as an unsigned key in the same order, both zeros the same
__device__ __forceinline__ uint32_t order_key(float v) {
    const int32_t b = __float_as_int(v + 0.0f);
    return (uint32_t)(b < 0 ? ~b : b | (int32_t)0x80000000);
}

template <class F>
__device__ __forceinline__ float block_reduce(float v, float* sh, F f) {
    for (int o = 32; o; o >>= 1) v = f(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
    for (int w = 1; w < kBlock / 64; ++w) v = f(v, sh[w]);
    return v;
}

template <class T>
__global__ void __launch_bounds__(kBlock)
k_label_logprob(const T* __restrict__ logits, int64_t n, int64_t classes, int64_t row_stride,
                const int64_t* __restrict__ labels, int64_t ignore, int k, float* __restrict__ log_prob,
                float* __restrict__ entropy, float* __restrict__ stats, float* __restrict__ top_lp,
                int64_t* __restrict__ top_idx) {
    __shared__ float sh[kBlock / 64];
    __shared__ unsigned long long sk[kBlock / 64];
    const auto add = [](float a, float b) { return a + b; };
    for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
        const T* z = logits + r * row_stride;
        float m = -kInf, bad = 0.f;
        for (int64_t j = threadIdx.x; j < classes; j += kBlock) {
            const float v = to_f32(z[j]);
            m = fmaxf(m, v);
            bad += !(v < kInf) ? 1.f : 0.f;
        }
        m = block_reduce(m, sh, [](float a, float b) { return fmaxf(a, b); });
        bad = block_reduce(bad, sh, add);
        float s = 0.f, t = 0.f;
        for (int64_t j = threadIdx.x; j < classes; j += kBlock) {
            const float d = to_f32(z[j]) - m;
            if (d > -kInf) {
                const float e = expf(d);
                s += e;
                t += e * d;
            }
        }
        s = block_reduce(s, sh, add);
        t = block_reduce(t, sh, add);
        const bool dead = !bad && m == -kInf;
        const float ls = bad ? NAN : dead ? 0.f : logf(s);
        if (bad) m = NAN;
        if (threadIdx.x == 0) {
            const int64_t y = labels[r];
            float lp = 0.f;
            if (y != ignore) {
                lp = y < 0 || y >= classes ? NAN : dead ? -kInf : (to_f32(z[y]) - m) - ls;
            }
            log_prob[r] = lp;
            entropy[r] = bad ? NAN : dead ? 0.f : ls - t / s;
            if (stats) {
                stats[2 * r] = m;
                stats[2 * r + 1] = ls;
            }
        }
        // the k largest (value, then the lower class): a round finds the largest below the last
        unsigned long long last = ~0ull;
        for (int q = 0; q < k; ++q) {
            unsigned long long best = 0;
            for (int64_t j = threadIdx.x; j < classes; j += kBlock) {
                const unsigned long long key = ((unsigned long long)order_key(to_f32(z[j])) << 32) | (uint32_t)~(uint32_t)j;
                if (key < last && key > best) best = key;
            }
            for (int o = 32; o; o >>= 1) {
                const unsigned long long b = __shfl_xor(best, o);
                best = b > best ? b : best;
            }
            __syncthreads();
            if ((threadIdx.x & 63) == 0) sk[threadIdx.x >> 6] = best;
            __syncthreads();
            for (int w = 0; w < kBlock / 64; ++w) best = sk[w] > best ? sk[w] : best;
            last = best;
            if (threadIdx.x == 0) {
                const int64_t j = (uint32_t)~(uint32_t)best;
                top_idx[r * k + q] = bad ? -1 : j;
                top_lp[r * k + q] = bad ? NAN : dead ? -kInf : (to_f32(z[j]) - m) - ls;
            }
        }
        __syncthreads();
    }
}

template <class T>
__global__ void __launch_bounds__(kBlock)
k_label_logprob_bwd(const T* __restrict__ logits, int64_t n, int64_t classes, int64_t row_stride,
                    const int64_t* __restrict__ labels, int64_t ignore, int k, const int64_t* __restrict__ top_idx,
                    const float* __restrict__ stats, const float* __restrict__ entropy,
                    const float* __restrict__ d_lp, const float* __restrict__ d_ent, const float* __restrict__ d_top,
                    T* __restrict__ out) {
    for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
        const T* z = logits + r * row_stride;
        const int64_t y = labels[r];
        const float m = stats[2 * r], ls = stats[2 * r + 1], h = entropy[r];
        float g_lp = d_lp && y != ignore ? d_lp[r] : 0.f;
        if (d_lp && y != ignore && (y < 0 || y >= classes)) g_lp = NAN;
        const float g_h = d_ent ? d_ent[r] : 0.f;
        float g = g_lp;
        if (d_top)
            for (int q = 0; q < k; ++q) g += d_top[r * k + q];
        const bool dead = m == -kInf;
        for (int64_t j = threadIdx.x; j < classes; j += kBlock) {
            const float d = to_f32(z[j]) - m, lp = d - ls, p = expf(lp);
            float v = -p * g;
            if (p != 0.f) v -= g_h * (p * (lp + h));
            if (j == y) v += g_lp;
            if (d_top)
                for (int q = 0; q < k; ++q) v += top_idx[r * k + q] == j ? d_top[r * k + q] : 0.f;
            from_f32(dead ? 0.f : v, out[r * classes + j]);
        }
    }
}

bool bad_args(const void* logits, int32_t dtype, int64_t n, int64_t classes, int64_t row_stride,
              const int64_t* labels, int32_t k) {
    if (dtype < PIN_TYPE_F32 || dtype > PIN_TYPE_BF16 || n < 0 || classes < 1 || classes > PIN_LABEL_CLASSES_MAX ||
        row_stride < 0 || k < 0 || k > PIN_LABEL_TOP_MAX || k > classes)
        return true;
    return n > 0 && (!logits || !labels || ((uintptr_t)logits & (dtype == PIN_TYPE_F32 ? 3 : 1)));
}

}  // namespace

extern "C" {

int64_t pin_label_logprob_workspace_bytes(int64_t n, int64_t classes, int32_t dtype, int32_t top_k) {
    (void)n;
    (void)classes;
    (void)dtype;
    (void)top_k;
    return 0;
}

int pin_label_logprob(const void* logits, int32_t dtype, int64_t n, int64_t classes, int64_t row_stride,
                      const int64_t* labels, int64_t ignore_index, int32_t top_k, float* log_prob, float* entropy,
                      float* row_stats, float* top_log_prob, int64_t* top_index, void* workspace, void* stream) {
    if (bad_args(logits, dtype, n, classes, row_stride, labels, top_k)) return PIN_ERR_ARG;
    if (n == 0) return PIN_OK;
    if (!log_prob || !entropy || (top_k > 0 && (!top_log_prob || !top_index))) return PIN_ERR_ARG;
    (void)workspace;
    const dim3 grid((unsigned)(n < (1 << 20) ? n : (1 << 20)));
    const hipStream_t st = as_stream(stream);
    if (dtype == PIN_TYPE_F32)
        hipLaunchKernelGGL(k_label_logprob<float>, grid, dim3(kBlock), 0, st, (const float*)logits, n, classes, row_stride,
                           labels, ignore_index, (int)top_k, log_prob, entropy, row_stats, top_log_prob, top_index);
    else if (dtype == PIN_TYPE_F16)
        hipLaunchKernelGGL(k_label_logprob<__half>, grid, dim3(kBlock), 0, st, (const __half*)logits, n, classes, row_stride,
                           labels, ignore_index, (int)top_k, log_prob, entropy, row_stats, top_log_prob, top_index);
    else
        hipLaunchKernelGGL(k_label_logprob<__hip_bfloat16>, grid, dim3(kBlock), 0, st, (const __hip_bfloat16*)logits, n,
                           classes, row_stride, labels, ignore_index, (int)top_k, log_prob, entropy, row_stats,
                           top_log_prob, top_index);
    return launch_status();
}

int pin_label_logprob_bwd(const void* logits, int32_t dtype, int64_t n, int64_t classes, int64_t row_stride,
                          const int64_t* labels, int64_t ignore_index, int32_t top_k, const int64_t* top_index,
                          const float* row_stats, const float* entropy, const float* d_log_prob,
                          const float* d_entropy, const float* d_top, void* d_logits, void* stream) {
    if (bad_args(logits, dtype, n, classes, row_stride, labels, top_k)) return PIN_ERR_ARG;
    if (n == 0) return PIN_OK;
    if (!row_stats || !entropy || !d_logits || (d_top && top_k > 0 && !top_index)) return PIN_ERR_ARG;
    const dim3 grid((unsigned)(n < (1 << 20) ? n : (1 << 20)));
    const hipStream_t st = as_stream(stream);
    const float* dt = top_k > 0 ? d_top : nullptr;
    if (dtype == PIN_TYPE_F32)
        hipLaunchKernelGGL(k_label_logprob_bwd<float>, grid, dim3(kBlock), 0, st, (const float*)logits, n, classes,
                           row_stride, labels, ignore_index, (int)top_k, top_index, row_stats, entropy, d_log_prob,
                           d_entropy, dt, (float*)d_logits);
    else if (dtype == PIN_TYPE_F16)
        hipLaunchKernelGGL(k_label_logprob_bwd<__half>, grid, dim3(kBlock), 0, st, (const __half*)logits, n, classes,
                           row_stride, labels, ignore_index, (int)top_k, top_index, row_stats, entropy, d_log_prob,
                           d_entropy, dt, (__half*)d_logits);
    else
        hipLaunchKernelGGL(k_label_logprob_bwd<__hip_bfloat16>, grid, dim3(kBlock), 0, st, (const __hip_bfloat16*)logits, n,
                           classes, row_stride, labels, ignore_index, (int)top_k, top_index, row_stats, entropy,
                           d_log_prob, d_entropy, dt, (__hip_bfloat16*)d_logits);
    return launch_status();
}

}  // extern "C"
