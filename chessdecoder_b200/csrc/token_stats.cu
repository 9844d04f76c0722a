// Statistics of given tokens under a row of logits: log-probability, entropy and
// the best alternatives, and the gradient of the first two (the log_softmax and
// gather of chessdecoder/rl/log_probs.py:58-101, with what a policy-gradient step
// with an entropy term and a scoring interface want beside it).
//
// With m = max x, s = sum e^(x - m), t = sum e^(x - m) (x - m):
//   L = m + log s,  lp = x_target - L,  entropy = log s - t / s
//   dx_j = g (1[j = target] - p_j) - h p_j (log p_j + entropy)
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "cdk.h"
#include "cdk_common.cuh"

using namespace cdk;

namespace {

constexpr int kMaxTop = 32;

template <bool BF16>
__device__ __forceinline__ float load_logit(const void* row, long long j) {
  return BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[j])
              : reinterpret_cast<const float*>(row)[j];
}

// Order of the alternatives as one integer: larger value first, then smaller
// index.  The float's bits are mapped to an unsigned integer that orders like the
// value (-0 as +0, NaN above +inf); the index enters inverted.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t j) {
  uint32_t u = __float_as_uint(x + 0.f);
  if (x != x) u = 0x7fffffffu;
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)~j;
}

// One block per row; three passes and one more per alternative.
template <bool BF16>
__global__ void __launch_bounds__(256)
    token_logprobs_kernel(const void* __restrict__ logits, long long ldl, long long ncls,
                          const int32_t* __restrict__ target, float* __restrict__ lp, float* __restrict__ entropy,
                          float* __restrict__ lse_out, int32_t* __restrict__ top_ids, float* __restrict__ top_lp,
                          int k) {
  const long long r = blockIdx.x;
  const char* row = reinterpret_cast<const char*>(logits) + r * ldl * (BF16 ? 2 : 4);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ float red[8], red2[8];
  __shared__ uint64_t redk[8];
  float m = -INFINITY;
  for (long long j = tid; j < ncls; j += 256) m = fmaxf(m, load_logit<BF16>(row, j));
  m = warp_max(m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
  m = red[0];
  for (int w = 1; w < 8; ++w) m = fmaxf(m, red[w]);
  __syncthreads();
  float s = 0.f, t = 0.f;
  bool nan = false;
  for (long long j = tid; j < ncls; j += 256) {
    const float x = load_logit<BF16>(row, j);
    nan |= x != x;
    if (x == -INFINITY) continue;
    const float z = x - m, e = expf(z);
    s += e;
    t += e * z;
  }
  if (nan) s = __uint_as_float(0x7fc00000u);
  s = warp_sum(s);
  t = warp_sum(t);
  if (lane == 0) {
    red[warp] = s;
    red2[warp] = t;
  }
  __syncthreads();
  s = t = 0.f;
  for (int w = 0; w < 8; ++w) {
    s += red[w];
    t += red2[w];
  }
  __syncthreads();
  const bool none = s == 0.f;  // every logit -inf
  const float lse = none ? -INFINITY : m + logf(s);
  if (tid == 0) {
    const int tg = target[r];
    lp[r] = (tg < 0 || tg >= ncls) ? 0.f : none ? -INFINITY : (load_logit<BF16>(row, tg) - m) - logf(s);
    if (entropy) entropy[r] = none ? 0.f : logf(s) - t / s;
    if (lse_out) lse_out[r] = lse;
  }
  uint64_t last = ~0ull;
  for (int i = 0; i < k; ++i) {
    uint64_t best = 0;
    for (long long j = tid; j < ncls; j += 256) {
      const uint64_t key = rank_key(load_logit<BF16>(row, j), (uint32_t)j);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    if (lane == 0) redk[warp] = best;
    __syncthreads();
    for (int w = 0; w < 8; ++w) best = redk[w] > best ? redk[w] : best;
    __syncthreads();
    last = best;
    if (tid == 0) {
      const uint32_t j = ~(uint32_t)best;
      top_ids[r * k + i] = (int32_t)j;
      top_lp[r * k + i] = none ? -INFINITY : (load_logit<BF16>(row, j) - m) - logf(s);
    }
  }
}

template <bool BF16>
__global__ void __launch_bounds__(256)
    token_logprobs_bwd_kernel(const void* logits, long long ldl, long long ncls,
                              const int32_t* __restrict__ target, const float* __restrict__ lse,
                              const float* __restrict__ entropy, const float* __restrict__ dlp,
                              const float* __restrict__ dentropy, void* dlogits, long long ldd) {
  const long long r = blockIdx.x;
  const char* row = reinterpret_cast<const char*>(logits) + r * ldl * (BF16 ? 2 : 4);
  const int tg = target[r];
  const float g = dlp && tg >= 0 && tg < ncls ? dlp[r] : 0.f;
  const float h = dentropy ? dentropy[r] : 0.f;
  const float L = lse[r], H = dentropy ? entropy[r] : 0.f;
  for (long long j = threadIdx.x; j < ncls; j += 256) {
    float d = 0.f;
    if (L != -INFINITY) {
      const float z = load_logit<BF16>(row, j) - L, p = expf(z);
      if (p != 0.f) d = -p * (g + h * (z + H));
      if (j == tg) d += g;
    }
    if (BF16) reinterpret_cast<__nv_bfloat16*>(dlogits)[r * ldd + j] = __float2bfloat16_rn(d);
    else reinterpret_cast<float*>(dlogits)[r * ldd + j] = d;
  }
}

inline int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : (int)e;
}

inline bool al(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

}  // namespace

extern "C" int cdk_token_logprobs(const void* logits, int dtype, int64_t ldl, int64_t rows, int64_t ncls,
                                  const int32_t* target, float* lp, float* entropy, float* lse, int32_t* top_ids,
                                  float* top_lp, int64_t k, void* stream) {
  if (rows == 0) return 0;
  if (!logits || !target || !lp || rows < 0 || rows > 0x7fffffff) return -1;
  if (dtype != 0 && dtype != 1) return -2;
  if (ncls <= 0 || ncls >= 0x7fffffe0 || ldl < ncls) return -3;
  if (!al(logits, dtype ? 2 : 4)) return -4;
  if (!top_ids != !top_lp) return -5;
  if (!top_ids) k = 0;
  if (k < 0 || k > kMaxTop || k > ncls) return -6;
  auto* st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype)
    token_logprobs_kernel<true><<<(unsigned)rows, 256, 0, st>>>(logits, ldl, ncls, target, lp, entropy, lse, top_ids,
                                                                top_lp, (int)k);
  else
    token_logprobs_kernel<false><<<(unsigned)rows, 256, 0, st>>>(logits, ldl, ncls, target, lp, entropy, lse, top_ids,
                                                                 top_lp, (int)k);
  return launched();
}

extern "C" int cdk_token_logprobs_bwd(const void* logits, int dtype, int64_t ldl, int64_t rows, int64_t ncls,
                                      const int32_t* target, const float* lse, const float* entropy, const float* dlp,
                                      const float* dentropy, void* dlogits, int64_t ldd, void* stream) {
  if (rows == 0) return 0;
  if (!logits || !target || !lse || !dlogits || rows < 0 || rows > 0x7fffffff) return -1;
  if (dtype != 0 && dtype != 1) return -2;
  if (ncls <= 0 || ncls >= 0x7fffffe0 || ldl < ncls || ldd < ncls) return -3;
  if (!al(logits, dtype ? 2 : 4) || !al(dlogits, dtype ? 2 : 4)) return -4;
  if (dentropy && !entropy) return -5;
  if (logits == dlogits && ldl != ldd) return -6;
  auto* st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype)
    token_logprobs_bwd_kernel<true><<<(unsigned)rows, 256, 0, st>>>(logits, ldl, ncls, target, lse, entropy, dlp,
                                                                    dentropy, dlogits, ldd);
  else
    token_logprobs_bwd_kernel<false><<<(unsigned)rows, 256, 0, st>>>(logits, ldl, ncls, target, lse, entropy, dlp,
                                                                     dentropy, dlogits, ldd);
  return launched();
}
