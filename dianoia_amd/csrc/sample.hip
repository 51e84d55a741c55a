// Sampling: rows of logits to tokens, from given random numbers. No
// counterpart in the reference, whose answer is the greedy one.
//
// With the row's largest logit M and temperature T, token j weighs
//   w_j = e^((l_j - M) / T).
// In the order of falling logits, of equal ones the lowest index first: the
// first top_k tokens; of these the shortest beginning that holds top_p of their
// weight; of these the tokens with w_j >= min_p. The answer is the first kept
// token, in the order of indices, up to which the weights' sum exceeds u times
// that of all.
//
// Weights are whole multiples of 2^-43, formed in 64 bits: whole numbers' sums
// do not depend on their order, whatever deals them to threads.

#include "common.h"
#include "dnx_kernels.h"

#include <math.h>

using namespace dnx;

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int64_t kMaxVocab = 1 << 20;   // the sum of a row's weights is below 2^64
constexpr int64_t kMaxRows = 1 << 16;

struct SampleArgs {
  const float *logits, *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* out;
  int64_t stride;
  int vocab;
};

// A row's request. T = 0: greedy.
struct Request {
  double inv_t, top_p, min_p;
  float u;
  int top_k;
  bool greedy;
};
DNX_DEV Request request(const SampleArgs& a, int row) {
  Request r;
  const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
  const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
  const float low = a.min_p != nullptr ? a.min_p[row] : 0.0f;
  const int k = a.top_k != nullptr ? a.top_k[row] : 0;
  const float u = a.u[row];
  r.greedy = !(t > 0.0f);
  r.inv_t = r.greedy ? 0.0 : 1.0 / (double)t;
  r.top_p = p < 1.0f ? fmax((double)p, 0.0) : 1.0;
  r.min_p = low > 0.0f ? fmin((double)low, 1.0) : 0.0;
  r.top_k = k > 0 && k < a.vocab ? k : 0;
  r.u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
  return r;
}

// Keys that rise as logits fall (+0 and -0 are one, NaN is -inf).
constexpr uint32_t kNothing = 0xff800000u;   // of -inf
DNX_DEV uint32_t falling_key(float v) {
  uint32_t b = __float_as_uint(v);
  if (v == 0.0f) b = 0;
  if (v != v) b = 0xff800000u;
  return (b & 0x80000000u) ? b : ~b & 0x7fffffffu;
}

// A token's weight in multiples of 2^-43.
DNX_DEV uint64_t weight(float l, float top, const Request& r) {
  if (!(l > -INFINITY)) return 0;
  if (l == top) return 1ull << 43;
  const double d = ((double)l - (double)top) * r.inv_t;
  if (!(d > -31.0)) return 0;
  const double w = exp(d);
  if (w < r.min_p) return 0;
  return (uint64_t)(w * 0x1p43 + 0.5);
}

DNX_DEV uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// The workgroup's sum, in every thread.
DNX_DEV uint64_t block_sum(uint64_t v, uint64_t* part) {
  v = wave_sum_u64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < kWaves; i++) v += part[i];
  return v;
}

// One workgroup a row: cuts are found by their order keys, eight bits at a
// time, each step counting and weighing the tokens that share the bits found.
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
  __shared__ uint64_t part[kWaves];
  __shared__ uint64_t mass[256];
  __shared__ uint32_t count[256];
  __shared__ uint64_t found[3];
  const int row = blockIdx.x, tid = threadIdx.x;
  const float* x = a.logits + row * a.stride;
  const Request r = request(a, row);

  uint64_t best = 0;
  for (int j = tid; j < a.vocab; j += kThreads) {
    const uint64_t k = (uint64_t)~falling_key(x[j]) << 32 | (uint32_t)~j;
    best = k > best ? k : best;
  }
  best = wave_max_u64(best);
  if ((tid & 63) == 0) part[tid >> 6] = best;
  __syncthreads();
  for (int i = 0; i < kWaves; i++) best = part[i] > best ? part[i] : best;
  const int first = (int)~(uint32_t)best;
  if (~(uint32_t)(best >> 32) == kNothing) {
    if (tid == 0) a.out[row] = -1;
    return;
  }
  if (r.greedy) {
    if (tid == 0) a.out[row] = first;
    return;
  }
  const float top = x[first];
  Request all = r;
  all.min_p = 0.0;

  // The last key of the first `tokens` tokens, or of the shortest beginning of
  // that weight; `within`: among keys up to that one. Its weight too.
  auto cut = [&](uint64_t within, uint32_t tokens, uint64_t target, uint64_t& weighs) {
    uint64_t prefix = 0, before = 0;
    uint32_t n_before = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kThreads) mass[i] = 0, count[i] = 0;
      __syncthreads();
      for (int j = tid; j < a.vocab; j += kThreads) {
        const uint64_t k = (uint64_t)falling_key(x[j]) << 32 | (uint32_t)j;
        if (k > within || (shift < 56 && (k ^ prefix) >> (shift + 8) != 0)) continue;
        atomicAdd(&count[k >> shift & 255], 1u);
        atomicAdd((unsigned long long*)&mass[k >> shift & 255],
                  (unsigned long long)weight(x[j], top, all));
      }
      __syncthreads();
      if (tid == 0) {
        int b = 0;
        uint64_t m = before;
        uint32_t n = n_before;
        int last = 0;
        for (; b < 256; b++) {
          if (count[b] == 0) continue;
          last = b;
          if (tokens > 0 ? n + count[b] >= tokens : m + mass[b] >= target) break;
          m += mass[b];
          n += count[b];
        }
        if (b == 256) {   // all of them
          b = last;
          m -= mass[b];
          n -= count[b];
        }
        found[0] = prefix | (uint64_t)b << shift;
        found[1] = m;
        found[2] = n;
        mass[0] = mass[b];
      }
      __syncthreads();
      prefix = found[0];
      before = found[1];
      n_before = (uint32_t)found[2];
      weighs = before + mass[0];
      __syncthreads();
    }
    return prefix;
  };

  uint64_t within = ~0ull, total = 0;
  if (r.top_k > 0) within = cut(within, (uint32_t)r.top_k, 0, total);
  if (r.top_p < 1.0) {
    if (r.top_k == 0) {
      for (int j = tid; j < a.vocab; j += kThreads) total += weight(x[j], top, all);
      total = block_sum(total, part);
    }
    const double target = ceil(r.top_p * (double)total);
    within = cut(within, 0, (uint64_t)target, total);
  }

  auto kept = [&](int j) -> uint64_t {
    if (j >= a.vocab || ((uint64_t)falling_key(x[j]) << 32 | (uint32_t)j) > within) return 0;
    return weight(x[j], top, r);
  };
  total = 0;
  for (int j = tid; j < a.vocab; j += kThreads) total += kept(j);
  total = block_sum(total, part);
  uint64_t target = (uint64_t)((double)r.u * (double)total);
  target = target < total ? target : total - 1;
  uint64_t before = 0;
  for (int j0 = 0; j0 < a.vocab; j0 += kThreads) {
    const uint64_t w = kept(j0 + tid);
    uint64_t upto = w;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t y = __shfl_up(upto, o);
      if ((tid & 63) >= o) upto += y;
    }
    __syncthreads();
    if ((tid & 63) == 63) part[tid >> 6] = upto;
    __syncthreads();
    uint64_t at = before;
    for (int i = 0; i < kWaves; i++) {
      if (i < tid >> 6) at += part[i];
      before += part[i];
    }
    upto += at;
    if (w > 0 && upto > target && upto - w <= target) a.out[row] = j0 + tid;
    if (before > target) return;
  }
}

}  // namespace

extern "C" {

int64_t dnx_sample_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 0 || rows > kMaxRows || vocab < 1 || vocab > kMaxVocab) return -1;
  return 0;
}

int dnx_sample(const float* logits, int64_t stride, const float* u, const float* temperature,
               const int32_t* top_k, const float* top_p, const float* min_p, int32_t* out,
               int64_t rows, int64_t vocab, void* workspace, int64_t workspace_bytes,
               dnx_stream_t stream) {
  const int64_t need = dnx_sample_workspace_bytes(rows, vocab);
  if (need < 0) return DNX_EINVAL;
  if (rows == 0) return DNX_OK;
  const uintptr_t all = (uintptr_t)logits | (uintptr_t)u | (uintptr_t)temperature |
                        (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)out;
  if (logits == nullptr || u == nullptr || out == nullptr || (all & 3) != 0 || stride < vocab ||
      stride > (int64_t)1 << 40 || workspace_bytes < need ||
      (need > 0 && (workspace == nullptr || ((uintptr_t)workspace & 15) != 0))) {
    return DNX_EINVAL;
  }
  const SampleArgs a{logits, u, temperature, top_p, min_p, top_k, out, stride, (int)vocab};
  hipLaunchKernelGGL(sample_kernel, dim3((unsigned)rows), dim3(kThreads), 0, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? DNX_OK : DNX_ELAUNCH;
}

}  // extern "C"
