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

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int64_t kMaxVocab = 1 << 20;   // the sum of a row's weights is below 2^64
constexpr int64_t kMaxRows = 1 << 16;
constexpr int kBins = 1024, kBinsPerUnit = 32;   // of l / T: 32 in all
constexpr int kMaxChunks = 128;
constexpr int kChunkFound = 1024;        // tokens of the bins in question, of a chunk
constexpr int kListed = 8192;            // of a row, that are held in LDS
constexpr int kFound = 2048;             // that are sorted at once
constexpr int kParts = 2048;             // of a span of order keys that holds more

struct SampleArgs {
  const float *logits, *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* out;
  int64_t stride;
  int vocab, chunks, wide;   // wide: rows may be read 16 bytes at a time
  // Of each row and chunk:
  uint64_t* hist;      // [kBins]: counts (the upper 16 bits) and weights
  uint64_t* sums;      // [3]: of weights
  uint64_t* found;     // [kChunkFound] order keys
  float* tops;         // the largest logit
  uint32_t* founds;    // how many tokens were found
  int32_t* cuts;       // [4] of each row: the bins in question
};

// A row's request. Greedy: of a steep T, the first token.
struct Request {
  double rate, top_p, min_p;   // rate: log2(e) / T
  float u, inv;                // inv: 1 / T of the bins, finite
  int top_k;
  bool cut;            // by rank or weight
};
DNX_DEV Request request(const SampleArgs& a, int row) {
  Request r;
  const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
  const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
  const float low = a.min_p != nullptr ? a.min_p[row] : 0.0f;
  const int k = a.top_k != nullptr ? a.top_k[row] : 0;
  const float u = a.u[row];
  const bool greedy = !(t > 0.0f);
  const double inv = greedy ? 0x1p40 : 1.0 / (double)t;
  r.rate = inv * 1.4426950408889634;
  r.inv = (float)fmax(fmin(inv, 1e37), 1e-41);   // an infinity times it is one
  r.top_p = !greedy && p < 1.0f ? fmax((double)p, 0.0) : 1.0;
  r.min_p = !greedy && low > 0.0f ? fmin((double)low, 1.0) : 0.0;
  r.top_k = greedy ? 1 : k > 0 && k < a.vocab ? k : 0;
  r.u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
  r.cut = r.top_k > 0 || r.top_p < 1.0;
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
DNX_DEV float of_key(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k : ~k & 0x7fffffffu);
}
DNX_DEV uint64_t order_key(float v, int j) { return (uint64_t)falling_key(v) << 32 | (uint32_t)j; }

// A token's weight in multiples of 2^-43, and whether that is enough. 2^x by the
// Taylor series about the nearest whole number: |z| <= ln 2 / 2, whose 12th term
// is below 2^-47. Adding 3 2^51 rounds to a whole number and leaves it in the lower
// bits, adding 2^52 rounds the result: conversions between 64 bits and whole
// numbers run at a quarter of the rate.
DNX_DEV uint64_t weight(float l, float top, double rate) {
  const double x = ((double)l - (double)top) * rate, m = x + 0x1.8p52;
  const double z = (x - (m - 0x1.8p52)) * 0.6931471805599453;
  double p = 1.0 / 39916800.0;
  p = fma(p, z, 1.0 / 3628800.0);
  p = fma(p, z, 1.0 / 362880.0);
  p = fma(p, z, 1.0 / 40320.0);
  p = fma(p, z, 1.0 / 5040.0);
  p = fma(p, z, 1.0 / 720.0);
  p = fma(p, z, 1.0 / 120.0);
  p = fma(p, z, 1.0 / 24.0);
  p = fma(p, z, 1.0 / 6.0);
  p = fma(p, z, 0.5);
  p = fma(p, z, 1.0);
  p = fma(p, z, 1.0);
  const bool some = x > -45.0 && l > -INFINITY;      // no NaN, no exponent out of range
  const int n = some ? (int)(uint32_t)__builtin_bit_cast(uint64_t, m) : 0;
  const double w = __builtin_bit_cast(
      double, __builtin_bit_cast(uint64_t, p) + ((uint64_t)(uint32_t)(n + 43) << 52));
  const uint64_t whole = __builtin_bit_cast(uint64_t, w + 0x1p52) & ((1ull << 52) - 1);
  return l == top ? (l > -INFINITY ? 1ull << 43 : 0) : some ? whole : 0;
}
DNX_DEV uint64_t at_least(uint64_t w, const Request& r) {
  return (double)w >= r.min_p * 0x1p43 ? w : 0;
}

// Bins of l / T, an eighth wide: whole numbers that do not fall as logits rise,
// the same for every chunk of a row. Far-off values are as the last ones (no
// difference of two is then an infinity).
DNX_DEV float scaled(float l, float inv) {
  return __builtin_amdgcn_fmed3f(l * inv, -1e37f, 1e37f) * (float)kBinsPerUnit;
}
// The bin below the one that the row's (or the chunk's) largest logit lies in;
// kBins and more: no weight.
DNX_DEV int bin_of(float l, float top, float place, float inv) {
  if (l == top) return 0;
  const float d = place - floorf(scaled(l, inv));    // NaN: of a logit NaN
  return l > -INFINITY && d < (float)kBins ? (int)fmaxf(d, 0.0f) : kBins;
}

DNX_DEV uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
template <typename V>
DNX_DEV V wave_scan(V v) {   // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V y = __shfl_up(v, o);
    if (lane >= o) v += y;
  }
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

// The sum of the threads' values before this one's; the workgroup's in `all`.
DNX_DEV uint64_t block_before(uint64_t v, uint64_t* part, uint64_t& all) {
  const uint64_t upto = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = upto;
  __syncthreads();
  uint64_t before = upto - v;
  all = 0;
  for (int i = 0; i < kWaves; i++) {
    if (i < (int)threadIdx.x >> 6) before += part[i];
    all += part[i];
  }
  return before;
}

// The row's largest logit, of its chunks'.
DNX_DEV float row_top(const SampleArgs& a, int row) {
  const int lane = threadIdx.x & 63;
  float top = -INFINITY;
  for (int c = lane; c < a.chunks; c += 64) top = fmaxf(top, a.tops[(int64_t)row * a.chunks + c]);
  return wave_max_dpp(top);
}

// A chunk's logits: a thread has four in a row of each 4 kThreads.
template <int E>
DNX_DEV int index_of(int chunk, int e) {
  return chunk * (kThreads * E) + e / 4 * (4 * kThreads) + 4 * threadIdx.x + e % 4;
}
template <int E>
DNX_DEV void load_chunk(const SampleArgs& a, int row, int chunk, float* l) {
  const float* x = a.logits + row * a.stride;
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const int j = index_of<E>(chunk, e);
    if (a.wide && j + 3 < a.vocab) {
      const float4 v = *(const float4*)(x + j);
      l[e] = v.x, l[e + 1] = v.y, l[e + 2] = v.z, l[e + 3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) l[e + i] = j + i < a.vocab ? x[j + i] : -INFINITY;
    }
  }
}

// ---- Step 1, a workgroup a chunk of a row: its largest logit, and (for a row
// that is cut) how many tokens and how much weight each bin holds, the weights
// relative to the bin's lower end.
template <int E>
DNX_DEV void count_chunk(const SampleArgs& a, int row, int chunk) {
  __shared__ unsigned long long hist[kBins];
  __shared__ float part[kWaves];
  const int tid = threadIdx.x;
  float l[E];
  load_chunk<E>(a, row, chunk, l);
  const Request r = request(a, row);
  for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
  float top = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; e++) top = fmaxf(top, l[e]);
  top = wave_max_dpp(top);
  if ((tid & 63) == 0) part[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; i++) top = fmaxf(top, part[i]);
  const int64_t at = (int64_t)row * a.chunks + chunk;
  if (tid == 0) a.tops[at] = top;
  if (!r.cut) return;
  const float place = floorf(scaled(top, r.inv));
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int b = bin_of(l[e], top, place, r.inv);
    if (b < kBins) {
      const float y = scaled(l[e], r.inv);
      const float w = __builtin_amdgcn_exp2f((y - floorf(y)) * (1.44269504088896341f / kBinsPerUnit));
      atomicAdd(&hist[b], (1ull << 48) | (unsigned long long)(uint32_t)(w * 0x1p26f + 0.5f));
    }
  }
  __syncthreads();
  for (int i = tid; i < kBins; i += kThreads) a.hist[at * kBins + i] = hist[i];
}

// a.cuts: the cut by weight lies in bins lo .. hi, that by rank in bin k, before
// which there are so many tokens; lo <= hi <= k, which is kBins without one. Without
// either lo is kBins too.

// Step 2, a workgroup a row: its chunks' bins added, their running sums, and where
// these reach the cuts. The weights of bins are off by 2^-22 or, for large l / T,
// by the rounding of that; where a cut by weight may lie takes this in.
DNX_DEV void find_cuts(const SampleArgs& a, int row) {
  constexpr int P = kBins / kThreads, U = 8;       // bins a thread, chunks at once
  __shared__ uint64_t mass[kBins];
  __shared__ uint32_t count[kBins];
  __shared__ uint64_t part[kWaves];
  __shared__ int32_t shift[kMaxChunks], found[3];
  const int tid = threadIdx.x;
  const int64_t base = (int64_t)row * a.chunks;
  const float mine = tid < a.chunks ? a.tops[base + tid] : -INFINITY;
  const Request r = request(a, row);
  const float top = row_top(a, row);
  int lo = kBins, hi = kBins, bin_k = kBins, before_k = 0;
  if (r.cut && top > -INFINITY) {
    const float place = floorf(scaled(top, r.inv));
    if (tid < kMaxChunks) shift[tid] = bin_of(mine, top, place, r.inv);   // a chunk's first bin
    if (tid < 3) found[tid] = kBins;
    __syncthreads();
    uint64_t w[P] = {};
    uint32_t n[P] = {};
    for (int c0 = 0; c0 < a.chunks; c0 += U) {
      uint64_t h[U][P];
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int k = 0; k < P; k++) {
          const int i = c0 + u < a.chunks ? P * tid + k - shift[c0 + u] : -1;
          h[u][k] = a.hist[(base + (i < 0 ? 0 : c0 + u)) * kBins + (i < 0 ? 0 : i)];
          h[u][k] = i < 0 ? 0 : h[u][k];
        }
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int k = 0; k < P; k++) {
          w[k] += h[u][k] & ((1ull << 48) - 1);
          n[k] += (uint32_t)(h[u][k] >> 48);
        }
    }
    // Below 2^(26 + 20 + 1): in whole multiples, whose running sums rise.
    uint64_t ws = 0, ns = 0, all, tokens;
#pragma unroll
    for (int k = 0; k < P; k++) {
      w[k] = (uint64_t)((double)w[k] * exp((double)(P * tid + k) * (-1.0 / kBinsPerUnit)) * 0x1p15);
      ws += w[k];
      ns += n[k];
    }
    uint64_t wb = block_before(ws, part, all), nb = block_before(ns, part, tokens);
#pragma unroll
    for (int k = 0; k < P; k++) {
      mass[P * tid + k] = wb += w[k];
      count[P * tid + k] = (uint32_t)(nb += n[k]);
    }
    __syncthreads();
    if (r.top_k > 0) {
#pragma unroll
      for (int k = P - 1; k >= 0; k--) {
        const int b = P * tid + k;
        if (count[b] >= (uint32_t)r.top_k && (b == 0 || count[b - 1] < (uint32_t)r.top_k)) found[2] = b;
      }
      __syncthreads();
      bin_k = found[2];
      if (bin_k > 0 && bin_k < kBins) before_k = (int)count[bin_k - 1];
      lo = hi = bin_k;
    }
    if (r.top_p < 1.0) {
      const double slack = 0x1p-17 + fabs((double)place) * 0x1p-27;
      const double least = (double)(bin_k == kBins ? all : bin_k == 0 ? 0 : mass[bin_k - 1]);
      const double most = (double)(bin_k == kBins ? all : mass[bin_k]);
      const double from = r.top_p * least * (1.0 - slack), to = r.top_p * most * (1.0 + slack);
#pragma unroll
      for (int k = 0; k < P; k++) {
        const int b = P * tid + k;
        const double upto = (double)mass[b], before = b == 0 ? -1.0 : (double)mass[b - 1];
        if (upto >= from && before < from) found[0] = b;
        if (upto >= to && before < to) found[1] = b;
      }
      __syncthreads();
      const int last = min(bin_k, kBins - 1);
      lo = min(found[0], last);
      hi = min(found[1], last);
    }
  }
  if (tid == 0) {
    int32_t* to = a.cuts + 4 * (int64_t)row;
    to[0] = lo, to[1] = hi, to[2] = bin_k, to[3] = before_k;
  }
}

// Step 3, a workgroup a chunk: the weights of the tokens before the bins in
// question (before lo; before k; before lo and of min_p), and the keys of the
// tokens in them.
template <int E>
DNX_DEV void weigh_chunk(const SampleArgs& a, int row, int chunk) {
  __shared__ uint64_t part[kWaves];
  __shared__ uint32_t found;
  const int tid = threadIdx.x;
  float l[E];
  load_chunk<E>(a, row, chunk, l);
  const int32_t* cut = a.cuts + 4 * (int64_t)row;
  const int lo = cut[0], hi = cut[1], bin_k = cut[2];
  const Request r = request(a, row);
  const float top = row_top(a, row);
  const int64_t at = (int64_t)row * a.chunks + chunk;
  if (tid == 0) found = 0;
  __syncthreads();
  const float place = floorf(scaled(top, r.inv));
  uint64_t before_lo = 0, before_k = 0, kept = 0;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int b = r.cut ? bin_of(l[e], top, place, r.inv) : l[e] > -INFINITY ? 0 : kBins;
    if (b < bin_k) {
      const uint64_t w = weight(l[e], top, r.rate);
      before_k += w;
      if (b < lo) {
        before_lo += w;
        kept += at_least(w, r);
      }
    }
    if (b < kBins && ((b >= lo && b <= hi) || b == bin_k)) {
      const uint32_t i = atomicAdd(&found, 1u);
      if (i < kChunkFound) a.found[at * kChunkFound + i] = order_key(l[e], index_of<E>(chunk, e));
    }
  }
  kept = block_sum(kept, part);
  if (r.cut) {
    before_lo = block_sum(before_lo, part);
    before_k = block_sum(before_k, part);
  }
  if (tid == 0) {
    a.sums[3 * at] = before_lo;
    a.sums[3 * at + 1] = before_k;
    a.sums[3 * at + 2] = kept;
    a.founds[at] = found;
  }
}

// Keys in rising order: N a power of two, those past n above all.
DNX_DEV void sort_keys(uint64_t* keys, int n) {
  const int tid = threadIdx.x;
  if (n <= 128) {           // each to its rank
    __syncthreads();
    const uint64_t mine = tid < n ? keys[tid] : 0;
    int rank = 0;
    if (tid < n)
      for (int i = 0; i < n; i++) rank += keys[i] < mine;
    __syncthreads();
    if (tid < n) keys[rank] = mine;
    __syncthreads();
    return;
  }
  int size = 256;
  while (size < n) size *= 2;
  for (int i = n + tid; i < size; i += kThreads) keys[i] = ~0ull;
  for (int k = 2; k <= size; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      __syncthreads();
      for (int t = tid; t < size / 2; t += kThreads) {
        const int i = 2 * t - (t & (j - 1)), p = i + j;
        const uint64_t x = keys[i], y = keys[p];
        if ((x > y) == ((i & k) == 0)) keys[i] = y, keys[p] = x;
      }
    }
  __syncthreads();
}

// What step 4 keeps in LDS: the order keys of the bins in question, those of them
// that are sorted, and the running sums of their weights, or the counts and weights
// of a span's parts.
static_assert(kFound <= kParts, "upto serves both");
struct PickShared {
  uint64_t list[kListed], keys[kFound], upto[kParts];
  uint64_t part[kWaves], ends[2];
  unsigned long long sums[kMaxChunks];
  int begin[kMaxChunks + 1], at[2], n;
};

// n keys of sh.keys in order, and the running sums of their weights.
DNX_DEV void order_keys(PickShared& sh, int n, float top, const Request& r) {
  const int tid = threadIdx.x;
  sort_keys(sh.keys, n);
  const int per = (n + kThreads - 1) / kThreads;    // in a row a thread
  uint64_t sum = 0, all;
  for (int i = tid * per; i < min(n, (tid + 1) * per); i++) {
    sh.upto[i] = weight(of_key((uint32_t)(sh.keys[i] >> 32)), top, r.rate);
    sum += sh.upto[i];
  }
  uint64_t before = block_before(sum, sh.part, all);
  for (int i = tid * per; i < min(n, (tid + 1) * per); i++) sh.upto[i] = before += sh.upto[i];
  __syncthreads();
}

// Of the tokens that `each` gives in bins lo .. hi, the order key of the one of
// that rank (from 1), or with rank 0 of the first up to which the weights,
// `before` among them, reach the target. upto: the weights up to it, `before`
// among them. Where they are too many to be sorted, the span of their keys is
// cut into parts until the one in question holds few enough: equal logits have
// different keys. false: the weights do not reach the target here.
template <typename Each>
DNX_DEV bool find_key(PickShared& sh, Each each, float top, const Request& r, int lo, int hi,
                      uint64_t rank, uint64_t target, uint64_t before, uint64_t& key,
                      uint64_t& upto) {
  const int tid = threadIdx.x;
  const float place = floorf(scaled(top, r.inv));
  uint64_t first = ~0ull, last = 0, n = 0;
  each([&](uint64_t k) {
    const int b = bin_of(of_key((uint32_t)(k >> 32)), top, place, r.inv);
    if (b < lo || b > hi) return;
    first = k < first ? k : first;
    last = k > last ? k : last;
    n++;
  });
  n = block_sum(n, sh.part);
  first = ~wave_max_u64(~first);
  last = wave_max_u64(last);
  __syncthreads();
  if (tid < 2) sh.ends[tid] = tid == 0 ? ~0ull : 0;
  __syncthreads();
  if ((tid & 63) == 0) {
    atomicMin((unsigned long long*)&sh.ends[0], (unsigned long long)first);
    atomicMax((unsigned long long*)&sh.ends[1], (unsigned long long)last);
  }
  __syncthreads();
  first = sh.ends[0];
  last = sh.ends[1];
  if (n == 0) return false;
  uint32_t* count = (uint32_t*)sh.keys;
  uint64_t rank_before = 0;
  while (n > kFound) {
    const int shift = max(0, 64 - 11 - __builtin_clzll(last - first));
    __syncthreads();
    for (int i = tid; i < kParts; i += kThreads) count[i] = 0, sh.upto[i] = 0;
    __syncthreads();
    each([&](uint64_t k) {
      if (k < first || k > last) return;
      const int i = (int)((k - first) >> shift);
      atomicAdd(&count[i], 1u);
      atomicAdd((unsigned long long*)&sh.upto[i],
                (unsigned long long)weight(of_key((uint32_t)(k >> 32)), top, r.rate));
    });
    __syncthreads();
    constexpr int P = kParts / kThreads;
    uint64_t c[P], w[P], cs = 0, ws = 0, all;
#pragma unroll
    for (int i = 0; i < P; i++) {
      cs += c[i] = count[P * tid + i];
      ws += w[i] = sh.upto[P * tid + i];
    }
    uint64_t cb = block_before(cs, sh.part, all) + rank_before;
    uint64_t wb = block_before(ws, sh.part, all) + before;
    if (tid == 0) sh.n = -1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < P; i++) {
      const bool here = rank > 0 ? cb < rank && cb + c[i] >= rank : wb < target && wb + w[i] >= target;
      if (here) {
        sh.n = P * tid + i;
        sh.ends[0] = cb;
        sh.ends[1] = wb;
        sh.part[0] = c[i];
      }
      cb += c[i];
      wb += w[i];
    }
    __syncthreads();
    if (sh.n < 0) return false;
    rank_before = sh.ends[0];
    before = sh.ends[1];
    n = sh.part[0];
    first += (uint64_t)sh.n << shift;
    const uint64_t width = (1ull << shift) - 1;
    last = last - first > width ? first + width : last;
  }
  __syncthreads();
  if (tid == 0) sh.n = 0;
  __syncthreads();
  each([&](uint64_t k) {
    const int b = bin_of(of_key((uint32_t)(k >> 32)), top, place, r.inv);
    if (k < first || k > last || b < lo || b > hi) return;
    sh.keys[atomicAdd(&sh.n, 1)] = k;
  });
  __syncthreads();
  const int found = sh.n;
  order_keys(sh, found, top, r);
  if (tid == 0) sh.at[0] = rank > 0 ? (int)(rank - rank_before) - 1 : kFound;
  __syncthreads();
  if (rank == 0)
    for (int i = tid; i < found; i += kThreads)
      if (before + sh.upto[i] >= target && (i == 0 || before + sh.upto[i - 1] < target)) sh.at[0] = i;
  __syncthreads();
  const int i = sh.at[0];
  if (i >= found || (rank == 0 && before >= target)) return false;
  key = sh.keys[i];
  upto = before + sh.upto[i];
  __syncthreads();
  return true;
}

// Step 4, a workgroup a row: the tokens of the bins in question in order, where
// among them the cuts lie, the kept weights of each chunk, and the token in its
// chunk.
template <int E>
DNX_DEV void pick(const SampleArgs& a, int row) {
  constexpr int kChunk = kThreads * E;
  __shared__ PickShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* x = a.logits + row * a.stride;
  const int64_t base = (int64_t)row * a.chunks;
  const float top = row_top(a, row);
  if (!(top > -INFINITY)) {
    if (tid == 0) a.out[row] = -1;
    return;
  }
  const Request r = request(a, row);
  uint64_t before_lo = 0, before_k = 0;
  for (int c = tid; c < kMaxChunks; c += kThreads) {
    sh.sums[c] = c < a.chunks ? a.sums[3 * (base + c) + 2] : 0;
    if (r.cut && c < a.chunks) {
      before_lo += a.sums[3 * (base + c)];
      before_k += a.sums[3 * (base + c) + 1];
    }
  }
  uint64_t within = ~0ull;
  bool whole = false;       // the chunks' sums have to be formed again
  const int32_t* cut = a.cuts + 4 * (int64_t)row;
  const int lo = cut[0], hi = cut[1], bin_k = cut[2], rank_k = r.top_k - cut[3];
  const float place = floorf(scaled(top, r.inv));
  if (lo < kBins) {
    before_lo = block_sum(before_lo, sh.part);
    before_k = block_sum(before_k, sh.part);
    if (wave == 0) {        // where each chunk's tokens begin
      int n[kMaxChunks / 64], sum = 0;
      bool over = false;
#pragma unroll
      for (int i = 0; i < kMaxChunks / 64; i++) {
        const int c = kMaxChunks / 64 * lane + i;
        n[i] = c < a.chunks ? (int)a.founds[base + c] : 0;
        over |= n[i] > kChunkFound;
        sum += n[i];
      }
      int b = wave_scan(sum) - sum;
#pragma unroll
      for (int i = 0; i < kMaxChunks / 64; i++) {
        sh.begin[kMaxChunks / 64 * lane + i] = b;
        b += n[i];
      }
      over = __any(over);
      if (lane == 63) sh.begin[kMaxChunks] = over ? -1 : b;
    }
    if (tid < 2) sh.at[tid] = kFound;
    __syncthreads();
    const int n = sh.begin[kMaxChunks];     // -1: more than a chunk's list holds
    uint64_t total = before_k;
    bool done = n > 0 && n <= kFound;
    if (n > 0 && n <= kListed) {
      uint64_t* to = done ? sh.keys : sh.list;
      for (int c = wave; c < a.chunks; c += kWaves) {
        const int b = sh.begin[c], m = sh.begin[c + 1] - b;
        const uint64_t* from = a.found + (base + c) * kChunkFound;
        for (int i0 = 0; i0 < m; i0 += 256) {
          uint64_t k[4];
#pragma unroll
          for (int u = 0; u < 4; u++) k[u] = from[min(i0 + 64 * u + lane, m - 1)];
#pragma unroll
          for (int u = 0; u < 4; u++)
            if (i0 + 64 * u + lane < m) to[b + i0 + 64 * u + lane] = k[u];
        }
      }
      __syncthreads();
    }
    if (done) {
      order_keys(sh, n, top, r);
      // The first token of bin k, and the last one by rank.
      auto bin_at = [&](int i) {
        return bin_of(of_key((uint32_t)(sh.keys[i] >> 32)), top, place, r.inv);
      };
      int last = n - 1, end = n;          // end: of the tokens up to bin hi
      if (bin_k < kBins) {
        for (int i = tid; i < n; i += kThreads)
          if (bin_at(i) == bin_k && (i == 0 || bin_at(i - 1) < bin_k)) sh.at[0] = i;
        __syncthreads();
        const int first = sh.at[0];
        last = min(first + rank_k - 1, n - 1);
        total += sh.upto[last] - (first > 0 ? sh.upto[first - 1] : 0);
        if (hi < bin_k) end = first;
      }
      if (r.top_p < 1.0) {
        const uint64_t target = max((uint64_t)ceil(r.top_p * (double)total), (uint64_t)1);
        for (int i = tid; i < end; i += kThreads)
          if (before_lo + sh.upto[i] >= target && (i == 0 || before_lo + sh.upto[i - 1] < target))
            sh.at[1] = i;
        __syncthreads();
        done = before_lo < target && sh.at[1] < kFound;    // or the bins' weights misled
        last = min(last, sh.at[1]);
        total = before_k;
      }
      if (done) {
        within = sh.keys[last];
        for (int i = tid; i <= last; i += kThreads) {
          const uint64_t w = at_least(sh.upto[i] - (i > 0 ? sh.upto[i - 1] : 0), r);
          if (w > 0) atomicAdd(&sh.sums[(uint32_t)sh.keys[i] / kChunk], (unsigned long long)w);
        }
      }
    }
    if (!done) {
      whole = n <= 0 || n > kListed;
      const auto any = [&](auto f) {
        for (int j0 = tid; j0 < a.vocab; j0 += 8 * kThreads) {
          float l[8];
#pragma unroll
          for (int u = 0; u < 8; u++) l[u] = x[min(j0 + u * kThreads, a.vocab - 1)];
#pragma unroll
          for (int u = 0; u < 8; u++)
            if (j0 + u * kThreads < a.vocab && l[u] > -INFINITY) f(order_key(l[u], j0 + u * kThreads));
        }
      };
      const auto listed = [&](auto f) {
        if (whole) return any(f);
        for (int i = tid; i < n; i += kThreads) f(sh.list[i]);
      };
      uint64_t key = ~0ull, upto;
      if (bin_k < kBins &&
          find_key(sh, listed, top, r, bin_k, bin_k, rank_k, 0, before_k, key, upto)) {
        within = key;
        total = upto;
      }
      if (r.top_p < 1.0) {
        const uint64_t target = max((uint64_t)ceil(r.top_p * (double)total), (uint64_t)1);
        if (!find_key(sh, listed, top, r, lo, hi, 0, target, before_lo, key, upto)) {
          whole = true;           // the bins' weights misled
          find_key(sh, any, top, r, 0, kBins - 1, 0, target, 0, key, upto);
        }
        within = key < within ? key : within;
      }
      for (int c = wave; c < a.chunks && !whole; c += kWaves) {
        uint64_t s = 0;
        for (int i = sh.begin[c] + lane; i < sh.begin[c + 1]; i += 64) {
          const uint64_t k = sh.list[i];
          if (k <= within) s += at_least(weight(of_key((uint32_t)(k >> 32)), top, r.rate), r);
        }
        s = wave_sum_u64(s);
        if (lane == 0) sh.sums[c] += s;
      }
    }
  }
  auto kept = [&](int j) -> uint64_t {
    if (j >= a.vocab) return 0;
    const float l = x[j];
    return order_key(l, j) <= within ? at_least(weight(l, top, r.rate), r) : 0;
  };
  __syncthreads();
  if (whole) {
    for (int c = wave; c < a.chunks; c += kWaves) {
      uint64_t s = 0;
#pragma unroll 4
      for (int e = 0; e < kChunk / 64; e++) s += kept(c * kChunk + e * 64 + lane);
      s = wave_sum_u64(s);
      if (lane == 0) sh.sums[c] = s;
    }
    __syncthreads();
  }
  // The chunk, by every wave alike.
  uint64_t s[kMaxChunks / 64], mine = 0;
#pragma unroll
  for (int i = 0; i < kMaxChunks / 64; i++) mine += s[i] = sh.sums[kMaxChunks / 64 * lane + i];
  const uint64_t all = wave_scan(mine), total = __shfl(all, 63);
  uint64_t target = (uint64_t)((double)r.u * (double)total), before = all - mine;
  target = target < total ? target : total - 1;
  int chunk = 0;
  uint64_t chunk_before = 0;
  bool here = false;
#pragma unroll
  for (int i = 0; i < kMaxChunks / 64; i++) {
    if (before <= target && target < before + s[i]) {
      here = true;
      chunk = kMaxChunks / 64 * lane + i;
      chunk_before = before;
    }
    before += s[i];
  }
  const int from = __builtin_ctzll(__ballot(here));
  chunk = __shfl(chunk, from);
  before = __shfl(chunk_before, from);
  // Its tokens in order: a wave 64 E of them.
  const int j0 = chunk * kChunk + wave * (64 * E) + lane;
  uint64_t w[E], of_wave = 0;
#pragma unroll
  for (int e = 0; e < E; e++) of_wave += w[e] = kept(j0 + 64 * e);
  of_wave = wave_sum_u64(of_wave);
  if (lane == 0) sh.part[wave] = of_wave;
  __syncthreads();
  for (int i = 0; i < wave; i++) before += sh.part[i];
  if (target < before || target >= before + of_wave) return;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const uint64_t to = before + wave_scan(w[e]);
    if (to > target && to - w[e] <= target) a.out[row] = j0 + 64 * e;
    before = __shfl(to, 63);
  }
}

template <int E>
__global__ void __launch_bounds__(kThreads) count_kernel(SampleArgs a) {
  count_chunk<E>(a, blockIdx.x, blockIdx.y);
}
__global__ void __launch_bounds__(kThreads) cuts_kernel(SampleArgs a) {
  find_cuts(a, blockIdx.x);
}
template <int E>
__global__ void __launch_bounds__(kThreads) weigh_kernel(SampleArgs a) {
  weigh_chunk<E>(a, blockIdx.x, blockIdx.y);
}
template <int E>
__global__ void __launch_bounds__(kThreads) pick_kernel(SampleArgs a) {
  pick<E>(a, blockIdx.x);
}
// A row of one chunk: the steps by one workgroup.
template <int E>
__global__ void __launch_bounds__(kThreads) row_kernel(SampleArgs a) {
  count_chunk<E>(a, blockIdx.x, 0);
  __syncthreads();
  find_cuts(a, blockIdx.x);
  __syncthreads();
  weigh_chunk<E>(a, blockIdx.x, 0);
  __syncthreads();
  pick<E>(a, blockIdx.x);
}

// Tokens of a thread in a chunk: 16, or 4 where that leaves CUs without a
// workgroup.
int per_thread(int64_t rows, int64_t vocab) {
  const int64_t chunks = (vocab + 16 * kThreads - 1) / (16 * kThreads);
  return chunks > 1 && rows * chunks < 256 && vocab <= kMaxChunks * 4 * kThreads ? 4 : 16;
}
int64_t chunks_of(int64_t rows, int64_t vocab) {
  const int64_t chunk = kThreads * per_thread(rows, vocab);
  return (vocab + chunk - 1) / chunk;
}
constexpr int64_t kChunkBytes = 8 * (kBins + 3 + kChunkFound) + 8;

}  // namespace

extern "C" {

int64_t dnx_sample_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 0 || rows > kMaxRows || vocab < 1 || vocab > kMaxVocab) return -1;
  return rows * (chunks_of(rows, vocab) * kChunkBytes + 16);
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
      stride > (int64_t)1 << 40 || workspace_bytes < need || workspace == nullptr ||
      ((uintptr_t)workspace & 15) != 0) {
    return DNX_EINVAL;
  }
  const int64_t chunks = chunks_of(rows, vocab), n = rows * chunks;
  SampleArgs a{logits, u, temperature, top_p, min_p, top_k, out, stride, (int)vocab, (int)chunks,
               ((uintptr_t)logits & 15) == 0 && (stride % 4 == 0 || rows == 1)};
  a.hist = (uint64_t*)workspace;
  a.sums = a.hist + n * kBins;
  a.found = a.sums + 3 * n;
  a.tops = (float*)(a.found + n * kChunkFound);
  a.founds = (uint32_t*)(a.tops + n);
  a.cuts = (int32_t*)(a.founds + n);
  const bool few = per_thread(rows, vocab) == 4;
  const hipStream_t st = (hipStream_t)stream;
  const auto launch = [&](void (*k)(SampleArgs), int64_t y) {
    hipLaunchKernelGGL(k, dim3((unsigned)rows, (unsigned)y), dim3(kThreads), 0, st, a);
    return hipGetLastError() == hipSuccess;
  };
  if (chunks == 1) return launch(row_kernel<16>, 1) ? DNX_OK : DNX_ELAUNCH;
  const bool done = launch(few ? count_kernel<4> : count_kernel<16>, chunks) &&
                    launch(cuts_kernel, 1) &&
                    launch(few ? weigh_kernel<4> : weigh_kernel<16>, chunks) &&
                    launch(few ? pick_kernel<4> : pick_kernel<16>, 1);
  return done ? DNX_OK : DNX_ELAUNCH;
}

}  // extern "C"
