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
//
// Nothing is sorted but what lies at a cut. Four launches: (1) of each chunk of a row
// its largest logit and, in bins of l / T, the tokens and a rough weight; (2) of each
// row the bins in which the cuts lie; (3) of each unit (a wave's tokens) the exact
// weights before those bins and the tokens in them; (4) of each row these tokens in
// order, the cuts, the total, the unit and the token. Up to 256 rows of up to 8192
// tokens take one launch. The logits are read twice, the second time mostly from the caches.
//
// 64 rows of 151936, a mix of requests: 59 us (traced 15 + 6 + 23 + 16), where reading
// the logits once takes 8: the third step's 64-bit series (25 instructions a token) and
// the fourth's ten or so waits in turn for memory and for its workgroup. One row of
// 128000 with top-k and top-p 21, 13 rows of 32003 without filters 13: four launches,
// one to three load latencies each. Rows of nearly equal logits, whose bins hold more
// than lists do, 92 (32003) to 480 (64 of 151936).

#include <algorithm>

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
constexpr int kMaxUnits = 1024;
constexpr int kListed = 8192;            // of a row, that are held in LDS
constexpr int kFound = 256;              // that are sorted at once
constexpr int kParts = 2048;             // of a span of order keys that holds more

struct SampleArgs {
  const float *logits, *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* out;
  int64_t stride;
  int vocab, chunks, units, wide;   // wide: rows may be read 16 bytes at a time
  // Of each row and chunk (a workgroup's tokens in the first step):
  uint64_t* hist;      // [kBins]: counts (the upper 16 bits) and weights
  float* tops;         // the largest logit
  int32_t* cuts;       // [4] of each row: the bins in question
  // Of each row and unit (a wave's tokens in the third):
  uint64_t* sums;      // [3]: of weights
  uint64_t* found;     // [unit_found(E)] order keys
  uint32_t* founds;    // how many tokens were found
};

// A row's request. Greedy: of a steep T, the first token.
struct Request {
  double rate, top_p;          // rate: kPowers log2(e) / T
  uint64_t least;              // min_p in weights
  float u, inv;                // inv: bins per unit / T, finite and not zero
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
  r.rate = inv * (1.4426950408889634 * 128.0);
  r.inv = (float)fmax(fmin(inv * kBinsPerUnit, 1e38), 1e-41);   // an infinity times it is one
  r.top_p = !greedy && p < 1.0f ? fmax((double)p, 0.0) : 1.0;
  r.least = !greedy && low > 0.0f ? (uint64_t)ceil(fmin((double)low, 1.0) * 0x1p43) : 0;
  r.top_k = greedy ? 1 : k > 0 && k < a.vocab ? k : 0;
  r.u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
  r.cut = r.top_k > 0 || r.top_p < 1.0;
  return r;
}

// Keys that rise as logits fall (+0 and -0 are one, NaN is -inf).
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

// Powers 2^(j / kPowers), by the Taylor series: |z| < ln 2, whose 18th term is below
// 2^-62.
constexpr int kPowers = 128;
DNX_DEV void fill_powers(double* powers) {
  if (threadIdx.x >= kPowers) return;
  const double z = (double)threadIdx.x * (0.6931471805599453 / kPowers);
  double p = 1.0;
#pragma unroll
  for (int i = 17; i > 0; i--) p = fma(p * (1.0 / i), z, 1.0);
  powers[threadIdx.x] = p;
}

// A token's weight in multiples of 2^-43, and if that is enough for min_p. With
// x = kPowers log2 of it, its whole part selects a power of two and one from the
// table, the rest z is at most a half: the series in z ln 2 / kPowers, whose 5th
// term is below 2^-49. Adding 3 2^51 rounds to a whole number and leaves it in the
// lower bits, adding 2^52 rounds the result: conversions between 64 bits and whole
// numbers run at a quarter of the rate.
DNX_DEV uint64_t weight(float l, float top, double rate, const double* powers) {
  constexpr double c = 0.6931471805599453 / kPowers;
  const double d = ((double)l - (double)top) * rate, x = l == top ? 0.0 : d, m = x + 0x1.8p52;
  const double z = x - (m - 0x1.8p52);
  double p = c * c * c * c / 24.0;
  p = fma(p, z, c * c * c / 6.0);
  p = fma(p, z, c * c / 2.0);
  p = fma(p, z, c);
  p = fma(p, z, 1.0);
  const bool some = x > -45.0 * kPowers;   // no NaN (of -inf - -inf too), no exponent out of range
  const int n = some ? (int)(uint32_t)__builtin_bit_cast(uint64_t, m) : 0;
  p *= powers[n & (kPowers - 1)];
  const double w = __builtin_bit_cast(
      double, __builtin_bit_cast(uint64_t, p) + ((uint64_t)(uint32_t)((n >> 7) + 43) << 52));
  static_assert(kPowers == 1 << 7, "the shift");
  const uint64_t whole = __builtin_bit_cast(uint64_t, w + 0x1p52) & ((1ull << 52) - 1);
  return some ? whole : 0;
}
DNX_DEV uint64_t at_least(uint64_t w, const Request& r) { return w >= r.least ? w : 0; }

// Bins of l / T, 1 / kBinsPerUnit wide: whole numbers that do not fall as logits rise,
// the same for every chunk of a row. Far-off values are as the last ones (no
// difference of two is then an infinity).
DNX_DEV float scaled(float l, float inv) {
  return __builtin_amdgcn_fmed3f(l * inv, -1e38f, 1e38f);
}
// The bin below the one that the row's (or the chunk's) largest logit lies in;
// kBins and more: no weight.
DNX_DEV int bin_of(float l, float top, float place, float inv) {
  if (l == top) return 0;
  const float d = place - floorf(scaled(l, inv));    // NaN: of a logit NaN
  return l > -INFINITY && d < (float)kBins ? (int)fmaxf(d, 0.0f) : kBins;
}

// Running sums over a wave by DPP: within rows of 16 lanes, then the last lane of
// a row into the next one's, and of the first half into the second's.
template <int Ctrl, int Rows>
DNX_DEV uint64_t dpp_or_0(uint64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, Ctrl, Rows, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), Ctrl, Rows, 0xf, false);
  return (uint64_t)hi << 32 | lo;
}
DNX_DEV uint64_t wave_scan(uint64_t v) {   // inclusive
  constexpr int kShr = 0x110, kBcast15 = 0x142, kBcast31 = 0x143;
  v += dpp_or_0<kShr + 1, 0xf>(v);
  v += dpp_or_0<kShr + 2, 0xf>(v);
  v += dpp_or_0<kShr + 4, 0xf>(v);
  v += dpp_or_0<kShr + 8, 0xf>(v);
  v += dpp_or_0<kBcast15, 0xa>(v);
  v += dpp_or_0<kBcast31, 0xc>(v);
  return v;
}
DNX_DEV uint64_t lane_value(uint64_t v, int lane) {
  const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | lo;
}
DNX_DEV uint64_t wave_sum_u64(uint64_t v) { return lane_value(wave_scan(v), 63); }

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

// Logits of `threads` threads from token j0 on, E each: of each 4 threads tokens
// four in a row a thread.
DNX_DEV int index_of(int j0, int thread, int threads, int e) {
  return j0 + e / 4 * (4 * threads) + 4 * thread + e % 4;
}
template <int E>
DNX_DEV void load_logits(const SampleArgs& a, int row, int j0, int thread, int threads, float* l) {
  const float* x = a.logits + row * a.stride;
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const int j = index_of(j0, thread, threads, e);
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
  load_logits<E>(a, row, chunk * kThreads * E, tid, kThreads, l);
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
  constexpr int P = kBins / kThreads, U = 16;       // bins a thread, chunks at once
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
      w[k] = (uint64_t)((double)w[k] * __builtin_amdgcn_exp2f((float)(P * tid + k) * (-1.44269504f / kBinsPerUnit)) * 0x1p15);
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
      // Where |l / T| is so large that a float of it is wider than the bins' weights hold
      // for (from 2^22 on), the cut may lie in any bin up to the last.
      const double from = r.top_p * least * fmax(1.0 - slack, 0.0), to = r.top_p * most * (1.0 + slack);
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

// How many tokens of the bins in question a unit of 64 E may list.
constexpr int unit_found(int E) { return E == 16 ? 128 : 64; }

// Step 3, a wave units of 64 E tokens (`first` and each `step` further): the weights
// of the tokens before the bins in question (before lo; before k; before lo and of
// min_p), and the keys of the tokens in them. The next unit is requested before
// the present one is weighed.
template <int E>
DNX_DEV void weigh_units(const SampleArgs& a, int row, int first, int step,
                         const double* powers) {
  if (first >= a.units) return;
  const int lane = threadIdx.x & 63;
  float l[E], next[E];
  load_logits<E>(a, row, first * 64 * E, lane, 64, next);
  const int32_t* cut = a.cuts + 4 * (int64_t)row;
  const int lo = cut[0], hi = cut[1], bin_k = cut[2];
  const Request r = request(a, row);
  const float top = row_top(a, row);
  const float place = floorf(scaled(top, r.inv));
  // Without a cut every token's weight counts; without one by rank every bin's.
  const float f_lo = lo < kBins ? (float)lo : INFINITY, f_hi = lo < kBins ? (float)hi : -1.0f;
  const float f_k = bin_k < kBins ? (float)bin_k : INFINITY;
#pragma unroll 1
  for (int unit = first; unit < a.units; unit += step) {
#pragma unroll
    for (int e = 0; e < E; e++) l[e] = next[e];
    load_logits<E>(a, row, (unit + step) * 64 * E, lane, 64, next);   // none past the last
    const int64_t at = (int64_t)row * a.units + unit;
    uint64_t before_lo = 0, before_k = 0, kept = 0;
    uint32_t found = 0;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      bool first[4], weighs[4], here[4], some = false, asked = false;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float x = l[e + i], d = place - floorf(scaled(x, r.inv));   // its bin
        const bool one = x > -INFINITY;
        here[i] = one && ((d >= f_lo && d <= f_hi) || d == f_k);
        weighs[i] = one && d < f_k;
        first[i] = d < f_lo;
        some |= weighs[i];
        asked |= here[i];
      }
      if (__any(some)) {       // four at once: their series are independent
        uint64_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = weight(l[e + i], top, r.rate, powers);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          w[i] = weighs[i] ? w[i] : 0;
          before_k += w[i];
          w[i] = first[i] ? w[i] : 0;
          before_lo += w[i];
          kept += at_least(w[i], r);
        }
      }
      if (!__any(asked)) continue;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint64_t with = __ballot(here[i]);
        if (with == 0) continue;
        const uint32_t at_i =
            found + __builtin_amdgcn_mbcnt_hi((uint32_t)(with >> 32),
                                              __builtin_amdgcn_mbcnt_lo((uint32_t)with, 0));
        if (here[i] && at_i < unit_found(E))
          a.found[at * unit_found(E) + at_i] =
              order_key(l[e + i], index_of(unit * 64 * E, lane, 64, e + i));
        found += __builtin_popcountll(with);
      }
    }
    kept = wave_sum_u64(kept);
    if (r.cut) {
      before_lo = wave_sum_u64(before_lo);
      before_k = wave_sum_u64(before_k);
    }
    if (lane == 0) {
      a.sums[3 * at] = before_lo;
      a.sums[3 * at + 1] = before_k;
      a.sums[3 * at + 2] = kept;
      a.founds[at] = found;
    }
  }
}

// Up to kFound keys in rising order: each to its rank.
DNX_DEV void sort_keys(uint64_t* keys, int n) {
  const int tid = threadIdx.x;
  __syncthreads();
  const uint64_t mine = tid < n ? keys[tid] : 0;
  int rank = 0;
  if (tid < n) {
#pragma unroll 8
    for (int i = 0; i < n; i++) rank += keys[i] < mine;
  }
  __syncthreads();
  if (tid < n) keys[rank] = mine;
  __syncthreads();
}

// What step 4 keeps in LDS: the order keys of the bins in question, those of them
// that are sorted, and the running sums of their weights, or the counts and weights
// of a span's parts.
static_assert(kFound <= kParts && kFound <= kThreads, "upto serves both, a thread a key");
struct PickShared {
  uint64_t list[kListed], keys[kFound], upto[kParts];
  uint32_t count[kParts];
  double powers[kPowers];
  uint64_t part[kWaves], ends[2];
  unsigned long long sums[kMaxUnits];
  int begin[kMaxUnits + 1], at[2], n, unit;
  uint64_t before;
};

// n keys of sh.keys in order, and the running sums of their weights.
DNX_DEV void order_keys(PickShared& sh, int n, float top, const Request& r) {
  const int tid = threadIdx.x;
  sort_keys(sh.keys, n);
  uint64_t all;
  const uint64_t w = tid < n ? weight(of_key((uint32_t)(sh.keys[tid] >> 32)), top, r.rate, sh.powers) : 0;
  const uint64_t before = block_before(w, sh.part, all);
  if (tid < n) sh.upto[tid] = before + w;
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
  uint32_t* count = sh.count;
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
                (unsigned long long)weight(of_key((uint32_t)(k >> 32)), top, r.rate, sh.powers));
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
// among them the cuts lie, the kept weights of each unit, and the token in its
// unit.
template <int E>
DNX_DEV void pick(const SampleArgs& a, int row) {
  constexpr int kUnit = 64 * E, kUnitFound = unit_found(E), U = kMaxUnits / kThreads;
  __shared__ PickShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* x = a.logits + row * a.stride;
  const int64_t base = (int64_t)row * a.units;
  fill_powers(sh.powers);
  const int32_t* cut = a.cuts + 4 * (int64_t)row;
  const int lo = cut[0], hi = cut[1], bin_k = cut[2];
  // A thread's units: U in a row. All is requested before the first wait.
  uint64_t before_lo = 0, before_k = 0, mine[U];
  uint32_t counts[U];
#pragma unroll
  for (int i = 0; i < U; i++) {
    const int c = U * tid + i;
    const uint64_t* from = a.sums + 3 * (base + min(c, a.units - 1));
    const uint64_t s0 = from[0], s1 = from[1], s2 = from[2];
    const uint32_t n = a.founds[base + min(c, a.units - 1)];
    mine[i] = c < a.units ? s2 : 0;
    counts[i] = c < a.units ? n : 0;
    before_lo += c < a.units ? s0 : 0;
    before_k += c < a.units ? s1 : 0;
  }
  const Request r = request(a, row);
  const int rank_k = r.top_k - cut[3];
  const float top = row_top(a, row);
  if (!(top > -INFINITY)) {
    if (tid == 0) a.out[row] = -1;
    return;
  }
#pragma unroll
  for (int i = 0; i < U; i++) sh.sums[U * tid + i] = mine[i];
  uint64_t within = ~0ull;
  bool whole = false;       // the units' sums have to be formed again
  const float place = floorf(scaled(top, r.inv));
  if (lo < kBins) {
    before_lo = block_sum(before_lo, sh.part);
    before_k = block_sum(before_k, sh.part);
    // Where each unit's tokens begin in the list; a unit that found more than it
    // may list counts so that the list is too long.
    uint64_t sum = 0, all;
#pragma unroll
    for (int i = 0; i < U; i++) sum += counts[i] > kUnitFound ? kListed + 1 : counts[i];
    uint64_t b = block_before(sum, sh.part, all);
#pragma unroll
    for (int i = 0; i < U; i++) {
      sh.begin[U * tid + i] = (int)b;
      b += counts[i];
    }
    if (tid == 0) sh.begin[kMaxUnits] = (int)all;
    if (tid < 2) sh.at[tid] = kFound;
    __syncthreads();
    const int n = sh.begin[kMaxUnits];
    uint64_t total = before_k;
    bool done = n > 0 && n <= kFound;
    if (n <= kListed) {
      uint64_t* to = done ? sh.keys : sh.list;
      for (int i0 = tid; i0 < n; i0 += 4 * kThreads) {
        uint64_t k[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
          const int i = min(i0 + u * kThreads, n - 1);
          int c = 0;                        // the last unit that begins at or before i
#pragma unroll
          for (int step = kMaxUnits / 2; step > 0; step /= 2) c += sh.begin[c + step] <= i ? step : 0;
          k[u] = a.found[(base + c) * kUnitFound + i - sh.begin[c]];
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
          if (i0 + u * kThreads < n) to[i0 + u * kThreads] = k[u];
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
          if (w > 0) atomicAdd(&sh.sums[(uint32_t)sh.keys[i] / kUnit], (unsigned long long)w);
        }
      }
    }
    if (!done) {
      whole = n <= kFound || n > kListed;     // up to kFound were put into sh.keys, not sh.list
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
      __syncthreads();
      for (int i = tid; i < n && !whole; i += kThreads) {
        const uint64_t k = sh.list[i];
        const uint64_t w = k <= within ? at_least(weight(of_key((uint32_t)(k >> 32)), top, r.rate, sh.powers), r) : 0;
        if (w > 0) atomicAdd(&sh.sums[(uint32_t)k / kUnit], (unsigned long long)w);
      }
    }
  }
  // The kept weights of a lane's tokens of a unit.
  auto kept = [&](int unit, uint64_t* w) {
    float l[E];
    load_logits<E>(a, row, unit * kUnit, lane, 64, l);
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
      w[e] = order_key(l[e], index_of(unit * kUnit, lane, 64, e)) <= within
                 ? at_least(weight(l[e], top, r.rate, sh.powers), r) : 0;
      sum += w[e];
    }
    return sum;
  };
  __syncthreads();
  if (whole) {
    for (int c = wave; c < a.units; c += kWaves) {
      uint64_t w[E];
      const uint64_t s = wave_sum_u64(kept(c, w));
      if (lane == 0) sh.sums[c] = s;
    }
    __syncthreads();
  }
  // The unit.
  uint64_t s = 0, total;
#pragma unroll
  for (int i = 0; i < U; i++) s += mine[i] = sh.sums[U * tid + i];
  uint64_t before = block_before(s, sh.part, total);
  uint64_t target = (uint64_t)((double)r.u * (double)total);
  target = target < total ? target : total - 1;
#pragma unroll
  for (int i = 0; i < U; i++) {
    if (before <= target && target < before + mine[i]) {
      sh.unit = U * tid + i;
      sh.before = before;
    }
    before += mine[i];
  }
  __syncthreads();
  if (wave > 0) return;
  const int unit = sh.unit;
  before = sh.before;
  uint64_t w[E];
  kept(unit, w);
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const uint64_t four = w[e] + w[e + 1] + w[e + 2] + w[e + 3], upto = wave_scan(four);
    uint64_t at = before + upto - four;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (at <= target && target < at + w[e + i]) a.out[row] = index_of(unit * kUnit, lane, 64, e + i);
      at += w[e + i];
    }
    before += lane_value(upto, 63);
  }
}

template <int E>
__global__ void __launch_bounds__(kThreads) count_kernel(SampleArgs a) {
  count_chunk<E>(a, blockIdx.x, blockIdx.y);
}
__global__ void __launch_bounds__(kThreads) cuts_kernel(SampleArgs a) { find_cuts(a, blockIdx.x); }
constexpr int kUnitWaves = 4;
template <int E>
__global__ void __launch_bounds__(64 * kUnitWaves) weigh_kernel(SampleArgs a) {
  __shared__ double powers[kPowers];
  fill_powers(powers);
  __syncthreads();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  weigh_units<E>(a, blockIdx.x, blockIdx.y * kUnitWaves + wave, gridDim.y * kUnitWaves, powers);
}
template <int E>
__global__ void __launch_bounds__(kThreads) pick_kernel(SampleArgs a) {
  pick<E>(a, blockIdx.x);
}
// A row of one chunk: the steps by one workgroup.
__global__ void __launch_bounds__(kThreads) row_kernel(SampleArgs a) {
  count_chunk<16>(a, blockIdx.x, 0);
  __syncthreads();
  find_cuts(a, blockIdx.x);
  __syncthreads();
  __shared__ double powers[kPowers];
  fill_powers(powers);
  __syncthreads();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  weigh_units<16>(a, blockIdx.x, wave, kWaves, powers);
  __syncthreads();
  pick<16>(a, blockIdx.x);
}

// Tokens of a thread in a chunk: 32 where 16 would make more workgroups than the card
// holds at once (64 rows of 151936 logits: the first two steps take 19.4 us, with 16
// 21.4), else 16 (one row of 128000: 10.7; with 4 18). Tokens of a lane in a unit: 4
// where 16 would leave SIMDs without a wave (one row of 128000: 4.1 us).
constexpr int kManyChunks = 1024, kManyUnits = 1024;   // of all rows, by 16 tokens a thread or lane
struct Shape {
  int64_t chunks, units;
  int counted, tokens;
};
Shape shape_of(int64_t rows, int64_t vocab) {
  const auto parts = [&](int64_t size) { return (vocab + size - 1) / size; };
  const int counted = rows * parts(kThreads * 16) > kManyChunks && vocab > kThreads * 16 ? 32 : 16;
  const int64_t chunks = parts(kThreads * counted);
  const bool few = chunks > 1 && rows * parts(64 * 16) < kManyUnits && parts(64 * 4) <= kMaxUnits;
  return {chunks, parts(64 * (few ? 4 : 16)), counted, few ? 4 : 16};
}

}  // namespace

extern "C" {

int64_t dnx_sample_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 0 || rows > kMaxRows || vocab < 1 || vocab > kMaxVocab) return -1;
  // What the most demanding call of up to that many rows and tokens takes: few rows
  // are in more chunks and units each than many are.
  const auto parts = [&](int64_t size) { return (vocab + size - 1) / size; };
  const auto unit = [](int64_t e) { return 8 * (3 + unit_found((int)e)) + 4; };
  const int64_t chunks = std::max(rows * parts(kThreads * 32),
                                  std::min<int64_t>(rows * parts(kThreads * 16), kManyChunks));
  const int64_t units = std::max(rows * parts(64 * 16) * unit(16),
                                 std::min<int64_t>(rows * parts(64 * 4), 4 * kManyUnits) * unit(4));
  return chunks * (8 * kBins + 4) + units + rows * 16;
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
  const Shape s = shape_of(rows, vocab);
  SampleArgs a{logits, u, temperature, top_p, min_p, top_k, out, stride, (int)vocab, (int)s.chunks,
               (int)s.units, ((uintptr_t)logits & 15) == 0 && (stride % 4 == 0 || rows == 1)};
  a.hist = (uint64_t*)workspace;
  a.sums = a.hist + rows * s.chunks * kBins;
  a.found = a.sums + 3 * rows * s.units;
  a.tops = (float*)(a.found + rows * s.units * unit_found(s.tokens));
  a.founds = (uint32_t*)(a.tops + rows * s.chunks);
  a.cuts = (int32_t*)(a.founds + rows * s.units);
  const hipStream_t st = (hipStream_t)stream;
  const auto launch = [&](void (*k)(SampleArgs), int64_t y, int threads = kThreads) {
    hipLaunchKernelGGL(k, dim3((unsigned)rows, (unsigned)y), dim3(threads), 0, st, a);
    return hipGetLastError() == hipSuccess;
  };
  // One launch for a row of one chunk while each CU has at most one (a workgroup holds
  // most of its LDS): us against four launches, 2000 tokens with top-k and top-p, 1
  // row 20.8 / 23.1, 256 22.4 / 27.1, 2000 159 / 112.
  if (s.chunks == 1 && rows <= 256) return launch(row_kernel, 1) ? DNX_OK : DNX_ELAUNCH;
  const bool few = s.tokens == 4;
  // Four waves a SIMD, of at least a unit each.
  const int64_t weighers = std::min((s.units + kUnitWaves - 1) / kUnitWaves,
                                    std::max<int64_t>(1, 4096 / kUnitWaves / rows));
  const bool done = launch(s.counted == 32 ? count_kernel<32> : count_kernel<16>, s.chunks) && launch(cuts_kernel, 1) &&
                    launch(few ? weigh_kernel<4> : weigh_kernel<16>, weighers, 64 * kUnitWaves) &&
                    launch(few ? pick_kernel<4> : pick_kernel<16>, 1);
  return done ? DNX_OK : DNX_ELAUNCH;
}

}  // extern "C"
