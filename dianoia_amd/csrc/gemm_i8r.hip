// y[t][r] = xs[t] ws[r] sum_k xq[t][k] wq[r][k]: int8 rows times int8 weight
// rows with one scale each, on the int8 matrix cores. The sums are whole
// numbers, exact in int32 (|q| <= 128: K up to 131040), so no order of adding
// changes a result; each output is rounded to float32 three times (the sum,
// the product of the scales, their product).

#include "common.h"
#include "dnx_kernels.h"
#include "gemm_i8r_route.h"

using namespace dnx;

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

constexpr int64_t kMaxK = 131040;   // fewer than 2^17 products of 2^14 or less: below 2^31

struct I8RArgs {
  const int8_t* w;
  const float* w_scale;
  const int8_t* x;
  const float* x_scale;
  float* y;
  int rows, cols, n;
};

// ---- Few tokens (a decode batch of up to 16): what it costs is to read the
// weights once. A workgroup takes 16 or 32 weight rows (NR tiles) and all
// tokens, its eight waves an eighth of K each, both operands straight from
// memory into the fragments of v_mfma_i32_16x16x64_i8 (lane l: row l % 16, the
// 16 bytes at k = 16 (l / 16) of 64), four steps requested at once; the eight
// sums meet in LDS. 13 x 6144 x 2048: 5.1 us (5.8 on another card), 2.5 TB/s, of
// which about 2.0 us are an empty launch's; 16 x 128256 x 4096 128 us, 4.2 TB/s.
constexpr int kFewWaves = 8, kFewRows = 16, kFewSteps = 4;

template <int NR>
__global__ void __launch_bounds__(kFewWaves * 64) gemm_i8r_few_kernel(I8RArgs p) {
  __shared__ int part[kFewWaves][NR][16][16];
  const int lane = threadIdx.x & 63, l16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r0 = blockIdx.x * kFewRows * NR;
  const i32x4 wrs = buffer_rsrc(p.w + (size_t)r0 * p.cols,
                                (uint32_t)(min(kFewRows * NR, p.rows - r0) * p.cols));
  const i32x4 xrs = buffer_rsrc(p.x, (uint32_t)(p.n * p.cols));
  const int chunks = (p.cols + 63) / 64, per = (chunks + kFewWaves - 1) / kFewWaves;
  const int end = min(chunks, (wave + 1) * per);
  v4i acc[NR] = {};
  for (int c0 = wave * per; c0 < end; c0 += kFewSteps) {
    i32x4 wv[kFewSteps][NR], xv[kFewSteps];
#pragma unroll
    for (int u = 0; u < kFewSteps; u++) {
      // Past the row: past the resource (zeros), the next row's bytes follow.
      const int k = (c0 + u) * 64 + 16 * g4;
      const bool in = c0 + u < end && k < p.cols;
#pragma unroll
      for (int i = 0; i < NR; i++)
        wv[u][i] = dnx_raw_buffer_load_v4i32(wrs, in ? (16 * i + l16) * p.cols + k : -1, 0, kStream);
      xv[u] = dnx_raw_buffer_load_v4i32(xrs, in ? l16 * p.cols + k : -1, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);   // every load before the first product waits
#pragma unroll
    for (int u = 0; u < kFewSteps; u++)
#pragma unroll
      for (int i = 0; i < NR; i++)
        acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xv[u], wv[u][i], acc[i], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < NR; i++)
#pragma unroll
    for (int v = 0; v < 4; v++) part[wave][i][4 * g4 + v][l16] = acc[i][v];
  __syncthreads();
  for (int o = threadIdx.x; o < NR * 256; o += kFewWaves * 64) {
    const int c = o % (16 * NR), t = o / (16 * NR), r = r0 + c;
    if (t >= p.n || r >= p.rows) continue;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kFewWaves; w++) sum += part[w][c / 16][t][c % 16];
    p.y[(size_t)t * p.rows + r] = (float)sum * (p.x_scale[t] * p.w_scale[r]);
  }
}

// ---- Many tokens: tiles of TM tokens x TN weight rows through LDS. WM x WN
// waves, each MT x NT tiles of v_mfma_i32_32x32x32_i8 (lane l: row l % 32, the
// 16 bytes at k = 16 (l / 32) of 32).
//
// A stage is 64 bytes of K of all TM + TN rows, moved into one of RING buffers
// by DMA, RING - 1 stages ahead. LDS holds rows of four 16-byte pieces; piece
// c of row r lies at place c ^ (r / 4 % 4), so that a fragment's rows meet all
// banks (a DMA writes its lanes in order, so the lanes fetch in that order
// instead). The second half of a stage is read while the first is multiplied;
// the one barrier of a stage stands before its second half's products, where
// the next stage has arrived and this one's buffer is free again. Stages past
// the last are requested too, out of bounds (zeros, no memory), so that the
// count of requests in flight stays the same to the end. With KG > 1 as many
// groups of waves take a part of K each (with buffers of their own), where the
// tiles alone are too few to keep the chip busy; their sums are added in LDS.
//
// 2047 x 8192 x 4096 on 256 x 256 tiles of 16 waves: 73 to 76 us, 1.8 to 1.9
// POP/s (a library product of that size with int32 outputs takes 76). By the
// counters the matrix cores are busy 66 k of 106 k cycles, and the clock falls to
// about 1.5 GHz under them; LDS is busy 37 k cycles, without bank conflicts; the
// 67 MB of outputs are 5 us. Eight waves of twice the tile took
// 80 us (fewer waves to cover a barrier), four 85. 1024 x 4304 x 1152: 14 us.
constexpr int kStageK = 64;

// Waits until all but `vm` requests of this wave have arrived, then for the
// workgroup; nothing that reads or writes memory moves past it.
template <int vm>
DNX_DEV void wait_all() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" : : : "memory");
  __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(vm));
  __builtin_amdgcn_s_barrier();
  asm volatile("" : : : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <int WM, int WN, int MT, int NT, int RING, int KG>
__global__ void __launch_bounds__(KG * WM * WN * 64) gemm_i8r_tile_kernel(I8RArgs p, int tiles_t,
                                                                           int tiles) {
  constexpr int kWaves = WM * WN, TM = WM * MT * 32, TN = WN * NT * 32;   // of a group
  constexpr int kThreads = KG * kWaves * 64;
  constexpr int kPieces = (TM + TN) / 16 / kWaves;   // DMAs of 16 rows, per wave and stage
  constexpr int kStage = (TM + TN) * kStageK;
  constexpr int kRow = TN * 4 + 32;    // of the outputs in LDS: rows 4 apart meet other banks
  constexpr int PASSES = WM % 2 == 0 && TM * (kRow + 4) > KG * RING * kStage ? 2 : 1;
  constexpr int kPass = TM / PASSES, kOut = kPass * kRow + TM * 4;
  constexpr int kLds = KG * RING * kStage > kOut ? KG * RING * kStage : kOut;
  static_assert((TM + TN) / 16 % kWaves == 0, "whole DMAs per wave");
  static_assert(kLds <= 160 * 1024, "a CU's LDS");
  static_assert(RING >= 3 && (RING - 2) * kPieces < 64, "requests that vmcnt can count");
  __shared__ __align__(1024) uint8_t lds[kLds];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) % kWaves);
  const int group = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) / kWaves);
  // Workgroups go round the eight XCDs, each with an L2 of its own: each takes
  // a run of tiles, all tokens of one strip of weights after another.
  const int run = (tiles + 7) / 8;
  const int tile = blockIdx.x % 8 * run + blockIdx.x / 8;
  if (tile >= tiles) return;
  const int t0 = tile % tiles_t * TM, r0 = tile / tiles_t * TN;
  const i32x4 xrs = buffer_rsrc(p.x + (size_t)t0 * p.cols,
                                (uint32_t)(min(TM, p.n - t0) * p.cols));
  const i32x4 wrs = buffer_rsrc(p.w + (size_t)r0 * p.cols,
                                (uint32_t)(min(TN, p.rows - r0) * p.cols));
  uint8_t* ring = lds + group * RING * kStage;
  const uint32_t lds0 = lds_address(ring) + wave * 16 * kStageK;
  const int stages = ((p.cols + kStageK - 1) / kStageK + KG - 1) / KG;   // of a group
  const int dma_k = ((lane & 3) ^ (lane >> 4)) * 16;
  auto dma = [&](int s, int buf) {
    const int k = (group * stages + s) * kStageK + dma_k;
    const bool in = s < stages && k < p.cols;
#pragma unroll
    for (int e = 0; e < kPieces; e++) {
      const int row = (e * kWaves + wave) * 16;          // tokens first, then weight rows
      const bool tok = row < TM;
      const int at = (row - (tok ? 0 : TM) + (lane >> 2)) * p.cols;
      buffer_load16_to_lds(tok ? xrs : wrs, lds0 + buf * kStage + e * kWaves * 16 * kStageK,
                           in ? at + k : -1);
    }
  };
  const int l32 = lane & 31, half = lane >> 5, turn = (l32 >> 2) & 3;
  const int xm = (wave % WM) * MT * 32 + l32, wm = TM + (wave / WM) * NT * 32 + l32;
  i32x4 xf[2][MT], wf[2][NT];
  auto read = [&](int buf, int s) {
    const uint8_t* base = ring + buf * kStage + (((2 * s + half) ^ turn) * 16);
#pragma unroll
    for (int i = 0; i < MT; i++) xf[s][i] = *(const i32x4*)(base + (xm + 32 * i) * kStageK);
#pragma unroll
    for (int j = 0; j < NT; j++) wf[s][j] = *(const i32x4*)(base + (wm + 32 * j) * kStageK);
  };
  v16i acc[MT][NT] = {};
  auto multiply = [&](int s) {
#pragma unroll
    for (int a = 0; a < MT; a++)
#pragma unroll
      for (int b = 0; b < NT; b++)
        acc[a][b] =
            __builtin_amdgcn_mfma_i32_32x32x32_i8(xf[s][a], wf[s][b], acc[a][b], 0, 0, 0);
  };
#pragma unroll
  for (int s = 0; s < RING - 1; s++) dma(s, s);
  wait_all<(RING - 2) * kPieces>();
  read(0, 0);
  int buf = 0, next = RING - 1;      // the buffer of stage i, and of stage i + RING - 1
  for (int i = 0; i < stages; i++) {
    dma(i + RING - 1, next);
    next = buf;
    read(buf, 1);
    __builtin_amdgcn_sched_barrier(0);   // products pass no read, wait or barrier
    multiply(0);
    buf = buf + 1 == RING ? 0 : buf + 1;
    wait_all<(RING - 2) * kPieces>();
    read(buf, 0);                        // after the last stage: zeros, not used
    __builtin_amdgcn_sched_barrier(0);
    multiply(1);
  }
  // The outputs through LDS (PASSES runs of the tile's tokens, as many as its
  // buffers hold): whole rows are stored, by a loop of few instructions.
  // Straight-line stores of every register are some kilobytes of code that
  // runs once, and its way into the instruction cache took longer than the
  // products of a short K.
  float* scale = (float*)(lds + kPass * kRow);
  constexpr int kCols = TN / 4, kStep = kThreads / kCols;   // threads a row, rows at once
  // A thread's four columns: 16 bytes where every row of y starts on 16,
  // else one in each quarter of the row, so that a wave's stores stay whole.
  const bool whole = p.rows % 4 == 0 && ((uintptr_t)p.y & 15) == 0;
  const int tid = threadIdx.x, c = tid % kCols * (whole ? 4 : 1), dc = whole ? 1 : kCols;
  const i32x4 wsr = buffer_rsrc(p.w_scale + r0, (uint32_t)(min(TN, p.rows - r0) * 4));
  f32x4 ws;
#pragma unroll
  for (int j = 0; j < 4; j++)
    ws[j] = __int_as_float(dnx_raw_buffer_load_i32(wsr, (c + j * dc) * 4, 0, 0));
  const float xs = __int_as_float(dnx_raw_buffer_load_i32(
      buffer_rsrc(p.x_scale + t0, (uint32_t)(min(TM, p.n - t0) * 4)), tid * 4, 0, 0));
  wait_all<0>();   // the last DMAs too
  if (tid < TM) scale[tid] = xs;
#pragma unroll
  for (int pass = 0; pass < PASSES; pass++) {
    const int first = pass * kPass;
    const bool mine = PASSES == 1 || (wave % WM) * MT * 32 / kPass == pass;
    int* to = (int*)(lds + (xm - l32 - first + 4 * half) * kRow) + (wm - TM);
#pragma unroll
    for (int g = 0; g < KG; g++) {
      if (pass > 0 || g > 0) __syncthreads();
      if (mine && group == g) {
#pragma unroll
        for (int a = 0; a < MT; a++)
#pragma unroll
          for (int b = 0; b < NT; b++)
#pragma unroll
            for (int v = 0; v < 16; v++) {
              int* at = to + (32 * a + 8 * (v >> 2) + (v & 3)) * (kRow / 4) + 32 * b;
              *at = g > 0 ? *at + acc[a][b][v] : acc[a][b][v];
            }
      }
    }
    __syncthreads();
#pragma unroll 2
    for (int i = tid / kCols; i < kPass; i += kStep) {
      const int t = t0 + first + i;
      if (t >= p.n) break;
      const int* from = (const int*)(lds + i * kRow) + c;
      const float s = scale[first + i];
      float* at = p.y + (size_t)t * p.rows + r0 + c;
      if (whole) {
        const v4i sum = *(const v4i*)from;
        f32x4 y;
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = (float)sum[j] * (s * ws[j]);
        if (r0 + c < p.rows) __builtin_nontemporal_store(y, (f32x4*)at);
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (r0 + c + j * dc < p.rows)
            __builtin_nontemporal_store((float)from[j * dc] * (s * ws[j]), at + j * dc);
      }
    }
  }
}

template <int I, int WM, int WN, int MT, int NT, int RING>
int launch_tile(const I8RArgs& p, hipStream_t st) {
  constexpr I8RTile T = kI8RTiles[I];
  static_assert(T.tokens == WM * MT * 32 && T.rows == WN * NT * 32, "the route's tile");
  const int64_t tiles_t = (p.n + T.tokens - 1) / T.tokens;
  const int64_t tiles = tiles_t * ((p.rows + T.rows - 1) / T.rows);
  constexpr int kThreads = T.parts * WM * WN * 64;
  const int64_t grid = (tiles + 7) / 8 * 8;
  if (grid > kLaunchThreads / kThreads) return DNX_EINVAL;
  hipLaunchKernelGGL((gemm_i8r_tile_kernel<WM, WN, MT, NT, RING, T.parts>), dim3((unsigned)grid),
                     dim3(kThreads), 0, st, p, (int)tiles_t, (int)tiles);
  return hipGetLastError() == hipSuccess ? DNX_OK : DNX_ELAUNCH;
}

}  // namespace

extern "C" {

int dnx_gemm_i8r(const int8_t* w, const float* w_scale, const int8_t* x, const float* x_scale,
                 float* y, int64_t rows, int64_t cols, int64_t n, dnx_stream_t stream) {
  if (rows <= 0 || rows >= (1 << 22) || n < 0 || n >= (1 << 22) || cols <= 0 ||
      cols % kBlock != 0 || cols > kMaxK) {
    return DNX_EINVAL;
  }
  if (n == 0) return DNX_OK;
  if (w == nullptr || w_scale == nullptr || x == nullptr || x_scale == nullptr || y == nullptr ||
      (((uintptr_t)w | (uintptr_t)x) & 15) != 0 ||
      (((uintptr_t)w_scale | (uintptr_t)x_scale | (uintptr_t)y) & 3) != 0) {
    return DNX_EINVAL;
  }
  const I8RArgs p{w, w_scale, x, x_scale, y, (int)rows, (int)cols, (int)n};
  const hipStream_t st = (hipStream_t)stream;
  switch (i8r_route(n, rows, cols)) {
    case 0: return launch_tile<0, 1, 1, 1, 1, 4>(p, st);
    case 1: return launch_tile<1, 2, 1, 1, 1, 4>(p, st);
    case 2: return launch_tile<2, 2, 2, 1, 1, 6>(p, st);
    case 3: return launch_tile<3, 2, 2, 2, 1, 4>(p, st);
    case 4: return launch_tile<4, 2, 2, 2, 2, 4>(p, st);
    case 5: return launch_tile<5, 4, 2, 2, 2, 3>(p, st);
    case 6: return launch_tile<6, 4, 4, 2, 2, 5>(p, st);
  }
  const int tiles = i8r_few_tiles(n, rows);
  const int64_t wg_rows = kFewRows * tiles;
  hipLaunchKernelGGL(tiles == 2 ? gemm_i8r_few_kernel<2> : gemm_i8r_few_kernel<1>,
                     dim3((unsigned)((rows + wg_rows - 1) / wg_rows)), dim3(kFewWaves * 64), 0, st, p);
  return hipGetLastError() == hipSuccess ? DNX_OK : DNX_ELAUNCH;
}

}  // extern "C"
