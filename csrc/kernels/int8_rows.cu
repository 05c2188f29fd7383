// Rows in 8-bit integers (int8_rows.cuh), by themselves and from the norms around a decoder's block:
//
//   x' = a x + b g post(y)      post, pre: RMS norms with a weight, or nothing
//   h  = pre(x')                g: nothing, one value a channel, one a token and channel (or the sigmoid of it)
//
// x is the residual stream, y what a block wrote, h what the next one reads: in a float type, or as 8-bit rows for a product.  All of it in
// 32 bits from the loads to one rounding at each store; h is taken from x' before x' is rounded to the stream's type.
//
// Both are bound by the bytes they move.  A row stays in registers from its load to its last store, so nothing is read twice: a warp, or a
// block of as many threads as leave each at most kNormVec pieces of eight values.  Few rows (a decode step) take a piece a thread, as
// the time is then a chain of latencies -- load, three sums over the row, store -- and not bandwidth.
#include <stdint.h>

#include "common.cuh"
#include "int8_rows.cuh"
#include "ogb_kernels.h"

namespace ogb {

constexpr int kVec = 4;            // pieces of eight values that a thread keeps
constexpr int kMostThreads = 512;
constexpr int kNormMaxCols = kVec * 8 * kMostThreads;

// Sum (or largest) of v over the threads of a row: a warp of its own, or the block.  `part`: a word per warp, used by one call only.
template <bool WARP>
OGB_DEVICE float row_sum(float v, float* part) {
  v = warp_sum(v);
  if (WARP) return v;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) v += part[i];
  return v;
}
template <bool WARP>
OGB_DEVICE uint32_t row_max(uint32_t v, uint32_t* part) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (WARP) return v;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) v = max(v, part[i]);
  return v;
}

// ------------------------------------------------------------------------------------------
// rows to codes
// ------------------------------------------------------------------------------------------
struct QuantizeParams {
  const void* x;
  int8_t* q;
  float* factor;
  long long ldx, ldq;
  int rows, cols, elem, vec;
  unsigned int* counters;
  int num_counters;
};

template <int E, int V, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : kMostThreads) quantize_rows_kernel(const QuantizeParams p) {
  __shared__ uint32_t part[kMostThreads / 32];
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < p.num_counters; i += blockDim.x) p.counters[i] = 0;
  const int threads = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int row = WARP ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= p.rows) return;
  const void* x = after_wait(p.x);
  const size_t at = static_cast<size_t>(row) * p.ldx;
  const int step = threads * 8;
  Raw8<E> f[V];
  uint32_t peak = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) f[v].load(x, p.vec != 0, at, tid * 8 + v * step, p.cols);
#pragma unroll
  for (int v = 0; v < V; ++v) peak = f[v].peak(peak);
  // longer rows than the registers hold are read again below
  for (int i = tid * 8 + V * step; i < p.cols; i += step) {
    Raw8<E> t;
    t.load(x, p.vec != 0, at, i, p.cols);
    peak = t.peak(peak);
  }
  const RowCode code(row_max<WARP>(Raw8<E>::peak_float(peak), part));
  const size_t to = static_cast<size_t>(row) * p.ldq;
  float t[8];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = tid * 8 + v * step;
    f[v].get(t);
    if (i < p.cols) store_codes(p.q, to, i, code, t);
  }
  for (int i = tid * 8 + V * step; i < p.cols; i += step) {
    Raw8<E> r;
    r.load(x, p.vec != 0, at, i, p.cols);
    r.get(t);
    store_codes(p.q, to, i, code, t);
  }
  if (tid == 0) p.factor[row] = code.factor;
}

// Threads for a row of `cols` values: 32 (a warp, four rows a block) or a block of them.
static int row_threads(int rows, int cols) {
  const int pieces = (cols + 7) / 8;
  const int per = rows <= 2 * ogb_num_sms() ? 1 : kVec;
  int t = 32;
  while (t < kMostThreads && t * per < pieces) t *= 2;
  return t;
}

template <int E>
static int launch_quantize(const QuantizeParams& p, cudaStream_t stream) {
  const int t = row_threads(p.rows, p.cols), pieces = (p.cols + 7) / 8;
  const dim3 grid(t == 32 ? (p.rows + 3) / 4 : p.rows), block(t == 32 ? 128 : t);
  const bool one = pieces <= t, more = pieces > kVec * t;
  auto kernel = t == 32 ? (one ? quantize_rows_kernel<E, 1, true> : quantize_rows_kernel<E, kVec, true>)
                        : (one ? quantize_rows_kernel<E, 1, false> : more ? quantize_rows_kernel<E, 2 * kVec, false> : quantize_rows_kernel<E, kVec, false>);
  return static_cast<int>(launch_overlapped(kernel, grid, block, 0, stream, p));
}

int launch_quantize_rows(const void* x, int8_t* q, float* factor, int rows, int cols, long long ldx, long long ldq, int elem, unsigned int* counters,
                         int num_counters, cudaStream_t stream) {
  const QuantizeParams p{x, q, factor, ldx, ldq, rows, cols, elem, rows_aligned(x, ldx, elem), counters, num_counters};
  if (elem == kElemF32) return launch_quantize<kElemF32>(p, stream);
  if (elem == kElemBf16) return launch_quantize<kElemBf16>(p, stream);
  return launch_quantize<kElemF16>(p, stream);
}

// ------------------------------------------------------------------------------------------
// norms around a block
// ------------------------------------------------------------------------------------------
struct BlockNormParams {
  const void *x, *y, *gate, *post, *pre;
  void *x_out, *h;
  int8_t* q;
  float* factor;
  long long ldx, ldy, ldg, ldxo, ldh, ldq;    // ldg 0: one gate for all rows
  int rows, cols;
  int x_elem, y_elem, gate_elem, w_elem, h_elem;
  int x_vec, y_vec, gate_vec, post_vec, pre_vec, xo_vec, h_vec;
  int gate_sigmoid;
  float eps, x_scale, y_scale;
};

template <int V, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : kMostThreads) block_norm_kernel(const BlockNormParams p) {
  __shared__ float part_y[kMostThreads / 32], part_x[kMostThreads / 32];
  __shared__ uint32_t part_q[kMostThreads / 32];
  pdl_trigger();
  pdl_wait();
  const int threads = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int row = WARP ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= p.rows) return;
  const int n = p.cols, step = threads * 8, i0 = tid * 8;
  const float over = 1.f / static_cast<float>(n);
  const void *xp = after_wait(p.x), *yp = after_wait(p.y), *gp = after_wait(p.gate);
  float x[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v) load8(xp, p.x_elem, p.x_vec != 0, static_cast<size_t>(row) * p.ldx, i0 + v * step, n, x[v]);
  if (yp != nullptr) {
    float y[V][8];
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) load8(yp, p.y_elem, p.y_vec != 0, static_cast<size_t>(row) * p.ldy, i0 + v * step, n, y[v]);
    float ry = p.y_scale;
    if (p.post != nullptr) {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += y[v][j] * y[v][j];
      ry *= rsqrtf(row_sum<WARP>(sum, part_y) * over + p.eps);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = i0 + v * step;
      float t[8];
      if (p.post != nullptr) {
        load8(p.post, p.w_elem, p.post_vec != 0, 0, i, n, t);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[v][j] *= t[j];
      }
      if (gp != nullptr) {
        load8(gp, p.gate_elem, p.gate_vec != 0, static_cast<size_t>(row) * p.ldg, i, n, t);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[v][j] *= p.gate_sigmoid != 0 ? __fdividef(1.f, 1.f + __expf(-t[j])) : t[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) x[v][j] = fmaf(ry, y[v][j], p.x_scale * x[v][j]);
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[v][j] *= p.x_scale;
  }
  if (p.x_out != nullptr) {
#pragma unroll
    for (int v = 0; v < V; ++v) store8(p.x_out, p.x_elem, p.xo_vec != 0, static_cast<size_t>(row) * p.ldxo, i0 + v * step, n, x[v]);
  }
  if (p.h == nullptr && p.q == nullptr) return;
  if (p.pre != nullptr) {
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += x[v][j] * x[v][j];      // past the row's end: zeros
    const float rx = rsqrtf(row_sum<WARP>(sum, part_x) * over + p.eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float t[8];
      load8(p.pre, p.w_elem, p.pre_vec != 0, 0, i0 + v * step, n, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[v][j] *= rx * t[j];
    }
  }
  if (p.h != nullptr) {
#pragma unroll
    for (int v = 0; v < V; ++v) store8(p.h, p.h_elem, p.h_vec != 0, static_cast<size_t>(row) * p.ldh, i0 + v * step, n, x[v]);
  }
  if (p.q != nullptr) {
    uint32_t peak = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) peak = max(peak, peak_bits8(x[v]));
    const RowCode code(row_max<WARP>(peak, part_q));
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = i0 + v * step;
      if (i < n) store_codes(p.q, static_cast<size_t>(row) * p.ldq, i, code, x[v]);
    }
    if (tid == 0) p.factor[row] = code.factor;
  }
}

}  // namespace ogb

using namespace ogb;

extern "C" int ogb_quantize_rows(const void* x, void* q, float* factor, int rows, int cols, int64_t ldx, int64_t ldq, int elem, void* stream) {
  if (rows < 0 || cols < 0 || elem < 0 || elem >= kElemKinds) return -2;
  if (rows == 0) return 0;
  if (cols == 0 || ldx < 0 || ldq < cols || (ldq & 15) != 0 || (reinterpret_cast<uintptr_t>(q) & 15) != 0) return -3;
  return launch_quantize_rows(x, static_cast<int8_t*>(q), factor, rows, cols, ldx, ldq, elem, nullptr, 0, static_cast<cudaStream_t>(stream));
}

extern "C" int ogb_block_norm(const void* x, const void* y, const void* gate, const void* post, const void* pre, void* x_out, void* h, void* q,
                              float* factor, int64_t ldx, int64_t ldy, int64_t ldg, int64_t ldxo, int64_t ldh, int64_t ldq, int rows, int cols,
                              int x_elem, int y_elem, int gate_elem, int w_elem, int h_elem, int gate_sigmoid, float eps, float x_scale, float y_scale,
                              void* stream_) {
  for (const int e : {x_elem, y_elem, gate_elem, w_elem, h_elem})
    if (e < 0 || e >= kElemKinds) return -2;
  if (rows < 0 || cols < 1 || cols > kNormMaxCols) return -2;
  if (rows == 0) return 0;
  if (q != nullptr && (ldq < cols || (ldq & 15) != 0 || (reinterpret_cast<uintptr_t>(q) & 15) != 0 || factor == nullptr)) return -3;
  BlockNormParams p{x, y, gate, post, pre, x_out, h, static_cast<int8_t*>(q), factor, ldx, ldy, ldg, ldxo, ldh, ldq, rows, cols, x_elem, y_elem, gate_elem,
                    w_elem, h_elem, rows_aligned(x, ldx, x_elem), rows_aligned(y, ldy, y_elem), rows_aligned(gate, ldg, gate_elem),
                    rows_aligned(post, 0, w_elem), rows_aligned(pre, 0, w_elem), rows_aligned(x_out, ldxo, x_elem), rows_aligned(h, ldh, h_elem),
                    gate_sigmoid, eps, x_scale, y_scale};
  const int t = row_threads(rows, cols);
  const bool one = (cols + 7) / 8 <= t;
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  cudaError_t e;
  if (t == 32) {
    const dim3 grid((rows + 3) / 4), block(128);
    e = one ? launch_overlapped(block_norm_kernel<1, true>, grid, block, 0, stream, p) : launch_overlapped(block_norm_kernel<kVec, true>, grid, block, 0, stream, p);
  } else {
    const dim3 grid(rows), block(t);
    e = one ? launch_overlapped(block_norm_kernel<1, false>, grid, block, 0, stream, p) : launch_overlapped(block_norm_kernel<kVec, false>, grid, block, 0, stream, p);
  }
  return static_cast<int>(e);
}
