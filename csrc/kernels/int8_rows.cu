// Rows in 8-bit integers (int8_rows.cuh), by themselves and from the norms around a decoder's block:
//
//   x' = a x + b g post(y)      post, pre: RMS norms with a weight, or nothing
//   h  = pre(x')                g: nothing, one value a channel, one a token and channel (or the sigmoid of it)
//
// x is the residual stream, y what a block wrote, h what the next one reads: in a float type, or as 8-bit rows for a product.  All of it in
// 32 bits from the loads to one rounding at each store; h is taken from x' before x' is rounded to the stream's type.
//
// Both are bound by the bytes they move, and by the chain load - sums over the row - store where rows are few.  A row belongs to a block (short ones of
// many to a warp) and stays in registers from its load to its last store, so nothing is read twice.  Rows up to two an SM take one piece of eight
// values a thread, which makes the chain short; many rows take two or four, whose loads overlap.  The norm's next row comes through shared memory
// while this one is summed and stored: 8192 rows of 3584 with a 32-bit stream, bf16 y, gate and h take 74 us, 5.6 TB/s of a copy's 6.45 (with a
// row's loads behind the stores of the one before 82, with two whole rows in shared memory, and so fewer blocks, 106).
// To 8 bits they take 70 with the 32-bit stream and 64 with one in bf16 (to bf16 68 and 47).  Rows alone, 8192 x 18944: bf16 97, 4.8 TB/s; fp32, whose codes
// look for values near a half, 195, 4.0 TB/s.
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "int8_rows.cuh"
#include "ogb_kernels.h"

namespace ogb {

constexpr int kVec = 4;            // pieces of eight values that a thread keeps
constexpr int kMostThreads = 512;
constexpr int kNormMaxCols = kVec * 8 * kMostThreads;
constexpr int kNormSmem = 225 * 1024;

// Sum (or largest) of v over the threads of a row: a warp of its own, or the block.  `part`: a word per warp, used by one call only.
template <bool WARP>
OGB_DEVICE float row_sum(float v, float* part) {
  v = warp_sum(v);
  if (WARP) return v;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  v = 0.f;
  for (int i = 0; i < warps; i += 4) {
    const float4 t = *reinterpret_cast<const float4*>(part + i);
    v += t.x + (i + 1 < warps ? t.y : 0.f) + ((i + 2 < warps ? t.z : 0.f) + (i + 3 < warps ? t.w : 0.f));
  }
  return v;
}
template <bool WARP>
OGB_DEVICE uint32_t row_max(uint32_t v, uint32_t* part) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (WARP) return v;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  v = 0;
  for (int i = 0; i < warps; i += 4) {
    const uint4 t = *reinterpret_cast<const uint4*>(part + i);
    v = max(max(v, t.x), max(i + 1 < warps ? t.y : 0u, max(i + 2 < warps ? t.z : 0u, i + 3 < warps ? t.w : 0u)));
  }
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
  int rows, cols, elem, shifted;               // shifted: rows do not all begin at multiples of eight values
  unsigned int* counters;
  int num_counters;
};

template <int E, int V, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : kMostThreads, WARP ? 12 : (V <= kVec ? 2 : 1) + (E != kElemF32 ? 1 : 0)) quantize_rows_kernel(const QuantizeParams p) {
  __shared__ __align__(16) uint32_t part[kMostThreads / 32];
  extern __shared__ __align__(16) uint2 exchange[];             // codes of every piece and of one behind them, where rows are shifted
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < p.num_counters; i += blockDim.x) p.counters[i] = 0;
  const int threads = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int row = WARP ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= p.rows) return;
  const void* x = after_wait(p.x);
  const size_t at = static_cast<size_t>(row) * p.ldx, to = static_cast<size_t>(row) * p.ldq;
  const int step = threads * 8, shift = row_shift(row, p.ldx), i0 = tid * 8 - shift;
  Raw8<E> f[V];
  uint32_t peak = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) f[v].load(x, at, i0 + v * step, p.cols);
#pragma unroll
  for (int v = 0; v < V; ++v) peak = f[v].peak(peak);
  const RowCode code(row_max<WARP>(Raw8<E>::peak_float(peak), part));
  if (tid == 0) p.factor[row] = code.factor;
  uint2 codes[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float t[8];
    f[v].get(t);
    codes[v] = E == kElemF32 ? code.codes(t) : code.codes_short(t);
  }
  if (p.shifted == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (i0 + v * step < p.cols) store_codes(p.q, to, i0 + v * step, codes[v]);
    return;
  }
  uint2* mine = exchange + (WARP ? (threadIdx.x >> 5) * (32 * V + 1) : 0);
#pragma unroll
  for (int v = 0; v < V; ++v) mine[tid + v * threads] = codes[v];
  if (tid == 0) mine[V * threads] = make_uint2(0, 0);
  if (WARP) __syncwarp();
  else __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (tid * 8 + v * step < p.cols) store_codes(p.q, to, tid * 8 + v * step, shift_codes(codes[v], mine[tid + v * threads + 1], shift));
}

// Rows of any length and alignment.
template <int V, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : kMostThreads, WARP ? 8 : 2) quantize_any_rows_kernel(const QuantizeParams p) {
  __shared__ __align__(16) uint32_t part[kMostThreads / 32];
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < p.num_counters; i += blockDim.x) p.counters[i] = 0;
  const int threads = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int row = WARP ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= p.rows) return;
  const void* x = after_wait(p.x);
  const size_t at = static_cast<size_t>(row) * p.ldx, to = static_cast<size_t>(row) * p.ldq;
  float f[V][8];
  uint32_t peak = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) load_strided(x, p.elem, at, tid + v * 8 * threads, threads, p.cols, f[v]);
#pragma unroll
  for (int v = 0; v < V; ++v) peak = max(peak, peak_bits8(f[v]));
  // longer rows than the registers hold are read again below
  for (int i = tid + V * 8 * threads; i < p.cols; i += 8 * threads) {
    float t[8];
    load_strided(x, p.elem, at, i, threads, p.cols, t);
    peak = max(peak, peak_bits8(t));
  }
  const RowCode code(row_max<WARP>(peak, part));
  auto codes = [&](const float (&t)[8]) { return p.elem == kElemF32 ? code.codes(t) : code.codes_short(t); };
#pragma unroll
  for (int v = 0; v < V; ++v) store_codes_strided(p.q, to, tid + v * 8 * threads, threads, p.cols, codes(f[v]));
  for (int i = tid + V * 8 * threads; i < p.cols; i += 8 * threads) {
    float t[8];
    load_strided(x, p.elem, at, i, threads, p.cols, t);
    store_codes_strided(p.q, to, i, threads, p.cols, codes(t));
  }
  if (tid == 0) p.factor[row] = code.factor;
}

// Threads for a row of `cols` values, `most` pieces of eight each where rows are many: 32 (a warp, four rows a block) or a block of them.
static int row_threads(int rows, int cols, int most) {
  const int pieces = (cols + 7) / 8;
  const int per = rows <= 2 * ogb_num_sms() ? 1 : most;
  return std::min(kMostThreads, ((pieces + per - 1) / per + 31) / 32 * 32);
}

template <int E>
static int launch_quantize(const QuantizeParams& p, cudaStream_t stream) {
  const int cols = p.cols + (p.shifted != 0 ? 7 : 0), pieces = (cols + 7) / 8;
  int t = row_threads(p.rows, cols, kVec);
  const bool one = pieces <= t, more = pieces > kVec * t;
  if (more) t = row_threads(p.rows, cols, 2 * kVec);
  const int v = t == 32 ? (one ? 1 : kVec) : one ? 1 : more ? 2 * kVec : kVec;
  const dim3 grid(t == 32 ? (p.rows + 3) / 4 : p.rows), block(t == 32 ? 128 : t);
  const int smem = p.shifted != 0 ? 8 * (t == 32 ? 4 * (32 * v + 1) : v * t + 1) : 0;
  auto kernel = t == 32 ? (one ? quantize_rows_kernel<E, 1, true> : quantize_rows_kernel<E, kVec, true>)
                        : (one ? quantize_rows_kernel<E, 1, false> : more ? quantize_rows_kernel<E, 2 * kVec, false> : quantize_rows_kernel<E, kVec, false>);
  return static_cast<int>(launch_overlapped(kernel, grid, block, smem, stream, p));
}

int launch_quantize_rows(const void* x, int8_t* q, float* factor, int rows, int cols, long long ldx, long long ldq, int elem, unsigned int* counters,
                         int num_counters, cudaStream_t stream) {
  const QuantizeParams p{x, q, factor, ldx, ldq, rows, cols, elem, ldx % 8 != 0 ? 1 : 0, counters, num_counters};
  // rows that stay in registers, and a matrix that begins at a multiple of eight values
  if (!starts_aligned(x, elem) || cols + 7 > 2 * kVec * 8 * kMostThreads) {
    const int t = row_threads(rows, cols, 2);
    const dim3 grid(t == 32 ? (rows + 3) / 4 : rows), block(t == 32 ? 128 : t);
    auto kernel = t == 32 ? quantize_any_rows_kernel<2, true> : (cols <= 8 * t ? quantize_any_rows_kernel<1, false> : quantize_any_rows_kernel<2, false>);
    return static_cast<int>(launch_overlapped(kernel, grid, block, 0, stream, p));
  }
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
  int gate_sigmoid;
  int shifted;                                 // rows do not all begin at multiples of eight values
  float eps, x_scale, y_scale;
};

// Blocks an SM holds at least, which bounds the registers: 80 a thread with four pieces, 64 with fewer.
constexpr int norm_blocks(int v, int t) { return 65536 / ((v < kVec ? 64 : 80) * (t == 32 ? 128 : t)); }

// Any types, sizes and alignments.  T: most threads of a block, 32: a warp a row.
template <int V, int T>
__global__ void __launch_bounds__(T == 32 ? 128 : T, V < kVec ? norm_blocks(V, T) : 1) block_norm_kernel(const BlockNormParams p) {
  __shared__ __align__(16) float part_y[2][kMostThreads / 32], part_x[2][kMostThreads / 32];
  __shared__ __align__(16) uint32_t part_q[2][kMostThreads / 32];
  constexpr bool WARP = T == 32;
  constexpr int N = 8 * V;
  pdl_trigger();
  pdl_wait();
  const int step = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int warps = WARP ? blockDim.x >> 5 : 1, rows_step = gridDim.x * warps;
  const int n = p.cols;
  const float over = 1.f / static_cast<float>(n);
  const void *xp = after_wait(p.x), *yp = after_wait(p.y), *gp = after_wait(p.gate);
  int turn = 0;
  for (int row = blockIdx.x * warps + (WARP ? threadIdx.x >> 5 : 0); row < p.rows; row += rows_step, turn ^= 1) {
    float x[N], t[N];
    load_strided(xp, p.x_elem, static_cast<size_t>(row) * p.ldx, tid, step, n, x);
    if (yp != nullptr) {
      float y[N], ry = p.y_scale, sum = 0.f;
      load_strided(yp, p.y_elem, static_cast<size_t>(row) * p.ldy, tid, step, n, y);
      if (gp != nullptr) load_strided(gp, p.gate_elem, static_cast<size_t>(row) * p.ldg, tid, step, n, t);
      if (p.post != nullptr) {
#pragma unroll
        for (int j = 0; j < N; ++j) sum = fmaf(y[j], y[j], sum);
      }
      if (gp != nullptr) {
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] *= p.gate_sigmoid != 0 ? __fdividef(1.f, 1.f + __expf(-t[j])) : t[j];
      }
      if (p.post != nullptr) {
        load_strided(p.post, p.w_elem, 0, tid, step, n, t);
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] *= t[j];
        ry *= rsqrtf(row_sum<WARP>(sum, part_y[turn]) * over + p.eps);
      }
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = fmaf(ry, y[j], p.x_scale * x[j]);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] *= p.x_scale;
    }
    if (p.x_out != nullptr) store_strided(p.x_out, p.x_elem, static_cast<size_t>(row) * p.ldxo, tid, step, n, x);
    if (p.h == nullptr && p.q == nullptr) continue;
    if (p.pre != nullptr) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j) sum = fmaf(x[j], x[j], sum);      // past the row's end: zeros
      load_strided(p.pre, p.w_elem, 0, tid, step, n, t);
      const float rx = rsqrtf(row_sum<WARP>(sum, part_x[turn]) * over + p.eps);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] *= rx * t[j];
    }
    if (p.h != nullptr) store_strided(p.h, p.h_elem, static_cast<size_t>(row) * p.ldh, tid, step, n, x);
    if (p.q != nullptr) {
      uint32_t peak = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) peak = max(peak, __float_as_uint(x[j]) & 0x7fffffffu);
      const RowCode code(row_max<WARP>(peak, part_q[turn]));
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = x[8 * v + j];
        store_codes_strided(p.q, static_cast<size_t>(row) * p.ldq, tid + v * 8 * step, step, n, code.codes(f));
      }
      if (tid == 0) p.factor[row] = code.factor;
    }
  }
}

// Eight floats as one store: a whole sector.
OGB_DEVICE void store32(float* to, const float (&f)[8]) {
  asm volatile("st.global.L1::no_allocate.L2::evict_first.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]),
               "f"(f[6]), "f"(f[7])
               : "memory");
}
// 1 / (1 + exp(-g)), off by a few 2^-23
OGB_DEVICE float sigmoid_approx(float g) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}

// Eight weights from column i on, wherever that is.
template <bool SHIFT>
OGB_DEVICE void load_weights(const void* p, int elem, int i, int n, float (&t)[8]) {
  if (SHIFT && (i & 7) != 0) {                                                          // rows that are shifted against them
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = i + j >= 0 && i + j < n ? load_elem(p, elem, i + j) : 0.f;
  } else if (elem == kElemF32) {
    Raw8<kElemF32> w;
    w.load(p, 0, i, n);
    w.get(t);
  } else if (elem == kElemBf16) {
    Raw8<kElemBf16> w;
    w.load(p, 0, i, n);
    w.get(t);
  } else {
    Raw8<kElemF16> w;
    w.load(p, 0, i, n);
    w.get(t);
  }
}
// Eight results from column i on, one by one at the ends of a row.
template <int E, bool SHIFT>
OGB_DEVICE void store_piece(void* p, size_t row, int i, int n, const float (&f)[8]) {
  if ((!SHIFT || i >= 0) && i + 8 <= n) {
    if (E == kElemF32) store32(static_cast<float*>(p) + row + i, f);
    else store8(p, E, true, row, i, n, f);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if ((!SHIFT || i + j >= 0) && i + j < n) store_elem(p, E, row + i + j, f[j]);
}

// The same for matrices that begin at multiples of eight values and share a row stride modulo eight (contiguous ones do): every row is taken in pieces of
// eight values that lie at such multiples in all of them.  XE: type of the stream, YE: of the block's output, a gate a token and h.  Weights meet the values
// before the sum over the row is known, so that what follows a sum is one product; the largest |h| is the largest |x' pre| times the root, so it joins the
// second sum's exchange.  A warp's pieces come through shared memory by copies of its own: those of the next row's y and gate start once this row's have been
// read, those of its stream once x' is formed, so that loads pass under the sums and stores.  SHIFT: rows do not all begin at multiples of
// eight values (8192 x 3583: 113 us; where they do, 3584: 74).
template <int XE, int YE, int V, int T, bool SHIFT>
__global__ void __launch_bounds__(T == 32 ? 128 : T, norm_blocks(V, T)) block_norm_usual_kernel(const BlockNormParams p) {
  __shared__ __align__(16) float part_y[2][kMostThreads / 32], part_x[2][kMostThreads / 32];
  __shared__ __align__(16) uint32_t part_q[2][kMostThreads / 32];
  extern __shared__ __align__(16) uint4 slots[];
  constexpr bool WARP = T == 32;
  constexpr int kX = XE == kElemF32 ? 2 : 1, kY = YE == kElemF32 ? 2 : 1;     // 16-byte words of a piece
  constexpr int kXBytes = XE == kElemF32 ? 4 : 2, kYBytes = YE == kElemF32 ? 4 : 2;
  pdl_trigger();
  pdl_wait();
  const int threads = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x, lane = threadIdx.x & 31;
  const int warps = WARP ? blockDim.x >> 5 : 1, rows_step = gridDim.x * warps;
  const int n = p.cols, step = threads * 8, all = blockDim.x;
  const float over = 1.f / static_cast<float>(n);
  const char *x = static_cast<const char*>(after_wait(p.x)), *y = static_cast<const char*>(after_wait(p.y)), *g = static_cast<const char*>(after_wait(p.gate));
  const bool has_y = y != nullptr, gate_row = g != nullptr && p.ldg != 0;
  const int words = V * (kX + (has_y ? kY : 0) + (gate_row ? kY : 0));
  uint4* mine = slots + threadIdx.x - lane;                                    // the warp's words
  const uint32_t base = smem_u32(mine);
  // (read once: first to leave L2)
  uint64_t once;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
  auto copy = [&](uint32_t to, const char* s) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(to), "l"(s), "l"(once) : "memory");
  };
  // A warp's 32 pieces of a matrix: 32 words, or of 32-bit values 64.  Lanes copy neighbouring words, so that no 32-byte sector is asked for twice, and
  // take two each from shared memory, where words trade places in every other eight to keep eight lanes on different banks.
  auto fetch_matrix = [&](auto bytes, uint32_t to, const char* s, size_t at, int shift) {
    constexpr int kBytes = decltype(bytes)::value, kW = kBytes / 2;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int h = 0; h < kW; ++h) {
        const int w = lane + 32 * h, piece = (tid - lane) * 8 + v * step - shift + 8 * (w / kW);
        if ((!SHIFT || piece >= 0) && piece + 8 <= n)
          copy(to + (v * kW * all + (kW == 2 ? w ^ (w >> 3 & 1) : w)) * 16, s + (at + piece) * kBytes + (w % kW) * 16);
      }
  };
  using XBytes = std::integral_constant<int, kXBytes>;
  using YBytes = std::integral_constant<int, kYBytes>;
  // (a warp's 64 words lie next to one another, a block's two sets of 32 a thread apart: every warp's begin at twice its first thread's)
  auto fetch_x = [&](int row) {
    fetch_matrix(XBytes(), base + (kX == 2 ? (threadIdx.x - lane) * 16 : 0), x, static_cast<size_t>(row) * p.ldx, SHIFT ? row_shift(row, p.ldx) : 0);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto fetch_y = [&](int row) {
    const int shift = SHIFT ? row_shift(row, p.ldx) : 0;
    const uint32_t to = base + V * kX * all * 16 + (kY == 2 ? (threadIdx.x - lane) * 16 : 0);
    if (has_y) fetch_matrix(YBytes(), to, y, static_cast<size_t>(row) * p.ldy, shift);
    if (gate_row) fetch_matrix(YBytes(), to + V * kY * all * 16, g, static_cast<size_t>(row) * p.ldg, shift);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // piece v of a matrix whose words begin at `from` of this warp's
  auto get = [&](auto elem, const uint4* from, int v, const char* s, size_t at, int i, float (&t)[8]) {
    constexpr int E = decltype(elem)::value;
    Raw8<E> r;
    if ((SHIFT && i < 0) || i + 8 > n) {
      r.edge(s, at, i, n);
    } else if constexpr (E == kElemF32) {
      const uint4* two = from + (threadIdx.x - lane) + v * 2 * all + 2 * lane;
      const int swap = lane >> 2 & 1;
      const uint4 lo = two[swap], hi = two[swap ^ 1];
      r = Raw8<E>{{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}};
    } else {
      const uint4 raw = from[v * all + lane];
      r = Raw8<E>{{raw.x, raw.y, raw.z, raw.w}};
    }
    r.get(t);
  };
  using XElem = std::integral_constant<int, XE>;
  using YElem = std::integral_constant<int, YE>;
  int row = blockIdx.x * warps + (WARP ? threadIdx.x >> 5 : 0);
  if (row < p.rows) {
    fetch_y(row);
    fetch_x(row);
  }
  for (int turn = 0; row < p.rows; row += rows_step, turn ^= 1) {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    const int i0 = tid * 8 - (SHIFT ? row_shift(row, p.ldx) : 0);
    float a[V][8], ry = p.y_scale;
    if (has_y) {
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = i0 + v * step;
        if (i < n) {
          float t[8];
          get(YElem(), mine + V * kX * all, v, y, static_cast<size_t>(row) * p.ldy, i, a[v]);
          if (p.post != nullptr) {
            load_weights<SHIFT>(p.post, p.w_elem, i, n, t);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              sum = fmaf(a[v][j], a[v][j], sum);
              a[v][j] *= t[j];
            }
          }
          if (g != nullptr) {
            if (gate_row) get(YElem(), mine + V * (kX + kY) * all, v, g, static_cast<size_t>(row) * p.ldg, i, t);
            else load_weights<SHIFT>(g, p.gate_elem, i, n, t);
            if (p.gate_sigmoid != 0) {
#pragma unroll
              for (int j = 0; j < 8; ++j) t[j] = sigmoid_approx(t[j]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) a[v][j] *= t[j];
          }
        }
      }
      __syncwarp();                                                           // the whole warp has read what the copies overwrite
      if (row + rows_step < p.rows) fetch_y(row + rows_step);
      else asm volatile("cp.async.commit_group;" ::: "memory");
      if (p.post != nullptr) ry *= rsqrtf(row_sum<WARP>(sum, part_y[turn]) * over + p.eps);
    } else {
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    float sum = 0.f;
    uint32_t peak = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = i0 + v * step;
      if (i < n) {
        float t[8];
        get(XElem(), mine, v, x, static_cast<size_t>(row) * p.ldx, i, t);      // zeros in front of a row and past its end, and so is x'
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          t[j] *= p.x_scale;
          if (has_y) t[j] = fmaf(ry, a[v][j], t[j]);
          a[v][j] = t[j];
        }
        if (p.x_out != nullptr) store_piece<XE, SHIFT>(p.x_out, static_cast<size_t>(row) * p.ldxo, i, n, a[v]);
        if (p.pre != nullptr) {
          load_weights<SHIFT>(p.pre, p.w_elem, i, n, t);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            sum = fmaf(a[v][j], a[v][j], sum);
            a[v][j] *= t[j];
          }
        }
        if (p.q != nullptr) peak = max(peak, peak_bits8(a[v]));
      }
    }
    __syncwarp();
    if (row + rows_step < p.rows) fetch_x(row + rows_step);
    if (p.h == nullptr && p.q == nullptr) continue;
    float rx = 1.f;
    if (p.q != nullptr) {
      // both at one exchange
      peak = __reduce_max_sync(0xffffffffu, peak);
      if (!WARP && lane == 0) part_q[turn][threadIdx.x >> 5] = peak;
    }
    if (p.pre != nullptr) rx = rsqrtf(row_sum<WARP>(sum, part_x[turn]) * over + p.eps);
    else if (!WARP && p.q != nullptr) __syncthreads();
    if (p.q == nullptr) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = i0 + v * step;
        if (i < n) {
#pragma unroll
          for (int j = 0; j < 8; ++j) a[v][j] *= rx;
          store_piece<YE, SHIFT>(p.h, static_cast<size_t>(row) * p.ldh, i, n, a[v]);
        }
      }
      continue;
    }
    if (!WARP)
      for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) peak = max(peak, part_q[turn][w]);
    // infinities and NaN stay above all values; a root that is not a number makes the row one
    const RowCode code(__float_as_uint(__uint_as_float(peak) * rx) & 0x7fffffffu);
    if (tid == 0) p.factor[row] = code.factor;
    uint2 codes[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      codes[v] = make_uint2(0, 0);
      if (i0 + v * step < n) {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[v][j] *= rx;
        codes[v] = code.codes(a[v]);
        if (!SHIFT) store_codes(p.q, static_cast<size_t>(row) * p.ldq, i0 + v * step, codes[v]);
      }
    }
    if (SHIFT) {
      // a word of q is made of two pieces: the next one is the next thread's
      uint2* exchange = reinterpret_cast<uint2*>(slots + words * all) + (WARP ? (threadIdx.x >> 5) * (32 * V + 1) : 0);
      if (WARP) __syncwarp();
      else __syncthreads();                                                   // of the row before
#pragma unroll
      for (int v = 0; v < V; ++v) exchange[tid + v * threads] = codes[v];
      if (tid == 0) exchange[V * threads] = make_uint2(0, 0);
      if (WARP) __syncwarp();
      else __syncthreads();
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (tid * 8 + v * step < n)
          store_codes(p.q, static_cast<size_t>(row) * p.ldq, tid * 8 + v * step, shift_codes(codes[v], exchange[tid + v * threads + 1], row_shift(row, p.ldx)));
    }
  }
}

// Launches `kernel` with rows of `threads` threads, V pieces each.
template <int V, int T, typename Kernel>
static int launch_norm_kernel(OncePerDevice& allowed, Kernel kernel, BlockNormParams p, int threads, cudaStream_t stream) {
  const int rc = allow_smem(allowed, kernel, kNormSmem);
  if (rc != 0) return rc;
  auto words = [](const void* m, int elem) { return m == nullptr ? 0 : elem == kElemF32 ? 2 : 1; };
  const int block = T == 32 ? 128 : threads;
  const int stage = 16 * block * V * (words(p.x, p.x_elem) + words(p.y, p.y_elem) + (p.ldg != 0 ? words(p.gate, p.gate_elem) : 0));
  // as many blocks as registers hold: the compiler's 56 a thread with up to two pieces are fewer than the kernel's bound
  const int most = std::max(1, 65536 / ((V < kVec ? 56 : 80) * block));
  const int exchange = p.q != nullptr && p.shifted != 0 ? (8 * (T == 32 ? 4 * (32 * V + 1) : V * block + 1) + 15) / 16 * 16 : 0;
  const int smem = stage + exchange;
  const int per_sm = std::max(1, std::min(kNormSmem / (smem + 1024), most));
  const int grid = std::min(T == 32 ? (p.rows + 3) / 4 : p.rows, ogb_num_sms() * per_sm);
  return static_cast<int>(launch_overlapped(kernel, dim3(grid), dim3(block), smem, stream, p));
}
template <int V, int T, bool SHIFT>
static int launch_usual(const BlockNormParams& p, int threads, cudaStream_t stream) {
  static OncePerDevice allowed[6];
#define OGB_NORM(AT, XE, YE) return launch_norm_kernel<V, T>(allowed[AT], block_norm_usual_kernel<XE, YE, V, T, SHIFT>, p, threads, stream)
  if (p.x_elem == kElemF32) {
    if (p.y_elem == kElemF32) OGB_NORM(0, kElemF32, kElemF32);
    if (p.y_elem == kElemBf16) OGB_NORM(1, kElemF32, kElemBf16);
    OGB_NORM(2, kElemF32, kElemF16);
  }
  if (p.y_elem == kElemF32) OGB_NORM(3, kElemBf16, kElemF32);
  if (p.y_elem == kElemBf16) OGB_NORM(4, kElemBf16, kElemBf16);
  OGB_NORM(5, kElemBf16, kElemF16);
#undef OGB_NORM
}
template <int V, int T>
static int launch_any(const BlockNormParams& p, int threads, cudaStream_t stream) {
  const int block = T == 32 ? 128 : threads;
  const int per_sm = V < kVec ? std::max(1, 65536 / (64 * block)) : std::max(1, 65536 / (128 * block));
  const int grid = std::min(T == 32 ? (p.rows + 3) / 4 : p.rows, ogb_num_sms() * per_sm);
  return static_cast<int>(launch_overlapped(block_norm_kernel<V, T>, dim3(grid), dim3(block), 0, stream, p));
}
static int launch_norm(BlockNormParams p, cudaStream_t stream) {
  // a type for the block's side of it: of what there is of its output, a gate a token and h
  int side = p.y != nullptr ? p.y_elem : p.h != nullptr ? p.h_elem : kElemBf16;
  auto goes = [&](const void* m, long long ld, int elem, int type) { return m == nullptr || (elem == type && starts_aligned(m, elem) && (ld - p.ldx) % 8 == 0); };
  auto vector = [](const void* m) { return (reinterpret_cast<uintptr_t>(m) & 15) == 0; };
  const bool usual = p.x_elem != kElemF16 && goes(p.x, p.ldx, p.x_elem, p.x_elem) && goes(p.x_out, p.ldxo, p.x_elem, p.x_elem) && goes(p.y, p.ldy, p.y_elem, side) &&
                     goes(p.h, p.ldh, p.h_elem, side) && (p.gate == nullptr || p.ldg == 0 || goes(p.gate, p.ldg, p.gate_elem, side)) && vector(p.post) &&
                     vector(p.pre) && (p.ldg != 0 || vector(p.gate)) && !(p.h != nullptr && p.q != nullptr) && p.cols + 7 <= kNormMaxCols;
  if (!usual) {
    const int t = row_threads(p.rows, p.cols, 2), pieces = (p.cols + 7) / 8;
    if (t == 32) return launch_any<2, 32>(p, t, stream);
    if (pieces <= t) return launch_any<1, kMostThreads>(p, t, stream);
    return pieces <= 2 * t ? launch_any<2, kMostThreads>(p, t, stream) : launch_any<kVec, kMostThreads>(p, t, stream);
  }
  p.y_elem = side;
  p.shifted = p.ldx % 8 != 0 ? 1 : 0;
  const int cols = p.cols + (p.shifted != 0 ? 7 : 0), t = row_threads(p.rows, cols, 2), pieces = (cols + 7) / 8;
  auto launch = [&](auto shifted) {
    constexpr bool S = decltype(shifted)::value;
    if (t == 32) return launch_usual<2, 32, S>(p, t, stream);
    if (pieces <= t) return launch_usual<1, kMostThreads, S>(p, t, stream);
    return pieces <= 2 * t ? launch_usual<2, kMostThreads, S>(p, t, stream) : launch_usual<kVec, kMostThreads, S>(p, t, stream);
  };
  return p.shifted != 0 ? launch(std::true_type()) : launch(std::false_type());
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
  const BlockNormParams p{x, y, gate, post, pre, x_out, h, static_cast<int8_t*>(q), factor, ldx, ldy, ldg, ldxo, ldh, ldq, rows, cols, x_elem, y_elem, gate_elem,
                          w_elem, h_elem, gate_sigmoid, 0, eps, x_scale, y_scale};
  return launch_norm(p, static_cast<cudaStream_t>(stream_));
}

// The same call with its arguments as 64-bit words, floating ones as doubles: see ogb_gemm_int8_args.
extern "C" int ogb_block_norm_args(const int64_t* a) {
  auto p = [&](int i) { return reinterpret_cast<void*>(a[i]); };
  auto n = [&](int i) { return static_cast<int>(a[i]); };
  auto f = [&](int i) { double d; memcpy(&d, a + i, 8); return static_cast<float>(d); };
  return ogb_block_norm(p(0), p(1), p(2), p(3), p(4), p(5), p(6), p(7), static_cast<float*>(p(8)), a[9], a[10], a[11], a[12], a[13], a[14], n(15), n(16), n(17),
                        n(18), n(19), n(20), n(21), n(22), f(23), f(24), f(25), p(26));
}
