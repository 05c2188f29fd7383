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
#include <string.h>

#include <algorithm>

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
  int rows, cols, elem, vec;
  unsigned int* counters;
  int num_counters;
};

template <int E, int V, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : kMostThreads, WARP ? 12 : (V <= kVec ? 2 : 1) + (E != kElemF32 ? 1 : 0)) quantize_rows_kernel(const QuantizeParams p) {
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
  auto store = [&](const Raw8<E>& r, int i) {
    float t[8];
    r.get(t);
    store_codes(p.q, to, i, E == kElemF32 ? code.codes(t) : code.codes_short(t));
  };
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (tid * 8 + v * step < p.cols) store(f[v], tid * 8 + v * step);
  for (int i = tid * 8 + V * step; i < p.cols; i += step) {
    Raw8<E> t;
    t.load(x, p.vec != 0, at, i, p.cols);
    store(t, i);
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
  int t = row_threads(p.rows, p.cols, kVec);
  const int pieces = (p.cols + 7) / 8;
  const bool one = pieces <= t, more = pieces > kVec * t;
  if (more) t = row_threads(p.rows, p.cols, 2 * kVec);
  const dim3 grid(t == 32 ? (p.rows + 3) / 4 : p.rows), block(t == 32 ? 128 : t);
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
  int xo_wide;                                 // rows of x_out begin at multiples of 32 bytes
  int stages;                                  // rows in shared memory: this one and the next, or this one
  float eps, x_scale, y_scale;
};

// A matrix that rows are read from, through shared memory: a thread fetches what it will use itself, so that a wait for its own copies is all
// the order there is.
struct RowSource {
  const void* p;
  int elem, vec;
  long long ld;
  OGB_DEVICE int words() const { return p == nullptr ? 0 : elem == kElemF32 ? 2 : 1; }        // 16-byte words a piece
  OGB_DEVICE void fetch(uint4* slot, int threads, int row, int i, int n) const {
    if (vec == 0 || i + 8 > n) return;
    const char* s = static_cast<const char*>(p) + (static_cast<size_t>(row) * ld + i) * (elem == kElemF32 ? 4 : 2);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(slot)), "l"(s) : "memory");
    if (elem == kElemF32) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(slot + threads)), "l"(s + 16) : "memory");
  }
  OGB_DEVICE void get(const uint4* slot, int threads, int row, int i, int n, float (&f)[8]) const {
    if (vec == 0 || i + 8 > n) {           // unaligned rows, and what a row's end leaves of a piece
      load8(p, elem, false, static_cast<size_t>(row) * ld, i, n, f);
      return;
    }
    const uint4 a = slot[0];
    if (elem == kElemF32) {
      const uint4 b = slot[threads];
      const Raw8<kElemF32> r{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
      r.get(f);
    } else if (elem == kElemBf16) {
      const Raw8<kElemBf16> r{{a.x, a.y, a.z, a.w}};
      r.get(f);
    } else {
      const Raw8<kElemF16> r{{a.x, a.y, a.z, a.w}};
      r.get(f);
    }
  }
};

// Blocks an SM holds at least, which bounds the registers: 80 a thread with four pieces, 64 with fewer.
constexpr int norm_blocks(int v, int t) { return 65536 / ((v < kVec ? 64 : 80) * (t == 32 ? 128 : t)); }

// T: most threads of a block, 32: a warp a row.
template <int V, int T>
__global__ void __launch_bounds__(T == 32 ? 128 : T, norm_blocks(V, T)) block_norm_kernel(const BlockNormParams p) {
  __shared__ __align__(16) float part_y[2][kMostThreads / 32], part_x[2][kMostThreads / 32];
  __shared__ __align__(16) uint32_t part_q[2][kMostThreads / 32];
  extern __shared__ __align__(16) uint4 slots[];
  constexpr bool WARP = T == 32;
  pdl_trigger();
  pdl_wait();
  const int threads = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int warps = WARP ? blockDim.x >> 5 : 1, rows_step = gridDim.x * warps;
  const int n = p.cols, step = threads * 8, i0 = tid * 8, all = blockDim.x;
  const float over = 1.f / static_cast<float>(n);
  const RowSource xs{after_wait(p.x), p.x_elem, p.x_vec, p.ldx};
  const RowSource ys{after_wait(p.y), p.y_elem, p.y_vec, p.ldy};
  const bool gate_row = p.gate != nullptr && p.ldg != 0;                      // a gate for all rows stays in cache
  const RowSource gs{gate_row ? after_wait(p.gate) : nullptr, p.gate_elem, p.gate_vec, p.ldg};
  const int wx = xs.words(), wy = ys.words(), wg = gs.words(), words = V * (wx + wy + wg);
  uint4* mine = slots + threadIdx.x;                                          // word w of a stage: mine[w * all]
  auto fetch = [&](int row, int stage) {
    uint4* to = mine + stage * words * all;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = i0 + v * step;
      xs.fetch(to + v * wx * all, all, row, i, n);
      if (wy != 0) ys.fetch(to + (V * wx + v * wy) * all, all, row, i, n);
      if (wg != 0) gs.fetch(to + (V * (wx + wy) + v * wg) * all, all, row, i, n);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int row = blockIdx.x * warps + (WARP ? threadIdx.x >> 5 : 0);
  if (p.stages == 2 && row < p.rows) fetch(row, 0);
  for (int turn = 0; row < p.rows; row += rows_step, turn ^= 1) {
    if (p.stages == 1) fetch(row, 0);
    else if (row + rows_step < p.rows) fetch(row + rows_step, turn ^ 1);
    if (p.stages == 2 && row + rows_step < p.rows) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
    const uint4* from = mine + (p.stages == 2 ? turn * words * all : 0);
    float ry = p.y_scale;
    if (p.post != nullptr) {
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float y[8];
        ys.get(from + (V * wx + v * wy) * all, all, row, i0 + v * step, n, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(y[j], y[j], sum);
      }
      ry *= rsqrtf(row_sum<WARP>(sum, part_y[turn]) * over + p.eps);
    }
    float x[V][8], sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = i0 + v * step;
      xs.get(from + v * wx * all, all, row, i, n, x[v]);
      if (wy != 0) {
        float y[8], t[8];
        ys.get(from + (V * wx + v * wy) * all, all, row, i, n, y);
        if (p.post != nullptr) {
          load8(p.post, p.w_elem, p.post_vec != 0, 0, i, n, t);
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] *= t[j];
        }
        if (p.gate != nullptr) {
          if (wg != 0) gs.get(from + (V * (wx + wy) + v * wg) * all, all, row, i, n, t);
          else load8(p.gate, p.gate_elem, p.gate_vec != 0, 0, i, n, t);
          if (p.gate_sigmoid != 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = __fdividef(y[j], 1.f + __expf(-t[j]));
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] *= t[j];
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[v][j] = fmaf(ry, y[j], p.x_scale * x[v][j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[v][j] *= p.x_scale;
      }
      if (p.x_out != nullptr) store8(p.x_out, p.x_elem, p.xo_vec != 0, static_cast<size_t>(row) * p.ldxo, i, n, x[v]);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(x[v][j], x[v][j], sum);      // past the row's end: zeros
    }
    if (p.h == nullptr && p.q == nullptr) continue;
    if (p.pre != nullptr) {
      const float rx = rsqrtf(row_sum<WARP>(sum, part_x[turn]) * over + p.eps);
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
      const RowCode code(row_max<WARP>(peak, part_q[turn]));
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = i0 + v * step;
        if (i < n) store_codes(p.q, static_cast<size_t>(row) * p.ldq, i, code.codes(x[v]));
      }
      if (tid == 0) p.factor[row] = code.factor;
    }
  }
}

// Eight floats as one store: a whole sector.
OGB_DEVICE void store32(float* to, const float (&f)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]),
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

// The same for the usual types and layouts: rows and weights at multiples of 16 bytes, cols a multiple of eight, a stream of type XE, bf16 from the
// block and to the next one (or 8-bit rows), weights and a gate a channel of type WE.  Weights meet the values before the sum over the row is known,
// so that what follows a sum is one product; the largest |h| is the largest |x' pre| times the root, so it joins the second sum's exchange.
template <int XE, int WE, int V, int T>
__global__ void __launch_bounds__(T == 32 ? 128 : T, norm_blocks(V, T)) block_norm_usual_kernel(const BlockNormParams p) {
  __shared__ __align__(16) float part_y[2][kMostThreads / 32], part_x[2][kMostThreads / 32];
  __shared__ __align__(16) uint32_t part_q[2][kMostThreads / 32];
  extern __shared__ __align__(16) uint4 slots[];
  constexpr bool WARP = T == 32;
  constexpr int kX = XE == kElemF32 ? 2 : 1;                                  // 16-byte words of a piece of the stream
  pdl_trigger();
  pdl_wait();
  const int threads = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int warps = WARP ? blockDim.x >> 5 : 1, rows_step = gridDim.x * warps;
  const int n = p.cols, step = threads * 8, i0 = tid * 8, all = blockDim.x;
  const float over = 1.f / static_cast<float>(n);
  const char *x = static_cast<const char*>(after_wait(p.x)), *y = static_cast<const char*>(after_wait(p.y)), *g = static_cast<const char*>(after_wait(p.gate));
  const bool has_y = y != nullptr, gate_row = g != nullptr && p.ldg != 0;
  const int words = V * (kX + (has_y ? 1 : 0) + (gate_row ? 1 : 0));
  uint4* mine = slots + threadIdx.x;
  const uint32_t base = smem_u32(mine);
  auto copy = [](uint32_t to, const char* s) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(s) : "memory"); };
  auto fetch = [&](int row, int stage) {
    uint32_t to = base + stage * words * all * 16;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (i0 + v * step < n) {
        if (kX == 1) copy(to + v * all * 16, x + (static_cast<size_t>(row) * p.ldx + i0 + v * step) * 2);
        if (has_y) copy(to + (V * kX + v) * all * 16, y + (static_cast<size_t>(row) * p.ldy + i0 + v * step) * 2);
        if (gate_row) copy(to + (V * (kX + 1) + v) * all * 16, g + (static_cast<size_t>(row) * p.ldg + i0 + v * step) * 2);
      }
    }
    if (kX == 2) {
      // A warp's 32 pieces are 64 words.  Lanes copy neighbouring ones, so that no 32-byte sector is asked for twice, and take two each from shared
      // memory, where words trade places in every other eight to keep eight lanes on different banks.
      const int lane = threadIdx.x & 31;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int w = lane + 32 * h, i = (i0 - 8 * lane) + v * step + 4 * w;
          if (i < n)
            copy(base - lane * 16 + (stage * words * all + v * 2 * all + (threadIdx.x - lane) + (w ^ (w >> 3 & 1))) * 16,
                 x + (static_cast<size_t>(row) * p.ldx + i) * 4);
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int row = blockIdx.x * warps + (WARP ? threadIdx.x >> 5 : 0);
  if (p.stages == 2 && row < p.rows) fetch(row, 0);
  for (int turn = 0; row < p.rows; row += rows_step, turn ^= 1) {
    if (kX == 2) __syncwarp();                                                // what the copies overwrite has been read by the whole warp
    if (p.stages == 1) fetch(row, 0);
    else if (row + rows_step < p.rows) fetch(row + rows_step, turn ^ 1);
    if (p.stages == 2 && row + rows_step < p.rows) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (kX == 2) __syncwarp();
    const uint4* from = mine + (p.stages == 2 ? turn * words * all : 0);
    float a[V][8], ry = p.y_scale;
    if (has_y) {
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = i0 + v * step;
        if (i < n) {
          const uint4 raw = from[(V * kX + v) * all];
          Raw8<kElemBf16>{{raw.x, raw.y, raw.z, raw.w}}.get(a[v]);
          float t[8];
          if (p.post != nullptr) {
            Raw8<WE> w;
            w.load(p.post, true, 0, i, n);
            w.get(t);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              sum = fmaf(a[v][j], a[v][j], sum);
              a[v][j] *= t[j];
            }
          }
          if (gate_row) {
            const uint4 graw = from[(V * (kX + 1) + v) * all];
            Raw8<kElemBf16>{{graw.x, graw.y, graw.z, graw.w}}.get(t);
          } else if (g != nullptr) {
            Raw8<WE> w;
            w.load(g, true, 0, i, n);
            w.get(t);
          }
          if (g != nullptr) {
            if (p.gate_sigmoid != 0) {
#pragma unroll
              for (int j = 0; j < 8; ++j) t[j] = sigmoid_approx(t[j]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) a[v][j] *= t[j];
          }
        }
      }
      if (p.post != nullptr) ry *= rsqrtf(row_sum<WARP>(sum, part_y[turn]) * over + p.eps);
    }
    float sum = 0.f;
    uint32_t peak = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = i0 + v * step;
      if (i < n) {
        float t[8];
        if constexpr (kX == 2) {
          const int lane = threadIdx.x & 31, swap = lane >> 2 & 1;
          const uint4* two = from - lane + v * 2 * all + (threadIdx.x - lane) + 2 * lane;
          const uint4 lo = two[swap], hi = two[swap ^ 1];
          Raw8<kElemF32>{{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}}.get(t);
        } else {
          const uint4 raw = from[v * all];
          Raw8<kElemBf16>{{raw.x, raw.y, raw.z, raw.w}}.get(t);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          t[j] *= p.x_scale;
          if (has_y) t[j] = fmaf(ry, a[v][j], t[j]);
          a[v][j] = t[j];
        }
        if (p.x_out != nullptr) {
          if (XE == kElemF32 && p.xo_wide != 0)
            store32(static_cast<float*>(p.x_out) + static_cast<size_t>(row) * p.ldxo + i, a[v]);
          else
            store8(p.x_out, XE, true, static_cast<size_t>(row) * p.ldxo, i, n, a[v]);
        }
        if (p.pre != nullptr) {
          Raw8<WE> w;
          w.load(p.pre, true, 0, i, n);
          w.get(t);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            sum = fmaf(a[v][j], a[v][j], sum);
            a[v][j] *= t[j];
          }
        }
        if (p.q != nullptr) peak = max(peak, peak_bits8(a[v]));
      }
    }
    if (p.h == nullptr && p.q == nullptr) continue;
    float rx = 1.f;
    if (p.q != nullptr) {
      // both at one exchange
      peak = __reduce_max_sync(0xffffffffu, peak);
      if (!WARP && (threadIdx.x & 31) == 0) part_q[turn][threadIdx.x >> 5] = peak;
    }
    if (p.pre != nullptr) rx = rsqrtf(row_sum<WARP>(sum, part_x[turn]) * over + p.eps);
    else if (!WARP && p.q != nullptr) __syncthreads();
    if (p.q != nullptr) {
      if (!WARP)
        for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) peak = max(peak, part_q[turn][w]);
      // infinities and NaN stay above all values; a root that is not a number makes the row one
      const RowCode code(__float_as_uint(__uint_as_float(peak) * rx) & 0x7fffffffu);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = i0 + v * step;
        if (i < n) {
#pragma unroll
          for (int j = 0; j < 8; ++j) a[v][j] *= rx;
          store_codes(p.q, static_cast<size_t>(row) * p.ldq, i, code.codes(a[v]));
        }
      }
      if (tid == 0) p.factor[row] = code.factor;
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = i0 + v * step;
        if (i < n) {
#pragma unroll
          for (int j = 0; j < 8; ++j) a[v][j] *= rx;
          store8(p.h, kElemBf16, true, static_cast<size_t>(row) * p.ldh, i, n, a[v]);
        }
      }
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
  // The next row's copies pass under this row's sums where shared memory holds both rows of as many blocks as registers do; else more blocks do
  // better (8192 rows of 3584, stream in 32 bits with a gate a token: 106 us with three blocks of two rows, 92 with four of one).
  const int most = std::max(1, 65536 / ((V < kVec ? 64 : 80) * block));
  p.stages = (2 * stage + 1024) * most <= kNormSmem ? 2 : 1;
  const int smem = p.stages * stage;
  const int per_sm = std::max(1, std::min(kNormSmem / (smem + 1024), most));
  const int grid = std::min(T == 32 ? (p.rows + 3) / 4 : p.rows, ogb_num_sms() * per_sm);
  return static_cast<int>(launch_overlapped(kernel, dim3(grid), dim3(block), smem, stream, p));
}
template <int V, int T>
static int launch_norm(const BlockNormParams& p, int threads, cudaStream_t stream) {
  static OncePerDevice allowed[5];
  const bool aligned = p.x_vec != 0 && p.y_vec != 0 && p.gate_vec != 0 && p.post_vec != 0 && p.pre_vec != 0 && p.xo_vec != 0 && p.h_vec != 0;
  const bool bf16 = (p.y == nullptr || p.y_elem == kElemBf16) && (p.gate == nullptr || p.gate_elem == (p.ldg != 0 ? kElemBf16 : p.w_elem)) &&
                    (p.h == nullptr || p.h_elem == kElemBf16) && (p.h == nullptr || p.q == nullptr);
  if (aligned && bf16 && p.cols % 8 == 0 && p.x_elem != kElemF16 && p.w_elem != kElemF16) {
    if (p.x_elem == kElemF32)
      return p.w_elem == kElemF32 ? launch_norm_kernel<V, T>(allowed[0], block_norm_usual_kernel<kElemF32, kElemF32, V, T>, p, threads, stream)
                                  : launch_norm_kernel<V, T>(allowed[1], block_norm_usual_kernel<kElemF32, kElemBf16, V, T>, p, threads, stream);
    return p.w_elem == kElemF32 ? launch_norm_kernel<V, T>(allowed[2], block_norm_usual_kernel<kElemBf16, kElemF32, V, T>, p, threads, stream)
                                : launch_norm_kernel<V, T>(allowed[3], block_norm_usual_kernel<kElemBf16, kElemBf16, V, T>, p, threads, stream);
  }
  return launch_norm_kernel<V, T>(allowed[4], block_norm_kernel<V, T>, p, threads, stream);
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
                    gate_sigmoid, (reinterpret_cast<uintptr_t>(x_out) & 31) == 0 && ldxo % 8 == 0 ? 1 : 0, 2, eps, x_scale, y_scale};
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int t = row_threads(rows, cols, 2), pieces = (cols + 7) / 8;
  if (t == 32) return launch_norm<2, 32>(p, t, stream);
  if (pieces <= t) return launch_norm<1, kMostThreads>(p, t, stream);
  return pieces <= 2 * t ? launch_norm<2, kMostThreads>(p, t, stream) : launch_norm<kVec, kMostThreads>(p, t, stream);
}

// The same call with its arguments as 64-bit words, floating ones as doubles: see ogb_gemm_int8_args.
extern "C" int ogb_block_norm_args(const int64_t* a) {
  auto p = [&](int i) { return reinterpret_cast<void*>(a[i]); };
  auto n = [&](int i) { return static_cast<int>(a[i]); };
  auto f = [&](int i) { double d; memcpy(&d, a + i, 8); return static_cast<float>(d); };
  return ogb_block_norm(p(0), p(1), p(2), p(3), p(4), p(5), p(6), p(7), static_cast<float*>(p(8)), a[9], a[10], a[11], a[12], a[13], a[14], n(15), n(16), n(17),
                        n(18), n(19), n(20), n(21), n(22), f(23), f(24), f(25), p(26));
}
