// Log probability of a given token per row of logits, the entropy of the row, how many tokens are more likely, and the `top` likeliest.
//
//   m = max x,  s = sum exp(x - m),  t = sum exp(x - m) (x - m)
//   log p(i) = x_i - m - log s,   entropy = log s - t / s,   rank = |{j : x_j > x_token}|
//
// One pass over the row: every thread carries (m, s, t) of its values, m being a value near their maximum, and rescales them when one turns up that
// is 2 above it.  The states of threads, warps and CTAs join by the same rule.  What bounds it is the stream of logits from HBM (2 bytes
// a value), with exp(x - m) -- one a value, 16 a clock and SM -- and the issue of instructions close behind: differences, products and sums
// go two values at a time, maxima and comparisons of 16-bit logits too.
//
// The likeliest values come from the same pass.  A value's key is its order as a whole number above its inverted index, so that no two are equal and
// ties go to the lower index.  Threads leave the maximum of every 32-byte piece of the row in shared memory; the top-th best of their own best is a bound
// that at least `top` values reach, and then only pieces whose maximum reaches it are read again, about as many as `top`.  A row on which
// many do (the largest values all in the columns of few threads) has its pieces taken in rounds, each of which keeps the best `top` and raises the
// bound; among the threads of a round the bound of their best keys holds again, so it adds at most top * kPer keys: such rows cost
// time, never space.
//
// A row is split over a cluster of CTAs where rows are few; the parts join over distributed shared memory.
//
// Measured, bf16: 3500 rows of 152064 170 us (6.2 TB/s), with entropies 192, with these and the 20 likeliest 239; 256 rows 21 and 30; one row 8.
//
// Logits may be minus infinity (masked): they weigh nothing.  A row of them has NaN for log probability and entropy, as a row that holds a NaN
// or plus infinity has; among the likeliest NaN comes last.
#include <cooperative_groups.h>
#include <stdint.h>

#include "common.cuh"
#include "int8_rows.cuh"
#include "ogb_kernels.h"

namespace ogb {

namespace cg = cooperative_groups;

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpMaxTop = 32;
constexpr int kLpMaxSplit = 8;             // the portable cluster size
constexpr int kLpSmem = 200 * 1024;        // maxima of a CTA's pieces, at most
constexpr int kLpQuick = 64;               // pieces that are read again at once, at most
constexpr float kLpSlack = 2.f;

struct LogprobsParams {
  const void* logits;
  const int* tokens;
  float *logprob, *entropy, *top_logprob;
  int *rank, *top_ids;
  long long ld;
  int rows, vocab, top, splits;
  int* status;
};

struct LpState {
  float m, s, t;
};
OGB_DEVICE LpState lp_join(const LpState& a, const LpState& b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return LpState{m, a.s + b.s, a.t + b.t};   // nothing yet: zeros, or the NaN of a value
  const float da = a.m - m, db = b.m - m;                          // zero or below; minus infinity for a part without weight
  const float ra = __expf(da), rb = __expf(db);
  return LpState{m, ra * a.s + rb * b.s, ra * fmaf(fmaxf(da, -1000.f), a.s, a.t) + rb * fmaf(fmaxf(db, -1000.f), b.s, b.t)};
}

// Order of values as whole numbers; both zeros alike, NaN below all.
OGB_DEVICE unsigned long long lp_key(float x, int index) {
  const uint32_t b = __float_as_uint(x + 0.f);
  const uint32_t o = (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
  return static_cast<unsigned long long>(x == x ? o : 0u) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}
OGB_DEVICE int lp_index(unsigned long long key) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key)); }
OGB_DEVICE float lp_value(unsigned long long key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  if (o == 0) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((o & 0x80000000u) != 0 ? o & 0x7fffffffu : ~o);
}

OGB_DEVICE float ex2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Logits of a type: 32 bytes of them in eight words.
template <typename T>
struct LpType;
template <>
struct LpType<float> {
  static constexpr int kPer = 8, kElem = kElemF32;
  using Max = float;                                       // as a piece's maximum is kept
  OGB_DEVICE static float max_of(const uint32_t (&w)[8]) {
    float m = __uint_as_float(w[0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) m = fmaxf(m, __uint_as_float(w[j]));
    return m;
  }
  template <typename F>
  OGB_DEVICE static void pairs(const uint32_t (&w)[8], F&& f) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) f(Float2(__uint_as_float(w[j]), __uint_as_float(w[j + 1])));
  }
  OGB_DEVICE static int above(const uint32_t (&w)[8], float given) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) n += __uint_as_float(w[j]) > given ? 1 : 0;
    return n;
  }
  OGB_DEVICE static float value(const uint32_t (&w)[8], int j) { return __uint_as_float(w[j]); }
  static constexpr uint32_t kNothing = 0xff800000u;        // a word of minus infinities
};
template <>
struct LpType<__nv_bfloat16> {
  static constexpr int kPer = 16, kElem = kElemBf16;
  using Max = __nv_bfloat16;
  OGB_DEVICE static __nv_bfloat162 two(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
  OGB_DEVICE static float max_of(const uint32_t (&w)[8]) {
    __nv_bfloat162 m = two(w[0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) m = __hmax2(m, two(w[j]));
    const __nv_bfloat16 one = __hmax(m.x, m.y);
    return __bfloat162float(one);
  }
  template <typename F>
  OGB_DEVICE static void pairs(const uint32_t (&w)[8], F&& f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f(Float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u)));
  }
  OGB_DEVICE static int above(const uint32_t (&w)[8], float given) {
    const __nv_bfloat162 g = __float2bfloat162_rn(given);
    __nv_bfloat162 n = __hgt2(two(w[0]), g);
#pragma unroll
    for (int j = 1; j < 8; ++j) n = __hadd2(n, __hgt2(two(w[j]), g));
    const float2 f = __bfloat1622float2(n);
    return static_cast<int>(f.x + f.y);
  }
  OGB_DEVICE static float value(const uint32_t (&w)[8], int j) { return __uint_as_float((j & 1) != 0 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16); }
  static constexpr uint32_t kNothing = 0xff80ff80u;
};
template <>
struct LpType<__half> {
  static constexpr int kPer = 16, kElem = kElemF16;
  using Max = __half;
  OGB_DEVICE static __half2 two(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
  OGB_DEVICE static float max_of(const uint32_t (&w)[8]) {
    __half2 m = two(w[0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) m = __hmax2(m, two(w[j]));
    const float2 f = __half22float2(m);
    return fmaxf(f.x, f.y);
  }
  template <typename F>
  OGB_DEVICE static void pairs(const uint32_t (&w)[8], F&& f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 t = __half22float2(two(w[j]));
      f(Float2(t.x, t.y));
    }
  }
  OGB_DEVICE static int above(const uint32_t (&w)[8], float given) {
    const __half2 g = __float2half2_rn(given);
    __half2 n = __hgt2(two(w[0]), g);
#pragma unroll
    for (int j = 1; j < 8; ++j) n = __hadd2(n, __hgt2(two(w[j]), g));
    const float2 f = __half22float2(n);
    return static_cast<int>(f.x + f.y);
  }
  OGB_DEVICE static float value(const uint32_t (&w)[8], int j) {
    const float2 t = __half22float2(two(w[j >> 1]));
    return (j & 1) != 0 ? t.y : t.x;
  }
  static constexpr uint32_t kNothing = 0xfc00fc00u;
};
OGB_DEVICE float lp_float(float v) { return v; }
OGB_DEVICE float lp_float(__nv_bfloat16 v) { return __bfloat162float(v); }
OGB_DEVICE float lp_float(__half v) { return __half2float(v); }

template <typename T>
struct LpShared {
  static constexpr int kPer = LpType<T>::kPer;
  static constexpr int kMost = (kLpMaxTop > kLpQuick ? kLpMaxTop : kLpQuick) * kPer + kLpMaxTop;
  __align__(16) unsigned long long keys[kMost + 8];           // the best so far, behind them what was added, and zeros to a multiple of eight
  __align__(16) unsigned long long best[kLpThreads];          // of each thread; then the list in order
  unsigned long long bound;
  LpState part[kLpWarps];
  int rank_part[kLpWarps];
  int count, reach;
  int pieces[kLpQuick];
  LpState total;
  int rank_total;
};

// The place of `key` among n keys in shared memory, n a multiple of eight: how many are above it.
OGB_DEVICE int lp_place(const unsigned long long* keys, int n, unsigned long long key) {
  int above = 0;
  for (int i = 0; i < n; i += 8) {
    ulonglong2 k[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const ulonglong2*>(keys + i + 2 * j);
#pragma unroll
    for (int j = 0; j < 4; ++j) above += (k[j].x > key ? 1 : 0) + (k[j].y > key ? 1 : 0);
  }
  return above;
}

// Read once, so first to leave L2 (256 rows: 21.6 us without that, 20.9 with it).
// The piece of a row of `vocab` logits that begins at value i0 (below zero or past the end where the row's ends are not at multiples of 32 bytes).
template <typename T>
OGB_DEVICE void lp_load(const T* x, int i0, int vocab, uint32_t (&w)[8]) {
  using Type = LpType<T>;
  if (i0 >= 0 && i0 + Type::kPer <= vocab) {
    asm volatile("ld.global.L1::no_allocate.L2::evict_first.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(x + i0));
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    w[j] = Type::kNothing;
    if constexpr (Type::kPer == 8) {
      if (i0 + j >= 0 && i0 + j < vocab) w[j] = __float_as_uint(x[i0 + j]);
    } else {
      const int i = i0 + 2 * j;
      const uint16_t* s = reinterpret_cast<const uint16_t*>(x);
      if (i >= 0 && i < vocab) w[j] = (w[j] & 0xffff0000u) | s[i];
      if (i + 1 >= 0 && i + 1 < vocab) w[j] = (w[j] & 0xffffu) | static_cast<uint32_t>(s[i + 1]) << 16;
    }
  }
}

template <typename T, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(kLpThreads, TOP ? 4 : 5) logprobs_kernel(const LogprobsParams p) {
  using Type = LpType<T>;
  constexpr int kPer = Type::kPer;                              // values of a 32-byte piece
  __shared__ LpShared<T> sh;
  extern __shared__ __align__(16) uint8_t dynamic_smem[];
  typename Type::Max* piece_max = reinterpret_cast<typename Type::Max*>(dynamic_smem);
  const int split = p.splits > 1 ? static_cast<int>(cg::this_cluster().block_rank()) : 0;
  const int row = blockIdx.x / p.splits, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = static_cast<const T*>(p.logits) + static_cast<size_t>(row) * p.ld;
  const int token = p.tokens[row];
  const bool known = token >= 0 && token < p.vocab;
  const float given = known ? load_elem(x, Type::kElem, token) : INFINITY;

  // 32-byte pieces that the row touches, an equal share of them to every CTA of the cluster
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 31) / sizeof(T));
  const int pieces = (off + p.vocab + kPer - 1) / kPer;
  const int each = (pieces + p.splits - 1) / p.splits;
  const int b0 = min(pieces, split * each), n_pieces = min(pieces, b0 + each) - b0;
  const int first = b0 * kPer - off;                        // value at which this CTA's share begins
  auto is_edge = [&](int i0) { return i0 < 0 || i0 + kPer > p.vocab; };

  // ---- the pass ----
  float ref = -INFINITY, neg = 0.f;                         // m; minus m, zero as long as there is no value
  Float2 s2(0.f), t2(0.f);
  int rank = 0;
  const Float2 log2e(1.4426950408889634f);
  // the next piece is on its way while this one is summed
  uint32_t next[8];
  auto fetch = [&](int piece) {
    if (piece < n_pieces) lp_load(x, first + piece * kPer, p.vocab, next);
  };
  fetch(tid);
  for (int piece = tid; piece < n_pieces; piece += kLpThreads) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = next[j];
    fetch(piece + kLpThreads);
    const float top = Type::max_of(w);
    if (top - ref > kLpSlack || (ref == -INFINITY && top > -INFINITY)) {
      if (ref != -INFINITY) {
        const float d = fmaxf(ref - top, -1000.f);          // a type's lowest value is minus infinity apart, in effect
        const Float2 r(__expf(d));
        t2 = r * fma2(Float2(d), s2, t2);
        s2 = r * s2;
      }
      ref = top;
      neg = -top;
    }
    const Float2 minus(neg);
    Type::pairs(w, [&](Float2 v) {
      const Float2 d = v + minus, a = d * log2e;
      const Float2 e(ex2_approx(a.lo()), ex2_approx(a.hi()));
      s2 = s2 + e;
      if (ENTROPY) t2 = fma2(e, Float2(fmaxf(d.lo(), -1000.f), fmaxf(d.hi(), -1000.f)), t2);
    });
    if (top > given) rank += Type::above(w, given);
    if (TOP) {
      float kept = top;
      const int i0 = first + piece * kPer;
      if (is_edge(i0)) {                                    // without what is not there
        kept = __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (i0 + j >= 0 && i0 + j < p.vocab) kept = fmaxf(kept, Type::value(w, j));
      }
      if constexpr (Type::kElem == kElemF32) piece_max[piece] = kept;
      else if constexpr (Type::kElem == kElemBf16) piece_max[piece] = __float2bfloat16(kept);
      else piece_max[piece] = __float2half_rn(kept);
    }
  }
  LpState st{ref, s2.lo() + s2.hi(), t2.lo() + t2.hi()};

  // ---- the likeliest of this CTA's share, and perhaps some more, kLpMaxTop of them at most, at the head of sh.keys ----
  int held = 0;
  if (TOP) {
    // the best key of a piece is at most that of its maximum at its first value, at least that at its last
    auto upper = [&](int piece) { return lp_key(lp_float(piece_max[piece]), max(0, first + piece * kPer)); };
    auto add_piece = [&](int piece, unsigned long long floor_key) {
      uint32_t w[8];
      const int i0 = first + piece * kPer;
      lp_load(x, i0, p.vocab, w);
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (i0 + j >= 0 && i0 + j < p.vocab) {
          const unsigned long long key = lp_key(Type::value(w, j), i0 + j);
          if (key > floor_key) sh.keys[held + atomicAdd(&sh.count, 1)] = key;
        }
    };
    // keeps the best of held + count keys; the least of them when there are enough, else the floor as it was
    auto keep_best = [&](unsigned long long floor_key) {
      const int n = held + sh.count, padded = (n + 7) / 8 * 8;
      if (tid < padded - n) sh.keys[n + tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kLpThreads) {
        const unsigned long long key = sh.keys[i];
        const int place = lp_place(sh.keys, padded, key);
        if (place < p.top) sh.best[place] = key;
      }
      __syncthreads();
      held = min(n, p.top);
      if (tid < held) sh.keys[tid] = sh.best[tid];
      if (tid == 0) sh.count = 0;
      if (n >= p.top) floor_key = sh.best[p.top - 1];
      __syncthreads();
      return floor_key;
    };
    float best = -INFINITY;
    int best_piece = -1;
    for (int b = tid; b < n_pieces; b += kLpThreads) {
      const float m = lp_float(piece_max[b]);
      if (m > best || (best_piece < 0 && m == m)) { best = m; best_piece = b; }      // nothing but NaN: no bound from this thread
    }
    unsigned long long own_best = best_piece >= 0 ? lp_key(best, min(p.vocab - 1, first + best_piece * kPer + kPer - 1)) : 0;
    // where every thread has several pieces, four threads' best is bound enough, and 64 keys take a sixteenth of the comparisons
    const int group = n_pieces >= 2 * kLpThreads ? 4 : 1;
    if (group == 4) {
#pragma unroll
      for (int o = 1; o <= 2; o <<= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, own_best, o);
        own_best = other > own_best ? other : own_best;
      }
    }
    if (tid % group == 0) sh.best[tid / group] = own_best;
    if (tid == 0) { sh.count = 0; sh.reach = 0; sh.bound = 0; }
    __syncthreads();
    if (tid % group == 0 && own_best != 0 && lp_place(sh.best, kLpThreads / group, own_best) == p.top - 1) sh.bound = own_best;
    __syncthreads();
    unsigned long long floor_key = sh.bound != 0 ? sh.bound - 1 : 0;          // fewer threads than `top` have a value: every value may be one
    const float floor_value = lp_value(floor_key + 1);
    auto reaches = [&](int b) { return !(lp_float(piece_max[b]) < floor_value) && upper(b) > floor_key; };
    for (int b = tid; b < n_pieces; b += kLpThreads)
      if (reaches(b)) {
        const int at = atomicAdd(&sh.reach, 1);
        if (at < kLpQuick) sh.pieces[at] = b;
      }
    __syncthreads();
    if (sh.reach <= kLpQuick) {
      // a value a thread, all of them at one latency
      for (int e = tid; e < sh.reach * kPer; e += kLpThreads) {
        const int i = first + sh.pieces[e / kPer] * kPer + e % kPer;
        if (i >= 0 && i < p.vocab) {
          const unsigned long long key = lp_key(load_elem(x, Type::kElem, i), i);
          if (key > floor_key) sh.keys[atomicAdd(&sh.count, 1)] = key;
        }
      }
      __syncthreads();
      if (sh.count <= kLpMaxTop) held = sh.count;           // the join puts them in order
      else keep_best(floor_key);
    } else {
      for (int b = 0; b < n_pieces; b += kLpThreads) {
        // a round: a piece a thread.  At most `top` threads keep one whose best key reaches the bound of this round.
        bool in = b + tid < n_pieces && upper(b + tid) > floor_key;
        const int threads = __syncthreads_count(in);
        if (threads == 0) continue;
        unsigned long long own = 0;
        if (in) {
          uint32_t w[8];
          const int i0 = first + (b + tid) * kPer;
          lp_load(x, i0, p.vocab, w);
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (i0 + j >= 0 && i0 + j < p.vocab) {
              const unsigned long long key = lp_key(Type::value(w, j), i0 + j);
              own = key > own ? key : own;
            }
          if (own <= floor_key) own = 0;
        }
        sh.best[tid] = own;
        if (tid == 0) sh.bound = 0;
        __syncthreads();
        if (own != 0 && lp_place(sh.best, kLpThreads, own) == p.top - 1) sh.bound = own;
        __syncthreads();
        if (sh.bound != 0) floor_key = sh.bound - 1;
        if (own > floor_key) add_piece(b + tid, floor_key);
        __syncthreads();
        floor_key = keep_best(floor_key);
      }
    }
  }

  // ---- threads -> warps -> the CTA ----
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const LpState other{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.t, o)};
    st = lp_join(st, other);
  }
  rank = __reduce_add_sync(0xffffffffu, rank);
  if (lane == 0) { sh.part[warp] = st; sh.rank_part[warp] = rank; }
  __syncthreads();
  if (tid == 0) {
    st = sh.part[0];
    rank = sh.rank_part[0];
    for (int w = 1; w < kLpWarps; ++w) { st = lp_join(st, sh.part[w]); rank += sh.rank_part[w]; }
    sh.total = st;
    sh.rank_total = rank;
    sh.count = held;
  }
  if (p.splits > 1) cg::this_cluster().sync();
  else __syncthreads();
  if (split == 0) {
    // every thread of the first CTA joins the parts for itself
    st = sh.total;
    rank = sh.rank_total;
    int n = held;
    if (p.splits > 1) {
      const LpShared<T>& peer = *cg::this_cluster().map_shared_rank(&sh, min(lane, p.splits - 1));
      const LpState theirs = peer.total;
      const int their_rank = peer.rank_total, their_count = TOP ? peer.count : 0;
      n = 0;
      int base = 0;                                          // the list of CTA r goes behind those before it, a warp a CTA
#pragma unroll
      for (int r = 0; r < kLpMaxSplit; ++r) {
        const LpState other{__shfl_sync(0xffffffffu, theirs.m, r), __shfl_sync(0xffffffffu, theirs.s, r), __shfl_sync(0xffffffffu, theirs.t, r)};
        const int more = __shfl_sync(0xffffffffu, their_rank, r), count = __shfl_sync(0xffffffffu, their_count, r);
        if (r == warp) base = n;
        if (r < p.splits) n += count;
        if (r > 0 && r < p.splits) { st = lp_join(st, other); rank += more; }
      }
      if (TOP && warp > 0 && warp < p.splits) {
        const LpShared<T>& from = *cg::this_cluster().map_shared_rank(&sh, warp);
        if (lane < __shfl_sync(0xffffffffu, their_count, warp)) sh.keys[base + lane] = from.keys[lane];
      }
    }
    const float log_s = logf(st.s);
    if (tid == 0) {
      if (token >= p.vocab) atomicOr(p.status, kStatusIndexOutOfRange);
      p.logprob[row] = known ? given - st.m - log_s : token < 0 ? 0.f : __uint_as_float(0x7fc00000u);
      if (p.rank != nullptr) p.rank[row] = known ? rank : -1;
      if (ENTROPY) p.entropy[row] = log_s - st.t / st.s;
    }
    if (TOP) {
      const int padded = (n + 7) / 8 * 8;
      if (tid < padded - n) sh.keys[n + tid] = 0;
      __syncthreads();
      const unsigned long long key = tid < n ? sh.keys[tid] : 0;
      const int place = key != 0 ? lp_place(sh.keys, padded, key) : p.top;
      if (place < p.top) {
        p.top_ids[static_cast<size_t>(row) * p.top + place] = lp_index(key);
        p.top_logprob[static_cast<size_t>(row) * p.top + place] = lp_value(key) - st.m - log_s;
      }
    }
  }
  if (p.splits > 1) cg::this_cluster().sync();          // nobody leaves while its shared memory is being read
}

template <typename T>
static int launch_logprobs(const LogprobsParams& p, cudaStream_t stream) {
  constexpr int kPer = LpType<T>::kPer;
  static OncePerDevice allowed[2];
  int smem = 0;
  if (p.top > 0) {
    const long long pieces = (static_cast<long long>(p.vocab) + 2 * kPer - 2) / kPer;
    const long long bytes = ((pieces + p.splits - 1) / p.splits * static_cast<long long>(sizeof(typename LpType<T>::Max)) + 15) / 16 * 16;
    if (bytes > kLpSmem) return -9;
    smem = static_cast<int>(bytes);
    const int rc = p.entropy != nullptr ? allow_smem(allowed[0], logprobs_kernel<T, true, true>, kLpSmem) : allow_smem(allowed[1], logprobs_kernel<T, false, true>, kLpSmem);
    if (rc != 0) return rc;
  }
  auto kernel = p.top > 0 ? (p.entropy != nullptr ? logprobs_kernel<T, true, true> : logprobs_kernel<T, false, true>)
                          : (p.entropy != nullptr ? logprobs_kernel<T, true, false> : logprobs_kernel<T, false, false>);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * p.splits);
  cfg.blockDim = dim3(kLpThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 ? 1 : 0;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, p));
}

}  // namespace ogb

using namespace ogb;

extern "C" int ogb_token_logprobs(const void* logits, const int* tokens, float* logprob, float* entropy, int* rank, int* top_ids, float* top_logprob,
                                  int rows, int vocab, int64_t ld, int top, int elem, int* status, void* stream_) {
  if (rows < 0 || vocab < 1 || ld < 0 || elem < 0 || elem >= kElemKinds) return -2;
  if (top < 0 || top > kLpMaxTop || top > vocab || (rows > 0 && top > 0 && (top_ids == nullptr || top_logprob == nullptr))) return -3;
  if (rows == 0) return 0;
  if (vocab > (1 << 30) || rows >= (1 << 28)) return -2;      // a grid of up to kLpMaxSplit CTAs a row has 31 bits
  LogprobsParams p{logits, tokens, logprob, entropy, top_logprob, rank, top_ids, ld, rows, vocab, top, 1, status};
  const int sms = ogb_num_sms();
  // parts of a row: until every SM has a few CTAs, as long as each keeps a piece or so a thread; more where the maxima of its pieces would not fit
  const long long round = kLpThreads * 32 / elem_bytes(elem);
  const long long fits = static_cast<long long>(kLpSmem) * 32 / elem_bytes(elem) / elem_bytes(elem) - 64;
  while (p.splits < kLpMaxSplit && ((static_cast<long long>(rows) * p.splits < 2 * sms && p.splits * round < vocab) || (top > 0 && p.splits * fits < vocab))) p.splits *= 2;
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (elem == kElemF32) return launch_logprobs<float>(p, stream);
  if (elem == kElemBf16) return launch_logprobs<__nv_bfloat16>(p, stream);
  return launch_logprobs<__half>(p, stream);
}

// The same call with its arguments as 64-bit words: see ogb_gemm_int8_args.
extern "C" int ogb_token_logprobs_args(const int64_t* a) {
  auto p = [&](int i) { return reinterpret_cast<void*>(a[i]); };
  auto n = [&](int i) { return static_cast<int>(a[i]); };
  return ogb_token_logprobs(p(0), static_cast<const int*>(p(1)), static_cast<float*>(p(2)), static_cast<float*>(p(3)), static_cast<int*>(p(4)),
                            static_cast<int*>(p(5)), static_cast<float*>(p(6)), n(7), n(8), a[9], n(10), n(11), static_cast<int*>(p(12)), p(13));
}
