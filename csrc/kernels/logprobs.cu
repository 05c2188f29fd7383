// Log probability of a given token per row of logits, the entropy of the row, how many tokens are more likely, and the `top` likeliest.
//
//   m = max x,  s = sum exp(x - m),  t = sum exp(x - m) (x - m)
//   log p(i) = x_i - m - log s,   entropy = log s - t / s,   rank = |{j : x_j > x_token}|
//
// One pass over the row: every thread carries (m, s, t) of its values and rescales them when a new maximum turns up; the states of threads,
// warps and CTAs join by the same rule.  What bounds it is the stream of logits from HBM (2 bytes a value), with exp(x - m) -- one a value,
// 16 a clock and SM -- close behind.
//
// The likeliest values are found in the same pass.  A value's key is its order as a whole number above its inverted index, so that no two are
// equal and ties go to the lower index.  A CTA holds the best `top` keys so far; only a piece whose maximum reaches the last of them is looked
// at.  Among the threads of a CTA with such a piece, the top-th best of their best keys bounds the row's top-th best from below, so
// at most `top` threads hold anything above that bound: a round adds at most top * kPiece keys whatever the order of the values (a row that rises from
// end to end costs rounds, never space).
//
// A row is split over a cluster of CTAs where rows are few; the parts join over distributed shared memory.
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
constexpr int kLpBlocks = 2;               // 16-byte blocks a thread takes per round
constexpr int kLpMaxTop = 32;
constexpr int kLpMaxSplit = 8;             // the portable cluster size

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

template <typename T>
struct LpType;
template <> struct LpType<float> { static constexpr int kPer = 4, kElem = kElemF32; };
template <> struct LpType<__nv_bfloat16> { static constexpr int kPer = 8, kElem = kElemBf16; };
template <> struct LpType<__half> { static constexpr int kPer = 8, kElem = kElemF16; };

template <typename T>
struct LpShared {
  static constexpr int kPiece = LpType<T>::kPer * kLpBlocks;          // values of a thread in a round
  static constexpr int kMost = kLpMaxTop * kPiece + kLpMaxTop;
  unsigned long long keys[kMost];                 // the best so far, and behind them what a round added
  unsigned long long best[kLpThreads];            // of each thread in a round; then the list in order
  unsigned long long bound;
  LpState part[kLpWarps];
  int rank_part[kLpWarps];
  int count;
  LpState total;
  int rank_total;
};

// The place of `key` among n keys in shared memory: how many are above it.
OGB_DEVICE int lp_place(const unsigned long long* keys, int n, unsigned long long key) {
  int above = 0;
  for (int i = 0; i < n; ++i) above += keys[i] > key ? 1 : 0;
  return above;
}

template <typename T, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(kLpThreads) logprobs_kernel(const LogprobsParams p) {
  using Type = LpType<T>;
  constexpr int kPer = Type::kPer;
  __shared__ LpShared<T> sh;
  const int split = p.splits > 1 ? static_cast<int>(cg::this_cluster().block_rank()) : 0;
  const int row = blockIdx.x / p.splits, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = static_cast<const T*>(p.logits) + static_cast<size_t>(row) * p.ld;
  const int token = p.tokens[row];
  const bool known = token >= 0 && token < p.vocab;
  const float given = known ? load_elem(x, Type::kElem, token) : INFINITY;

  // 16-byte blocks that the row touches; those it does not fill (its ends, where it is not aligned) are read value by value
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int blocks = (off + p.vocab + kPer - 1) / kPer;
  const int each = (blocks + p.splits - 1) / p.splits;
  const int b0 = split * each, b1 = min(blocks, b0 + each);
  const uint4* base = reinterpret_cast<const uint4*>(x - off);
  auto load = [&](int b, float (&f)[kPer]) {
    const int i0 = b * kPer - off;
    if (b < b1 && i0 >= 0 && i0 + kPer <= p.vocab) {
      const uint4 v = __ldcs(base + b);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (kPer == 4) {
          f[j] = __uint_as_float(w[j]);
        } else {
          const float2 t = Type::kElem == kElemBf16 ? unpack_bf16(w[j]) : __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          f[2 * j] = t.x;
          f[2 * j + 1] = t.y;
        }
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) f[j] = b < b1 && i0 + j >= 0 && i0 + j < p.vocab ? load_elem(x, Type::kElem, i0 + j) : -INFINITY;
  };

  LpState st{-INFINITY, 0.f, 0.f};
  int rank = 0;
  unsigned long long floor_key = 0;      // nothing at or below it is among the best
  float floor_value = -INFINITY;
  int held = 0;                          // keys in the list
  if (TOP && tid == 0) sh.count = 0;
  if (TOP) __syncthreads();

  for (int b = b0; b < b1; b += kLpThreads * kLpBlocks) {
    float f[kLpBlocks][kPer];
#pragma unroll
    for (int u = 0; u < kLpBlocks; ++u) load(b + u * kLpThreads + tid, f[u]);
    float top = f[0][0];
#pragma unroll
    for (int u = 0; u < kLpBlocks; ++u)
#pragma unroll
      for (int j = 0; j < kPer; ++j) top = fmaxf(top, f[u][j]);
    if (top > st.m) {
      if (st.m != -INFINITY) {
        const float d = fmaxf(st.m - top, -1000.f), r = __expf(d);     // a type's lowest value is minus infinity apart, in effect
        st.t = r * fmaf(d, st.s, st.t);
        st.s *= r;
      }
      st.m = top;
    }
    const float m = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int u = 0; u < kLpBlocks; ++u)
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const float d = f[u][j] - m, e = __expf(d);
        st.s += e;
        if (ENTROPY) st.t = fmaf(e, fmaxf(d, -1000.f), st.t);
        rank += f[u][j] > given ? 1 : 0;
      }
    if (TOP) {
      unsigned long long mine = 0;
      if (!(top < floor_value)) {
#pragma unroll
        for (int u = 0; u < kLpBlocks; ++u)
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const int i = (b + u * kLpThreads + tid) * kPer - off + j;
            const unsigned long long key = b + u * kLpThreads + tid < b1 && i >= 0 && i < p.vocab ? lp_key(f[u][j], i) : 0;
            mine = key > mine ? key : mine;
          }
        if (mine <= floor_key) mine = 0;
      }
      const int threads = __syncthreads_count(mine != 0);
      if (threads == 0) continue;
      if (threads > p.top) {
        sh.best[tid] = mine;
        __syncthreads();
        const int place = mine != 0 ? lp_place(sh.best, kLpThreads, mine) : kLpThreads;
        if (place == p.top - 1) sh.bound = mine;
        __syncthreads();
        floor_key = sh.bound - 1;                                    // the bound itself is kept
      }
      if (mine > floor_key) {
#pragma unroll
        for (int u = 0; u < kLpBlocks; ++u)
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const int i = (b + u * kLpThreads + tid) * kPer - off + j;
            if (b + u * kLpThreads + tid < b1 && i >= 0 && i < p.vocab) {
              const unsigned long long key = lp_key(f[u][j], i);
              if (key > floor_key) sh.keys[held + atomicAdd(&sh.count, 1)] = key;
            }
          }
      }
      __syncthreads();
      const int n = held + sh.count;
      if (n >= p.top) {
        for (int i = tid; i < n; i += kLpThreads) {
          const unsigned long long key = sh.keys[i];
          const int place = lp_place(sh.keys, n, key);
          if (place < p.top) sh.best[place] = key;
        }
        __syncthreads();
        if (tid < p.top) sh.keys[tid] = sh.best[tid];
        held = p.top;
        floor_key = sh.best[p.top - 1];
        floor_value = lp_value(floor_key);
      } else {
        held = n;
      }
      if (tid == 0) sh.count = 0;
      __syncthreads();
    }
  }

  // threads -> warps -> the CTA
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
    for (int r = 1; r < p.splits; ++r) {
      const LpShared<T>& peer = *cg::this_cluster().map_shared_rank(&sh, r);
      st = lp_join(st, peer.total);
      rank += peer.rank_total;
      if (TOP) {
        const int more = peer.count;
        if (tid < more) sh.keys[n + tid] = peer.keys[tid];
        n += more;
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
      __syncthreads();
      for (int i = tid; i < n; i += kLpThreads) {
        const unsigned long long key = sh.keys[i];
        const int place = lp_place(sh.keys, n, key);
        if (place < p.top) {
          p.top_ids[static_cast<size_t>(row) * p.top + place] = lp_index(key);
          p.top_logprob[static_cast<size_t>(row) * p.top + place] = lp_value(key) - st.m - log_s;
        }
      }
    }
  }
  if (p.splits > 1) cg::this_cluster().sync();          // nobody leaves while its shared memory is being read
}

template <typename T>
static int launch_logprobs(const LogprobsParams& p, cudaStream_t stream) {
  auto kernel = p.top > 0 ? (p.entropy != nullptr ? logprobs_kernel<T, true, true> : logprobs_kernel<T, false, true>)
                          : (p.entropy != nullptr ? logprobs_kernel<T, true, false> : logprobs_kernel<T, false, false>);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * p.splits);
  cfg.blockDim = dim3(kLpThreads);
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
  if (vocab > (1 << 30) || rows > (1 << 28)) return -2;
  LogprobsParams p{logits, tokens, logprob, entropy, top_logprob, rank, top_ids, ld, rows, vocab, top, 1, status};
  const int sms = ogb_num_sms();
  // parts of a row: until every SM has work, as long as a part keeps a round's worth of values
  const int round = kLpThreads * kLpBlocks * 16 / elem_bytes(elem);
  while (p.splits < kLpMaxSplit && static_cast<long long>(rows) * p.splits < sms && static_cast<long long>(p.splits) * round < vocab) p.splits *= 2;
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (elem == kElemF32) return launch_logprobs<float>(p, stream);
  if (elem == kElemBf16) return launch_logprobs<__nv_bfloat16>(p, stream);
  return launch_logprobs<__half>(p, stream);
}
