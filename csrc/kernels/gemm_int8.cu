// Products in 8-bit integers:  y[t, n] = s[t] c[n] sum_k q[t, k] w[n, k]  (+ bias)(+ residual) | silu(gate) up.
//
// q are rows of activations in 8 bits with a factor s each (int8_rows.cuh), w a weight with a factor c per channel.  The sums are whole
// numbers in 32 bits, exact for K up to 131072 (q is -127 to 127, w may be -128: 127 * 128 * K < 2^31), so their order does not matter and a
// product may be cut along K wherever it pays; one rounding to the type of the result follows the factors, the bias and the residual.
//
// What bounds it: few rows, the stream of w from HBM (half of bf16's); many, the tensor cores, kind::i8 at twice the rate of
// kind::f16 for the same bytes of operands.
//
// W is the M side of tcgen05.mma -- 128 channels a tile, TW = 2: 128 gate and their 128 up channels, two accumulators -- and the rows are its N
// side, padded to a multiple of 16 only, up to 256 (128 when gated).  So one kernel serves three rows, whose stage of the ring is W almost
// alone, and thousands, 128 x 256 to a tile (PAIR: 256 x 256 to two CTAs).  Warp 0 issues the TMA loads, warp 1 the products, warps 2 - 9 are two groups of
// the epilogue: sums leave TMEM for shared memory 32 rows at a time and come back a row per warp, so that 128 channels of a row are stored
// together.
//
// Division of the work (i8_plan):
//   * no more tiles than SMs: a cluster of up to 8 CTAs shares a tile, each takes a part of K; the parts are summed over distributed shared
//     memory;
//   * else: whole tiles, dealt to one CTA (or pair) per SM in rounds, the epilogue of a tile under the products of the next (two accumulators).
//     Where K is long the tiles left for the last round, which would leave most SMs idle, are cut along K into one range per SM; CTAs that
//     share a tile leave their sums in a workspace, and whichever comes last adds them up.  Ranges come first, so that those sums pass under
//     whole tiles;
//   * one or two rows of a weight of moderate size: no tensor cores (gemv_int8_kernel).
//
// Measured with weights from HBM, 8-bit rows made by the call: 64 rows against 3584 x 18944 with a residual 22.6 us (28 tiles in clusters of four: as many of
// five do not fit the SMs' groups at once, and 36 SMs idle); 77, gated 37888 x 3584 32; 8192, 3584 x 18944 rows 97 and product 329 to 349, 3.2 to 3.4
// POP/s, by the clock that the power limit leaves; one row of 4608 x 3584 9.5.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "gemm_common.cuh"
#include "gemm_rows.cuh"
#include "int8_rows.cuh"
#include "ogb_kernels.h"


namespace ogb {

int make_tmap_u8_2d(CUtensorMap* out, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows, uint32_t box_cols);

constexpr int kI8K = 128;                    // 128 bytes: a row of the 128-byte swizzle
constexpr int kI8Threads = 320;              // TMA, MMA, two groups of four epilogue warps
constexpr int kI8MaxK = 131072;
constexpr int kI8Group = 16;                 // tiles of W that go together against all rows
constexpr int kI8Groups = 2;                 // of epilogue warps, every other chunk of a tile's rows each
template <int TW>
constexpr int kI8Chunk = 32 / TW;            // rows of a chunk: 16 KB of sums, of both accumulators
constexpr int kI8Stage = 32 * 128 * 4;       // staging of a group

struct Int8Params {
  void* out;
  const float* factor;                       // s
  const float* channel;                      // c
  const float* bias;                         // or null
  const void* residual;                      // or null
  long long ldc, ldr;
  int vec;                                   // results and residuals in pieces of four
  int pair;                                  // 1: two CTAs on 256 channels
  int M, N, mn;                              // mn: rows of a tile, a multiple of 16 (32)
  int n_tiles, m_tiles, tiles, k_blocks, stages;
  int splits;                                // CTAs (a cluster) per tile; 0: whole tiles and ranges
  int cut;                                   // the first `cut` tiles are cut into ranges of
  int range, longer;                         //   `range` k-blocks a CTA, and one more for the first `longer`; of a cluster's tile likewise
  int* status;
  int* ws;                                   // [CTA][2][TW][4 quarters][rows / 4][32 channels][4 rows]
  unsigned int* counters;                    // [CTA], zero when the kernel starts
};

template <bool PAIR>
OGB_DEVICE void umma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (PAIR) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}
// A pair's barriers.  What both CTAs report (bytes that have landed, accumulators that have been read) is counted by the first one's, which issues the products;
// what its products report (operands read, sums complete) arrives at the same barrier of both.
OGB_DEVICE uint32_t i8_pair_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
OGB_DEVICE uint32_t i8_first_addr(const void* p) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}
OGB_DEVICE void i8_first_arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(i8_first_addr(bar)) : "memory"); }
OGB_DEVICE bool i8_pair_wait(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = global_timer_ns();
  for (uint32_t spins = 0;; ++spins) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred P;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, P;\n\t}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok != 0) return true;
    if ((spins & 0x3ff) == 0x3ff && global_timer_ns() - t0 > kWaitLimitNs) return false;
  }
}
template <bool PAIR>
OGB_DEVICE bool i8_wait(uint64_t* bar, uint32_t parity) { return PAIR ? i8_pair_wait(bar, parity) : mbar_wait(bar, parity); }
template <bool PAIR>
OGB_DEVICE void i8_commit(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"(static_cast<uint16_t>(3)) : "memory");
  else umma_commit(bar);
}
template <bool PAIR>
OGB_DEVICE void i8_load(void* to, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  if constexpr (PAIR)
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(smem_u32(to)), "l"(reinterpret_cast<uint64_t>(map)), "r"(i8_first_addr(bar)), "r"(x), "r"(y) : "memory");
  else tma_load_2d(to, map, bar, x, y);
}
OGB_DEVICE void i8_pair_sync() { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); }
// kind::i8: signed 8-bit A and B, both K-major, 32-bit sums that wrap (they never get that far).
__host__ __device__ constexpr uint32_t make_idesc_i8(int m, int n) {
  return (2u << 4)                      // D format: s32
         | (1u << 7) | (1u << 10)       // A, B format: signed
         | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// Tiles in groups of kI8Group tiles of W: within a group W goes fastest, so that the tiles under way at one time (about 148) share both operands
// in L2.
OGB_DEVICE void i8_tile(const Int8Params& p, int tile, int& nt, int& mt) {
  if (p.m_tiles == 1) {
    nt = tile;
    mt = 0;
  } else {
    const int g = tile / (kI8Group * p.m_tiles), first = g * kI8Group;
    const int wide = min(kI8Group, p.n_tiles - first), t = tile - first * p.m_tiles;
    nt = first + t % wide;
    mt = t / wide;
  }
  if (p.pair != 0) nt = 2 * nt + (blockIdx.x & 1);
}

OGB_DEVICE int i8_cluster_index() {
  int i;
  asm("mov.u32 %0, %%clusterid.x;" : "=r"(i));
  return i;
}
// First k-block of a CTA's range, and the CTA whose range holds one.
OGB_DEVICE int i8_range_begin(const Int8Params& p, int cta) { return cta * p.range + min(cta, p.longer); }
OGB_DEVICE int i8_range_owner(const Int8Params& p, int i) {
  const int edge = (p.range + 1) * p.longer;
  return i < edge ? i / (p.range + 1) : p.longer + (i - edge) / p.range;
}

// The parts of tiles that a CTA computes, in order: of its range the tile it shares with the CTA before it, the one it shares with the CTA
// after it and the whole ones; then its whole tiles.  In a cluster one part of one tile, which takes no division: the first loads wait for this.  (Fewer than 200 tiles of at most 1024 k-blocks are cut: 32 bits hold their sum.)
struct Int8Segs {
  int it0, it1, first_end, last_begin, mid;
  int k_blocks, state = 0, tile, tiles, stride;
  OGB_DEVICE explicit Int8Segs(const Int8Params& p) : k_blocks(p.k_blocks), tiles(p.tiles) {
    const int unit = blockIdx.x >> p.pair;
    stride = gridDim.x >> p.pair;
    if (p.splits > 0) {
      state = 3;
      tile = p.splits == 1 ? blockIdx.x : i8_cluster_index();
      const int rank = p.splits == 1 ? 0 : cooperative_groups::this_cluster().block_rank();
      it0 = i8_range_begin(p, rank);
      it1 = i8_range_begin(p, rank + 1);
      return;
    }
    tile = p.cut + unit;
    it0 = i8_range_begin(p, unit);
    it1 = i8_range_begin(p, unit + 1);
    first_end = it0;
    last_begin = it1;
    if (it1 > it0) {
      const int t0 = it0 / k_blocks, t1 = it1 / k_blocks;
      if (it0 != t0 * k_blocks) first_end = min(it1, (t0 + 1) * k_blocks);
      if (it1 != t1 * k_blocks) last_begin = max(first_end, t1 * k_blocks);
    }
    mid = first_end;
  }
  OGB_DEVICE bool next(int& t, int& kb0, int& kb1) {
    if (state >= 3) {
      t = tile; kb0 = it0; kb1 = it1;
      return state++ == 3;
    }
    int a = 0, b = 0;
    if (state == 0) { a = it0; b = first_end; state = 1; }
    if (state == 1 && a >= b) { a = last_begin; b = it1; state = 2; }
    if (state == 2 && a >= b) {
      if (mid < last_begin) {
        a = mid;
        b = mid = mid + k_blocks;
      } else {
        if (tile >= tiles) return false;
        t = tile; kb0 = 0; kb1 = k_blocks;
        tile += stride;
        return true;
      }
    }
    t = a / k_blocks;
    kb0 = a - t * k_blocks;
    kb1 = b - t * k_blocks;
    return true;
  }
};
// The k-blocks of a CTA one by one, with their tile's place.
struct Int8Cursor {
  const Int8Params& p;
  Int8Segs segs;
  int nt = 0, mt = 0, kb = 0, kb1 = 0;
  bool more;
  OGB_DEVICE explicit Int8Cursor(const Int8Params& params) : p(params), segs(params) { part(); }
  OGB_DEVICE void part() {
    int tile;
    more = segs.next(tile, kb, kb1);
    if (more) i8_tile(p, tile, nt, mt);
  }
  OGB_DEVICE void step() {
    if (++kb == kb1) part();
  }
};

// What a lane needs of its four channels for all rows of a tile: neighbouring ones, or where rows of the result are not at multiples of four values
// every 32nd, so that a warp stores neighbours together.
template <int TW>
struct Int8Channels {
  int n, step, n_out;                         // first column of the result, way to the next, and how many there are
  float c[TW][4], b[TW][4];
  OGB_DEVICE Int8Channels(const Int8Params& p, int nt) {
    const int lane = threadIdx.x & 31;
    step = p.vec != 0 ? 1 : 32;
    n = nt * 128 + (p.vec != 0 ? 4 * lane : lane);
    n_out = p.N / TW;
#pragma unroll
    for (int w = 0; w < TW; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = min((nt * TW + w) * 128 + n - nt * 128 + i * step, p.N - 1);
        c[w][i] = __ldg(p.channel + at);
        b[w][i] = p.bias != nullptr ? __ldg(p.bias + at) : 0.f;
      }
  }
  // a lane's four sums of a row of 128
  OGB_DEVICE int4 sums(const int* row) const {
    const int lane = threadIdx.x & 31;
    if (step == 1) return *reinterpret_cast<const int4*>(row + 4 * lane);
    return make_int4(row[lane], row[lane + 32], row[lane + 64], row[lane + 96]);
  }
};
// A lane's four residuals of a row, fetched ahead of the sums they are added to.
template <int OUT>
struct Int8Residual {
  uint32_t raw[OUT == kElemF32 ? 4 : 2];
  template <int TW>
  OGB_DEVICE void load(const Int8Params& p, const Int8Channels<TW>& ch, int m) {
    const size_t from = static_cast<size_t>(m) * p.ldr + ch.n;
    if (p.vec != 0 && ch.n + 4 <= ch.n_out) {
      if constexpr (OUT == kElemF32) {
        const uint4 r = *reinterpret_cast<const uint4*>(static_cast<const float*>(p.residual) + from);
        raw[0] = r.x; raw[1] = r.y; raw[2] = r.z; raw[3] = r.w;
      } else {
        const uint2 r = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.residual) + from);
        raw[0] = r.x; raw[1] = r.y;
      }
      return;
    }
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = ch.n + i * ch.step < ch.n_out;
      if constexpr (OUT == kElemF32) v[i] = in ? static_cast<const uint32_t*>(p.residual)[from + i * ch.step] : 0;
      else v[i] = in ? static_cast<const uint16_t*>(p.residual)[from + i * ch.step] : 0;
    }
    if constexpr (OUT == kElemF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = v[i];
    } else {
      raw[0] = v[0] | v[1] << 16;
      raw[1] = v[2] | v[3] << 16;
    }
  }
  OGB_DEVICE void add(float (&v)[4]) const {
    if constexpr (OUT == kElemF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += __uint_as_float(raw[i]);
    } else {
      const float2 lo = OUT == kElemBf16 ? unpack_bf16(raw[0]) : __half22float2(*reinterpret_cast<const __half2*>(&raw[0]));
      const float2 hi = OUT == kElemBf16 ? unpack_bf16(raw[1]) : __half22float2(*reinterpret_cast<const __half2*>(&raw[1]));
      v[0] += lo.x; v[1] += lo.y; v[2] += hi.x; v[3] += hi.y;
    }
  }
};
// Sums of R rows (and of their up halves) -> the stored results; row j is m0 + j * step, there if below `end`.  All rows are computed before the first is
// stored: one after the other each took a chain of 500 cycles.
template <int TW, int OUT, int R>
OGB_DEVICE void i8_store(const Int8Params& p, const Int8Channels<TW>& ch, int m0, int step, int end, const float (&s)[R], const int4 (&a)[R],
                         const int4 (&u)[R], const Int8Residual<OUT> (&res)[R]) {
  float v[R][4];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int raw[4] = {a[j].x, a[j].y, a[j].z, a[j].w}, up[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[j][i] = fmaf(static_cast<float>(raw[i]) * s[j], ch.c[0][i], ch.b[0][i]);
      if constexpr (TW == 2) {
        const float w = fmaf(static_cast<float>(up[i]) * s[j], ch.c[TW - 1][i], ch.b[TW - 1][i]);
        v[j][i] = __fdividef(v[j][i], 1.f + __expf(-v[j][i])) * w;
      }
    }
  }
  if (TW == 1 && p.residual != nullptr) {
#pragma unroll
    for (int j = 0; j < R; ++j) res[j].add(v[j]);
  }
  if (p.vec != 0 && ch.n + 4 <= ch.n_out) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int m = m0 + j * step;
      const size_t at = static_cast<size_t>(m) * p.ldc + ch.n;
      if (m < end) {
        if constexpr (OUT == kElemF32)
          *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
        else
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
              OUT == kElemBf16 ? make_uint2(pack_bf16(v[j][0], v[j][1]), pack_bf16(v[j][2], v[j][3])) : make_uint2(pack_f16(v[j][0], v[j][1]), pack_f16(v[j][2], v[j][3]));
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int m = m0 + j * step;
    const size_t at = static_cast<size_t>(m) * p.ldc + ch.n;
    if (m < end) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (ch.n + i * ch.step < ch.n_out) store_elem(p.out, OUT, at + i * ch.step, v[j][i]);
    }
  }
}

// 32 lanes x 32 / TW consecutive columns of an accumulator
template <int TW>
OGB_DEVICE void i8_tmem_ld(uint32_t addr, uint32_t (&r)[kI8Chunk<TW>]) {
  if constexpr (TW == 1) {
    tmem_ld_32x32(addr, r);
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
  }
}
// Barriers of the epilogue warps: all of them, or a group's.
OGB_DEVICE void i8_epi_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
OGB_DEVICE void i8_group_sync(int group) { asm volatile("bar.sync %0, 128;" ::"r"(2 + group) : "memory"); }
OGB_DEVICE bool i8_group_all(int group, bool v) { return barrier_all(2 + group, 128, v); }

// The epilogue warps, where whole tiles and ranges are computed.  Warp index mod 4: the quarter of TMEM's lanes, 32 channels of a tile; each of the
// two groups takes every other chunk of rows.
template <int TW, int OUT, bool PAIR>
OGB_DEVICE void i8_epilogue(const Int8Params& p, uint32_t tmem_base, int bufs, int acc_cols, RowsBars* bars, int* staging) {
  constexpr int kChunk = kI8Chunk<TW>;
  const int warp = (threadIdx.x >> 5) - 2, q = (threadIdx.x >> 5) & 3, group = warp >> 2, lane = threadIdx.x & 31;
  const int slot = TW * 4 * acc_cols * 32;
  int* stage = staging + group * (kI8Stage / 4);
  volatile int* abort_flag = &bars->abort_flag;
  volatile uint32_t* shared_last = &bars->shared_last;
  pdl_wait();
  const float* factor = after_wait(p.factor);
  bool ok = true;
  // this warp has read an accumulator
  auto release = [&](int buf) {
    if (lane == 0) PAIR ? i8_first_arrive(&bars->tmem_empty[buf]) : mbar_arrive(&bars->tmem_empty[buf]);
  };
  Int8Segs segs(p);
  int tile, kb0, kb1;
  for (int seg = 0; segs.next(tile, kb0, kb1); ++seg) {
    const bool head = kb0 == 0, whole = head && kb1 == p.k_blocks;
    const int buf = bufs == 2 ? (seg & 1) : 0;
    const uint32_t buf_phase = (bufs == 2 ? seg >> 1 : seg) & 1;
    int nt, mt;
    i8_tile(p, tile, nt, mt);
    const int row0 = mt * p.mn, rows = min(p.mn, p.M - row0);
    // what the tile's epilogue needs besides its sums, while they are under way
    const Int8Channels<TW> ch(p, nt);
    // the factors of a chunk's rows, a lane each
    auto chunk_factor = [&](int c) { return lane < kChunk && c + lane < rows ? factor[row0 + c + lane] : 0.f; };
    Int8Residual<OUT> res[kChunk / 4];
    auto chunk_residual = [&](int c) {
      if (TW == 1 && p.residual != nullptr) {
#pragma unroll
        for (int j = 0; j < kChunk / 4; ++j)
          if (c + q * (kChunk / 4) + j < rows) res[j].load(p, ch, row0 + c + q * (kChunk / 4) + j);
      }
    };
    float f = chunk_factor(group * kChunk);
    chunk_residual(group * kChunk);
    // Every lane polls (each needs the acquire); the vote keeps the warp converged for tcgen05.ld.  Each warp's wait has a clock of its own, so the warps
    // of a group settle together whether it ended (specs/epilogue_votes.py).  After one that ran out they go on to arrive on the counters of their shared tiles.
    if (ok && !i8_group_all(group, __all_sync(0xffffffffu, i8_wait<PAIR>(&bars->tmem_full[buf], buf_phase)))) {
      ok = false;
      if (lane == 0) { atomicOr(p.status, kStatusWaitTimeout); *abort_flag = 1; }
    }
    tc_fence_after();
    const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * TW * acc_cols;
    int c_lo = 0, c_hi = 0;                                   // the CTAs that share the tile
    if (!whole) {
      c_lo = i8_range_owner(p, tile * p.k_blocks);
      c_hi = i8_range_owner(p, (tile + 1) * p.k_blocks - 1) + 1;
      if (ok) {
        int4* dst = reinterpret_cast<int4*>(p.ws + static_cast<size_t>(blockIdx.x * 2 + (head ? 1 : 0)) * slot) + q * acc_cols * 8 + lane;
#pragma unroll
        for (int w = 0; w < TW; ++w) {
#pragma unroll 1
          for (int c = group * kChunk; c < rows; c += kI8Groups * kChunk) {
            uint32_t r[kChunk];
            i8_tmem_ld<TW>(t_addr + w * acc_cols + c, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < kChunk; j += 4)
              if (c + j < rows) __stcg(dst + (w * 4 * acc_cols + c + j) * 8, make_int4(r[j], r[j + 1], r[j + 2], r[j + 3]));
          }
        }
      }
      tc_fence_before();
      __threadfence();
      i8_epi_sync();
      release(buf);
      if (warp == 0 && lane == 0) {
        *shared_last = atomicAdd(p.counters + (PAIR ? 2 * c_lo + (blockIdx.x & 1) : c_lo), 1u) == static_cast<unsigned int>(c_hi - c_lo - 1);
        __threadfence();
      }
      i8_epi_sync();
      const bool last = *shared_last != 0;
      i8_epi_sync();
      if (!__all_sync(0xffffffffu, ok && last)) continue;     // both alike in all warps of the group
    } else if (!ok) {
      continue;
    }
#pragma unroll 1
    for (int c = group * kChunk; c < rows; c += kI8Groups * kChunk) {
      const float f_next = chunk_factor(c + kI8Groups * kChunk);
#pragma unroll
      for (int w = 0; w < TW; ++w) {
        int v[kChunk];
        if (whole) {
          uint32_t r[kChunk];
          i8_tmem_ld<TW>(t_addr + w * acc_cols + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < kChunk; ++j) v[j] = static_cast<int>(r[j]);
        } else {
#pragma unroll
          for (int j = 0; j < kChunk; ++j) v[j] = 0;
          // two CTAs at a time
#pragma unroll 1
          for (int x = c_lo; x < c_hi; x += 2) {
            int4 t[2][kChunk / 4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              // the first CTA of a tile holds its head (slot 1), the others a later part (slot 0)
              const int from = min(x + i, c_hi - 1);
              const int cta = PAIR ? 2 * from + (blockIdx.x & 1) : from;
              const int4* src = reinterpret_cast<const int4*>(p.ws + static_cast<size_t>(cta * 2 + (from == c_lo ? 1 : 0)) * slot) +
                                ((w * 4 + q) * acc_cols + c) * 8 + lane;
#pragma unroll
              for (int j = 0; j < kChunk / 4; ++j) t[i][j] = __ldcg(src + j * 32);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (x + i < c_hi) {
#pragma unroll
                for (int j = 0; j < kChunk / 4; ++j) {
                  v[4 * j] += t[i][j].x; v[4 * j + 1] += t[i][j].y; v[4 * j + 2] += t[i][j].z; v[4 * j + 3] += t[i][j].w;
                }
              }
          }
        }
#pragma unroll
        for (int j = 0; j < kChunk; ++j) stage[(w * kChunk + j) * 128 + q * 32 + lane] = v[j];
      }
      i8_group_sync(group);
      float s[kChunk / 4];
      int4 a[kChunk / 4], u[kChunk / 4];
#pragma unroll
      for (int j = 0; j < kChunk / 4; ++j) {
        const int m = q * (kChunk / 4) + j;
        s[j] = __shfl_sync(0xffffffffu, f, m);
        a[j] = ch.sums(stage + m * 128);
        u[j] = TW == 2 ? ch.sums(stage + ((TW - 1) * kChunk + m) * 128) : a[j];
      }
      i8_store<TW, OUT>(p, ch, row0 + c + q * (kChunk / 4), 1, row0 + rows, s, a, u, res);
      chunk_residual(c + kI8Groups * kChunk);
      i8_group_sync(group);
      f = f_next;
    }
    if (whole) {
      tc_fence_before();
      __syncwarp();
      release(buf);
    }
  }
}

// All threads of a CTA, after their parts of the main loop: the epilogue of a tile that a cluster shares.  smem: the ring, free by then.
template <int TW, int OUT>
OGB_DEVICE void i8_finish_cluster(const Int8Params& p, uint32_t tmem_base, int acc_cols, RowsBars* bars, uint8_t* smem, int ring_bytes) {
  constexpr int kChunk = kI8Chunk<TW>;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* stage = reinterpret_cast<int*>(smem);
  bool ok = true;
  pdl_wait();
  const float* factor = after_wait(p.factor);
  const int rank = p.splits == 1 ? 0 : cooperative_groups::this_cluster().block_rank();
  const int tile = p.splits == 1 ? blockIdx.x : i8_cluster_index();
  int nt, mt;
  i8_tile(p, tile, nt, mt);
  const int row0 = mt * p.mn, rows = min(p.mn, p.M - row0);
  // Row k of those this warp will store is rank + splits * (warp + warps * k); their factors, a lane each, and the channels come while the
  // products are still under way.
  const Int8Channels<TW> ch(p, nt);
  const int first = rank + p.splits * warp, stride = p.splits * warps;
  float f = first + stride * lane < rows ? factor[row0 + first + stride * lane] : 0.f;
  if (warp >= 2) {
    ok = __all_sync(0xffffffffu, mbar_wait(&bars->tmem_full[0], 0));      // every product has retired: the ring is free
    if (!ok && lane == 0) { atomicOr(p.status, kStatusWaitTimeout); *reinterpret_cast<volatile int*>(&bars->abort_flag) = 1; }
    tc_fence_after();
    if (ok) {
      // all sums of the tile fit the ring: [accumulator][row][128]
      const int q = warp & 3, group = (warp - 2) >> 2;
#pragma unroll
      for (int w = 0; w < TW; ++w) {
#pragma unroll 1
        for (int c = group * kChunk; c < rows; c += kI8Groups * kChunk) {
          uint32_t r[kChunk];
          i8_tmem_ld<TW>(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + w * acc_cols + c, r);
          tmem_ld_wait();
          int* dst = stage + (w * acc_cols + c) * 128 + q * 32 + lane;
#pragma unroll
          for (int j = 0; j < kChunk; ++j) dst[j * 128] = static_cast<int>(r[j]);
        }
      }
    }
  }
  if (p.splits > 1) cooperative_groups::this_cluster().sync();
  else __syncthreads();
  constexpr int kRows = 2;                   // at a time
#pragma unroll 1
  for (int m0 = first, k = 0; m0 < rows; m0 += stride * kRows, k += kRows) {
    float s[kRows];
    int4 sum[TW][kRows];
    Int8Residual<OUT> res[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      s[j] = __shfl_sync(0xffffffffu, f, (k + j) & 31);
      if (TW == 1 && p.residual != nullptr && m0 + stride * j < rows) res[j].load(p, ch, row0 + m0 + stride * j);
    }
    // two CTAs at a time, in a loop: a launch runs this code once or twice, and unrolled it waits for instructions
#pragma unroll
    for (int w = 0; w < TW; ++w)
#pragma unroll
      for (int j = 0; j < kRows; ++j) sum[w][j] = make_int4(0, 0, 0, 0);
#pragma unroll 1
    for (int x = 0; x < p.splits; x += 2) {
      int4 t[2][TW][kRows];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int w = 0; w < TW; ++w)
#pragma unroll
          for (int j = 0; j < kRows; ++j) {
            const int* src = stage + (w * acc_cols + min(m0 + stride * j, rows - 1)) * 128;
            t[i][w][j] = ch.sums(p.splits > 1 ? cooperative_groups::this_cluster().map_shared_rank(src, min(x + i, p.splits - 1)) : src);
          }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (x + i < p.splits) {
#pragma unroll
          for (int w = 0; w < TW; ++w)
#pragma unroll
            for (int j = 0; j < kRows; ++j) {
              sum[w][j].x += t[i][w][j].x; sum[w][j].y += t[i][w][j].y; sum[w][j].z += t[i][w][j].z; sum[w][j].w += t[i][w][j].w;
            }
        }
    }
    i8_store<TW, OUT>(p, ch, row0 + m0, stride, row0 + rows, s, sum[0], sum[TW - 1], res);
  }
  // nobody leaves what is being read
  if (p.splits > 1) cooperative_groups::this_cluster().sync();
}

template <int TW, bool PAIR>
OGB_DEVICE bool i8_issue_mma(const Int8Params& p, uint8_t* smem, int stage_bytes, uint32_t tmem_base, int bufs, int acc_cols, RowsBars* bars) {
  const uint32_t idesc = make_idesc_i8(PAIR ? 256 : 128, p.mn);
  int stage = 0;
  uint32_t phase = 0;
  Int8Segs segs(p);
  int tile, kb0, kb1;
  for (int seg = 0; segs.next(tile, kb0, kb1); ++seg) {
    const int buf = bufs == 2 ? (seg & 1) : 0;
    const uint32_t buf_phase = (bufs == 2 ? seg >> 1 : seg) & 1;
    if (!i8_wait<PAIR>(&bars->tmem_empty[buf], buf_phase ^ 1)) return false;
    tc_fence_after();
    const uint32_t d_addr = tmem_base + buf * TW * acc_cols;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!i8_wait<PAIR>(&bars->full[stage], phase)) return false;
      tc_fence_after();
      const uint32_t sw = smem_u32(smem + stage * stage_bytes);
      const uint64_t db = make_kmajor_sw128_desc(sw + TW * 128 * kI8K);
#pragma unroll
      for (int w = 0; w < TW; ++w) {
        const uint64_t da = make_kmajor_sw128_desc(sw + w * 128 * kI8K);
        // 32 values of K an instruction: +2 in the (>> 4) address field
#pragma unroll
        for (int k = 0; k < kI8K / 32; ++k) umma_i8<PAIR>(d_addr + w * acc_cols, da + 2 * k, db + 2 * k, idesc, (kb > kb0 || k > 0) ? 1u : 0u);
      }
      i8_commit<PAIR>(&bars->empty[stage]);
      if (++stage == p.stages) { stage = 0; phase ^= 1; }
    }
    i8_commit<PAIR>(&bars->tmem_full[buf]);
  }
  return true;
}

template <int TW, int OUT, bool PAIR>
__global__ void __launch_bounds__(kI8Threads, 1)
gemm_int8_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_q, const Int8Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr int kStageW = TW * 128 * kI8K;
  const int half = PAIR ? p.mn / 2 : p.mn;                     // rows that this CTA brings
  const int stage_bytes = kStageW + half * kI8K;
  const int ring_bytes = p.stages * stage_bytes;
  RowsBars* bars = reinterpret_cast<RowsBars*>(smem + ring_bytes);
  int* staging = reinterpret_cast<int*>(smem + ring_bytes + kRowsBarBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int acc_cols = (p.mn + 31) / 32 * 32;                  // the reads take 32 columns at a time
  const int bufs = p.splits == 0 && 2 * TW * acc_cols <= 512 ? 2 : 1;
  uint32_t tmem_cols = 32;
  while (static_cast<int>(tmem_cols) < bufs * TW * acc_cols) tmem_cols *= 2;
  // The thread that issues the loads makes the barriers, and has the first ring of W on its way before anything else is set up -- and before
  // the kernel ahead, which makes the rows, has ended.
  int ahead = 0;
  const uint32_t rank = PAIR ? i8_pair_rank() : 0;
  auto load_w = [&](const Int8Cursor& c, int st) {
    if (rank == 0) mbar_expect_tx(&bars->full[st], PAIR ? 2 * stage_bytes : stage_bytes);
#pragma unroll
    for (int w = 0; w < TW; ++w)
      i8_load<PAIR>(smem + st * stage_bytes + w * 128 * kI8K, &tmap_w, &bars->full[st], c.kb * kI8K, (c.nt * TW + w) * 128);
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->tmem_full[i], 1);
      mbar_init(&bars->tmem_empty[i], (PAIR ? 2 : 1) * 4 * kI8Groups);
    }
    bars->abort_flag = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
    if (!PAIR)
      for (Int8Cursor c(p); c.more && ahead < p.stages; c.step()) load_w(c, ahead++);
  }
  if constexpr (PAIR) i8_pair_sync();                          // both CTAs run: tensor memory is allocated on both SMs, and loads of either report to the first one's barriers
  if (warp == 1) {
    if constexpr (PAIR) {
      __syncwarp();
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_slot)), "r"(tmem_cols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(&bars->tmem_slot, tmem_cols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) i8_pair_sync();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_slot;
  pdl_trigger();

  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      if (PAIR)
        for (Int8Cursor c(p); c.more && ahead < p.stages; c.step()) load_w(c, ahead++);
      pdl_wait();
      for (Int8Cursor c(p); c.more; c.step()) {
        if (ahead > 0) {
          --ahead;
        } else {
          if (!i8_wait<PAIR>(&bars->empty[stage], phase ^ 1)) { ok = false; break; }
          load_w(c, stage);
        }
        i8_load<PAIR>(smem + stage * stage_bytes + kStageW, &tmap_q, &bars->full[stage], c.kb * kI8K, c.mt * p.mn + static_cast<int>(rank) * half);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
      // a CTA stays for what the other one's products still report to it
      for (int i = 0; PAIR && ok && i < p.stages; ++i) {
        ok = i8_wait<PAIR>(&bars->empty[stage], phase ^ 1);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
      if (!ok) { atomicOr(p.status, kStatusWaitTimeout); *reinterpret_cast<volatile int*>(&bars->abort_flag) = 1; }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------ MMA issuer ------------------------------
    if (lane == 0 && rank == 0 && !i8_issue_mma<TW, PAIR>(p, smem, stage_bytes, tmem_base, bufs, acc_cols, bars)) {
      atomicOr(p.status, kStatusWaitTimeout);
      *reinterpret_cast<volatile int*>(&bars->abort_flag) = 1;
    }
    __syncwarp();
  } else if (p.splits == 0) {
    i8_epilogue<TW, OUT, PAIR>(p, tmem_base, bufs, acc_cols, bars, staging);
  }
  if constexpr (PAIR) {
    tc_fence_before();
    __syncthreads();
    i8_pair_sync();
    if (*reinterpret_cast<volatile int*>(&bars->abort_flag) != 0 && threadIdx.x == 0) {
      // a wait ran out: copies that may still be in flight get a bounded time to land
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
    __syncthreads();
    i8_pair_sync();
    if (warp == 1) {
      tc_fence_after();
      __syncwarp();
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(tmem_cols) : "memory");
    }
    i8_pair_sync();                                            // neither leaves before the other has given its share back
  } else {
    if (p.splits > 0) i8_finish_cluster<TW, OUT>(p, tmem_base, acc_cols, bars, smem, ring_bytes);
    rows_teardown(bars, tmem_base, tmem_cols);
  }
}

// ----------------------------------------------------------------------------------------
// a handful of rows in one launch
// ----------------------------------------------------------------------------------------
// One user's token leaves the tensor cores idle and the time is launches and latencies: two kernels, barriers, tensor memory, a cluster's sum.
// Here every block turns the rows into 8 bits for itself, in shared memory, while its first weights are on their way, and a warp takes a
// pair of channels (or a gate and its up channel): 16 bytes of each a lane, four products an instruction, a sum over the warp in one more.
constexpr int kGemvThreads = 256;
constexpr int kGemvPieces = 4;               // 16-byte pieces of each channel that a lane has in flight

struct GemvParams {
  const void* x;
  const int8_t* q;                           // or x
  const float* factor;
  const int8_t* w;
  const float* channel;
  const float* bias;
  const void* residual;
  void* out;
  long long ldx, ldq, ldw, ldr, ldc;
  int x_elem, out_elem, x_vec, M, N, K, gated;
};

// 16 bytes of a row of weights from byte k on; what lies past its end is zero.
OGB_DEVICE uint4 gemv_weights(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return __ldcs(reinterpret_cast<const uint4*>(row + k));
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (k + j < K) v[j >> 2] |= (static_cast<uint32_t>(row[k + j]) & 255u) << (8 * (j & 3));
  return make_uint4(v[0], v[1], v[2], v[3]);
}
OGB_DEVICE int dot16(const uint4& a, const uint4& b, int sum) {
  sum = __dp4a(static_cast<int>(a.x), static_cast<int>(b.x), sum);
  sum = __dp4a(static_cast<int>(a.y), static_cast<int>(b.y), sum);
  sum = __dp4a(static_cast<int>(a.z), static_cast<int>(b.z), sum);
  return __dp4a(static_cast<int>(a.w), static_cast<int>(b.w), sum);
}

// ROWS: rows held, at least M.
template <int ROWS>
__global__ void __launch_bounds__(kGemvThreads, 3) gemv_int8_kernel(const GemvParams p) {
  extern __shared__ __align__(16) int8_t codes[];                  // [ROWS][K to a multiple of 16]
  __shared__ uint32_t part[kGemvThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = gridDim.x * (kGemvThreads / 32);
  const int pitch = (p.K + 15) / 16 * 16, n_out = p.gated != 0 ? p.N / 2 : p.N;
  const int pairs = p.gated != 0 ? n_out : (p.N + 1) / 2;
  int pair = blockIdx.x * (kGemvThreads / 32) + warp;
  auto rows_of = [&](int i, int& a, int& b) {
    if (p.gated != 0) {
      a = (i >> 7) * 256 + (i & 127);
      b = a + 128;
    } else {
      a = 2 * i;
      b = min(a + 1, p.N - 1);
    }
  };
  uint4 wa[kGemvPieces], wb[kGemvPieces];
  auto fetch = [&](int i, int k0) {
    int a, b;
    rows_of(i, a, b);
#pragma unroll
    for (int u = 0; u < kGemvPieces; ++u) {
      const int k = k0 + (u * 32 + lane) * 16;
      if (k < p.K) {
        wa[u] = gemv_weights(p.w + static_cast<size_t>(a) * p.ldw, k, p.K);
        wb[u] = gemv_weights(p.w + static_cast<size_t>(b) * p.ldw, k, p.K);
      }
    }
  };
  pdl_trigger();
  if (pair < pairs) fetch(pair, 0);
  pdl_wait();

  // ---- rows to codes ----
  const void* x = after_wait(p.x);
  const int8_t* q = after_wait(p.q);
  float s[ROWS];
  if (q == nullptr) {
    // all rows at once, an equal share of the warps each
    constexpr int kWarps = kGemvThreads / 32 / ROWS, kLanes = 32 * kWarps;
    const int m = warp / kWarps, t = tid - m * kLanes;
    const size_t row = static_cast<size_t>(m) * p.ldx;
    uint32_t peak = 0;
    if (m < p.M) {
#pragma unroll 4
      for (int i = t * 8; i < p.K; i += kLanes * 8) {
        float f[8];
        load8(x, p.x_elem, p.x_vec != 0, row, i, p.K, f);
        peak = max(peak, peak_bits8(f));
      }
    }
    peak = __reduce_max_sync(0xffffffffu, peak);
    if (lane == 0) part[warp] = peak;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      uint32_t top = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = max(top, part[r * kWarps + w]);
      const RowCode code(top);
      s[r] = code.factor;
      if (r == m && m < p.M) {
#pragma unroll 2
        for (int i = t * 8; i < p.K; i += kLanes * 8) {
          float f[8];
          load8(x, p.x_elem, p.x_vec != 0, row, i, p.K, f);
          store_codes(codes, static_cast<size_t>(m) * pitch, i, p.x_elem == kElemF32 ? code.codes(f) : code.codes_short(f));
        }
      }
    }
  } else {
    const float* factor = after_wait(p.factor);
#pragma unroll
    for (int m = 0; m < ROWS; ++m)
      if (m < p.M) {
        s[m] = factor[m];
        for (int i = tid * 16; i < p.K; i += kGemvThreads * 16)
          *reinterpret_cast<uint4*>(codes + static_cast<size_t>(m) * pitch + i) = gemv_weights(q + static_cast<size_t>(m) * p.ldq, i, p.K);
      }
  }
  // store_codes writes eight at a time: the last eight of the pitch may be nobody's
  if (q == nullptr && tid < ROWS && pitch - (p.K + 7) / 8 * 8 == 8 && tid < p.M)
    *reinterpret_cast<uint2*>(codes + static_cast<size_t>(tid) * pitch + pitch - 8) = make_uint2(0, 0);
  __syncthreads();

  for (; pair < pairs; pair += warps) {
    int sum_a[ROWS], sum_b[ROWS];
#pragma unroll
    for (int m = 0; m < ROWS; ++m) sum_a[m] = sum_b[m] = 0;
    for (int k0 = 0; k0 < p.K; k0 += kGemvPieces * 512) {
#pragma unroll
      for (int u = 0; u < kGemvPieces; ++u) {
        const int k = k0 + (u * 32 + lane) * 16;
        if (k < p.K) {
#pragma unroll
          for (int m = 0; m < ROWS; ++m)
            if (m < p.M) {
              const uint4 c = *reinterpret_cast<const uint4*>(codes + static_cast<size_t>(m) * pitch + k);
              sum_a[m] = dot16(wa[u], c, sum_a[m]);
              sum_b[m] = dot16(wb[u], c, sum_b[m]);
            }
        }
      }
      // the next pieces: of this pair, or of the next one
      if (k0 + kGemvPieces * 512 < p.K) fetch(pair, k0 + kGemvPieces * 512);
      else if (pair + warps < pairs) fetch(pair + warps, 0);
    }
    int a, b;
    rows_of(pair, a, b);
    const float ca = __ldg(p.channel + a), cb = __ldg(p.channel + b);
    const float ba = p.bias != nullptr ? __ldg(p.bias + a) : 0.f, bb = p.bias != nullptr ? __ldg(p.bias + b) : 0.f;
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
      sum_a[m] = __reduce_add_sync(0xffffffffu, sum_a[m]);
      sum_b[m] = __reduce_add_sync(0xffffffffu, sum_b[m]);
      if (m >= p.M || lane != m) continue;                        // a lane a row
      float va = fmaf(static_cast<float>(sum_a[m]) * s[m], ca, ba), vb = fmaf(static_cast<float>(sum_b[m]) * s[m], cb, bb);
      const size_t at = static_cast<size_t>(m) * p.ldc, from = static_cast<size_t>(m) * p.ldr;
      if (p.gated != 0) {
        store_elem(p.out, p.out_elem, at + pair, __fdividef(va, 1.f + __expf(-va)) * vb);
        continue;
      }
      if (p.residual != nullptr) {
        va += load_elem(p.residual, p.out_elem, from + a);
        vb += load_elem(p.residual, p.out_elem, from + b);
      }
      store_elem(p.out, p.out_elem, at + a, va);
      if (2 * pair + 1 < p.N) store_elem(p.out, p.out_elem, at + b, vb);
    }
  }
}

// Rows and sizes that this kernel takes (times in us with weights from HBM, tensor cores -> this one).  One row: 1152 x 896 7.8 -> 3.2, 4608 x 3584 11.5 ->
// 7.4, gated 9728 x 896 8.8 -> 5.9, 20000 x 2048 16.2 -> 12.8; but 37888 x 3584 26.7 -> 34.7 and 3584 x 11008, whose blocks all round a long
// row, 15.6 -> 19.3.  Two: 3584 x 3584 10.4 -> 9.3, 20000 x 2048 16.2 -> 14.7.  Four: 4608 x 3584 11.6 -> 14.1.
static bool gemv_applies(int M, int N, int K) { return M <= 2 && M * K <= 8192 && static_cast<long long>(N) * K <= (48ll << 20); }

template <int ROWS>
static int launch_gemv(const GemvParams& p, cudaStream_t stream) {
  const int smem = ROWS * ((p.K + 15) / 16 * 16);
  const int pairs = p.gated != 0 ? p.N / 2 : (p.N + 1) / 2;
  const int grid = std::min((pairs + kGemvThreads / 32 - 1) / (kGemvThreads / 32), 3 * ogb_num_sms());
  return static_cast<int>(launch_overlapped(gemv_int8_kernel<ROWS>, dim3(grid), dim3(kGemvThreads), smem, stream, p));
}

// ----------------------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------------------
// How a product is divided, from its sizes alone.
// Two CTAs, an SM each, share the products of 256 channels and 256 rows: each brings its own channels and half of the rows, so that a k-block
// of 128 x 256 results draws 32 KB through L2 instead of 48, which is what bounds whole tiles (96 bytes a cycle and SM at the tensor cores'
// rate).  It pays where main loops are long and rounds many, us with pairs and without: 8192 rows, 3584 x 18944 347 and 380, 8192 x 8192 335 and 400; 4096,
// 4096 x 4096 52 and 56; 600, 37888 x 3584 70 and 74; but 1024, 8192 x 8192, 1.7 rounds, 70 and 66; 4096, 8192 x 1024 53 and 49, where
// both CTAs' epilogues are waited for.  Gated tiles are no wider for it, having two accumulators each: 2048, 37888 x 3584 240 and 225.
static bool i8_pairs(int M, int N, int K, bool gated, int sms) {
  return !gated && M > 256 && K >= 24 * kI8K && static_cast<long long>((N + 255) / 256) * ((M + 255) / 256) >= 3 * (sms / 2);
}
struct Int8Plan {
  int mn, m_tiles, n_tiles, tiles, k_blocks, cut, units;
  bool clusters, pair;
  long long counter_bytes, ws_bytes;
};
// The rows of a tile come from a score that ranks its heights and is no forecast of times: a k-block of a full tile (128 x 256) counts 0.43, of which 0.1
// are W's; an epilogue 1 and, over 256 rows, 2 more; a cluster's sum 1.5.  It leaves out the stream of W from HBM and counts an epilogue that
// nothing hides too low (5.8 us a tile of 128 x 256, measured at K = 128): 64 rows against 3584 x 18944 score 8.5 and take 19 to 23 us, 1333 against
// 1001 x 2039 4.9 and 12.3, 8192 against 3584 x 18944 423 and 329 to 349.  What stands below is what chose the numbers.  Whole rounds
// waste what the last leaves idle; ranges cost about 80 k-blocks (partial sums written, awaited and added).  What that chooses, and what as few tiles as
// possible take:
//   700 rows against 4608 x 3584: four tiles of 176 rows 17.8 us, three of 240 20.4;  1333, 1001 x 2039: 17 of 80 rows 11.6, six of 224 14.1
//   1000, gated 9728 x 896: eleven of 96 rows 25.6, eight of 128 30.4
//   ranges: 1500, 3584 x 18944 123 -> 93, 8192 419 -> 401; but 2000, 3584 x 3584 49 -> 62, 4096, 8192 x 8192 193 -> 203
static Int8Plan i8_plan(int M, int N, int K, bool gated, int all) {
  Int8Plan r{};
  const int tw = gated ? 2 : 1, most = 256 / tw;
  r.pair = i8_pairs(M, N, K, gated, all);
  const int sms = r.units = r.pair ? all / 2 : all, wide = r.pair ? 2 : 1;
  r.n_tiles = (N + 128 * tw * wide - 1) / (128 * tw * wide);
  r.k_blocks = (K + kI8K - 1) / kI8K;
  const int fewest = (M + most - 1) / most;
  float best = 0.f;
  for (int m_tiles = fewest; m_tiles <= fewest + 24; ++m_tiles) {
    const int mn = ((M + m_tiles - 1) / m_tiles + 16 * wide - 1) / (16 * wide) * (16 * wide);
    const long long tiles = static_cast<long long>(r.n_tiles) * ((M + mn - 1) / mn);
    if (m_tiles > fewest && (tiles > 4 * sms || mn < 32)) break;
    const float part = static_cast<float>(tw * mn) / 256.f, block = 0.1f * tw + 0.33f * part, epilogue = 1.f + 2.f * part;
    float us;
    int cut = 0;
    if (tiles <= sms) {
      const int splits = std::max(1, std::min({kRowsMaxSplit, static_cast<int>(sms / tiles), r.k_blocks / 2}));
      us = static_cast<float>((r.k_blocks + splits - 1) / splits) * block + epilogue + (splits > 1 ? 1.5f : 0.f);
    } else {
      const int rest = static_cast<int>(tiles % sms);
      cut = (sms - rest) * r.k_blocks > 80 * sms && rest > 0 ? rest : 0;
      const float rounds = cut > 0 ? static_cast<float>(tiles) / static_cast<float>(sms) + 80.f / static_cast<float>(r.k_blocks)
                                   : static_cast<float>((tiles + sms - 1) / sms);
      us = rounds * std::max(static_cast<float>(r.k_blocks) * block, epilogue) + epilogue;
    }
    if (m_tiles == fewest || us < 0.97f * best) {
      best = us;
      r.mn = mn;
      r.m_tiles = (M + mn - 1) / mn;
      r.cut = cut;
    }
  }
  r.tiles = r.m_tiles * r.n_tiles;
  r.clusters = !r.pair && r.tiles <= sms;
  if (r.cut > 0) {
    r.counter_bytes = (static_cast<long long>(all) * 4 + 1023) / 1024 * 1024;
    r.ws_bytes = 2ll * all * tw * 128 * ((r.mn + 31) / 32 * 32) * 4;
  }
  return r;
}

template <int TW, int OUT, bool PAIR>
static int launch_int8(const Int8Plan& plan, Int8Params p, const void* q, long long ldq, const void* w, long long ldw, int K, bool early, cudaStream_t stream) {
  auto kernel = gemm_int8_kernel<TW, OUT, PAIR>;
  static OncePerDevice allowed;
  int rc = allow_smem(allowed, kernel, kRowsSmemMax);
  if (rc != 0) return rc;
  const int rows = PAIR ? p.mn / 2 : p.mn, stage_bytes = TW * 128 * kI8K + rows * kI8K;
  const int extra = kRowsBarBytes + (plan.clusters ? 0 : kI8Groups * kI8Stage);
  p.stages = std::min(kRowsMaxStages, (kRowsSmemMax - extra) / stage_bytes);
  const int smem = p.stages * stage_bytes + extra;
  int grid = PAIR ? 2 * plan.units : plan.units;
  if (plan.clusters) {
    p.splits = rows_pick_splits(kernel, kI8Threads, smem, p.tiles, p.k_blocks);
    p.range = p.k_blocks / p.splits;
    p.longer = p.k_blocks % p.splits;
    grid = p.tiles * p.splits;
  }
  CUtensorMap mw, mq;
  rc = make_tmap_u8_2d(&mw, w, p.N, K, ldw, 128, kI8K);
  if (rc != 0) return rc;
  rc = make_tmap_u8_2d(&mq, q, p.M, K, ldq, rows, kI8K);
  if (rc != 0) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kI8Threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (PAIR || p.splits > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = PAIR ? 2 : p.splits;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (early && !PAIR) {      // a pair starts when the kernel ahead has ended: it needs two SMs at once, and is long
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, mw, mq, p));
}

}  // namespace ogb

using namespace ogb;

// Bytes of workspace that a product needs: for its rows (when they come in a float type), its counters and the sums of shared tiles.
static long long i8_rows_bytes(int M, int K) { return (static_cast<long long>(M) * ((K + 15) / 16 * 16) + 255) / 256 * 256; }
static long long i8_factor_bytes(int M) { return (static_cast<long long>(M) * 4 + 255) / 256 * 256; }

extern "C" int64_t ogb_gemm_int8_workspace(int M, int N, int K, int gated, int quantize) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (gemv_applies(M, N, K)) return 0;
  const Int8Plan plan = i8_plan(M, N, K, gated != 0, ogb_num_sms());
  return plan.counter_bytes + plan.ws_bytes + (quantize != 0 ? i8_rows_bytes(M, K) + i8_factor_bytes(M) : 0);
}

extern "C" int ogb_gemm_int8(const void* x, int x_elem, int64_t ldx, const void* q, const float* factor, int64_t ldq, const void* w, int64_t ldw,
                             const float* channel, const float* bias, const void* residual, int64_t ldr, void* out, int64_t ldc, int out_elem, int M, int N,
                             int K, int gated, void* ws, int64_t ws_bytes, int* status, void* stream_) {
  if (M < 0 || N < 0 || K < 1 || K > kI8MaxK || out_elem < 0 || out_elem >= kElemKinds) return -2;
  if (M == 0 || N == 0) return 0;
  if ((x == nullptr) == (q == nullptr) || (x != nullptr && (x_elem < 0 || x_elem >= kElemKinds)) || (q != nullptr && factor == nullptr)) return -5;
  if ((ldw & 15) != 0 || ldw < K || (reinterpret_cast<uintptr_t>(w) & 15) != 0) return -4;
  if (q != nullptr && ((ldq & 15) != 0 || ldq < K || (reinterpret_cast<uintptr_t>(q) & 15) != 0)) return -4;
  if (gated != 0 && (N % 256) != 0) return -6;
  if (static_cast<long long>((M + 15) / 16) * ((N + 127) / 128) > (1 << 30)) return -2;
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (gemv_applies(M, N, K)) {
    const GemvParams p{x, static_cast<const int8_t*>(q), factor, static_cast<const int8_t*>(w), channel, bias, residual, out, ldx, ldq, ldw, ldr, ldc,
                       x_elem, out_elem, rows_aligned(x, ldx, x_elem), M, N, K, gated};
    return M == 1 ? launch_gemv<1>(p, stream) : launch_gemv<2>(p, stream);
  }
  const int sms = ogb_num_sms();
  const Int8Plan plan = i8_plan(M, N, K, gated != 0, sms);
  const bool quantize = q == nullptr;
  const long long rows_bytes = quantize ? i8_rows_bytes(M, K) : 0, factor_bytes = quantize ? i8_factor_bytes(M) : 0;
  if (ws_bytes < rows_bytes + factor_bytes + plan.counter_bytes + plan.ws_bytes || (reinterpret_cast<uintptr_t>(ws) & 255) != 0) return -8;
  uint8_t* at = static_cast<uint8_t*>(ws);
  Int8Params p{};
  p.counters = reinterpret_cast<unsigned int*>(at + rows_bytes + factor_bytes);
  p.ws = reinterpret_cast<int*>(at + rows_bytes + factor_bytes + plan.counter_bytes);
  const int counters = plan.counter_bytes > 0 ? sms : 0;
  bool early = launch_overlap();
  if (quantize) {
    ldq = (K + 15) / 16 * 16;
    float* f = reinterpret_cast<float*>(at + rows_bytes);
    const int rc = launch_quantize_rows(x, reinterpret_cast<int8_t*>(at), f, M, K, ldx, ldq, x_elem, p.counters, counters, stream);
    if (rc != 0) return rc;
    q = at;
    factor = f;
    early = true;          // nothing but the kernel just launched is still running when this one starts: see pdl_wait
  } else if (counters > 0) {
    OGB_CUDA_CHECK(cudaMemsetAsync(p.counters, 0, static_cast<size_t>(counters) * 4, stream));
    early = false;
  }
  p.out = out; p.factor = factor; p.channel = channel; p.bias = bias; p.residual = residual;
  p.ldc = ldc; p.ldr = ldr;
  const int piece = 4 * elem_bytes(out_elem);
  p.vec = (reinterpret_cast<uintptr_t>(out) % piece == 0 && ldc % 4 == 0 &&
           (residual == nullptr || (reinterpret_cast<uintptr_t>(residual) % piece == 0 && ldr % 4 == 0))) ? 1 : 0;
  p.M = M; p.N = N; p.mn = plan.mn; p.n_tiles = plan.n_tiles; p.m_tiles = plan.m_tiles; p.tiles = plan.tiles; p.k_blocks = plan.k_blocks;
  p.pair = plan.pair ? 1 : 0;
  p.cut = plan.cut; p.range = plan.cut * plan.k_blocks / plan.units; p.longer = plan.cut * plan.k_blocks % plan.units; p.status = status;
  auto launch = [&](auto out_type) {
    constexpr int E = decltype(out_type)::value;
    if (gated != 0) return launch_int8<2, E, false>(plan, p, q, ldq, w, ldw, K, early, stream);
    return plan.pair ? launch_int8<1, E, true>(plan, p, q, ldq, w, ldw, K, early, stream) : launch_int8<1, E, false>(plan, p, q, ldq, w, ldw, K, early, stream);
  };
  if (out_elem == kElemF32) return launch(std::integral_constant<int, kElemF32>());
  if (out_elem == kElemBf16) return launch(std::integral_constant<int, kElemBf16>());
  return launch(std::integral_constant<int, kElemF16>());
}

// The same call with its arguments as 64-bit words in their order: a binding that converts every argument by itself spends as long on these as on a
// launch.
extern "C" int ogb_gemm_int8_args(const int64_t* a) {
  auto p = [&](int i) { return reinterpret_cast<void*>(a[i]); };
  auto n = [&](int i) { return static_cast<int>(a[i]); };
  return ogb_gemm_int8(p(0), n(1), a[2], p(3), static_cast<const float*>(p(4)), a[5], p(6), a[7], static_cast<const float*>(p(8)), static_cast<const float*>(p(9)),
                       p(10), a[11], p(12), a[13], n(14), n(15), n(16), n(17), n(18), p(19), a[20], static_cast<int*>(p(21)), p(22));
}
