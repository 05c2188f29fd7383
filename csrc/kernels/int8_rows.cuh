// Rows of 8-bit integers with one factor each, the left side of the products of gemm_int8.cu.
//
//   factor = max |x| / 127,   q = round(127 x / max |x|), halves to even
//
// A row of zeros has factor 0; a row that holds an infinity or a NaN has factor NaN and zeros, so that whatever is multiplied by it is NaN.
#pragma once
#include "common.cuh"

namespace ogb {

enum Elem : int { kElemF32 = 0, kElemBf16 = 1, kElemF16 = 2 };
constexpr int kElemKinds = 3;
inline int elem_bytes(int elem) { return elem == kElemF32 ? 4 : 2; }
// every row of a matrix begins at a multiple of 16 bytes
inline int rows_aligned(const void* p, long long ld, int elem) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * elem_bytes(elem) & 15) == 0 ? 1 : 0;
}
// A matrix begins at a multiple of eight values.  Its rows then begin (row * ld) mod 8 values past one, and are taken in pieces of eight that lie at
// such multiples, the first of them so many values in front of the row.
inline bool starts_aligned(const void* p, int elem) { return (reinterpret_cast<uintptr_t>(p) & (8 * elem_bytes(elem) - 1)) == 0; }
OGB_DEVICE int row_shift(int row, long long ld) { return static_cast<int>((static_cast<unsigned>(row) * static_cast<unsigned>(ld & 7)) & 7u); }

OGB_DEVICE float load_elem(const void* p, int elem, size_t at) {
  if (elem == kElemF32) return static_cast<const float*>(p)[at];
  if (elem == kElemBf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
  return __half2float(static_cast<const __half*>(p)[at]);
}
// Eight neighbouring values from column i on of a row that begins at value `row` and has n; zeros past its end.
OGB_DEVICE void load8(const void* p, int elem, bool vec, size_t row, int i, int n, float (&f)[8]) {
  if (vec && i + 8 <= n) {
    if (elem == kElemF32) {
      const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + row + i);
      const float4 a = s[0], b = s[1];
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
      return;
    }
    const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + row + i);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = elem == kElemBf16 ? unpack_bf16(w[j]) : __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      f[2 * j] = t.x;
      f[2 * j + 1] = t.y;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = i + j < n ? load_elem(p, elem, row + i + j) : 0.f;
}
OGB_DEVICE void store_elem(void* p, int elem, size_t at, float v) {
  if (elem == kElemF32) static_cast<float*>(p)[at] = v;
  else if (elem == kElemBf16) static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16(v);
  else static_cast<__half*>(p)[at] = __float2half_rn(v);
}
OGB_DEVICE uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
OGB_DEVICE void store8(void* p, int elem, bool vec, size_t row, int i, int n, const float (&f)[8]) {
  if (vec && i + 8 <= n) {
    if (elem == kElemF32) {
      float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + row + i);
      d[0] = make_float4(f[0], f[1], f[2], f[3]);
      d[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else if (elem == kElemBf16) {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + row + i) =
          make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
    } else {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + row + i) =
          make_uint4(pack_f16(f[0], f[1]), pack_f16(f[2], f[3]), pack_f16(f[4], f[5]), pack_f16(f[6], f[7]));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (i + j < n) store_elem(p, elem, row + i + j, f[j]);
}

// Where rows do not begin at multiples of 16 bytes a thread takes every `step`-th value instead of neighbours, so that a warp's accesses still meet
// whole sectors.  N values from column i on of a row that begins at value `row` and has n; zeros past its end.
template <int N>
OGB_DEVICE void load_strided(const void* p, int elem, size_t row, int i, int step, int n, float (&f)[N]) {
  if (elem == kElemF32) {
    const float* s = static_cast<const float*>(p) + row;
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = i + j * step < n ? s[i + j * step] : 0.f;
  } else if (elem == kElemBf16) {
    const __nv_bfloat16* s = static_cast<const __nv_bfloat16*>(p) + row;
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = i + j * step < n ? __bfloat162float(s[i + j * step]) : 0.f;
  } else {
    const __half* s = static_cast<const __half*>(p) + row;
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = i + j * step < n ? __half2float(s[i + j * step]) : 0.f;
  }
}
template <int N>
OGB_DEVICE void store_strided(void* p, int elem, size_t row, int i, int step, int n, const float (&f)[N]) {
  if (elem == kElemF32) {
    float* d = static_cast<float*>(p) + row;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i + j * step < n) d[i + j * step] = f[j];
  } else if (elem == kElemBf16) {
    __nv_bfloat16* d = static_cast<__nv_bfloat16*>(p) + row;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i + j * step < n) d[i + j * step] = __float2bfloat16(f[j]);
  } else {
    __half* d = static_cast<__half*>(p) + row;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i + j * step < n) d[i + j * step] = __float2half_rn(f[j]);
  }
}

// Eight neighbouring values as they lie in memory.
template <int E>
struct Raw8 {
  static constexpr int kWords = E == kElemF32 ? 8 : 4;
  uint32_t w[kWords];
  // from column i on of a row that begins at value `row` and has n, at a multiple of eight values; zeros in front of it and past its end
  OGB_DEVICE void load(const void* p, size_t row, int i, int n) {
    if (i >= 0 && i + 8 <= n) {
      const uint4* s = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + (row + i) * (E == kElemF32 ? 4 : 2));
      const uint4 a = s[0];
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
      if constexpr (E == kElemF32) {
        const uint4 b = s[1];
        w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
      }
      return;
    }
    edge(p, row, i, n);
  }
  OGB_DEVICE void edge(const void* p, size_t row, int i, int n) {
#pragma unroll
    for (int j = 0; j < kWords; ++j) w[j] = 0;
    if (i + 8 <= 0 || i >= n) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (i + j < 0 || i + j >= n) continue;
      if constexpr (E == kElemF32) w[j] = static_cast<const uint32_t*>(p)[row + i + j];
      else w[j >> 1] |= static_cast<uint32_t>(static_cast<const uint16_t*>(p)[row + i + j]) << (16 * (j & 1));
    }
  }
  OGB_DEVICE void get(float (&f)[8]) const {
    if constexpr (E == kElemF32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(w[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 t = E == kElemBf16 ? unpack_bf16(w[j]) : __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        f[2 * j] = t.x;
        f[2 * j + 1] = t.y;
      }
    }
  }
  // the larger of `m` and the bits of the largest |value|, of both halves of a word for themselves in 16-bit types
  OGB_DEVICE uint32_t peak(uint32_t m) const {
#pragma unroll
    for (int j = 0; j < kWords; ++j) m = E == kElemF32 ? max(m, w[j] & 0x7fffffffu) : __vmaxu2(m, w[j] & 0x7fff7fffu);
    return m;
  }
  // the bits of that as a float; infinities and NaN stay what they are
  OGB_DEVICE static uint32_t peak_float(uint32_t m) {
    if constexpr (E == kElemF32) return m;
    const uint32_t h = max(m >> 16, m & 0xffffu);
    return E == kElemBf16 ? h << 16 : __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(h))));
  }
};

// Two 32-bit floats in one instruction.
struct Float2 {
  unsigned long long v;
  OGB_DEVICE Float2(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
  OGB_DEVICE explicit Float2(float both) : Float2(both, both) {}
  OGB_DEVICE explicit Float2(unsigned long long bits) : v(bits) {}
  OGB_DEVICE float lo() const { return __uint_as_float(static_cast<uint32_t>(v)); }
  OGB_DEVICE float hi() const { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
};
OGB_DEVICE Float2 operator*(Float2 a, Float2 b) { unsigned long long d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a.v), "l"(b.v)); return Float2(d); }
OGB_DEVICE Float2 operator+(Float2 a, Float2 b) { unsigned long long d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a.v), "l"(b.v)); return Float2(d); }
OGB_DEVICE Float2 fma2(Float2 a, Float2 b, Float2 c) { unsigned long long d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a.v), "l"(b.v), "l"(c.v)); return Float2(d); }

// What a row's values are multiplied by.  `peak` holds the bits of max |x|: as whole numbers they are ordered like the values, with
// infinities and NaN above.
struct RowCode {
  float power;       // of two, keeps the row within the range of the type
  float scale;       // 127 times that
  float peak, inv;   // max |x| times that power, and its reciprocal
  float factor;
  bool none;         // zeros, or not a number
  OGB_DEVICE explicit RowCode(uint32_t peak_bits) {
    const bool bad = peak_bits >= 0x7f800000u;
    const float top = bad ? 0.f : __uint_as_float(peak_bits);
    none = !(top > 0.f);
    factor = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(top, 127.f);
    power = top > 0x1p60f ? 0x1p-40f : top < 0x1p-60f ? 0x1p70f : 1.f;
    scale = 127.f * power;
    peak = top * power;
    inv = none ? 0.f : __frcp_rn(peak);
  }
  // Adding 3 * 2^22 rounds to a whole number, halves to even, and leaves it in the low byte of the sum (conversions run at an eighth of the rate
  // of additions).
  static constexpr float kMagic = 12582912.f;
  OGB_DEVICE static uint2 bytes(const uint32_t (&u)[8]) {
    return make_uint2(__byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410));
  }
  // Eight codes of values of 11 bits or fewer (bf16, fp16).  127 x is exact; r, the product with the reciprocal, is within 2^-22 of the quotient, and
  // r + inv (127 x - peak r), whose middle is exact, within a rounding: a quotient that is a half is found as one, and no other comes nearer
  // to a half than 2^-20 of itself (127 x and half * peak are whole multiples of one unit with 19 bits).
  OGB_DEVICE uint2 codes_short(const float (&f)[8]) const {
    uint32_t u[8];
    const Float2 s(scale), v(inv), m(-peak), magic(kMagic);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const Float2 x = Float2(f[j], f[j + 1]) * s, r = x * v;
      const Float2 q = fma2(fma2(m, r, x), v, r) + magic;
      u[j] = __float_as_uint(q.lo());
      u[j + 1] = __float_as_uint(q.hi());
    }
    return none ? make_uint2(0, 0) : bytes(u);
  }
  // Eight codes of any values.  The product with 127 / max |x| is off by less than 2^-15; only where it lies that near to a half is the
  // sign of 127 x - half * peak taken, exactly: both products are split into what they round to and the rest.
  OGB_DEVICE uint2 codes(const float (&f)[8]) const {
    constexpr float kNear = 0.5f - 0x1p-14f;
    float s[8], far = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float r = f[j] * scale * inv;
      s[j] = r + kMagic;
      far = fmaxf(far, fabsf(r - (s[j] - kMagic)));
    }
    if (far > kNear) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = f[j] * power, r = f[j] * scale * inv;
        if (fabsf(r - (s[j] - kMagic)) > kNear) {
          const float below = floorf(r), half = below + 0.5f;
          const float a = x * 127.f, a_rest = fmaf(x, 127.f, -a), b = half * peak, b_rest = fmaf(half, peak, -b);
          const float d = (a - b) + (a_rest - b_rest);       // a - b is exact, the two being that near
          const float even = 2.f * rintf(0.5f * half);       // the even one of the two neighbours
          s[j] = (d > 0.f ? below + 1.f : d < 0.f ? below : even) + kMagic;
        }
      }
    }
    uint32_t u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = __float_as_uint(s[j]);
    return none ? make_uint2(0, 0) : bytes(u);
  }
};
// Eight codes from column i on; rows of q are a multiple of 16 bytes long, so that the last ones may pass the row's end.
OGB_DEVICE void store_codes(int8_t* q, size_t row, int i, uint2 codes) { *reinterpret_cast<uint2*>(q + row + i) = codes; }
// The codes of a row whose pieces begin `shift` values in front of it: the eight of one piece from its `shift`-th on, then of the next.
OGB_DEVICE uint2 shift_codes(uint2 a, uint2 b, int shift) {
  const int bits = 8 * (shift & 3);
  if (shift < 4) return make_uint2(__funnelshift_r(a.x, a.y, bits), __funnelshift_r(a.y, b.x, bits));
  return make_uint2(__funnelshift_r(a.y, b.x, bits), __funnelshift_r(b.x, b.y, bits));
}
OGB_DEVICE void store_codes_strided(int8_t* q, size_t row, int i, int step, int n, uint2 codes) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (i + j * step < n) q[row + i + j * step] = static_cast<int8_t>((j < 4 ? codes.x >> (8 * j) : codes.y >> (8 * (j - 4))) & 255u);
}
OGB_DEVICE uint32_t peak_bits8(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(f[j]) & 0x7fffffffu);
  return m;
}

// Launches the kernel that turns rows of x into codes (int8_rows.cu).  counters: words it sets to zero for the kernel behind it.
int launch_quantize_rows(const void* x, int8_t* q, float* factor, int rows, int cols, long long ldx, long long ldq, int elem, unsigned int* counters,
                         int num_counters, cudaStream_t stream);

}  // namespace ogb
