// Rows as e4m3 codes with a 32-bit scale for each block of 128 elements: what the kernels that leave such rows share
// (quantize_fp8.hip, gemm_fp8.hip).  A row of K elements has whole blocks of codes, zeros behind its end; the scale of block b
// of row r lies at scales[b * ld + r], block by block, so that a product's 16 rows find a block's scales side by side.
//
//   m = max(max |x|, 448 * 2^-126),  scale = m / 448,  code = e4m3(448 x / m), rounded to nearest even
//
// The quotient is the 32-bit number nearest to 448 x / m: the factor 448 / m stays in two parts (with its rounded value alone, or with
// the rounded scale, elements that lie halfway between two codes go to either: of rows of bfloat16 numbers, which have many of those, 1 in
// 2,000, and their values were 2e-3 of the rows' norm off the definition's).  A block of zeros has the scale 2^-126, no quotient
// overflows, and every route to a row gives the same bits.  A block with an infinity or NaN has an infinite or NaN scale and
// NaN for codes: everything in it stands for NaN.
#pragma once

#include "common.h"

#define BW_FP8_BLOCK 128

// The largest of non-negative floats by their bits, which puts NaN above infinity (a float maximum would drop it).
__device__ __forceinline__ uint32_t max_bits(uint32_t a, uint32_t b) { return a > b ? a : b; }

// over the 16 lanes of a row of lanes
__device__ __forceinline__ uint32_t row16_max_bits(uint32_t v) {
  v = max_bits(v, __float_as_uint(lane_xor<8>(__uint_as_float(v))));
  v = max_bits(v, __float_as_uint(lane_xor<4>(__uint_as_float(v))));
  v = max_bits(v, __float_as_uint(lane_xor<2>(__uint_as_float(v))));
  return max_bits(v, __float_as_uint(lane_xor<1>(__uint_as_float(v))));
}

// A block's scale, and 448 / m = hi + lo (off by 2^-47 of it).
struct Fp8Scale {
  float scale, hi, lo;
};

__device__ __forceinline__ Fp8Scale fp8_scale_of(uint32_t amax_bits) {
  const float m = __uint_as_float(max_bits(amax_bits, __float_as_uint(448.0f * 0x1p-126f)));
  const float hi = 448.0f / m;
  return {m / 448.0f, hi, (fmaf(-hi, m, 448.0f) * (1.0f / 448.0f)) * hi};
}

// Four codes of four values.
__device__ __forceinline__ uint32_t fp8_codes4(float a, float b, float c, float d, const Fp8Scale& s) {
  auto quotient = [&](float x) { return fmaf(x, s.hi, x * s.lo); };
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(a), quotient(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(quotient(c), quotient(d), v, true);
}

// Eight consecutive elements as they come from memory: 16 bytes of bfloat16 or 32 of floats.  The load is a step of its own, so
// that a caller can ask for everything before anything is waited for.
struct Raw8 {
  u32x4 a, b;
};

// Elements e .. e + 7 of ``p``, those from ``end`` on as zeros.  VEC: 16-byte loads (aligned, ``end`` a multiple of 8);
// otherwise one element at a time, left as floats.
template <bool VEC>
__device__ __forceinline__ Raw8 load_raw8(const void* p, int is_bf16, size_t row_at, int e, int end) {
  Raw8 r;
  r.a = r.b = (u32x4){0u, 0u, 0u, 0u};
  if constexpr (VEC) {
    if (e < end) {
      if (is_bf16) {
        r.a = *reinterpret_cast<const u32x4*>((const bf16_t*)p + row_at + e);
      } else {
        r.a = *reinterpret_cast<const u32x4*>((const float*)p + row_at + e);
        r.b = *reinterpret_cast<const u32x4*>((const float*)p + row_at + e + 4);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t v = 0u;
      if (e + i < end) v = is_bf16 ? (uint32_t)((const bf16_t*)p)[row_at + e + i] << 16 : ((const uint32_t*)p)[row_at + e + i];
      if (i < 4) r.a[i] = v;
      else r.b[i - 4] = v;
    }
  }
  return r;
}

template <bool VEC>
__device__ __forceinline__ void raw8_floats(const Raw8& r, int is_bf16, float (&v)[8]) {
  if (VEC && is_bf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(r.a[i] << 16);
      v[2 * i + 1] = __uint_as_float(r.a[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = __uint_as_float(r.a[i]);
      v[4 + i] = __uint_as_float(r.b[i]);
    }
  }
}

__device__ __forceinline__ uint32_t largest8(const float (&v)[8]) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max_bits(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

// 1 / (1 + exp(-g)) within two units in the last place: codes are rounded from it, and what is more off moves more of them to
// a neighbour.  The exponential through the hardware exp2, its argument in two parts; the quotient through the hardware
// reciprocal and one Newton step.  Beyond 88 the argument stays there, which gives 1.  For g of -87 and more: below, the quotient lies
// under the normal numbers, which the reciprocal does not give.  NaN gives a number.
__device__ __forceinline__ float sigmoid_from_87(float g) {
  const float x = fminf(fmaxf(-g, -88.0f), 88.0f);
  const float hi = x * 0x1.715476p+0f;
  const float lo = fmaf(x, 0x1.715476p+0f, -hi) + x * 0x1.4ae0cp-26f;
  const float d = fmaf(__builtin_amdgcn_exp2f(hi), fmaf(lo, 0x1.62e43p-1f, 1.0f), 1.0f);
  const float r = __builtin_amdgcn_rcpf(d);
  return fmaf(fmaf(-d, r, 1.0f), r, r);
}

// The same for g under -87, where it is exp(g) but for e^-87 of it: 2^96 times that, scaled by one product, which rounds it to within the
// least number.  Beyond -112 the argument stays there: less than half of the least number.
__device__ __forceinline__ float sigmoid_under_87(float g) {
  const float x = fmaxf(g, -112.0f);
  const float hi = x * 0x1.715476p+0f;
  const float lo = fmaf(x, 0x1.715476p+0f, -hi) + x * 0x1.4ae0cp-26f;
  return (__builtin_amdgcn_exp2f(96.0f + hi) * fmaf(lo, 0x1.62e43p-1f, 1.0f)) * 0x1p-96f;
}

// use(i, sigmoid(g(i))) for i below N, all numbers.  Gates under -87 are rare: a wave looks for them once for all N.  (Chosen element by
// element without a branch, silu behind 39 x 12032 x 1012 took 13.2 us for 12.6, behind 2048 x 8192 x 512 57.6 for 54.0.)
template <int N, typename G, typename Use>
__device__ __forceinline__ void with_sigmoids(G g, Use use) {
  float least = g(0);
#pragma unroll
  for (int i = 1; i < N; ++i) least = fminf(least, g(i));
  if (__builtin_amdgcn_ballot_w64(least < -87.0f) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) use(i, sigmoid_from_87(g(i)));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) use(i, g(i) < -87.0f ? sigmoid_under_87(g(i)) : sigmoid_from_87(g(i)));
  }
}

// ------------------------------------------------------------------------------ where a call's matrices lie (host)

// ``rows`` rows of ``wide`` bytes that begin ``apart`` bytes from one another, in elements of ``size`` bytes; at null: not there.
struct Lies {
  const void* at;
  long long apart, wide;
  long long rows;
  int size;
};

// Whether two share memory.  Rows an equal distance apart may lie beside one another, as columns of one wider matrix.
static inline bool meet(const Lies& a, const Lies& b) {
  if (a.at == nullptr || b.at == nullptr || a.rows < 1 || b.rows < 1) return false;
  const long long a0 = (long long)(uintptr_t)a.at, b0 = (long long)(uintptr_t)b.at;
  if (a0 + (a.rows - 1) * a.apart + a.wide <= b0 || b0 + (b.rows - 1) * b.apart + b.wide <= a0) return false;
  const long long apart = a.rows > 1 ? a.apart : b.apart;
  if ((a.rows == 1 && b.rows == 1) || (a.rows > 1 && b.rows > 1 && a.apart != b.apart) || apart <= 0) return true;
  const long long behind = ((b0 - a0) % apart + apart) % apart;
  return behind < a.wide || behind + b.wide > apart;
}

// Whether an output keeps out of what a kernel reads element by element: apart from it, or in its place, element for element.
static inline bool in_place_or_apart(const Lies& out, const Lies& in) {
  return !meet(out, in) || (out.at == in.at && out.size == in.size && out.wide == in.wide && (out.rows == 1 || out.apart == in.apart));
}
