// Rows of an activation as e4m3 codes with a scale for each block of 128, by themselves and behind the norms around a sublayer.
#include "rows_fp8.h"
#include "api.h"

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// ------------------------------------------------------------------------------ rows

// 16 lanes a block of a row, eight elements each; a wave takes one block of four rows (their scales are four neighbours in
// memory), a workgroup of 16.  Memory bounds it: every element is read once, by one wide load a lane, and nothing is waited for but that
// load.  2048 rows of 4096 bfloat16 elements 6.2 us (25.4 MB: 4.1 TB/s; a copy reaches 4.9), one row 2.4 us, which is a launch.
template <bool VEC>
__global__ __launch_bounds__(256) void quantize_fp8_kernel(const void* __restrict__ x, int x_is_bf16, int ldx, uint8_t* __restrict__ codes,
                                                           int ldq, float* __restrict__ scales, int lds, int rows, int width) {
  const int row = (int)blockIdx.y * 16 + (int)(threadIdx.x >> 4), l = threadIdx.x & 15;
  const int block = blockIdx.x, e = block * BW_FP8_BLOCK + 8 * l;
  const bool in = row < rows;
  const Raw8 raw = load_raw8<VEC>(x, x_is_bf16, (size_t)(in ? row : 0) * ldx, e, width);
  float v[8];
  raw8_floats<VEC>(raw, x_is_bf16, v);
  const Fp8Scale s = fp8_scale_of(row16_max_bits(largest8(v)));
  if (!in) return;
  *reinterpret_cast<u32x2*>(codes + (size_t)row * ldq + e) = (u32x2){fp8_codes4(v[0], v[1], v[2], v[3], s), fp8_codes4(v[4], v[5], v[6], v[7], s)};
  if (l == 0) scales[(size_t)block * lds + row] = s.scale;
}

// ------------------------------------------------------------------------------ the norms around a sublayer

struct NormAddNormArgs {
  const float* x;            // the stream as it was
  const void* y;             // the sublayer's output, or null: the stream is only normed
  const void* post_weight;   // of the norm behind the sublayer, or null
  const void* gate;          // [rows, dim] (ldg > 0) or [dim] (ldg == 0), or null
  const void* scale_vec;     // [dim], or null: the number
  const void* weight;        // of the norm in front of the next sublayer
  float* stream;             // the new stream (may be x)
  void* out;
  float* scales;             // codes: their scales
  int ldx, ldy, ldg, ldst, ldo, lds;
  int y_bf16, post_bf16, gate_bf16, gate_sigmoid, scale_bf16, weight_bf16, out_kind;       // out_kind: 0 float, 1 bfloat16, 2 codes
  float scale, eps, post_eps;
  int dim;
};

enum { OUT_F32 = 0, OUT_BF16 = 1, OUT_FP8 = 2 };

template <bool VEC>
__device__ __forceinline__ void branch_step(const NormAddNormArgs& a, const float (&y)[8], float inv, const Raw8& rp, const Raw8& rg, const Raw8& rs,
                                            float (&x)[8]) {
  float p[8], g[8], s[8];
  if (a.post_weight != nullptr) raw8_floats<VEC>(rp, a.post_bf16, p);
  if (a.gate != nullptr) raw8_floats<VEC>(rg, a.gate_bf16, g);
  if (a.scale_vec != nullptr) raw8_floats<VEC>(rs, a.scale_bf16, s);
  if (a.gate != nullptr && a.gate_sigmoid) {
    // (one by one: eight at a time take registers past 64, and rows of 8,192 their second workgroup a unit: 500 of them 17.0 us for 14.6)
#pragma unroll
    for (int k = 0; k < 8; ++k) with_sigmoids<1>([&](int) { return g[k]; }, [&](int, float open) { g[k] = g[k] != g[k] ? g[k] : open; });
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float z = y[i];
    if (a.post_weight != nullptr) z = (z * inv) * p[i];
    if (a.gate != nullptr) z *= g[i];
    x[i] = fmaf(a.scale_vec != nullptr ? s[i] : a.scale, z, x[i]);
  }
}

template <bool VEC>
__device__ __forceinline__ void store_stream(const NormAddNormArgs& a, size_t row, int e, const float (&x)[8]) {
  float* to = a.stream + row * a.ldst + e;
  if constexpr (VEC) {
    if (e < a.dim) {
      reinterpret_cast<f32x4*>(to)[0] = (f32x4){x[0], x[1], x[2], x[3]};
      reinterpret_cast<f32x4*>(to)[1] = (f32x4){x[4], x[5], x[6], x[7]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e + i < a.dim) to[i] = x[i];
  }
}

// (codes: every lane of a row of 16 lanes comes here, those behind the row's end with zeros)
template <bool VEC>
__device__ __forceinline__ void store_normed(const NormAddNormArgs& a, size_t row, int e, int whole, const float (&x)[8], float inv, const Raw8& rw) {
  float w[8], h[8];
  raw8_floats<VEC>(rw, a.weight_bf16, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = (x[i] * inv) * w[i];
  if (a.out_kind == OUT_FP8) {
    const Fp8Scale s = fp8_scale_of(row16_max_bits(largest8(h)));
    if (e < whole) {
      *reinterpret_cast<u32x2*>((uint8_t*)a.out + row * a.ldo + e) = (u32x2){fp8_codes4(h[0], h[1], h[2], h[3], s), fp8_codes4(h[4], h[5], h[6], h[7], s)};
      if ((e & (BW_FP8_BLOCK - 1)) == 0) a.scales[(size_t)(e / BW_FP8_BLOCK) * a.lds + row] = s.scale;
    }
  } else if (a.out_kind == OUT_BF16) {
    bf16_t* to = (bf16_t*)a.out + row * a.ldo + e;
    if constexpr (VEC) {
      if (e < a.dim)
        *reinterpret_cast<u32x4*>(to) = (u32x4){pack_bf16x2(h[0], h[1]), pack_bf16x2(h[2], h[3]), pack_bf16x2(h[4], h[5]), pack_bf16x2(h[6], h[7])};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e + i < a.dim) to[i] = f32_to_bf16(h[i]);
    }
  } else {
    float* to = (float*)a.out + row * a.ldo + e;
    if constexpr (VEC) {
      if (e < a.dim) {
        reinterpret_cast<f32x4*>(to)[0] = (f32x4){h[0], h[1], h[2], h[3]};
        reinterpret_cast<f32x4*>(to)[1] = (f32x4){h[4], h[5], h[6], h[7]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e + i < a.dim) to[i] = h[i];
    }
  }
}

__device__ __forceinline__ float sumsq8(const float (&v)[8], float acc) {
#pragma unroll
  for (int i = 0; i < 8; ++i) acc = fmaf(v[i], v[i], acc);
  return acc;
}

__device__ __forceinline__ float row_inverse(float acc, float* part, int dim, float eps) {
  acc = wave_sum(acc);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = acc;
  __syncthreads();
  float total = part[0];
  for (int v = 1; v < (int)(blockDim.x >> 6); ++v) total += part[v];
  return 1.0f / sqrtf(total / (float)dim + eps);
}

// A workgroup a row.  WHOLE: as many threads as the row has eights of elements: all loads are asked for first, everything is read
// once.  Otherwise (rows of more than 8,192) thread t has the eights t, t + 1024, ... in passes, and reads the stream back that it
// wrote.  Memory bounds it, and for a few rows the two sums over a row, each behind a barrier: 2048 rows of 4096 with a gate and codes behind
// them 25.9 us (109 MB: 4.2 TB/s; 256 threads with up to four eights each took 30.0), eight rows 4.1 us.
template <bool WHOLE, bool VEC>
__global__ __launch_bounds__(1024) void norm_add_norm_kernel(NormAddNormArgs a) {
  __shared__ float part[2][16];
  const size_t row = blockIdx.x;
  const int whole = a.out_kind == OUT_FP8 ? (a.dim + BW_FP8_BLOCK - 1) / BW_FP8_BLOCK * BW_FP8_BLOCK : a.dim;
  const Raw8 none = {(u32x4){0u, 0u, 0u, 0u}, (u32x4){0u, 0u, 0u, 0u}};
  if constexpr (WHOLE) {
    const int e = 8 * (int)threadIdx.x;
    const Raw8 ry = a.y != nullptr ? load_raw8<VEC>(a.y, a.y_bf16, row * a.ldy, e, a.dim) : none;
    const Raw8 rx = load_raw8<VEC>(a.x, 0, row * a.ldx, e, a.dim);
    const Raw8 rg = a.gate != nullptr ? load_raw8<VEC>(a.gate, a.gate_bf16, row * a.ldg, e, a.dim) : none;
    const Raw8 rp = a.post_weight != nullptr ? load_raw8<VEC>(a.post_weight, a.post_bf16, 0, e, a.dim) : none;
    const Raw8 rs = a.scale_vec != nullptr ? load_raw8<VEC>(a.scale_vec, a.scale_bf16, 0, e, a.dim) : none;
    const Raw8 rw = load_raw8<VEC>(a.weight, a.weight_bf16, 0, e, a.dim);
    float x[8];
    raw8_floats<VEC>(rx, 0, x);
    if (a.y != nullptr) {
      float y[8], inv = 0.0f;
      raw8_floats<VEC>(ry, a.y_bf16, y);
      if (a.post_weight != nullptr) inv = row_inverse(sumsq8(y, 0.0f), part[0], a.dim, a.post_eps);
      branch_step<VEC>(a, y, inv, rp, rg, rs, x);
      store_stream<VEC>(a, row, e, x);
    }
    store_normed<VEC>(a, row, e, whole, x, row_inverse(sumsq8(x, 0.0f), part[1], a.dim, a.eps), rw);
  } else {
    float inv = 0.0f, acc = 0.0f;
    if (a.post_weight != nullptr) {
      for (int e = 8 * (int)threadIdx.x; e < a.dim; e += 8192) {
        float y[8];
        raw8_floats<VEC>(load_raw8<VEC>(a.y, a.y_bf16, row * a.ldy, e, a.dim), a.y_bf16, y);
        acc = sumsq8(y, acc);
      }
      inv = row_inverse(acc, part[0], a.dim, a.post_eps);
    }
    acc = 0.0f;
    for (int e = 8 * (int)threadIdx.x; e < a.dim; e += 8192) {
      float x[8];
      raw8_floats<VEC>(load_raw8<VEC>(a.x, 0, row * a.ldx, e, a.dim), 0, x);
      if (a.y != nullptr) {
        float y[8];
        raw8_floats<VEC>(load_raw8<VEC>(a.y, a.y_bf16, row * a.ldy, e, a.dim), a.y_bf16, y);
        branch_step<VEC>(a, y, inv, a.post_weight != nullptr ? load_raw8<VEC>(a.post_weight, a.post_bf16, 0, e, a.dim) : none,
                         a.gate != nullptr ? load_raw8<VEC>(a.gate, a.gate_bf16, row * a.ldg, e, a.dim) : none,
                         a.scale_vec != nullptr ? load_raw8<VEC>(a.scale_vec, a.scale_bf16, 0, e, a.dim) : none, x);
        store_stream<VEC>(a, row, e, x);
      }
      acc = sumsq8(x, acc);
    }
    const float inv2 = row_inverse(acc, part[1], a.dim, a.eps);
    const float* from = a.y != nullptr ? a.stream + row * a.ldst : a.x + row * a.ldx;
    for (int e = 8 * (int)threadIdx.x; e < ((whole + 127) & ~127); e += 8192) {      // (whole rows of 16 lanes)
      float x[8];
      raw8_floats<VEC>(load_raw8<VEC>(from, 0, 0, e, a.dim), 0, x);
      store_normed<VEC>(a, row, e, whole, x, inv2, load_raw8<VEC>(a.weight, a.weight_bf16, 0, e, a.dim));
    }
  }
}

}  // namespace

extern "C" int bw_quantize_fp8(const void* x, int x_is_bf16, int ldx, void* codes, int ldq, float* scales, int lds, int rows, int width, void* stream) {
  if (rows <= 0) return 0;
  const long long blocks = ((long long)width + BW_FP8_BLOCK - 1) / BW_FP8_BLOCK;
  if (width < 1 || blocks > 0x7fffff || (rows > 1 && (ldx < width || ldq < blocks * BW_FP8_BLOCK)) || lds < rows || rows > 16 * 65535) return -2;
  if (!aligned16(codes) || ldq % 16) return -3;
  const int size = x_is_bf16 ? 2 : 4;
  // (rows that others still read would be written over)
  const Lies at_x = {x, (long long)ldx * size, (long long)width * size, rows, size}, at_codes = {codes, ldq, blocks * BW_FP8_BLOCK, rows, 1},
             at_scales = {scales, 4ll * lds, 4ll * rows, blocks, 4};
  if (meet(at_codes, at_x) || meet(at_scales, at_x) || meet(at_scales, at_codes)) return -2;
  const bool vec = aligned16(x) && width % 8 == 0 && (rows == 1 || (long long)ldx * size % 16 == 0);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, (unsigned)((rows + 15) / 16)), dim3(256), 0, (hipStream_t)stream, x, x_is_bf16, ldx,
                       (uint8_t*)codes, ldq, scales, lds, rows, width);
  };
  if (vec) launch(quantize_fp8_kernel<true>);
  else launch(quantize_fp8_kernel<false>);
  return BW_LAUNCH_CHECK();
}

extern "C" int bw_norm_add_norm(const float* x, int ldx, const void* y, int y_is_bf16, int ldy, const void* post_weight, int post_is_bf16, float post_eps,
                                const void* gate, int gate_is_bf16, int ldg, int gate_sigmoid, const void* scale_vec, int scale_is_bf16, float scale,
                                float* stream_out, int ldst, const void* weight, int weight_is_bf16, float eps, void* out, int out_kind, int ldo,
                                float* scales, int lds, int rows, int dim, void* stream) {
  if (rows <= 0) return 0;
  if (dim < 1 || dim > (1 << 30) || rows > (1 << 21) || out_kind < 0 || out_kind > 2 || (y != nullptr && stream_out == nullptr) || (out_kind == OUT_FP8 && (scales == nullptr || lds < rows)))
    return -2;
  const int ends = out_kind == OUT_FP8 ? (dim + BW_FP8_BLOCK - 1) / BW_FP8_BLOCK * BW_FP8_BLOCK : dim;
  if (rows > 1 && (ldx < dim || ldo < ends || (y != nullptr && (ldy < dim || ldst < dim)) || (gate != nullptr && ldg != 0 && ldg < dim))) return -2;
  if (y == nullptr && (post_weight != nullptr || gate != nullptr || scale_vec != nullptr)) return -2;
  if (out_kind == OUT_FP8 && (!aligned16(out) || ldo % 16)) return -3;
  // A row is read before it is written, by one workgroup: results may lie in the place of what is read element by element, and nowhere else in it
  // (other workgroups still read the rows there), nor in one another.
  const int out_size = out_kind == OUT_FP8 ? 1 : out_kind == OUT_BF16 ? 2 : 4;
  auto rows_at = [&](const void* p, long long ld, long long n, int size) { return Lies{p, ld * size, n * size, rows, size}; };
  auto vector_at = [&](const void* p, int bf16) { return Lies{p, 0, (long long)dim * (bf16 ? 2 : 4), 1, bf16 ? 2 : 4}; };
  const Lies at_out = rows_at(out, ldo, ends, out_size), at_stream = rows_at(y != nullptr ? stream_out : nullptr, ldst, dim, 4),
             at_scales = {out_kind == OUT_FP8 ? scales : nullptr, 4ll * lds, 4ll * rows, (ends + BW_FP8_BLOCK - 1) / BW_FP8_BLOCK, 4};
  const Lies by_element[] = {rows_at(x, ldx, dim, 4), rows_at(y, ldy, dim, y_is_bf16 ? 2 : 4), rows_at(ldg != 0 ? gate : nullptr, ldg, dim, gate_is_bf16 ? 2 : 4)};
  const Lies by_all[] = {vector_at(weight, weight_is_bf16), vector_at(post_weight, post_is_bf16), vector_at(scale_vec, scale_is_bf16),
                         vector_at(ldg == 0 ? gate : nullptr, gate_is_bf16)};
  if (meet(at_out, at_stream) || meet(at_scales, at_out) || meet(at_scales, at_stream)) return -2;
  for (const Lies& in : by_element)
    if (!in_place_or_apart(at_out, in) || !in_place_or_apart(at_stream, in) || meet(at_scales, in)) return -2;
  for (const Lies& in : by_all)
    if (meet(at_out, in) || meet(at_stream, in) || meet(at_scales, in)) return -2;
  NormAddNormArgs a;
  a.x = x, a.y = y, a.post_weight = post_weight, a.gate = gate, a.scale_vec = scale_vec, a.weight = weight, a.stream = stream_out, a.out = out, a.scales = scales;
  a.ldx = ldx, a.ldy = ldy, a.ldg = ldg, a.ldst = ldst, a.ldo = ldo, a.lds = lds;
  a.y_bf16 = y_is_bf16, a.post_bf16 = post_is_bf16, a.gate_bf16 = gate_is_bf16, a.gate_sigmoid = gate_sigmoid, a.scale_bf16 = scale_is_bf16;
  a.weight_bf16 = weight_is_bf16, a.out_kind = out_kind, a.scale = scale, a.eps = eps, a.post_eps = post_eps, a.dim = dim;
  auto fits = [](const void* p, int bf16, long long ld) { return p == nullptr || (aligned16(p) && ld * (bf16 ? 2 : 4) % 16 == 0); };
  const bool vec = dim % 8 == 0 && fits(x, 0, ldx) && fits(y, y_is_bf16, ldy) && fits(post_weight, post_is_bf16, 0) && fits(gate, gate_is_bf16, ldg) &&
                   fits(scale_vec, scale_is_bf16, 0) && fits(weight, weight_is_bf16, 0) && fits(y != nullptr ? stream_out : nullptr, 0, ldst) &&
                   (out_kind == OUT_FP8 || fits(out, out_kind == OUT_BF16, ldo));
  // (whole waves; rows of codes end with whole blocks)
  const int threads = dim > 8192 ? 1024 : (dim + 511) / 512 * 64;
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(threads), 0, (hipStream_t)stream, a); };
  if (dim <= 8192) {
    if (vec) launch(norm_add_norm_kernel<true, true>);
    else launch(norm_add_norm_kernel<true, false>);
  } else {
    if (vec) launch(norm_add_norm_kernel<false, true>);
    else launch(norm_add_norm_kernel<false, false>);
  }
  return BW_LAUNCH_CHECK();
}
