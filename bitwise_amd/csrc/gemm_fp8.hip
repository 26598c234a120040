// Products of rows of e4m3 codes with matrices of e4m3 codes, a 32-bit scale for each 128 of a row's elements and for each
// 128 x 128 block of the matrix:
//
//   y[m][n] = sum over blocks b of  (xs[b][m] * ws[n / 128][b]) * (sum over k in b of x[m][k] * w[n][k])
//
// A block's inner sum is four v_mfma_f32_16x16x32_bf16 from zero, the outer sum one chain of 32-bit multiply-adds, b ascending.
// Whichever kernel runs decides only which outputs share their loads: a row's bits do not depend on the rows beside it.
//
// Why not the 8-bit matrix instructions, which are twice as fast: they add up eight products at a time with no bits below
// 2^-13 of the largest of the eight (measured: 2^16 + 2^3 is exact, 2^16 + 2^2 is not, with 16x16x32 as with 16x16x128 and 32x32x64),
// which leaves a sum of 128 normal products 1.2 to 2.7e-5 of their norm off, 100 times what 32-bit sums are off.  Codes are exact as
// bfloat16, and the bfloat16 instructions' sums of their products are off by 1e-8.  The conversion, two codes an instruction at the rate
// of a multiply-add, runs beside the matrix instructions.
//
// Rows of codes and of the matrix have whole blocks (zeros behind the inner size).
#include "rows_fp8.h"
#include "api.h"

namespace {

// What becomes of the sums.
enum { STORE_F32 = 0, STORE_BF16 = 1, SWIGLU_F32 = 2, SWIGLU_FP8 = 3 };

struct Fp8Args {
  const uint8_t* x;
  const float* xs;
  const uint8_t* w;
  const float* ws;
  const float* residual;     // added to the sums (STORE_F32), or null
  void* out;
  float* out_scales;         // SWIGLU_FP8
  int ldx, ldxs, ldr, ldo, lds;
  int M, N, K;               // N: output columns (gated: half the matrix's rows); K: the padded inner size
  int m_tiles, n_tiles;
};

// A block's 128 codes of 16 rows as the matrix instructions take them: lane (g, r) has row r's bytes 16 g and 64 + 16 g of the block
// (the same permutation of k on both sides), eight bytes for each of four instructions.
struct Frag {
  bf16x8 t[4];
};

__device__ __forceinline__ uint32_t codes_to_bf16x2(uint32_t four, bool upper) {
  // (the scale has to be a constant operand, the half a constant too)
  return upper ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, 1.0f, true))
               : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, 1.0f, false));
}

__device__ __forceinline__ Frag frag_of(u32x4 lo, u32x4 hi) {
  Frag f;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const u32x4 v = t < 2 ? lo : hi;
    const uint32_t a = v[2 * (t & 1)], b = v[2 * (t & 1) + 1];
    f.t[t] = as_bf16x8((u32x4){codes_to_bf16x2(a, false), codes_to_bf16x2(a, true), codes_to_bf16x2(b, false), codes_to_bf16x2(b, true)});
  }
  return f;
}

// One block's sums of 16 matrix rows and 16 rows of x: of the result, lane (g, r) has rows 4 g .. 4 g + 3 of the matrix for row r of x:
// four neighbouring outputs.
__device__ __forceinline__ f32x4 block_sums(const Frag& w, const Frag& x) {
  f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < 4; ++t) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.t[t], x.t[t], p, 0, 0, 0);
  return p;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const void* base, size_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
}

constexpr int OUTSIDE = 0x7fff0000;           // an offset behind every descriptor's end: reads as zeros, asks memory for nothing

__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);         // this wave's LDS work, not its loads
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <int EPI>
__device__ __forceinline__ void store_one(const Fp8Args& a, int m, int n, float y, float u) {
  if constexpr (EPI == STORE_BF16) {
    ((bf16_t*)a.out)[(size_t)m * a.ldo + n] = f32_to_bf16(y);
  } else if constexpr (EPI == SWIGLU_F32) {
    ((float*)a.out)[(size_t)m * a.ldo + n] = silu32_times(y, u);
  } else {
    if (a.residual != nullptr) y = a.residual[(size_t)m * a.ldr + n] + y;
    ((float*)a.out)[(size_t)m * a.ldo + n] = y;
  }
}

// ------------------------------------------------------------------------------ few rows

// Up to 64 rows: a workgroup of NW waves a strip of 16 matrix rows (gated: 16 gate and 16 up rows).  In round t wave v
// computes the sums of block t NW + v; they meet in LDS, where the threads that own the outputs walk them in order.
template <int WM, int EPI, int NW, int D>
__global__ __launch_bounds__(64 * NW) void gemm_fp8_few_kernel(Fp8Args a) {
  constexpr int NB = EPI == SWIGLU_F32 ? 2 : 1;
  constexpr int OWN = (WM * 256 + 64 * NW - 1) / (64 * NW);
  __shared__ __attribute__((aligned(16))) float part[2][NW][NB][WM][256];
  __shared__ float factor[2][NW][NB][WM * 16];
  const int wave = wave_index(), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, KB = a.K / BW_FP8_BLOCK;
  const int w_rows = min(16, a.N - n0);
  __amdgpu_buffer_rsrc_t rs_w[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) rs_w[b] = rows_of(a.w + ((size_t)b * a.N + n0) * a.K, (size_t)w_rows * a.K);
  const __amdgpu_buffer_rsrc_t rs_x = rows_of(a.x, (size_t)(a.M - 1) * a.ldx + a.K);
  const int voff_w = r * a.K + 16 * g;
  int voff_x[WM], row_m[WM];
#pragma unroll
  for (int i = 0; i < WM; ++i) {
    voff_x[i] = 16 * i + r < a.M ? (16 * i + r) * a.ldx + 16 * g : OUTSIDE;
    row_m[i] = min(16 * i + r, a.M - 1);
  }
  const float* ws_row[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) ws_row[b] = a.ws + ((size_t)(n0 / BW_FP8_BLOCK) + (size_t)b * ((a.N + BW_FP8_BLOCK - 1) / BW_FP8_BLOCK)) * KB;

  u32x4 wq[D][NB][2], xq[D][WM][2];
  float sx[D][WM], sw[D][NB];
  auto issue = [&](int d, int round) {
    const int blk = min(round * NW + wave, KB - 1);            // (past the end: the last block again, whose sums nobody takes)
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      wq[d][b][0] = __builtin_amdgcn_raw_buffer_load_b128(rs_w[b], voff_w, blk * BW_FP8_BLOCK, 0);
      wq[d][b][1] = __builtin_amdgcn_raw_buffer_load_b128(rs_w[b], voff_w + 64, blk * BW_FP8_BLOCK, 0);
    }
#pragma unroll
    for (int i = 0; i < WM; ++i) {
      xq[d][i][0] = __builtin_amdgcn_raw_buffer_load_b128(rs_x, voff_x[i], blk * BW_FP8_BLOCK, 0);
      xq[d][i][1] = __builtin_amdgcn_raw_buffer_load_b128(rs_x, voff_x[i] + 64, blk * BW_FP8_BLOCK, 0);
    }
#pragma unroll
    for (int i = 0; i < WM; ++i) sx[d][i] = a.xs[(size_t)blk * a.ldxs + row_m[i]];
#pragma unroll
    for (int b = 0; b < NB; ++b) sw[d][b] = ws_row[b][blk];
  };
  const int rounds = (KB + NW - 1) / NW;
#pragma unroll
  for (int d = 0; d < D; ++d) issue(d, d);
  __builtin_amdgcn_sched_barrier(0);
  float acc[NB][OWN];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int o = 0; o < OWN; ++o) acc[b][o] = 0.0f;
  for (int t0 = 0; t0 < rounds; t0 += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int t = t0 + d;
      if (t < rounds) {                                          // (scalar)
        const int buf = t & 1;
        Frag fw[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) fw[b] = frag_of(wq[d][b][0], wq[d][b][1]);
#pragma unroll
        for (int i = 0; i < WM; ++i) {
          const Frag fx = frag_of(xq[d][i][0], xq[d][i][1]);
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            *reinterpret_cast<f32x4*>(&part[buf][wave][b][i][4 * lane]) = block_sums(fw[b], fx);
            if (g == 0) factor[buf][wave][b][16 * i + r] = sx[d][i] * sw[d][b];
          }
        }
        issue(d, t + D);
        __builtin_amdgcn_sched_barrier(0);
        lds_barrier();
        const int here = min(NW, KB - t * NW);
#pragma unroll
        for (int o = 0; o < OWN; ++o) {
          const int at = (int)threadIdx.x + o * 64 * NW;
          if (at < WM * 256) {
            const int i = at >> 8, m = 16 * i + ((at >> 2) & 15);
            auto walk = [&](int v) {
#pragma unroll
              for (int b = 0; b < NB; ++b) acc[b][o] = fmaf(factor[buf][v][b][m], part[buf][v][b][i][at & 255], acc[b][o]);
            };
            if (here == NW) {
#pragma unroll
              for (int v = 0; v < NW; ++v) walk(v);
            } else {
              for (int v = 0; v < here; ++v) walk(v);
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int o = 0; o < OWN; ++o) {
    const int at = (int)threadIdx.x + o * 64 * NW;
    const int m = 16 * (at >> 8) + ((at >> 2) & 15), n = n0 + 4 * ((at >> 6) & 3) + (at & 3);
    if (at < WM * 256 && m < a.M && n < a.N) store_one<EPI>(a, m, n, acc[0][o], acc[NB - 1][o]);
  }
}

// ------------------------------------------------------------------------------ tiles

// A workgroup of eight waves computes BM rows times BN matrix rows (gated: BN / 2 gate and BN / 2 up rows) in steps of one
// block of 128; both operands travel from memory straight into LDS, some steps ahead.  The waves lie WY x 8 / WY over the tile,
// each with MI x NJ results of 16 x 16.  One load of a wave brings 8 rows of a step, 128 bytes each, into 1 KB of LDS, lane l's 16
// bytes to 16 l; slot c' of row r (within its block of 16 rows) holds the row's chunk c' ^ (r >> 1), so that the 16 lanes that
// read one chunk of 16 rows hit 16 different groups of banks.
template <int EPI, int WY_, int MI_, int NJ_>
struct Fp8Tile {
  static constexpr int WY = WY_, WX = 8 / WY_, MI = MI_, NJ = NJ_;
  static constexpr bool GLU = EPI == SWIGLU_FP8;
  static constexpr int BM = 16 * WY * MI, BN = 16 * WX * NJ, COLS = GLU ? BN / 2 : BN;
  static constexpr int A_SLOT = BM * 128, B_SLOT = BN * 128, STEP = A_SLOT + B_SLOT;
  static constexpr int LA = BM / 64, LB = BN / 64;
  static constexpr int ST = 160 * 1024 / STEP >= 4 ? 4 : 160 * 1024 / STEP;
  static constexpr int BYTES = ST * STEP;
  static_assert(BM % 64 == 0 && BN % 64 == 0 && ST >= 2 && 128 % (16 * (GLU ? NJ / 2 : NJ)) == 0 && (!GLU || COLS == 128), "tile shapes");
};

template <int EPI, int WY, int MI, int NJ>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void gemm_fp8_tiles_kernel(Fp8Args a) {
  using T = Fp8Tile<EPI, WY, MI, NJ>;
  constexpr bool GLU = T::GLU;
  constexpr int BM = T::BM, COLS = T::COLS, NH = GLU ? NJ / 2 : NJ, NB = GLU ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) unsigned char ring[];
  const int wave = wave_index(), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wy = wave / T::WX, wx = wave % T::WX;
  // consecutive workgroups go to different dies: die d takes a run of tiles, so that an n tile's workgroups share a die
  const int nblocks = a.m_tiles * a.n_tiles, die = blockIdx.x & 7;
  const int bid = die * (nblocks >> 3) + min(die, nblocks & 7) + (int)(blockIdx.x >> 3);
  const int m0 = (bid % a.m_tiles) * BM, n0 = (bid / a.m_tiles) * COLS;
  const int KB = a.K / BW_FP8_BLOCK;

  const int a_rows = min(BM, a.M - m0), b_rows = min(COLS, a.N - n0);
  const bool up = GLU && wave >= 4;
  const __amdgpu_buffer_rsrc_t rs_a = rows_of(a.x + (size_t)m0 * a.ldx, (size_t)(a_rows - 1) * a.ldx + a.K);
  const __amdgpu_buffer_rsrc_t rs_b = rows_of(a.w + ((size_t)(up ? a.N : 0) + n0) * a.K, (size_t)b_rows * a.K);
  const int lrow = lane >> 3, lslot = lane & 7;
  int voff_a[4], voff_b[4];
#pragma unroll
  for (int t = 0; t < T::LA; ++t) {
    const int row = 8 * (T::LA * wave + t) + lrow;
    voff_a[t] = row < a_rows ? row * a.ldx + 16 * (lslot ^ ((row & 15) >> 1)) : OUTSIDE;
  }
#pragma unroll
  for (int t = 0; t < T::LB; ++t) {
    const int row = 8 * (T::LB * wave + t) + lrow;
    voff_b[t] = (up ? row - COLS : row) * a.K + 16 * (lslot ^ ((row & 15) >> 1));
  }
  typedef __attribute__((address_space(3))) void* lds_ptr;
  auto issue = [&](int step, int slot) {
#pragma unroll
    for (int t = 0; t < T::LA; ++t)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_a, (lds_ptr)(ring + slot * T::STEP + (T::LA * wave + t) * 1024), 16,
                                               step < KB ? voff_a[t] : OUTSIDE, step * 128, 0, 0);
#pragma unroll
    for (int t = 0; t < T::LB; ++t)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_b, (lds_ptr)(ring + slot * T::STEP + T::A_SLOT + (T::LB * wave + t) * 1024), 16,
                                               step < KB ? voff_b[t] : OUTSIDE, step * 128, 0, 0);
  };
  // the scales of this wave's rows and columns for a step
  int row_m[8];
#pragma unroll
  for (int i = 0; i < MI; ++i) row_m[i] = min(m0 + 16 * (MI * wy + i) + r, a.M - 1);
  const float* ws_row[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
    ws_row[b] = a.ws + ((size_t)((n0 + 16 * NH * wx) / BW_FP8_BLOCK) + (size_t)b * ((a.N + BW_FP8_BLOCK - 1) / BW_FP8_BLOCK)) * KB;
  if (n0 + 16 * NH * wx >= a.N) {               // (columns past the matrix: any scale will do)
#pragma unroll
    for (int b = 0; b < NB; ++b) ws_row[b] = a.ws;
  }
  float sx[8], sw[2];
  auto scales = [&](int step) {
    const int s = min(step, KB - 1);
#pragma unroll
    for (int i = 0; i < MI; ++i) sx[i] = a.xs[(size_t)s * a.ldxs + row_m[i]];
#pragma unroll
    for (int b = 0; b < NB; ++b) sw[b] = ws_row[b][s];
  };

  f32x4 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int row_off = (r >> 3) * 1024 + (r & 7) * 128;
  int slot_off[2];
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) slot_off[kk] = row_off + (((4 * kk + g) ^ (r >> 1)) * 16);

  scales(0);
#pragma unroll
  for (int st = 0; st < T::ST - 1; ++st) issue(st, st);
  int slot = 0;
  for (int step = 0; step < KB; ++step) {
    // all but the loads of the ST - 2 steps behind this one
    __builtin_amdgcn_s_waitcnt(vmcnt_only((T::ST - 2) * (T::LA + T::LB)) & ~0x0f00);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    float f[8][2];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int b = 0; b < NB; ++b) f[i][b] = sx[i] * sw[b];
    scales(step + 1);
    issue(step + T::ST - 1, slot == 0 ? T::ST - 1 : slot - 1);
    const unsigned char* at_a = ring + slot * T::STEP;
    const unsigned char* at_b = at_a + T::A_SLOT;
    Frag fb[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int blk = GLU ? (NH * wx + j % NH) + (j / NH) * (T::BN / 32) : NJ * wx + j;
      fb[j] = frag_of(*reinterpret_cast<const u32x4*>(at_b + blk * 2048 + slot_off[0]), *reinterpret_cast<const u32x4*>(at_b + blk * 2048 + slot_off[1]));
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const unsigned char* at = at_a + (MI * wy + i) * 2048;
      const Frag fa = frag_of(*reinterpret_cast<const u32x4*>(at + slot_off[0]), *reinterpret_cast<const u32x4*>(at + slot_off[1]));
      f32x4 p[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) p[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < NJ; ++j) p[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j].t[t], fa.t[t], p[j], 0, 0, 0);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const float s = f[i][GLU ? j / NH : 0];
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[i][j][q] = fmaf(s, p[j][q], acc[i][j][q]);
      }
    }
    slot = slot + 1 == T::ST ? 0 : slot + 1;
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_only(0));                       // the padding loads too, before LDS is used again or the waves end

  if constexpr (GLU) {
    // silu(g) u, the largest magnitude of each row's 128 outputs over lanes and waves, codes
    __syncthreads();
    uint32_t* most = reinterpret_cast<uint32_t*>(ring);            // [WX][BM]
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      uint32_t mx = 0u;
#pragma unroll
      for (int j = 0; j < NH; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          acc[i][j][q] = silu32_times(acc[i][j][q], acc[i][NH + j][q]);
          mx = max_bits(mx, __float_as_uint(acc[i][j][q]) & 0x7fffffffu);
        }
      float lo, hi;
      lane_halves<32>(__uint_as_float(mx), lo, hi);
      mx = max_bits(__float_as_uint(lo), __float_as_uint(hi));
      lane_halves<16>(__uint_as_float(mx), lo, hi);
      mx = max_bits(__float_as_uint(lo), __float_as_uint(hi));
      if (g == 0) most[wx * BM + 16 * (MI * wy + i) + r] = mx;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int row = 16 * (MI * wy + i) + r, m = m0 + row;
      uint32_t mx = 0u;
#pragma unroll
      for (int v = 0; v < T::WX; ++v) mx = max_bits(mx, most[v * BM + row]);
      const float scale = fp8_scale_of(mx);
      const float inv = 1.0f / scale;
      if (m < a.M) {
#pragma unroll
        for (int j = 0; j < NH; ++j)
          *reinterpret_cast<uint32_t*>((uint8_t*)a.out + (size_t)m * a.ldo + n0 + 16 * (NH * wx + j) + 4 * g) =
              fp8_codes4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3], inv);
        if (wx == 0 && g == 0) a.out_scales[(size_t)(n0 / BW_FP8_BLOCK) * a.lds + m] = scale;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m = m0 + 16 * (MI * wy + i) + r;
      if (m >= a.M) continue;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n0 + 16 * (NJ * wx + j) + 4 * g + q;
          if (n < a.N) store_one<EPI>(a, m, n, acc[i][j][q], 0.0f);
        }
    }
  }
}

// ------------------------------------------------------------------------------ which kernel

template <int WM, int EPI>
void launch_few(const Fp8Args& a, hipStream_t s) {
  constexpr int NW = EPI == SWIGLU_F32 ? (WM == 1 ? 8 : 4) : (WM <= 2 ? 8 : 4);
  constexpr int D = WM == 1 ? 4 : 2;
  hipLaunchKernelGGL((gemm_fp8_few_kernel<WM, EPI, NW, D>), dim3((a.N + 15) / 16), dim3(64 * NW), 0, s, a);
}

template <int EPI>
int few_rows(const Fp8Args& a, hipStream_t s) {
  switch ((a.M + 15) / 16) {
    case 1: launch_few<1, EPI>(a, s); break;
    case 2: launch_few<2, EPI>(a, s); break;
    case 3: launch_few<3, EPI>(a, s); break;
    default: launch_few<4, EPI>(a, s); break;
  }
  return BW_LAUNCH_CHECK();
}

template <int EPI, int WY, int MI, int NJ>
int launch_tiles(Fp8Args a, hipStream_t s) {
  using T = Fp8Tile<EPI, WY, MI, NJ>;
  a.m_tiles = (a.M + T::BM - 1) / T::BM;
  a.n_tiles = (a.N + T::COLS - 1) / T::COLS;
  hipLaunchKernelGGL((gemm_fp8_tiles_kernel<EPI, WY, MI, NJ>), dim3((unsigned)(a.m_tiles * a.n_tiles)), dim3(512), T::BYTES, s, a);
  return BW_LAUNCH_CHECK();
}

bool aligned(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

constexpr int FEW_ROWS = 64;

// sizes that every entry point refuses
int sizes_wrong(const void* x, int ldx, int ldxs, const void* w, int rows, int N, int K) {
  if (N < 1 || K < BW_FP8_BLOCK || K % BW_FP8_BLOCK || K > (1 << 22) || N > (1 << 24) || rows > (1 << 22) || (rows > 1 && ldx < K) || ldxs < rows) return -2;
  if ((long long)256 * ldx > 0x7fff0000ll) return -2;            // (a tile's rows lie in one descriptor)
  if (!aligned(x, 16) || !aligned(w, 16) || ldx % 16) return -3;
  return 0;
}

}  // namespace

extern "C" int bw_gemm_fp8(const void* x, int ldx, const float* xs, int ldxs, const void* w, const float* ws, const float* residual, int ldr, void* out,
                           int ldo, int out_is_bf16, int rows, int N, int K, void* stream) {
  if (rows <= 0) return 0;
  if (const int bad = sizes_wrong(x, ldx, ldxs, w, rows, N, K)) return bad;
  if (rows > 1 && (ldo < N || (residual != nullptr && ldr < N))) return -2;
  if (out_is_bf16 && residual != nullptr) return -2;
  Fp8Args a = {};
  a.x = (const uint8_t*)x, a.xs = xs, a.w = (const uint8_t*)w, a.ws = ws, a.residual = residual, a.out = out;
  a.ldx = ldx, a.ldxs = ldxs, a.ldr = ldr, a.ldo = ldo, a.M = rows, a.N = N, a.K = K;
  hipStream_t s = (hipStream_t)stream;
  if (rows <= FEW_ROWS) return out_is_bf16 ? few_rows<STORE_BF16>(a, s) : few_rows<STORE_F32>(a, s);
  if (out_is_bf16) return launch_tiles<STORE_BF16, 2, 4, 4>(a, s);
  return launch_tiles<STORE_F32, 2, 4, 4>(a, s);
}

extern "C" int bw_gemm_fp8_swiglu(const void* x, int ldx, const float* xs, int ldxs, const void* w, const float* ws, float* sums, int ldsums, void* codes,
                                  int ldq, float* scales, int lds, int rows, int inter, int K, void* stream) {
  if (rows <= 0) return 0;
  if (const int bad = sizes_wrong(x, ldx, ldxs, w, rows, inter, K)) return bad;
  const int whole = (inter + BW_FP8_BLOCK - 1) / BW_FP8_BLOCK * BW_FP8_BLOCK;
  if ((rows > 1 && ldq < whole) || lds < rows) return -2;
  if (!aligned(codes, 16) || ldq % 16) return -3;
  Fp8Args a = {};
  a.x = (const uint8_t*)x, a.xs = xs, a.w = (const uint8_t*)w, a.ws = ws;
  a.ldx = ldx, a.ldxs = ldxs, a.M = rows, a.N = inter, a.K = K;
  hipStream_t s = (hipStream_t)stream;
  if (rows <= FEW_ROWS) {
    if (sums == nullptr || (rows > 1 && ldsums < inter)) return -2;
    a.out = sums, a.ldo = ldsums;
    if (const int bad = few_rows<SWIGLU_F32>(a, s)) return bad;
    return bw_quantize_fp8(sums, 0, ldsums, codes, ldq, scales, lds, rows, inter, stream);
  }
  a.out = codes, a.ldo = ldq, a.out_scales = scales, a.lds = lds;
  return launch_tiles<SWIGLU_FP8, 2, 4, 4>(a, s);
}
