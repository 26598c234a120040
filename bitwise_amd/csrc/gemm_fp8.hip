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
#include <type_traits>

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
  int vec_out;               // rows of out and residual can be taken 16 bytes at a time
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

__device__ __forceinline__ bf16x8 quarter_of(u32x4 half, int odd) {
  const uint32_t a = half[2 * odd], b = half[2 * odd + 1];
  return as_bf16x8((u32x4){codes_to_bf16x2(a, false), codes_to_bf16x2(a, true), codes_to_bf16x2(b, false), codes_to_bf16x2(b, true)});
}

__device__ __forceinline__ Frag frag_of(u32x4 lo, u32x4 hi) {
  Frag f;
#pragma unroll
  for (int t = 0; t < 4; ++t) f.t[t] = quarter_of(t < 2 ? lo : hi, t & 1);
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

// 16 bytes a lane from memory to LDS, lane l's to ``to`` + 16 l.
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t rs, unsigned char* to, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)to, 16, voff, soff, 0, 0);
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
    // (a NaN goes through the first product)
    with_sigmoids<1>([&](int) { return y; }, [&](int, float s) { y = (y * s) * u; });
    ((float*)a.out)[(size_t)m * a.ldo + n] = y;
  } else {
    if (a.residual != nullptr) y = a.residual[(size_t)m * a.ldr + n] + y;
    ((float*)a.out)[(size_t)m * a.ldo + n] = y;
  }
}

// ------------------------------------------------------------------------------ few rows

// What lies outside of what is read is told by a lane's own offset (behind the descriptor, whatever the scalar offset adds: rows past the
// matrices) or by a descriptor without a byte (blocks past K), never by the scalar offset, which not every range check counts.
// FAR: behind the descriptors of up to 64 rows of at most 2^23 bytes, with room for a strip's offset below 2^31.
constexpr int FAR = 0x40000000;

// How a wave gets its block's rows: straight into registers as the matrix instructions take them, or by way of LDS (a room of its own,
// 128 bytes a row as in the tiles below), where each load brings eight whole rows; ROOM8: with room for eight rows of x only.
enum { STRAIGHT = 0, ROOM16 = 1, ROOM8 = 2 };

constexpr int SIXTEEN = 100;                  // the choice of strips for up to 16 rows

// A workgroup of NW waves a block of 16 WM rows of x and NC strips of CW matrix rows (gated: as many gate and up rows).  The blocks of
// K go round the waves; their sums meet in LDS, where the threads that own the outputs walk them in order.  CW = 8 halves a strip
// (nothing is asked for for lanes with r >= 8): twice as many workgroups, for products with too few columns to give every compute unit 16.
// More strips a workgroup share x's loads and its conversion.
//
// Bound by the matrix's bytes where it is large (8 x 28672 x 4096 24.9 us, 4.7 TB/s), else by loads, start and end: of 43 x 4096 x 4096
// straight into registers 10.8 us, 2.7 went with the loads of x, 4.0 with the matrix's, nothing with conversions and walk.  Straight loads
// have 16 lanes in a row at 16 different lines, which the first cache looks up one by one, some 16 bytes a clock; by way of LDS eight lanes
// share a line: 8.4 us (64 x 2048 x 8192 13.6 -> 10.0, 8 x 28672 x 4096 27.9 -> 24.9).
template <int WM, int NC, int EPI, int NW, int CW, int VIA>
__global__ __launch_bounds__(64 * NW) void gemm_fp8_few_kernel(Fp8Args a) {
  constexpr int NB = EPI == SWIGLU_F32 ? 2 : 1, NS = NB * NC;                    // (strip c of gate or up b: c * NB + b)
  constexpr int PS = 16 * CW, OWNED = NC * WM * PS, OWN = (OWNED + 64 * NW - 1) / (64 * NW);
  constexpr int BX = VIA == ROOM8 ? 1 : 2 * WM, BW = CW * NS / 8, ROOM = VIA ? (BX + BW) * 1024 : 0;      // (BX, BW: eights of rows)
  static_assert(VIA != ROOM8 || WM == 1, "eight rows are one block of x");
  extern __shared__ __attribute__((aligned(16))) unsigned char room[];          // [NW][ROOM]
  float* part = reinterpret_cast<float*>(room + NW * ROOM);                     // [NW][NB][NC][WM][PS], then the factors
  float* factor = part + NW * NB * OWNED;                                       // [NW][NB][WM * 16]
  const int wave = wave_index(), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  // workgroups with the same strips and other rows are neighbours on one die (every eighth), which reads the strips once
  const int of_eight = blockIdx.x / (8 * a.m_tiles);
  const int n0 = (8 * of_eight + (int)(blockIdx.x & 7)) * (CW * NC), m0 = (int)(blockIdx.x / 8 - of_eight * a.m_tiles) * (16 * WM), KB = a.K / BW_FP8_BLOCK;
  if (n0 >= a.N) return;
  const int rows = min(16 * WM, a.M - m0);
  __amdgpu_buffer_rsrc_t rs_ws[NB];
  const int size_w = min(CW * NC, a.N - n0) * a.K, size_x = (rows - 1) * a.ldx + a.K;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    rs_ws[b] = rows_of(a.ws + ((size_t)(n0 / BW_FP8_BLOCK) + (size_t)b * ((a.N + BW_FP8_BLOCK - 1) / BW_FP8_BLOCK)) * KB, (size_t)KB * 4);
  }
  int row_m[WM];
#pragma unroll
  for (int i = 0; i < WM; ++i) row_m[i] = m0 + min(16 * i + r, rows - 1);
  // STRAIGHT: a lane's rows.  Otherwise: a load's row and slot of a lane (``via``), and where it reads its operands (of 16 rows, of 8).
  int voff_w = 0, voff_x[WM], via_x[2], via_w[2], from16[2], from8[2];
  unsigned char* const mine = room + wave * ROOM;
  if constexpr (VIA == STRAIGHT) {
    voff_w = r < CW ? r * a.K + 16 * g : FAR;
#pragma unroll
    for (int i = 0; i < WM; ++i) voff_x[i] = 16 * i + r < rows ? (16 * i + r) * a.ldx + 16 * g : FAR;
  } else {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int lrow = lane >> 3, chunk = 16 * ((lane & 7) ^ (4 * t + (lrow >> 1)));
      via_x[t] = lrow * a.ldx + chunk;
      via_w[t] = lrow * a.K + chunk;
      from16[t] = r * 128 + (((4 * t + g) ^ (r >> 1)) * 16);
      from8[t] = (r & 7) * 128 + (((4 * t + g) ^ ((r & 7) >> 1)) * 16);
    }
  }

  u32x4 wq[NS][2], xq[WM][2];
  float sx[WM], sw[NB];
  // (A wave whose turn lies behind the last block asks memory for nothing: 8 x 28672 x 4224, a block past whole passes, 31.5 -> 29.3 us.
  // All are vector loads, in one order everywhere and in the last pass not at all, so that what is waited for is never more than
  // needed.  Factors last were slower, 64 x 6144 x 4096 18.3 for 16.6.)
  auto issue = [&](int pass) {
    const int blk = pass * NW + wave, here = min(blk, KB - 1), at_k = here * BW_FP8_BLOCK;
    const bool live = blk < KB;
    const __amdgpu_buffer_rsrc_t rs_x = rows_of(a.x + (size_t)m0 * a.ldx, live ? size_x : 0);
    __amdgpu_buffer_rsrc_t rs_w[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) rs_w[b] = rows_of(a.w + ((size_t)b * a.N + n0) * a.K, live ? size_w : 0);
#pragma unroll
    for (int i = 0; i < WM; ++i) sx[i] = a.xs[(size_t)here * a.ldxs + row_m[i]];
#pragma unroll
    for (int b = 0; b < NB; ++b) sw[b] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs_ws[b], 0, here * 4, 0));
    if constexpr (VIA == STRAIGHT) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const int at = voff_w + c * CW * a.K;                  // (a strip past the matrix lies outside the descriptor)
          wq[c * NB + b][0] = __builtin_amdgcn_raw_buffer_load_b128(rs_w[b], at, at_k, 0);
          wq[c * NB + b][1] = __builtin_amdgcn_raw_buffer_load_b128(rs_w[b], at + 64, at_k, 0);
        }
#pragma unroll
      for (int i = 0; i < WM; ++i) {
        xq[i][0] = __builtin_amdgcn_raw_buffer_load_b128(rs_x, voff_x[i], at_k, 0);
        xq[i][1] = __builtin_amdgcn_raw_buffer_load_b128(rs_x, voff_x[i] + 64, at_k, 0);
      }
    } else {
      // (rows past the matrices lie outside the descriptors: zeros)
#pragma unroll
      for (int t = 0; t < BX; ++t) load_to_lds(rs_x, mine + t * 1024, via_x[t & 1] + 8 * t * a.ldx, at_k);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < BW / NB; ++t) load_to_lds(rs_w[b], mine + (BX + b * (BW / NB) + t) * 1024, via_w[CW == 16 ? t & 1 : 0] + 8 * t * a.K, at_k);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // the outputs that this thread owns
  auto owned = [&](int o, int& m, int& n) {
    const int e = (int)threadIdx.x + o * 64 * NW;
    m = m0 + 16 * (e / PS % WM) + ((e >> 2) & 15);
    n = n0 + CW * (e / (PS * WM)) + 4 * ((e % PS) >> 6) + (e & 3);
    return e < OWNED && m < a.M && n < a.N;
  };
  const int passes = (KB + NW - 1) / NW;
  issue(0);
  float acc[NB][OWN], old[OWN];                                  // (old: what the sums are added to, asked for early)
#pragma unroll
  for (int o = 0; o < OWN; ++o) {
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b][o] = 0.0f;
    int m, n;
    if (EPI == STORE_F32 && a.residual != nullptr && owned(o, m, n)) old[o] = a.residual[(size_t)m * a.ldr + n];
  }
  auto run = [&](int pass, auto is_last) {
    constexpr bool LAST = decltype(is_last)::value;
    if (!LAST || pass * NW + wave < KB) {                        // (scalar)
      if constexpr (VIA != STRAIGHT) {
        __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
        asm volatile("" ::: "memory");
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int i = 0; i < WM; ++i) xq[i][t] = *reinterpret_cast<const u32x4*>(mine + 2048 * i + (VIA == ROOM8 ? from8[t] : from16[t]));
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int b = 0; b < NB; ++b)
              wq[c * NB + b][t] = *reinterpret_cast<const u32x4*>(mine + (BX + (b * NC + c) * (CW / 8)) * 1024 + (CW == 16 ? from16[t] : from8[t]));
        }
      }
      float both[WM][NB];
#pragma unroll
      for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b) both[i][b] = sx[i] * sw[b];
      if constexpr (VIA != STRAIGHT && !LAST) {
        __builtin_amdgcn_s_waitcnt(0xc07f);                      // (the block has left its room)
        asm volatile("" ::: "memory");
        issue(pass + 1);
      }
      Frag fw[NS];
#pragma unroll
      for (int k = 0; k < NS; ++k) fw[k] = frag_of(wq[k][0], wq[k][1]);
#pragma unroll
      for (int i = 0; i < WM; ++i) {
        const Frag fx = frag_of(xq[i][0], xq[i][1]);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const f32x4 sums = block_sums(fw[c * NB + b], fx);
            if (CW == 16 || lane < 32) *reinterpret_cast<f32x4*>(part + (((wave * NB + b) * NC + c) * WM + i) * PS + 4 * lane) = sums;
          }
          if (g == 0) factor[(wave * NB + b) * (WM * 16) + 16 * i + r] = both[i][b];
        }
      }
    } else if constexpr (VIA != STRAIGHT) {
      __builtin_amdgcn_s_waitcnt(vmcnt_only(0));                 // (its last loads still go to the workgroup's LDS: not behind its end)
    }
    if (!LAST && VIA == STRAIGHT) issue(pass + 1);
    lds_barrier();
    const int here = LAST ? KB - pass * NW : NW;
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int e = (int)threadIdx.x + o * 64 * NW;
      if (e < OWNED) {
        const int m = 16 * (e / PS % WM) + ((e >> 2) & 15);
        auto walk = [&](int v) {
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[b][o] = fmaf(factor[(v * NB + b) * (WM * 16) + m], part[(v * NB + b) * OWNED + e], acc[b][o]);
        };
        if (!LAST || here == NW) {
#pragma unroll
          for (int v = 0; v < NW; ++v) walk(v);
        } else {
#pragma unroll 4
          for (int v = 0; v < here; ++v) walk(v);
        }
      }
    }
  };
  for (int pass = 0; pass < passes - 1; ++pass) {
    run(pass, std::false_type{});
    lds_barrier();                                               // (the pass's sums have been walked)
  }
  run(passes - 1, std::true_type{});
#pragma unroll
  for (int o = 0; o < OWN; ++o) {
    int m, n;
    if (!owned(o, m, n)) continue;
    if (EPI == STORE_F32) ((float*)a.out)[(size_t)m * a.ldo + n] = a.residual != nullptr ? old[o] + acc[0][o] : acc[0][o];
    else store_one<EPI>(a, m, n, acc[0][o], acc[NB - 1][o]);
  }
}

// ------------------------------------------------------------------------------ tiles

// A copy made where it is written.  (A plain assignment of what a load brings becomes a copy at the loop's end, and the wait for the
// load with it: nothing would be in flight across steps.)
__device__ __forceinline__ float taken(float v) {
  float r;
  asm volatile("v_mov_b32 %0, %1" : "=v"(r) : "v"(v));
  return r;
}

// A workgroup computes BM rows times BN matrix rows (gated: BN / 2 gate and BN / 2 up rows) in steps of one block of 128; both
// operands travel from memory straight into LDS, ST steps ahead.  The waves lie WY x WAVES / WY over the tile, each with MI x NJ
// results of 16 x 16.  One load of a wave brings 8 rows of a step, 128 bytes each, into 1 KB of LDS, lane l's 16
// bytes to 16 l; slot c' of row r (within its block of 16 rows) holds the row's chunk c' ^ (r >> 1), so that the 16 lanes that
// read one chunk of 16 rows hit 16 different groups of banks (conflicts: 1 % of LDS's busy cycles).
//
// What bounds it, of 2048 rows by gated 14336 columns, K = 4096, 407 us (1.18 PFLOP/s; in an unbroken row 450, 1.07; a plain bfloat16
// product of the library reaches 1.38): the matrix cores are busy 51 % of the cycles, and for 16 matrix instructions of a wave there are 54 others, of which 27 convert
// and 18 join chains.  Left out one at a time the conversions are worth 11 %, three quarters of the chains' multiply-adds 8 %, the reads
// from LDS 13 %, the loads 13 %, all together 30 %: no one of them is the bound, and the clock falls with the matrix cores' power
// (zeros for operands run 8 % faster).  So the tile is as large as a wave's registers allow: a step of 192 x 256 takes 2.04 us, of 128 x 128 for the same work 2.7.
template <int EPI, int WAVES_, int WY_, int MI_, int NJ_, int ST_>
struct Fp8Tile {
  static constexpr int WAVES = WAVES_, WY = WY_, WX = WAVES / WY_, MI = MI_, NJ = NJ_, ST = ST_;
  static constexpr bool GLU = EPI == SWIGLU_FP8;
  static constexpr int BM = 16 * WY * MI, BN = 16 * WX * NJ, COLS = GLU ? BN / 2 : BN;
  static constexpr int A_SLOT = BM * 128, B_SLOT = BN * 128, STEP = A_SLOT + B_SLOT;
  static constexpr int LA = BM / (8 * WAVES), LB = BN / (8 * WAVES);
  static constexpr int BYTES = ST * STEP;
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0 && ST >= 2 && BYTES <= 160 * 1024 && LA <= 8 && LB <= 8 && 128 % (16 * (GLU ? NJ / 2 : NJ)) == 0 && (!GLU || COLS == 128), "tile shapes");
};

template <int EPI, int WAVES, int WY, int MI, int NJ, int ST>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(2, 2))) void gemm_fp8_tiles_kernel(Fp8Args a) {
  using T = Fp8Tile<EPI, WAVES, WY, MI, NJ, ST>;
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
  const bool up = GLU && wave >= WAVES / 2;
  const uint8_t* const base_a = a.x + (size_t)m0 * a.ldx;
  const uint8_t* const base_b = a.w + ((size_t)(up ? a.N : 0) + n0) * a.K;
  const int size_a = (a_rows - 1) * a.ldx + a.K, size_b = b_rows * a.K;
  const int lrow = lane >> 3, lslot = lane & 7;
  int voff_a[8], voff_b[8];
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
  // (a step past the end: descriptors without a byte, no traffic, zeros into a slot that nobody reads)
  auto issue = [&](int step, int slot) {
    const bool live = step < KB;
    const __amdgpu_buffer_rsrc_t rs_a = rows_of(base_a, live ? size_a : 0), rs_b = rows_of(base_b, live ? size_b : 0);
    unsigned char* const to = ring + slot * T::STEP;
#pragma unroll
    for (int t = 0; t < T::LA; ++t)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_a, (lds_ptr)(to + (T::LA * wave + t) * 1024), 16, voff_a[t], step * 128, 0, 0);
#pragma unroll
    for (int t = 0; t < T::LB; ++t)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_b, (lds_ptr)(to + T::A_SLOT + (T::LB * wave + t) * 1024), 16, voff_b[t], step * 128, 0, 0);
  };
  // The scales of this wave's rows and columns for a step, asked for a step ahead (rows past M: zeros).
  const int xs_at = 4 * (m0 + 16 * MI * wy + r);
  const int NBLK = (a.N + BW_FP8_BLOCK - 1) / BW_FP8_BLOCK;
  const int my_block = min((n0 + 16 * NH * wx) / BW_FP8_BLOCK, NBLK - 1);       // (columns past the matrix: any scale will do)
  const float* xs_step = a.xs;
  const float* ws_step = a.ws + (size_t)my_block * KB;
  float sx[8], sw[2], sx_next[8], sw_next[2];
  auto scales = [&]() {
    const __amdgpu_buffer_rsrc_t rs = rows_of(xs_step, (size_t)a.M * 4);
#pragma unroll
    for (int i = 0; i < MI; ++i) sx_next[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, xs_at + 64 * i, 0, 0));
#pragma unroll
    for (int b = 0; b < NB; ++b) sw_next[b] = ws_step[(size_t)b * NBLK * KB];
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
  // Operands as they come from LDS (of a block of x, of a half of the wave's blocks of the matrix), converted, and the results of
  // the block of x at hand and of the one before.
  u32x4 ra[2], rb[NJ];
  Frag fa, fb[NJ];
  constexpr int PN = MI > 4 ? 1 : 2;
  f32x4 p[2][NJ];
  auto read_a = [&](int at_slot, int i, int kk) {
    ra[kk] = *reinterpret_cast<const u32x4*>(ring + at_slot * T::STEP + (MI * wy + i) * 2048 + slot_off[kk]);
  };
  auto read_b = [&](int at_slot, int kk) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int blk = GLU ? (NH * wx + j % NH) + (j / NH) * (T::BN / 32) : NJ * wx + j;
      rb[j] = *reinterpret_cast<const u32x4*>(ring + at_slot * T::STEP + T::A_SLOT + blk * 2048 + slot_off[kk]);
    }
  };
  auto add_up = [&](int i, int e) {                               // element e of block i's results joins its chain
    const int j = e >> 2, q = e & 3;
    acc[i][j][q] = fmaf(sx[i] * sw[GLU ? j / NH : 0], p[PN == 1 ? 0 : i & 1][j][q], acc[i][j][q]);
  };

  scales();
#pragma unroll
  for (int st = 0; st < T::ST; ++st) issue(st, st);
  __builtin_amdgcn_s_waitcnt(vmcnt_only((T::ST - 1) * (T::LA + T::LB)));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  read_b(0, 0);
  read_a(0, 0, 0);
  read_a(0, 0, 1);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int j = 0; j < NJ; ++j) fb[j].t[t] = quarter_of(rb[j], t);
#pragma unroll
  for (int t = 0; t < 3; ++t) fa.t[t] = quarter_of(ra[t >> 1], t & 1);
  read_b(0, 1);
  read_a(0, 1, 0);
#pragma unroll
  for (int i = 0; i < MI; ++i) sx[i] = 0.0f;                       // (the first block adds up a block that was none)
  sw[0] = sw[1] = 0.0f;
#pragma unroll
  for (int j = 0; j < NJ; ++j) p[PN - 1][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  int slot = 0;
  for (int step = 0; step < KB; ++step) {
    const int next = slot + 1 == T::ST ? 0 : slot + 1;
    // A step is MI blocks of x, a block four phases: a quarter of the block's k against the wave's NJ blocks of the matrix.  Under a
    // phase's matrix instructions a quarter of the block before joins the chains and what the phase before was the last to use is
    // replaced by what comes next (a quarter of the next block of x; in the step's last phases and the next one's first, of the
    // matrix's blocks).  The barrier stands a block and a half before the step's end, when the wave has its last operands of the step.
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        int valu = 0, reads = 0;
        __builtin_amdgcn_sched_barrier(0);
        if (i == MI - 2 && t == 2) {
          __builtin_amdgcn_s_waitcnt(vmcnt_only((T::ST - 2) * (T::LA + T::LB)) & ~0x0f00);
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          issue(step + T::ST, slot);
          __builtin_amdgcn_sched_barrier(0);
        }
        // reads: the next block of x, its second half two phases behind its first; the next step's halves of the matrix's blocks
        const int from = i + 1 < MI ? slot : next;
        if (t == 1) {
          read_a(from, (i + 1) % MI, 1);
          reads += 1;
        }
        if (t == 3) {
          read_a(i + 2 < MI ? slot : next, (i + 2) % MI, 0);
          reads += 1;
          if (i == MI - 2) {
            read_b(next, 0);
            reads += NJ;
          }
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          f32x4& pj = p[PN == 1 ? 0 : i & 1][j];
          if (PN == 1 && t == 0) {
#pragma unroll
            for (int q = 0; q < 4; ++q) add_up((i + MI - 1) % MI, 4 * j + q);
          }
          if (t == 0) pj = (f32x4){0.f, 0.f, 0.f, 0.f};
          pj = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j].t[t], fa.t[t], pj, 0, 0, 0);
        }
        if (PN == 2) {
#pragma unroll
          for (int e = t * NJ; e < (t + 1) * NJ; ++e) add_up((i + MI - 1) % MI, e);
          valu += NJ;
        } else if (t == 0) {
          valu += 4 * NJ;
        }
        // (the quarter that this phase's instructions are the last to use is replaced a phase later)
        const int was = (t + 3) & 3;
        fa.t[was] = quarter_of(ra[was >> 1], was & 1);
        valu += 4;
        if (i == MI - 1 && t == 1) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) fb[j].t[0] = quarter_of(rb[j], 0);
          valu += 4 * NJ;
        }
        if (i == MI - 1 && t == 2) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) fb[j].t[1] = quarter_of(rb[j], 1);
          valu += 4 * NJ;
        }
        if (i == MI - 1 && t == 3) {
          read_b(next, 1);
          reads += NJ;
        }
        if (i == 0 && t == 0) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) fb[j].t[2] = quarter_of(rb[j], 0);
          valu += 4 * NJ;
        }
        if (i == 0 && t == 1) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) fb[j].t[3] = quarter_of(rb[j], 1);
          valu += 4 * NJ;
        }
#pragma unroll
        for (int k = 0; k < NJ; ++k) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          if (k == 0 && reads) __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
          if (valu > 4 * NJ) __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
          else __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
        }
        if (i == 0 && t == 3) {
          // every result of the step before has joined its chain
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int k = 0; k < MI; ++k) sx[k] = taken(sx_next[k]);
#pragma unroll
          for (int b = 0; b < NB; ++b) sw[b] = taken(sw_next[b]);
          if (step + 1 < KB) {
            xs_step += a.ldxs;
            ws_step += 1;
          }
          scales();
        }
      }
    }
    slot = next;
  }
#pragma unroll
  for (int e = 0; e < 4 * NJ; ++e) add_up(MI - 1, e);
  __builtin_amdgcn_s_waitcnt(vmcnt_only(0));                       // the padding loads too, before LDS is used again or the waves end

  if constexpr (GLU) {
    // silu(g) u, the largest magnitude of each row's 128 outputs over lanes and waves, codes
    __syncthreads();
    uint32_t* most = reinterpret_cast<uint32_t*>(ring);            // [WX][BM]
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      uint32_t mx = 0u;
      with_sigmoids<4 * NH>([&](int k) { return acc[i][k / 4][k % 4]; }, [&](int k, float s) {
        acc[i][k / 4][k % 4] = (acc[i][k / 4][k % 4] * s) * acc[i][NH + k / 4][k % 4];
      });
#pragma unroll
      for (int k = 0; k < 4 * NH; ++k) mx = max_bits(mx, __float_as_uint(acc[i][k / 4][k % 4]) & 0x7fffffffu);
      float lo, hi;
      lane_halves<32>(__uint_as_float(mx), lo, hi);
      mx = max_bits(__float_as_uint(lo), __float_as_uint(hi));
      lane_halves<16>(__uint_as_float(mx), lo, hi);
      mx = max_bits(__float_as_uint(lo), __float_as_uint(hi));
      if (g == 0) most[wx * BM + 16 * (MI * wy + i) + r] = mx;
    }
    __syncthreads();
    // The codes of the tile's rows lie in LDS row by row (144 bytes apart, which spreads the columns' words over the banks) and
    // leave as whole lines.
    constexpr int CODES_AT = 4 * T::WX * BM, CLD = 144;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int row = 16 * (MI * wy + i) + r, m = m0 + row;
      uint32_t mx = 0u;
#pragma unroll
      for (int v = 0; v < T::WX; ++v) mx = max_bits(mx, most[v * BM + row]);
      const Fp8Scale s = fp8_scale_of(mx);
#pragma unroll
      for (int j = 0; j < NH; ++j)
        *reinterpret_cast<uint32_t*>(ring + CODES_AT + row * CLD + 16 * (NH * wx + j) + 4 * g) =
            fp8_codes4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3], s);
      if (m < a.M && wx == 0 && g == 0) a.out_scales[(size_t)(n0 / BW_FP8_BLOCK) * a.lds + m] = s.scale;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < BM * 8 / (64 * WAVES); ++e) {
      const int at = e * 64 * WAVES + (int)threadIdx.x, row = at >> 3, m = m0 + row;
      if (m < a.M)
        *reinterpret_cast<u32x4*>((uint8_t*)a.out + (size_t)m * a.ldo + n0 + 16 * (at & 7)) =
            *reinterpret_cast<const u32x4*>(ring + CODES_AT + row * CLD + 16 * (at & 7));
    }
  } else {
    // 16 rows of the wave's results at a time go through LDS of its own, so that a store covers whole rows of them: a lane holds
    // four neighbours of one of 16 rows.
    __syncthreads();
    constexpr int W = 16 * NJ, LDW = W + 4;
    float* const mine = reinterpret_cast<float*>(ring) + wave * 16 * LDW;
    const int nw = n0 + W * wx;
    constexpr int PER = EPI == STORE_BF16 ? 8 : 4, LANES = W / PER, ROWS = 64 / LANES;      // elements a lane, lanes a row, rows a store
    const bool vec = a.vec_out && nw + W <= a.N;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m1 = m0 + 16 * (MI * wy + i);
#pragma unroll
      for (int j = 0; j < NJ; ++j) *reinterpret_cast<f32x4*>(mine + r * LDW + 16 * j + 4 * g) = acc[i][j];
      __builtin_amdgcn_wave_barrier();
      if (vec) {
#pragma unroll
        for (int e = 0; e < 16 / ROWS; ++e) {
          const int row = e * ROWS + lane / LANES, c = PER * (lane % LANES), m = m1 + row;
          f32x4 y = *reinterpret_cast<const f32x4*>(mine + row * LDW + c);
          if constexpr (EPI == STORE_BF16) {
            const f32x4 z = *reinterpret_cast<const f32x4*>(mine + row * LDW + c + 4);
            if (m < a.M)
              *reinterpret_cast<u32x4*>((bf16_t*)a.out + (size_t)m * a.ldo + nw + c) =
                  (u32x4){pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(z[0], z[1]), pack_bf16x2(z[2], z[3])};
          } else if (m < a.M) {
            if (a.residual != nullptr) y = *reinterpret_cast<const f32x4*>(a.residual + (size_t)m * a.ldr + nw + c) + y;
            *reinterpret_cast<f32x4*>((float*)a.out + (size_t)m * a.ldo + nw + c) = y;
          }
        }
      } else {
        constexpr int RPS = 64 / W;                                  // rows a store of single elements
#pragma unroll 4
        for (int e = 0; e < 16 / RPS; ++e) {
          const int row = e * RPS + lane / W, c = lane % W;
          if (m1 + row < a.M && nw + c < a.N) store_one<EPI>(a, m1 + row, nw + c, mine[row * LDW + c], 0.0f);
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// ------------------------------------------------------------------------------ which kernel

template <int WM, int NC, int EPI, int NW, int CW, int VIA>
int launch_few(Fp8Args a, hipStream_t s) {
  constexpr int NB = EPI == SWIGLU_F32 ? 2 : 1, LDS = NW * (NB * WM * 16 * (CW * NC + 1) * 4 + (VIA ? (VIA == ROOM8 ? 8 : 16 * WM) + CW * NC * NB : 0) * 128);
  static_assert(LDS <= 160 * 1024 && 128 % (CW * NC) == 0, "a pass's sums fit LDS, a workgroup's columns one block's scale");
  a.m_tiles = (a.M + 16 * WM - 1) / (16 * WM);
  a.n_tiles = (a.N + CW * NC - 1) / (CW * NC);
  hipLaunchKernelGGL((gemm_fp8_few_kernel<WM, NC, EPI, NW, CW, VIA>), dim3((unsigned)((a.n_tiles + 7) / 8 * 8 * a.m_tiles)), dim3(64 * NW), LDS, s, a);
  return BW_LAUNCH_CHECK();
}

// Up to 16 rows: strips of 16 columns for the 256 compute units, K's blocks over the waves of one.  Eight waves a strip where there are
// strips for more than one workgroup a unit (8 rows of 5120 columns, K = 5120: 8.1 us, with 16 waves 10.1), 16 where there is at most
// one (4 of 4096, K = 14336: 12.7, with eight 14.2).  Up to 2048 columns strips of eight, so that every unit has one: of 2048
// columns, K = 8192, 6.4 us for 7.2; by eight waves where K has no work for more (K = 1024 2.7 for 2.9).  Up to eight rows leave eight waves room for
// a fourth workgroup a unit (2 x 16384 x 8192 30.1 -> 27.6 us); with sixteen, one a unit is better (4 x 4096 x 14336 12.7 for 14.5).
// Two strips a workgroup share x where there is more of it (16 x 28672 x 2048 14.8 -> 14.0, 16 x 6144 x 5120 11.6 -> 10.5, 16 x 28672 x 14336 89.9 ->
// 80.8), or where one workgroup a unit then takes all (8 x 6144 x 5120 9.8 -> 9.4, gated 3 x 5504 x 2048 9.8 -> 9.0; 1 x 28672 x 4096 24.2 -> 25.0).  Not
// where the matrix's rows lie a multiple of 8,192 bytes apart, so that twice as many of them meet in the same channels (12 x 8192 x 8192 15.9 ->
// 17.3, 8 x 6144 x 8192 13.2 -> 14.2, 16 x 20000 x 16384 67 -> 73; K = 8064 and 8320 gain 1.03 to 1.13, 12288 0.94 to 1.06, 24576 0.96 to 1.09).
template <int EPI, int VIA>
int sixteen_rows(const Fp8Args& a, hipStream_t s) {
  if constexpr (EPI != SWIGLU_F32) {
    if (a.N <= 2048) return a.K <= 8 * BW_FP8_BLOCK ? launch_few<1, 1, EPI, 8, 8, VIA>(a, s) : launch_few<1, 1, EPI, 16, 8, ROOM16>(a, s);
    if (a.N <= 4096) return launch_few<1, 1, EPI, 16, 16, ROOM16>(a, s);
    if (a.K % 8192 != 0 && (VIA == ROOM16 || a.N <= 8192)) return launch_few<1, 2, EPI, 8, 16, VIA>(a, s);
  } else {
    if (a.N > 4096 && a.N <= 8192) return launch_few<1, 2, EPI, 8, 16, VIA>(a, s);
  }
  return launch_few<1, 1, EPI, 8, 16, VIA>(a, s);
}

template <int EPI>
int by_strips(const Fp8Args& a, int shape, hipStream_t s) {
  if (shape == SIXTEEN) return a.M <= 8 ? sixteen_rows<EPI, ROOM8>(a, s) : sixteen_rows<EPI, ROOM16>(a, s);
  if constexpr (EPI != SWIGLU_F32) {
    switch (shape) {
      case 0: return launch_few<1, 1, EPI, 8, 16, ROOM16>(a, s);
      case 1: return launch_few<1, 2, EPI, 8, 16, ROOM16>(a, s);
      case 2: return launch_few<2, 1, EPI, 8, 16, ROOM16>(a, s);
      default: return launch_few<2, 2, EPI, 8, 16, ROOM16>(a, s);
    }
  } else {
    switch (shape) {
      case 0: return launch_few<2, 1, EPI, 8, 16, STRAIGHT>(a, s);
      case 1: return launch_few<2, 2, EPI, 8, 16, STRAIGHT>(a, s);
      case 2: return launch_few<3, 2, EPI, 8, 16, STRAIGHT>(a, s);
      default: return launch_few<4, 2, EPI, 8, 16, STRAIGHT>(a, s);
    }
  }
}

template <int EPI, int WAVES, int WY, int MI, int NJ, int ST>
int launch_tiles(Fp8Args a, hipStream_t s) {
  using T = Fp8Tile<EPI, WAVES, WY, MI, NJ, ST>;
  a.m_tiles = (a.M + T::BM - 1) / T::BM;
  a.n_tiles = (a.N + T::COLS - 1) / T::COLS;
  hipLaunchKernelGGL((gemm_fp8_tiles_kernel<EPI, WAVES, WY, MI, NJ, ST>), dim3((unsigned)(a.m_tiles * a.n_tiles)), dim3(64 * T::WAVES), T::BYTES, s, a);
  return BW_LAUNCH_CHECK();
}

// What a workgroup of a shape (rows x columns) takes, in us: its start and end, and a step of 128 of K, with the compute unit for
// itself and, where two fit (``per_cu`` 2), beside another.  Measured on normal values (the power of the matrix cores, and with it
// their clock, hangs on them): slopes over K = 2048 and 8192, grids of up to 256 workgroups and of one or two full rounds.
struct ShapeCost {
  int rows, columns, per_cu;
  double start, step, start_beside, step_beside;
};

double shape_us(const ShapeCost& c, int M, int N, int K) {
  const double steps = K / BW_FP8_BLOCK, alone = c.start + steps * c.step, beside = c.start_beside + steps * c.step_beside;
  const long long groups = (long long)((M + c.rows - 1) / c.rows) * ((N + c.columns - 1) / c.columns);
  const long long full = groups / (256 * c.per_cu), rest = groups % (256 * c.per_cu);
  return 2.0 + full * (c.per_cu == 2 ? beside : alone) + (rest == 0 ? 0.0 : rest <= 256 ? alone : beside);
}

template <int SHAPES>
int cheapest(const ShapeCost (&shapes)[SHAPES], int M, int N, int K, double* us) {
  int best = 0;
  *us = shape_us(shapes[0], M, N, K);
  for (int i = 1; i < SHAPES; ++i) {
    const double t = shape_us(shapes[i], M, N, K);
    if (t < *us) {
      *us = t;
      best = i;
    }
  }
  return best;
}

// Strips: each wave a block of K of its own, which hides what a tile's step waits for; x and the matrix come once a workgroup,
// though, so many rows and columns are cheaper by tiles (64 x 4096 x 4096 9.4 us by strips, 19.6 by tiles; 40 x 28672 x 4096 41 and 31).
constexpr ShapeCost STORE_STRIPS[] = {{16, 16, 2, 0.1, 0.104, 1.1, 0.154}, {16, 32, 2, 0.2, 0.171, 0.4, 0.306}, {32, 16, 2, 0.2, 0.133, 1.1, 0.225}, {32, 32, 1, 0.8, 0.208, 0, 0}};
constexpr ShapeCost GATED_STRIPS[] = {{32, 16, 2, 0.0, 0.285, 0.0, 0.47}, {32, 32, 1, 0.6, 0.43, 0, 0}, {48, 32, 1, 1.0, 0.55, 0, 0}, {64, 32, 1, 1.0, 0.70, 0, 0}};
// Tiles: a step's conversions a matrix instruction fall with the tile.  192 x 256 by eight waves does the most a us, 128 x 128 by four, two
// workgroups a unit, fills a round sooner, 64 x 128 and 64 x 64 give a few hundred rows of few columns more workgroups.
constexpr ShapeCost STORE_TILES[] = {{192, 256, 1, 6.5, 2.04, 0, 0}, {128, 128, 2, 5.8, 1.02, 6.5, 1.78}, {64, 128, 2, 2.9, 0.64, 3.1, 1.12}, {64, 64, 2, 2.5, 0.49, 3.2, 0.74}};
constexpr ShapeCost GATED_TILES[] = {{192, 128, 1, 11.0, 2.04, 0, 0}, {128, 128, 1, 5.5, 1.70, 0, 0}, {64, 128, 2, 3.5, 1.20, 9.5, 1.60}, {32, 128, 2, 2.5, 0.95, 4.5, 1.30}};

// The strips' prices hold for rounds of few rows; past this, products of few columns are as often faster by tiles (30 of them, 1,037 to 9,662 rows of
// 27 to 407 columns: by strips 1.08 of the time, 0.5 to 2.2 one by one).
constexpr int STRIPS_MOST_ROWS = 1024;

constexpr int FEW_ROWS = 64;                    // rows up to which a gated product has a buffer for its sums

// What runs: ``strips`` (of the tables above; SIXTEEN: up to 16 rows, the strips made for those), or -1 and ``tiles``, the last ``tail``
// rows behind the tiles by a launch of their own, which takes what a product of so many rows takes (``choose_stored`` again).
struct Choice {
  int strips, tiles, tail;
};

Choice choose_stored(int rows, int N, int K) {
  if (rows <= 16) return {SIXTEEN, 0, 0};
  double us, strips_us;
  int shape = cheapest(STORE_TILES, rows, N, K, &us), tail = 0;
  const int strips = cheapest(STORE_STRIPS, rows, N, K, &strips_us);
  if (rows > STRIPS_MOST_ROWS) strips_us = us + 1.0;
  // A few rows past whole tiles can cost a round of their own: then they go behind the tiles (777 x 5003 x 2000, of which 768 rows are one
  // round, 35.9 -> 32.7 us; 2100 x 2048 x 2048 31.5 -> 27.5).  Their price is that of strips, also where they then take small tiles (one such
  // launch in eight): priced as those, which a table of whole products puts too low behind others, 40 products that change took 1.07 of the time;
  // by strips after all, 40 such products took 1.03.  Up to 16 rows run strips that have no table: over 45 sizes 0.74 to 1.33 of the price, 1.08 in
  // the middle.
  double best = us < strips_us ? us : strips_us;
  for (int i = 0; i < 4; ++i) {
    const int rest = rows % STORE_TILES[i].rows;
    if (rest == 0 || rest == rows || rest > FEW_ROWS) continue;
    double rest_us;
    cheapest(STORE_STRIPS, rest, N, K, &rest_us);
    const double both = shape_us(STORE_TILES[i], rows - rest, N, K) + rest_us;
    if (both < best) {
      best = both;
      tail = rest;
      shape = i;
    }
  }
  if (tail == 0 && strips_us <= us) return {strips, 0, 0};
  return {-1, shape, tail};
}

Choice choose_gated(int rows, int inter, int K) {
  if (rows <= 16) return {SIXTEEN, 0, 0};
  double us, strips_us;
  const int shape = cheapest(GATED_TILES, rows, inter, K, &us), strips = cheapest(GATED_STRIPS, rows, inter, K, &strips_us);
  if (rows <= FEW_ROWS && strips_us + 2.5 <= us) return {strips, 0, 0};      // (the quantization of the sums is a launch of its own)
  return {-1, shape, 0};
}

template <int EPI>
int stored_by_tiles(const Fp8Args& a, int shape, hipStream_t s) {
  switch (shape) {
    case 0: return launch_tiles<EPI, 8, 2, 6, 4, 2>(a, s);
    case 1: return launch_tiles<EPI, 4, 2, 4, 4, 2>(a, s);
    case 2: return launch_tiles<EPI, 4, 2, 2, 4, 3>(a, s);
    default: return launch_tiles<EPI, 4, 2, 2, 2, 4>(a, s);
  }
}

int gated_by_tiles(const Fp8Args& a, int shape, hipStream_t s) {
  switch (shape) {
    case 0: return launch_tiles<SWIGLU_FP8, 8, 2, 6, 4, 2>(a, s);
    case 1: return launch_tiles<SWIGLU_FP8, 8, 2, 4, 4, 3>(a, s);
    case 2: return launch_tiles<SWIGLU_FP8, 4, 1, 4, 4, 2>(a, s);
    default: return launch_tiles<SWIGLU_FP8, 4, 1, 2, 4, 2>(a, s);
  }
}

bool aligned(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

// Whether a result lies in what workgroups beside its own still read: rows of codes with their scales, a matrix (``halves`` times N rows) with its.
bool in_operands(const Lies& out, const void* x, int ldx, const float* xs, int ldxs, const void* w, const float* ws, int rows, int N, int K, int halves) {
  const long long kb = K / BW_FP8_BLOCK, nb = (long long)halves * ((N + BW_FP8_BLOCK - 1) / BW_FP8_BLOCK);
  const Lies operands[] = {{x, ldx, K, rows, 1}, {xs, 4ll * ldxs, 4ll * rows, kb, 4}, {w, 0, (long long)halves * N * K, 1, 1}, {ws, 0, 4 * nb * kb, 1, 4}};
  for (const Lies& o : operands)
    if (meet(out, o)) return true;
  return false;
}

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
  const int size = out_is_bf16 ? 2 : 4;
  const Lies at_out = {out, (long long)ldo * size, (long long)N * size, rows, size}, at_residual = {residual, 4ll * ldr, 4ll * N, rows, 4};
  if (in_operands(at_out, x, ldx, xs, ldxs, w, ws, rows, N, K, 1) || !in_place_or_apart(at_out, at_residual)) return -2;
  Fp8Args a = {};
  a.x = (const uint8_t*)x, a.xs = xs, a.w = (const uint8_t*)w, a.ws = ws, a.residual = residual, a.out = out;
  a.ldx = ldx, a.ldxs = ldxs, a.ldr = ldr, a.ldo = ldo, a.M = rows, a.N = N, a.K = K;
  a.vec_out = aligned(out, 16) && (rows == 1 || (long long)ldo * (out_is_bf16 ? 2 : 4) % 16 == 0) &&
              (residual == nullptr || (aligned(residual, 16) && (rows == 1 || ldr % 4 == 0)));
  hipStream_t s = (hipStream_t)stream;
  const Choice c = choose_stored(rows, N, K);
  if (c.strips >= 0) return out_is_bf16 ? by_strips<STORE_BF16>(a, c.strips, s) : by_strips<STORE_F32>(a, c.strips, s);
  a.M = rows - c.tail;
  if (const int bad = out_is_bf16 ? stored_by_tiles<STORE_BF16>(a, c.tiles, s) : stored_by_tiles<STORE_F32>(a, c.tiles, s)) return bad;
  if (c.tail == 0) return 0;
  const size_t head = rows - c.tail;
  void* rest_out = out_is_bf16 ? (void*)((bf16_t*)out + head * ldo) : (void*)((float*)out + head * ldo);
  return bw_gemm_fp8((const uint8_t*)x + head * ldx, ldx, xs + head, ldxs, w, ws, residual == nullptr ? nullptr : residual + head * ldr, ldr, rest_out, ldo,
                     out_is_bf16, c.tail, N, K, stream);
}

// Which kernels a product's sizes lead to (``Choice``): strips, tiles, tail.
extern "C" int bw_gemm_fp8_choice(int rows, int N, int K, int gated, int* choice) {
  if (rows < 1 || N < 1 || K < BW_FP8_BLOCK) return -2;
  const Choice c = gated ? choose_gated(rows, N, K) : choose_stored(rows, N, K);
  choice[0] = c.strips, choice[1] = c.tiles, choice[2] = c.tail;
  return 0;
}

extern "C" int bw_gemm_fp8_swiglu(const void* x, int ldx, const float* xs, int ldxs, const void* w, const float* ws, float* sums, int ldsums, void* codes,
                                  int ldq, float* scales, int lds, int rows, int inter, int K, void* stream) {
  if (rows <= 0) return 0;
  if (const int bad = sizes_wrong(x, ldx, ldxs, w, rows, inter, K)) return bad;
  const int whole = (inter + BW_FP8_BLOCK - 1) / BW_FP8_BLOCK * BW_FP8_BLOCK;
  if ((rows > 1 && ldq < whole) || lds < rows) return -2;
  if (rows <= FEW_ROWS && (sums == nullptr || (rows > 1 && ldsums < inter))) return -2;
  if (!aligned(codes, 16) || ldq % 16) return -3;
  const Lies results[] = {{codes, ldq, whole, rows, 1}, {scales, 4ll * lds, 4ll * rows, whole / BW_FP8_BLOCK, 4},
                          {rows <= FEW_ROWS ? sums : nullptr, 4ll * ldsums, 4ll * inter, rows, 4}};
  for (const Lies& r : results)
    if (in_operands(r, x, ldx, xs, ldxs, w, ws, rows, inter, K, 2)) return -2;
  if (meet(results[0], results[1]) || meet(results[0], results[2]) || meet(results[1], results[2])) return -2;
  Fp8Args a = {};
  a.x = (const uint8_t*)x, a.xs = xs, a.w = (const uint8_t*)w, a.ws = ws;
  a.ldx = ldx, a.ldxs = ldxs, a.M = rows, a.N = inter, a.K = K;
  hipStream_t s = (hipStream_t)stream;
  const Choice c = choose_gated(rows, inter, K);
  if (c.strips >= 0) {
    a.out = sums, a.ldo = ldsums;
    if (const int bad = by_strips<SWIGLU_F32>(a, c.strips, s)) return bad;
    return bw_quantize_fp8(sums, 0, ldsums, codes, ldq, scales, lds, rows, inter, stream);
  }
  a.out = codes, a.ldo = ldq, a.out_scales = scales, a.lds = lds;
  return gated_by_tiles(a, c.tiles, s);
}
