// Matrix products of 8-bit floating-point codes with a scale for each block of 128 along the contraction (gfx950).
//
//   y[m][n] = sum_b 2^(ex[m][b] + ew[n/128][b]) * sum_{k in block b} qx[m][k] * qw[n][k]        qx, qw: e4m3 codes
//
// The scales are powers of two (e8m0 bytes): 2^e is the smallest power with amax <= 448 2^e over the block, so a code never saturates,
// scaling is exact and the only rounding of the format is the one to e4m3 (round to nearest even).  CDNA4's scaled matrix instruction
// takes such a scale per lane and 32 contraction steps: a block of 128 hands the same byte to its steps, and the scales cost no
// arithmetic of their own.  Accumulators are fp32 (what the 8-bit pipe adds into them, and which results avoid it: "which matrix pipe"
// below).  An infinity or NaN of the input becomes the NaN code (e4m3 has no infinity, and a saturated code would hide the overflow) and
// the block's scale comes from its finite values.
//
// Codes lie in tiles of 16 rows x 64 columns, 1 KiB each: [row tile][column tile][chunk of 16 columns][row][16 bytes].  One wave's load, store or
// LDS transfer moves whole tiles (row-major codes fill LDS at two thirds of that rate: the first 128 x 128 kernel took 627 us over them for 8192^3
// against 499), a matrix fragment is one 16-byte read per lane and tile, and the 16 lanes that LDS serves at once read 256 consecutive bytes.
// Scale bytes of activations: [block of 128 columns][rows padded to 16]; of weights: [block][groups of 32 rows].  Weights are padded with
// zeros to 256 rows, so a tile's loads need no bounds there.
#include "fp8.h"
#include "gemm.h"
#include <atomic>
#include <type_traits>

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(8))) __bf16 mfma_b8;

namespace {

// ---- the format ------------------------------------------------------------------------------------------------------------------
// biased exponent of the block scale: amax = 1.f * 2^p, 448 = 1.75 * 2^8 -> e = p - 8, one more if the significand exceeds 1.75
__device__ __forceinline__ int scale_byte(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < 0 ? 0 : e;
}
__device__ __forceinline__ float scale_up(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }   // 2^(127 - byte)
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.f;
}
// a scaled value within +-448, or the NaN that becomes the NaN code
__device__ __forceinline__ float code_in(float v, float up) {
  const float t = v * up;
  return fabsf(t) <= 448.f ? t : __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float up) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(code_in(a, up), code_in(b, up), 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(code_in(c, up), code_in(d, up), r, true);
  return (uint32_t)r;
}

// 16-byte accesses at any address that an element may have
typedef uint16_t u16x8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// eight consecutive elements of a row from column k on; columns >= K read as zero
template <typename T>
__device__ __forceinline__ void load8(const T* p, int k, int K, float v[8]) {
  if (k + 8 <= K) {
    if constexpr (sizeof(T) == 2) {
      const u16x8_any t = *(const u16x8_any*)(p + k);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = bf2f(t[i]);
    } else {
      const f32x4_any a = *(const f32x4_any*)(p + k), b = *(const f32x4_any*)(p + k + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 2) v[i] = k + i < K ? bf2f(p[k + i]) : 0.f;
      else v[i] = k + i < K ? (float)p[k + i] : 0.f;
    }
  }
}

// sixteen consecutive elements of a row from column k on, as load8
template <typename T>
__device__ __forceinline__ void load16(const T* p, int k, int K, float v[16]) {
  load8(p, k, K, v);
  load8(p, k + 8, K, v + 8);
}
// a block of 128 held by eight lanes, 16 values each, that differ in the lane bits o0, o1, o2: its scale byte.  Infinities are rare: they are
// seen in the maximum (fmax drops a NaN), only then replaced by NaN and the maximum taken again over the finite values; the values
// left are within +-448 after scaling, or NaN, which the conversion keeps
__device__ __forceinline__ int block_scale(float v[16], int o0, int o1, int o2) {
  float a = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < 16; ++i) a = fmaxf(a, fabsf(v[i]));
  auto over = [&](float t) {
    t = fmaxf(t, __shfl_xor(t, o0, 64));
    t = fmaxf(t, __shfl_xor(t, o1, 64));
    return fmaxf(t, __shfl_xor(t, o2, 64));
  };
  a = over(a);
  if (a > 3.402823466e38f) {
    a = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (fabsf(v[i]) > 3.402823466e38f) v[i] = __uint_as_float(0x7fc00000u);
      a = fmaxf(a, fabsf(v[i]));
    }
    a = over(a);
  }
  return scale_byte(a != a ? 0.f : a);             // (a block of nothing but NaN)
}
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
__device__ __forceinline__ uint4 codes16(const float v[16], float up) {
  return make_uint4(pack4(v[0] * up, v[1] * up, v[2] * up, v[3] * up), pack4(v[4] * up, v[5] * up, v[6] * up, v[7] * up),
                    pack4(v[8] * up, v[9] * up, v[10] * up, v[11] * up), pack4(v[12] * up, v[13] * up, v[14] * up, v[15] * up));
}

// ---- rows of activations -------------------------------------------------------------------------------------------------------------
// Four rows per workgroup; a wave takes 256 columns at a time, 16 per lane (four neighbouring lanes hold the four rows of one chunk and write
// 64 consecutive bytes).  NORM: y = x * rsqrt(mean(x^2) + eps) * w in fp32 first, each wave summing one row's squares.
template <typename T, bool NORM>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* x, int64_t ldx, const float* w, float eps, uint8_t* q, uint8_t* s, int64_t M,
                                                         int64_t Mp, int K, int Kb) {
  __shared__ float rs[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m0 = (int64_t)blockIdx.x * 4;
  if constexpr (NORM) {
    const T* row = x + (m0 + wave < M ? m0 + wave : M - 1) * ldx;
    float ss = 0.f, v[8];
#pragma unroll 4
    for (int k = lane * 8; k < K; k += 512) {
      load8(row, k, K, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
    }
    ss = wave_sum(ss);
    if (lane == 0) rs[wave] = 1.f / sqrtf(ss / (float)K + eps);
    __syncthreads();
  }
  const int r = lane & 3, c = lane >> 2;
  const int64_t m = m0 + r;
  const T* row = x + (m < M ? m : M - 1) * ldx;
  const int width = Kb * 128, cols = m < M ? K : 0;
  // two pieces of 256 columns in flight per wave: a grid of four rows x 2048 columns, or, behind a norm, all columns of the four rows
  const int first = NORM ? wave * 256 : blockIdx.y * 2048 + wave * 256, stop = NORM || first >= width ? width : first + 1;
  for (int k0 = first; k0 < stop; k0 += 2048) {
    float v[2][16], g[2][16];
#pragma unroll
    for (int h = 0; h < 2; ++h) load16(row, k0 + h * 1024 + c * 16, cols, v[h]);
    if constexpr (NORM) {
#pragma unroll
      for (int h = 0; h < 2; ++h) load16(w, k0 + h * 1024 + c * 16, K, g[h]);
      const float rr = rs[r];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) v[h][i] = v[h][i] * rr * g[h][i];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = k0 + h * 1024 + c * 16, byte = block_scale(v[h], 4, 8, 16);
      if (k < width) {
        *(uint4*)(q + ((m >> 4) * Kb * 2 + (k >> 6)) * 1024 + (c & 3) * 256 + (m & 15) * 16) = codes16(v[h], scale_up(byte));
        if ((c & 7) == 0) s[(k >> 7) * Mp + m] = (uint8_t)byte;
      }
    }
  }
}

// ---- weights: one workgroup per 128 x 128 block, codes in both orders (once per weight) --------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(const T* w, int64_t ldw, int N, int K, uint8_t* q, uint8_t* s, uint8_t* qt, uint8_t* st) {
  // (the grid covers both dimensions padded to 256: two blocks of 128)
  __shared__ uint8_t tile[128][132];
  __shared__ float part[4];
  const int nb = blockIdx.y, kb = blockIdx.x;
  const int Nb = (N + 127) >> 7, Kb = (K + 127) >> 7, Ng = ((N + 255) >> 8) * 8, Kg = ((K + 255) >> 8) * 8;
  auto at = [&](int r, int c) {
    const int n = nb * 128 + r, k = kb * 128 + c;
    float v = 0.f;
    if (n < N && k < K) {
      if constexpr (sizeof(T) == 2) v = bf2f(w[(int64_t)n * ldw + k]);
      else v = w[(int64_t)n * ldw + k];
    }
    return v;
  };
  float amax = 0.f;
  for (int i = threadIdx.x; i < 128 * 128; i += 256) amax = fmaxf(amax, finite_abs(at(i >> 7, i & 127)));
  amax = wave_max(amax);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = amax;
  __syncthreads();
  const int byte = scale_byte(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
  const float up = scale_up(byte);
  for (int i = threadIdx.x; i < 128 * 32; i += 256) {
    const int r = i >> 5, c = (i & 31) * 4;
    *(uint32_t*)&tile[r][c] = codes4(at(r, c), at(r, c + 1), at(r, c + 2), at(r, c + 3), up);
  }
  if (threadIdx.x < 4) {
    if (kb < Kb) s[(int64_t)kb * Ng + nb * 4 + threadIdx.x] = (uint8_t)byte;
    if (st && nb < Nb) st[(int64_t)nb * Kg + kb * 4 + threadIdx.x] = (uint8_t)byte;
  }
  __syncthreads();
  // 16-byte chunk i of the block's 16 tiles: row r, columns 16 c ..
  for (int i = threadIdx.x; i < 1024; i += 256) {
    const int r = i & 127, c = i >> 7;
    union { uint4 v; uint8_t b[16]; } u;
    const int rt = nb * 8 + (r >> 4);
    if (kb < Kb) {
#pragma unroll
      for (int e = 0; e < 16; ++e) u.b[e] = tile[r][c * 16 + e];
      *(uint4*)(q + ((int64_t)rt * Kb * 2 + kb * 2 + (c >> 2)) * 1024 + (c & 3) * 256 + (r & 15) * 16) = u.v;
    }
    const int ct = kb * 8 + (r >> 4);
    if (qt && nb < Nb) {
#pragma unroll
      for (int e = 0; e < 16; ++e) u.b[e] = tile[c * 16 + e][r];
      *(uint4*)(qt + ((int64_t)ct * Nb * 2 + nb * 2 + (c >> 2)) * 1024 + (c & 3) * 256 + (r & 15) * 16) = u.v;
    }
  }
}

// ---- which matrix pipe ------------------------------------------------------------------------------------------------------------
// The 8-bit pipe adds the products of eight consecutive contraction steps aligned to the largest of them and drops what lies 2^-13 below it
// (measured on crafted operands: of 448 - 448 + s in one group s = 2^-4 is left and 2^-6 is not; between such groups the sums are fp32): up to
// 2^-10 of each group's largest product, 1e-4 of a typical result, more where large products of one group cancel.  A bf16 result has
// 1.7e-3 of rounding and takes that pipe; so does the gated product, whose codes have 2^-4 (its feed-forward is 1.70e-3 from 64 bits
// where fp32 sums are 1.64e-3).  A result that is kept in fp32 takes the bf16 pipe (half the rate; products and sums are fp32; a code times its
// scale is exact in bf16 for scales from 2^-124 on, its last bits 2^-9 2^-124 being the smallest subnormal; smaller scales, of blocks up
// to 1e-35, round to multiples of 2^-133).
__device__ __forceinline__ mfma_b8 widen8(int lo, int hi, float scale) {   // eight codes times their block's scale, as bf16
  typedef __attribute__((ext_vector_type(2))) __bf16 b2;
  const b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return (mfma_b8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ float scale_of(uint32_t word) { return __uint_as_float((word & 0xff) << 23); }

// ---- the tile kernel ---------------------------------------------------------------------------------------------------------------
// global -> LDS without a register: lane i of the wave fetches 16 (4) bytes from base + off and they land at lds + 16 i (4 i)
__device__ __forceinline__ void dma16(const void* base, unsigned off, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "v"(off), "s"(base), "s"(lds));
}
__device__ __forceinline__ void dma4(const void* ptr, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "v"(ptr), "s"(lds));
}
// all but the N newest of this wave's transfers have landed, and its LDS reads have returned
template <int N>
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ i32x8 join(uint4 a, uint4 b) {
  return (i32x8){(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}
__device__ __forceinline__ float act_of(int act, float v) {
  switch (act) {
    case ACT_SILU: return silu_f(v);
    case ACT_RELU: return fmaxf(v, 0.f);
    case ACT_GELU: return gelu_f(v);
    case ACT_GELU_TANH: return gelu_tanh_fast(v);
    default: return v;
  }
}

// eight consecutive columns of one row, rows of odd lengths included (turned round in LDS and stored by single columns, 4096 x 4100 x 4096 took
// 147 us instead of 79): the residual (16 bytes of bf16, 32 of fp32) ...
template <bool F32>
__device__ __forceinline__ void load_res8(const Fp8GemmArgs& a, int m, int n, uint4 r[F32 ? 2 : 1]) {
  const char* p = (const char*)a.residual + ((int64_t)m * a.ldr + n) * (F32 ? 4 : 2);
#pragma unroll
  for (int i = 0; i < (F32 ? 2 : 1); ++i) {
    const u32x4_any t = *(const u32x4_any*)(p + 16 * i);
    r[i] = make_uint4(t[0], t[1], t[2], t[3]);
  }
}
// ... and sums + bias, activation, + residual, stored
template <bool F32>
__device__ __forceinline__ void store8(const Fp8GemmArgs& a, int m, int n, float v[8], const uint4 r[F32 ? 2 : 1]) {
  if (a.bias) {
    const f32x4_any p = *(const f32x4_any*)(a.bias + n), q = *(const f32x4_any*)(a.bias + n + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] += p[i];
      v[4 + i] += q[i];
    }
  }
  if (a.act) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_of(a.act, v[i]);
  }
  if constexpr (F32) {
    if (a.residual) {
      v[0] += __uint_as_float(r[0].x); v[1] += __uint_as_float(r[0].y); v[2] += __uint_as_float(r[0].z); v[3] += __uint_as_float(r[0].w);
      v[4] += __uint_as_float(r[1].x); v[5] += __uint_as_float(r[1].y); v[6] += __uint_as_float(r[1].z); v[7] += __uint_as_float(r[1].w);
    }
    float* c = (float*)a.C + (int64_t)m * a.ldc + n;
    *(f32x4_any*)c = (f32x4_any){v[0], v[1], v[2], v[3]};
    *(f32x4_any*)(c + 4) = (f32x4_any){v[4], v[5], v[6], v[7]};
  } else {
    if (a.residual) {
      const uint32_t t[4] = {r[0].x, r[0].y, r[0].z, r[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] += __uint_as_float(t[i] << 16);
        v[2 * i + 1] += __uint_as_float(t[i] & 0xffff0000u);
      }
    }
    *(u32x4_any*)((bf16_t*)a.C + (int64_t)m * a.ldc + n) = (u32x4_any){pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7])};
  }
}
__device__ __forceinline__ void store1(const Fp8GemmArgs& a, int m, int n, float v) {
  v = act_of(a.act, a.bias ? v + a.bias[n] : v);
  if (a.out_f32) {
    if (a.residual) v += ((const float*)a.residual)[(int64_t)m * a.ldr + n];
    ((float*)a.C)[(int64_t)m * a.ldc + n] = v;
  } else {
    if (a.residual) v += bf2f(((const bf16_t*)a.residual)[(int64_t)m * a.ldr + n]);
    ((bf16_t*)a.C)[(int64_t)m * a.ldc + n] = f2bf(v);
  }
}

// BM x BN output tile, WM x WN waves, v_mfma_scale_f32_32x32x64 with W's rows as the first operand (lane l then holds output row l & 31 and
// runs of four columns).
//
// A stage is 64 contraction steps: 64 bytes of every row, in a ring of four LDS slots filled by LDS-DMA up to three stages ahead (an
// operand that another XCD has not touched yet comes from memory: about 2000 clocks, more than a stage's products).  A stage is MF
// steps (32 rows of X, NF products each); the fragments of step s + AHEAD are read while step s is multiplied.  Where that reading
// crosses into the next stage the waves hand over: the stage behind has been read by all, the next one has landed, and the slot behind
// is refilled by pieces spread over the following steps (in one burst they would block the wave until the address unit, 64 B a
// clock, has taken them).
//
// Workgroups are persistent: a work item is one tile's contraction, or one of equal segments of at most SEG blocks of a long one, and the
// ring runs on into the next item, so a tile's epilogue is spent with the next tile's first stages on their way (a launch of one
// workgroup per tile lost 11 us a tile at 256 x 256 x 4096).  An item's scale bytes are fetched during the item before, into the other of
// two panels.  The last tile row is moved up to end at the last row of X; the rows it shares with its neighbour are not stored twice.
constexpr int BAND = 4;                                               // tile rows walked together (4 and 8 measure alike)
constexpr int SEG = 48;                                              // blocks of 128 per item
constexpr int fp8_segments(int kb) { return (kb + SEG - 1) / SEG; }
constexpr int fp8_segment(int kb) { return (kb + fp8_segments(kb) - 1) / fp8_segments(kb); }
// LDS: the ring, two panels of scales ([block][BM rows of X | 8 groups of W]; the last transfer into one may be whole), and the
// gated form's maxima, one per row and wave column
constexpr int fp8_panel(int BM, int kb) { return (kb < SEG ? kb : SEG) * (BM + 8) + 256; }
constexpr int fp8_smem(int BM, int BN, int WM, int WN, bool gated, int kb) {
  return 4 * (BM + BN) * 64 + 2 * fp8_panel(BM, kb) + (gated ? BM * WN * 4 : 0);
}

template <int BM, int BN, int WM, int WN, bool GATED, bool WIDE>
__global__ __launch_bounds__(WM * WN * 64, 2) void fp8_tile_kernel(const Fp8GemmArgs a, int row0, int tilesM, int tilesN) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int NW = WM * WN, MF = BM / WM / 32, NF = BN / WN / 32, STAGE = (BM + BN) * 64;
  constexpr int AP = BM / 16 / NW, WP = BN / 16 / NW, PIECES = AP + WP;   // 1 KiB pieces (16 rows) per wave and stage
  constexpr int AHEAD = MF >= 2 ? 2 : 1, RING = 2 * MF >= 4 ? 4 : 2, BURST = (PIECES + MF - 1) / MF, LATE = AHEAD * BURST < PIECES ? AHEAD * BURST : PIECES;
  static_assert(AP >= 1 && WP >= 1 && NW % 4 == 0 && (!GATED || (NF == 2 && BN == 256)), "tile shape");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN, half = lane >> 5, j = lane & 31;
  const int total = tilesM * tilesN, G = gridDim.x;
  const unsigned panel = (unsigned)a.Kb * 2048;                       // bytes of one row tile of codes
  const int Mt = (a.M + 15) >> 4, len = fp8_segment(a.Kb);
  const int64_t Mp = (int64_t)Mt * 16, Ng = (int64_t)((a.N + 255) >> 8) * 8;

  // block b runs on XCD b % 8: give each XCD a contiguous range of tiles of a column-first walk through bands of BAND tile rows (the
  // tiles in flight on an XCD share a few panels of X and of W)
  struct Item { int v, m0, mt, n0, kb0, stages; };                    // mt: first row tile of X that is loaded
  auto place = [&](Item& it) {
    const int xcd = it.v & 7, qd = total >> 3, rem = total & 7;
    const int t = (xcd < rem ? xcd * (qd + 1) : rem * (qd + 1) + (xcd - rem) * qd) + (it.v >> 3);
    const int band = t / (BAND * tilesN), in = t - band * BAND * tilesN, rows = tilesM - band * BAND < BAND ? tilesM - band * BAND : BAND;
    it.m0 = row0 + (band * BAND + in % rows) * BM;
    it.n0 = (in / rows) * BN;
    it.mt = it.m0 >> 4;
    if (it.mt > Mt - BM / 16) it.mt = Mt > BM / 16 ? Mt - BM / 16 : 0;
  };
  auto cut = [&](Item& it) { it.stages = 2 * (it.kb0 + len < a.Kb ? len : a.Kb - it.kb0); };
  auto x_of = [&](const Item& it) { return a.X + (int64_t)it.mt * panel + (int64_t)it.kb0 * 2048; };
  // gated: the tile's rows alternate between 32 of W and the same 32 features of W2; a wave's pieces are all of one of them
  const bool second = GATED && ((wave >> 1) & 1);
  auto w_of = [&](const Item& it) {
    return (second ? a.W2 : a.W) + (int64_t)(GATED ? it.n0 >> 5 : it.n0 >> 4) * panel + (int64_t)it.kb0 * 2048;
  };
  unsigned xoff[AP], woff[WP];
#pragma unroll
  for (int p = 0; p < AP; ++p) {
    const int r = p * NW + wave;
    xoff[p] = (unsigned)(r < Mt ? r : Mt - 1) * panel + lane * 16;
  }
#pragma unroll
  for (int p = 0; p < WP; ++p) {
    const int r = p * NW + wave;
    woff[p] = (unsigned)(GATED ? (r >> 2) * 2 + (r & 1) : r) * panel + lane * 16;
  }

  const unsigned lds0 = (unsigned)(uintptr_t)((__attribute__((address_space(3))) char*)smem);
  const int panel_bytes = fp8_panel(BM, a.Kb);
  auto fetch_scales = [&](const Item& it, int which) {                // four bytes per lane, 64 lanes per transfer
    constexpr int per = BM / 4 + 2;
    const int count = (it.stages >> 1) * per;
    for (int e0 = wave * 64; e0 < count; e0 += NW * 64) {
      const int e = e0 + lane < count ? e0 + lane : count - 1, kb = e / per, r = e - kb * per;
      const uint8_t* src;
      if (r < BM / 4) {
        const int64_t m = (int64_t)it.mt * 16 + r * 4;
        src = a.sx + (it.kb0 + kb) * Mp + (m < Mp ? m : Mp - 4);
      } else {
        const int64_t g = GATED ? (it.n0 >> 8) * 4 : (it.n0 >> 7) * 4 + (r - BM / 4) * 4;
        src = (GATED && r > BM / 4 ? a.sw2 : a.sw) + (it.kb0 + kb) * Ng + (g < Ng ? g : Ng - 4);
      }
      dma4(src, (unsigned)__builtin_amdgcn_readfirstlane(lds0 + 4 * STAGE + which * panel_bytes + e0 * 4));
    }
  };

  f32x16 acc[NF][MF];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int k = 0; k < MF; ++k) acc[i][k] = (f32x16){};
  i32x8 x[RING], w[2][NF];
  mfma_b8 wide[WIDE ? NF : 1][4];
  int sx[MF], sw[NF], nsx[MF], nsw[NF];
  auto frag = [&](int slot, int row) {            // rows row + (0 .. 31), columns 32 half + (0 .. 31) of a stage
    const char* r = smem + (slot & 3) * STAGE + row * 64 + (j >> 4) * 1024 + half * 512 + (j & 15) * 16;
    return join(*(const uint4*)r, *(const uint4*)(r + 256));
  };
  auto read_step = [&](int slot, int s) {         // step s of the two stages of a block, and on into the next block's
    if (s % MF == 0) {
#pragma unroll
      for (int i = 0; i < NF; ++i) w[s / MF & 1][i] = frag(slot + s / MF, BM + wn * (BN / WN) + i * 32);
    }
    x[s % RING] = frag(slot + s / MF, wm * (BM / WM) + (s % MF) * 32);
  };
  auto multiply = [&](int s) {
    const int k = s % MF, ks = s / MF;
    if constexpr (!WIDE) {
#pragma unroll
      for (int i = 0; i < NF; ++i)
        acc[i][k] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[ks][i], x[s % RING], acc[i][k], 0, 0, 0, sw[i], 0, sx[k]);
    } else {
      if (k == 0) {
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) wide[i][q] = widen8(w[ks][i][2 * q], w[ks][i][2 * q + 1], scale_of(sw[i]));
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const mfma_b8 xb = widen8(x[s % RING][2 * q], x[s % RING][2 * q + 1], scale_of(sx[k]));
#pragma unroll
        for (int i = 0; i < NF; ++i) acc[i][k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wide[i][q], xb, acc[i][k], 0, 0, 0);
      }
    }
  };
  // scale bytes of an item's block kb.  W's eight bytes: four 32-row groups of W, then the next four or, gated, those of W2
  auto read_scales = [&](const Item& it, int which, int kb) {
    const char* q = smem + 4 * STAGE + which * panel_bytes + kb * (BM + 8);
#pragma unroll
    for (int i = 0; i < MF; ++i) nsx[i] = *(const uint8_t*)(q + wm * (BM / WM) + i * 32 + j);
#pragma unroll
    for (int i = 0; i < NF; ++i) nsw[i] = *(const uint8_t*)(q + BM + (GATED ? i * 4 + wn : (BN < 128 ? (it.n0 >> 5) & 3 : 0) + wn * NF + i));
  };

  auto epilogue = [&](const Item& it) {
    const int mw = it.mt * 16 + wm * (BM / WM), nw = it.n0 + wn * (BN / WN);
    if constexpr (GATED) {
      // the tile's 128 features are one block of the next product's contraction: amax per row over the four waves of a row group
      float* red = (float*)(smem + 4 * STAGE + 2 * panel_bytes);      // [BM][WN]
      float h[MF][16];
#pragma unroll
      for (int k = 0; k < MF; ++k) {
        float m = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int f = it.n0 / 2 + wn * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
          h[k][r] = f < a.N ? gelu_tanh_fast(acc[0][k][r]) * acc[1][k][r] : 0.f;
          m = fmaxf(m, finite_abs(h[k][r]));
        }
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        if (half == 0) red[(wm * (BM / WM) + k * 32 + j) * WN + wn] = m;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < MF; ++k) {
        const int row = wm * (BM / WM) + k * 32 + j, m = it.mt * 16 + row;
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < WN; ++i) mx = fmaxf(mx, red[row * WN + i]);
        const int byte = scale_byte(mx);
        const float up = scale_up(byte);
        uint32_t d[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) d[r] = codes4(h[k][4 * r], h[k][4 * r + 1], h[k][4 * r + 2], h[k][4 * r + 3], up);
        // lanes l and l + 32 hold alternating runs of four features: exchange so that each has 16 consecutive ones
        const auto e0 = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false);
        const auto e1 = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
        if (m >= it.m0 && m < a.M) {
          const int nb = (a.N + 127) >> 7, blk = it.n0 >> 8;
          *(uint4*)(a.H + ((int64_t)(m >> 4) * nb * 2 + blk * 2 + (wn >> 1)) * 1024 + ((wn & 1) * 2 + half) * 256 + (m & 15) * 16) =
              make_uint4(e0[0], e0[1], e1[0], e1[1]);
          if (half == 0 && wn == 0) a.sh[(int64_t)blk * Mp + m] = (uint8_t)byte;
        }
      }
      __syncthreads();                                                // (red is written again by the next tile)
    } else {
      // lanes l and l + 32 hold alternating runs of four columns: exchange so that each has eight consecutive ones.  The residual of the next
      // 32 rows is asked for before these are stored (C may be the residual, so the compiler keeps loads behind the stores before them;
      // 8192^3 with a residual: 457 us without, 441 with the loads ahead)
      uint4 res[2][NF][2][WIDE ? 2 : 1];
      auto fetch = [&](int k) {
        const int m = mw + k * 32 + j;
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int n = nw + i * 32 + r * 16 + half * 8;
            if (m >= it.m0 && m < a.M && n + 8 <= a.N) load_res8<WIDE>(a, m, n, res[k & 1][i][r]);
          }
      };
      if (a.residual) fetch(0);
#pragma unroll
      for (int k = 0; k < MF; ++k) {
        if (a.residual && k + 1 < MF) fetch(k + 1);
        const int m = mw + k * 32 + j;
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float v[8];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const auto e = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[i][k][8 * r + t]), __float_as_uint(acc[i][k][8 * r + 4 + t]),
                                                              false, false);
              v[t] = __uint_as_float(e[0]);
              v[4 + t] = __uint_as_float(e[1]);
            }
            const int n = nw + i * 32 + r * 16 + half * 8;
            if (m >= it.m0 && m < a.M) {
              if (n + 8 <= a.N) store8<WIDE>(a, m, n, v, res[k & 1][i][r]);
              else {                                                  // the last columns of a row, one by one (unrolled, the 256 x 256
#pragma unroll 1                                                      // tile spills over it: 16384 x 10240 x 4096 in 597 us instead of 526)
                for (int c = n; c < a.N; ++c) {
                  store1(a, m, c, v[0]);
#pragma unroll
                  for (int t = 0; t < 7; ++t) v[t] = v[t + 1];
                }
              }
            }
          }
      }
    }
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int k = 0; k < MF; ++k) acc[i][k] = (f32x16){};
  };

  Item cur;
  cur.v = blockIdx.x;
  cur.kb0 = 0;
  place(cur);
  cut(cur);
  int slot = 0, which = 0;                        // ring position of the item's first stage; its panel
  const uint8_t* xb = x_of(cur);
  const uint8_t* wb = w_of(cur);
  auto piece_at = [&](const uint8_t* xk, const uint8_t* wk, int at, int p) {
    const unsigned to = (unsigned)__builtin_amdgcn_readfirstlane(lds0 + (at & 3) * STAGE + wave * 1024);
    if (p < AP) dma16(xk, xoff[p < AP ? p : 0], to + p * NW * 1024);
    else dma16(wk, woff[p < AP ? 0 : p - AP], to + BM * 64 + (p - AP) * NW * 1024);
  };
  fetch_scales(cur, 0);
#pragma unroll
  for (int h = 0; h < 4; ++h)
#pragma unroll
    for (int p = 0; p < (h < 3 ? PIECES : LATE); ++p) {    // (the loop's first steps issue the rest of the fourth)
      const int64_t k = (int64_t)(h < cur.stages ? h : cur.stages - 1) * 1024;
      piece_at(xb + k, wb + k, h, p);
    }
  dma_wait<2 * PIECES + LATE>();                  // (the scales are older: landed too)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) read_step(0, s);
  while (true) {
    Item nxt = cur;
    nxt.kb0 += len;
    bool more = nxt.kb0 < a.Kb;
    const bool done = !more;                      // the tile ends with this item
    if (done) {
      nxt.kb0 = 0;
      nxt.v += G;
      more = nxt.v < total;
      if (more) place(nxt);
    }
    // where the stages behind this item's lie: the next item's, or its own last one over and over
    int64_t xd = (int64_t)(cur.stages - 1) * 1024, wd = xd;
    int step = 0;
    if (more) {
      cut(nxt);
      fetch_scales(nxt, which ^ 1);
      xd = x_of(nxt) - xb;
      wd = w_of(nxt) - wb;
      step = 1024;
    }
    read_scales(cur, which, 0);
    const int blocks = cur.stages >> 1;
    for (int kb = 0; kb < blocks; ++kb) {         // (no branch in this body: the compiler would sink the products past it)
#pragma unroll
      for (int i = 0; i < MF; ++i) sx[i] = nsx[i];
#pragma unroll
      for (int i = 0; i < NF; ++i) sw[i] = nsw[i];
#pragma unroll
      for (int s = 0; s < 2 * MF; ++s) {
        if (s % MF == MF - AHEAD) {               // hand over
          dma_wait<2 * PIECES>();
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
        read_step(slot + 2 * kb, s + AHEAD);
        if (s == 0) read_scales(cur, which, kb + 1 < blocks ? kb + 1 : kb);
        if constexpr (MF < 4) __builtin_amdgcn_sched_barrier(0);   // (8192^3: 464 us with it at 128 x 128, 482 without; 256 x 256: 395, 390)
        multiply(s);
        const int u = (s + AHEAD) % MF, h = 2 * kb + (s + AHEAD) / MF + 3;   // burst u since the hand-over to stage h - 3
        const int over = h - cur.stages;
        const int64_t in = over >> 31, own = (int64_t)h * 1024, far = (int64_t)over * step;
        const int64_t kx = (in & own) | (~in & (xd + far)), kw = (in & own) | (~in & (wd + far));
#pragma unroll
        for (int p = u * BURST; p < (u + 1) * BURST && p < PIECES; ++p) piece_at(xb + kx, wb + kw, slot + h, p);
      }
    }
    if (done) epilogue(cur);
    if (!more) break;
    slot += cur.stages;
    which ^= 1;
    cur = nxt;
    xb = x_of(cur);
    wb = w_of(cur);
  }
  dma_wait<0>();                                  // no transfer may be on its way when the workgroup's LDS is released
}

// the kernel's allowance of dynamic LDS, asked for once per device (`done`: one bit for each)
int allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  FDMI_HIP(hipGetDevice(&dev));
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return 0;
  FDMI_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return 0;
}

// the rows from row0 on (a multiple of 16), `rows` of them (a multiple of BM, or all)
template <int BM, int BN, int WM, int WN, bool GATED, bool WIDE>
int launch_tile(const Fp8GemmArgs& a, hipStream_t st, int row0 = 0, int rows = 0) {
  constexpr int most = fp8_smem(BM, BN, WM, WN, GATED, SEG);
  static_assert(most <= 160 * 1024, "LDS");
  static std::atomic<uint64_t> allowed;
  const int smem = fp8_smem(BM, BN, WM, WN, GATED, a.Kb);
  const int64_t tilesM = ((int64_t)(rows ? rows : a.M - row0) + BM - 1) / BM, tilesN = ((int64_t)a.N * (GATED ? 2 : 1) + BN - 1) / BN;
  FDMI_CHECK(tilesM * tilesN < (1ll << 30), "gemm_fp8: too many tiles");
  // as many workgroups as fit (a multiple of the 8 XCDs); one per tile where an item is too short for the ring to run across items
  int fit = 160 * 1024 / smem;
  if (fit > 2048 / (WM * WN * 64)) fit = 2048 / (WM * WN * 64);
  const int64_t room = (int64_t)256 * fit, total = tilesM * tilesN;
  const int64_t grid = a.Kb < 2 || total < room ? total : room;
  FDMI_CHECK(grid * (WM * WN * 64) <= FDMI_LAUNCH_THREADS, "gemm_fp8: too many tiles for one launch");
  if (const int rc = allow_lds((const void*)fp8_tile_kernel<BM, BN, WM, WN, GATED, WIDE>, most, allowed)) return rc;
  hipLaunchKernelGGL((fp8_tile_kernel<BM, BN, WM, WN, GATED, WIDE>), dim3((unsigned)grid), dim3(WM * WN * 64), smem, st, a, row0, (int)tilesM,
                     (int)tilesN);
  FDMI_HIP(hipGetLastError());
  return 0;
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------------
// A product of few rows is bound by streaming the weight once.  A workgroup takes 16 NT rows of W and 16 MT rows of X; its eight waves share
// out the contraction (block kb goes to wave kb % 8), fetch whole tiles straight into matrix fragments -- a lane's two 16-byte reads of
// a 16 x 128 pair of tiles are v_mfma_scale_f32_16x16x128's operand -- DEPTH blocks at a time, and join their sums through LDS in the
// order of the waves.  No split over workgroups: N / 16 of them fill the chip from N = 4096 on, and smaller weights sit in L2.
constexpr int FUSE = 1 << 16;            // bytes of codes that a workgroup quantises for itself
constexpr int fp8_stream_smem(int MT, int NT) { return 8 * MT * 16 * (NT * 16 + 4) * 4; }

template <int MT, int NT, bool WIDE, typename RAW>
__global__ __launch_bounds__(512) void fp8_stream_kernel(const Fp8GemmArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int DEPTH = MT * 2 + NT * 2 <= 4 ? 4 : MT * 2 + NT * 2 <= 8 ? 2 : 1, LD = NT * 16 + 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t panel = (int64_t)a.Kb * 2048;
  const int Mt = (a.M + 15) >> 4, across = (a.N + NT * 16 - 1) / (NT * 16), mt0 = blockIdx.x / across * MT, nt0 = blockIdx.x % across * NT;
  const int64_t Mp = (int64_t)Mt * 16, Ng = (int64_t)((a.N + 255) >> 8) * 8;
  constexpr bool FUSED = !std::is_void<RAW>::value;
  static_assert(!FUSED || MT == 1, "sixteen rows");
  const uint8_t* wp[NT];
  const uint8_t* xp[MT];
  const uint8_t* sxp[MT];
#pragma unroll
  for (int i = 0; i < NT; ++i) wp[i] = a.W + (nt0 + i) * panel + lane * 16;
#pragma unroll
  for (int k = 0; k < MT; ++k) {
    const int mt = mt0 + k < Mt ? mt0 + k : Mt - 1;                  // (rows past the last tile repeat it and are not stored)
    xp[k] = a.X + mt * panel + lane * 16;
    sxp[k] = a.sx + mt * 16 + (lane & 15);
  }
  const uint8_t* swp = a.sw + (nt0 >> 1);
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int k = 0; k < MT; ++k) acc[i][k] = (f32x4){0.f, 0.f, 0.f, 0.f};
  i32x8 w[DEPTH][NT], x[DEPTH][MT];
  int sw[DEPTH], sx[DEPTH][MT];
  auto fetch_w = [&](int kb0) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int kb = kb0 + 8 * d < a.Kb ? kb0 + 8 * d : kb0;
#pragma unroll
      for (int i = 0; i < NT; ++i) w[d][i] = join(*(const uint4*)(wp[i] + (int64_t)kb * 2048), *(const uint4*)(wp[i] + (int64_t)kb * 2048 + 1024));
      sw[d] = swp[kb * Ng];                                            // (16 NT rows lie in one group of 32)
    }
  };
  if constexpr (FUSED) {
    // the rows come unquantised: every workgroup quantises all of them into LDS, [chunk of 16 columns][row][16 bytes] and scales behind
    // (at most FUSE bytes of codes; one launch instead of two), while its first tiles of W are on their way
    if (wave < a.Kb) fetch_w(wave);
    const int per = a.Kb * 8;
    uint8_t* sq = (uint8_t*)smem + a.M * per * 16;
    for (int u = threadIdx.x; u < a.M * per; u += 512) {
      const int m = u / per, c = u - m * per;
      float v[16];
      load16((const RAW*)a.x + (int64_t)m * a.ldxr, c * 16, a.K, v);
      const int byte = block_scale(v, 1, 2, 4);
      *(uint4*)(smem + (c * a.M + m) * 16) = codes16(v, scale_up(byte));
      if ((c & 7) == 0) sq[(c >> 3) * a.M + m] = (uint8_t)byte;
    }
    __syncthreads();
  }
  for (int kb0 = wave; kb0 < a.Kb; kb0 += 8 * DEPTH) {
    if (!FUSED || kb0 != wave) fetch_w(kb0);
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int kb = kb0 + 8 * d < a.Kb ? kb0 + 8 * d : kb0;
      if constexpr (FUSED) {
        const int m = (lane & 15) < a.M ? lane & 15 : a.M - 1, c = kb * 8 + (lane >> 4);
        x[d][0] = join(*(const uint4*)(smem + (c * a.M + m) * 16), *(const uint4*)(smem + ((c + 4) * a.M + m) * 16));
        sx[d][0] = ((const uint8_t*)smem)[a.M * a.Kb * 128 + kb * a.M + m];
      } else {
        const int64_t o = (int64_t)kb * 2048;
#pragma unroll
        for (int k = 0; k < MT; ++k) x[d][k] = join(*(const uint4*)(xp[k] + o), *(const uint4*)(xp[k] + o + 1024));
#pragma unroll
        for (int k = 0; k < MT; ++k) sx[d][k] = sxp[k][kb * Mp];
      }
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (kb0 + 8 * d >= a.Kb) break;
      if constexpr (!WIDE) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int k = 0; k < MT; ++k)
            acc[i][k] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[d][i], x[d][k], acc[i][k], 0, 0, 0, sw[d], 0, sx[d][k]);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          mfma_b8 wb[NT];
#pragma unroll
          for (int i = 0; i < NT; ++i) wb[i] = widen8(w[d][i][2 * q], w[d][i][2 * q + 1], scale_of(sw[d]));
#pragma unroll
          for (int k = 0; k < MT; ++k) {
            const mfma_b8 xb = widen8(x[d][k][2 * q], x[d][k][2 * q + 1], scale_of(sx[d][k]));
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[i][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[i], xb, acc[i][k], 0, 0, 0);
          }
        }
      }
    }
  }
  // lane l holds output row l & 15 and columns 4 (l >> 4) + 0 .. 3 of each fragment
  float* red = (float*)smem;
  if constexpr (FUSED) __syncthreads();                                // (the codes lie there)
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int k = 0; k < MT; ++k)
      *(f32x4*)(red + ((wave * MT + k) * 16 + (lane & 15)) * LD + i * 16 + (lane >> 4) * 4) = acc[i][k];
  __syncthreads();
  for (int e = threadIdx.x; e < MT * 16 * NT * 16; e += 512) {
    const int r = e / (NT * 16), c = e % (NT * 16), m = mt0 * 16 + r, n = nt0 * 16 + c;
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) v += red[(q * MT * 16 + r) * LD + c];
    if (m < a.M && n < a.N) store1(a, m, n, v);
  }
}

template <int MT, int NT, bool WIDE, typename RAW>
int launch_stream(const Fp8GemmArgs& a, hipStream_t st) {
  constexpr int join = fp8_stream_smem(MT, NT), most = std::is_void<RAW>::value ? join : FUSE + FUSE / 128;
  static_assert(join <= most && most <= 160 * 1024, "LDS");
  static std::atomic<uint64_t> allowed;
  const int codes = std::is_void<RAW>::value ? 0 : a.M * a.Kb * 129, smem = join > codes ? join : codes;
  const int64_t grid = (int64_t)cdiv(a.N, NT * 16) * cdiv(a.M, MT * 16);   // (in one dimension: the second holds 65535)
  FDMI_CHECK(grid * 512 <= FDMI_LAUNCH_THREADS, "gemm_fp8: too many tiles for one launch");
  if (const int rc = allow_lds((const void*)fp8_stream_kernel<MT, NT, WIDE, RAW>, most, allowed)) return rc;
  hipLaunchKernelGGL((fp8_stream_kernel<MT, NT, WIDE, RAW>), dim3((unsigned)grid), dim3(512), smem, st, a);
  FDMI_HIP(hipGetLastError());
  return 0;
}

}  // namespace

int launch_quant_fp8(const void* x, int x_f32, int64_t ldx, const float* norm, float eps, uint8_t* q, uint8_t* s, int64_t M, int K,
                     hipStream_t st) {
  if (M == 0) return 0;
  const int Kb = cdiv(K, 128);
  const int64_t Mp = (M + 15) / 16 * 16;
  FDMI_CHECK(cdiv(Kb, 16) < 65536, "quant_fp8: too many columns");
  constexpr int64_t SLICE = 1ll << 25;             // rows of one launch (256 threads for four of them)
  for (int64_t m0 = 0; m0 < M; m0 += SLICE) {
    const int64_t rows = M - m0 < SLICE ? M - m0 : SLICE;
    const dim3 grid((unsigned)((rows + 3) / 4), norm ? 1 : cdiv(Kb, 16));
    const char* from = (const char*)x + m0 * ldx * (x_f32 ? 4 : 2);
    uint8_t* to = q + m0 * Kb * 128;
#define FP8_QUANT(T, NORM) hipLaunchKernelGGL((quant_rows_kernel<T, NORM>), grid, dim3(256), 0, st, (const T*)from, ldx, norm, eps, to, s + m0, rows, Mp, K, Kb)
    if (norm) { if (x_f32) FP8_QUANT(float, true); else FP8_QUANT(bf16_t, true); }
    else { if (x_f32) FP8_QUANT(float, false); else FP8_QUANT(bf16_t, false); }
#undef FP8_QUANT
    FDMI_HIP(hipGetLastError());
  }
  return 0;
}

int launch_pack_fp8(const void* w, int w_f32, int64_t ldw, int N, int K, uint8_t* q, uint8_t* s, uint8_t* qt, uint8_t* st, hipStream_t stream) {
  const dim3 grid(qt ? cdiv(K, 256) * 2 : cdiv(K, 128), cdiv(N, 256) * 2);
  if (w_f32) hipLaunchKernelGGL(pack_kernel<float>, grid, dim3(256), 0, stream, (const float*)w, ldw, N, K, q, s, qt, st);
  else hipLaunchKernelGGL(pack_kernel<bf16_t>, grid, dim3(256), 0, stream, (const bf16_t*)w, ldw, N, K, q, s, qt, st);
  FDMI_HIP(hipGetLastError());
  return 0;
}

// Which kernel: the least of the times that formulas in the problem's sizes give (microseconds), their constants fitted to times of every kernel on drawn
// problems.  On 147 others (16 .. 16384 rows, 64 .. 12288 columns, K 64 .. 10240, half of them large; every kernel's time for each in
// profiles/fp8_kernel_choice.csv) the chosen one is 4.5% slower than the best on average for a bf16 result and 5.8% for fp32; by more
// than 1.4 times in seven of 294, six of them below 5 us and 1588 x 2584 x 3584 in fp32 (69.9 us, 44.7 with 128 x 128 tiles).  A tile kernel spends `block` + `share` * w on a block of 128 and `fixed` + `tile` * w beside, w = tiles per CU
// rounded up; a grid that leaves CUs idle runs its blocks up to `idle` faster.  The streaming kernel is bound by what its workgroups read
// from L2 (a short grid leaves some CUs idle) or by the weight from memory, and pays for each further turn of 1024 workgroups.
// For example (us; 64 / 128 / 128 x 256 / 256 tile, stream): 1 x 4096 x 4096: 11.2 / 15.7 / 22.8 / 36, 4.3;  1920 x 4096 x 4096:
// 57 / 33.6 / 32.9 / 47, 86;  1920 x 10240 x 4096: 123 / 75.5 / 83.9 / 93, 246;  8192^3: 935 / 469 / 477 / 403, 2234.
struct Fp8Cost { int BM, BN; double block, share, fixed, tile, idle; };
double fp8_cost(int64_t M, int64_t N, int Kb, const Fp8Cost& c) {
  const double tiles = double((M + c.BM - 1) / c.BM) * ((N + c.BN - 1) / c.BN), w = (double)(int64_t)((tiles + 255) / 256);
  return c.fixed + c.tile * w + Kb * (c.block + c.share * w * (tiles < 256 ? 1. - c.idle * (1. - tiles / 256) : 1.));
}
double fp8_stream_cost(const Fp8GemmArgs& a, int rows) {   // `rows` rows of X and of W per workgroup
  const double groups = double(((int64_t)a.M + rows - 1) / rows) * ((a.N + rows - 1) / rows), more = (double)(int64_t)((groups - 1) / 1024);
  if (groups * 512 > FDMI_LAUNCH_THREADS) return 1e30;     // (more than one launch holds)
  const double l2 = (groups < 256 ? 256 : groups) * 2 * rows * a.Kb * 128 / 24e6, hbm = double(a.N) * a.Kb * 128 / 4.5e6;
  return (rows == 16 ? 3.5 + .5 * more : 3. + 1.3 * more) + (l2 > hbm ? l2 : hbm);
}
constexpr double FP8_LAUNCH = 1.5;                         // a second launch on the same stream
// The largest tiles are the fastest per product and leave the most CUs idle in the last turn.  The rows that fill whole turns of 256 x 256
// tiles; the others may go to a second launch of smaller ones (gated 1920 x 4096 -> 10240: 153 us on 128-row tiles, 111 + 33 on 1536 rows of the
// large and 384 of the small; 3500 x 5120 x 2048: 49 us)
int fp8_whole(int64_t M, int64_t N) {
  const int64_t cols = (N + 255) / 256, turns = M / 256 * cols / 256;
  return (int)(turns * 256 / cols * 256);
}

// whether a product of unquantised rows quantises them inside the streaming kernel
bool fp8_fused(int64_t M, int K) { return M <= 16 && M * cdiv(K, 128) * 128 <= FUSE; }

int launch_gemm_fp8(const Fp8GemmArgs& a, hipStream_t st) {
  if (a.M == 0) return 0;
  if (a.x) {   // unquantised rows without scratch (fp8_fused)
    if (a.x_f32) return a.out_f32 ? launch_stream<1, 1, true, float>(a, st) : launch_stream<1, 1, false, float>(a, st);
    return a.out_f32 ? launch_stream<1, 1, true, bf16_t>(a, st) : launch_stream<1, 1, false, bf16_t>(a, st);
  }
  static const Fp8Cost narrow[] = {{64, 64, .08, .174, 2.4, .63, 0.}, {128, 128, .06, .384, 3.3, 1.8, .27}, {128, 256, .07, .744, .9, 4.3, .34},
                                   {256, 256, .10, 1.39, .2, 7.5, .39}};
  static const Fp8Cost wide[] = {{64, 64, .20, .265, 2., .95, 0.}, {128, 128, .27, .69, 2., 3.25, .37}, {256, 256, .33, 2.74, 0., 9.8, .43}};
  if (a.H) {
    // A tile is 128 features.  While 128-row ones leave half of the CUs without work, twice as many of 64 rows end sooner (K = 4096: 768 x 2560,
    // 120 against 240 workgroups, 26.3 and 19.7 us; 120 x 10240, 80 against 160: 25.4 and 18.5), from there on they do not (1024 x 2560, 160 against
    // 320: 26.9 and 34.6; 200 x 10240: 27.1 and 34.5; profiles/fp8_gated_choice.csv)
    const int64_t cols = ((int64_t)a.N + 127) / 128 * 256;
    if (((int64_t)a.M + 127) / 128 * (cols / 256) < 128) return launch_tile<64, 256, 1, 4, true, false>(a, st);
    const int whole = fp8_whole(a.M, cols), rest = a.M - whole;
    const double small = fp8_cost(a.M, cols, a.Kb, narrow[2]), large = fp8_cost(a.M, cols, a.Kb, narrow[3]);
    const double both = whole && rest ? fp8_cost(whole, cols, a.Kb, narrow[3]) + FP8_LAUNCH + fp8_cost(rest, cols, a.Kb, narrow[2]) : 1e30;
    if (small <= large && small <= both) return launch_tile<128, 256, 2, 4, true, false>(a, st);
    if (large <= both) return launch_tile<256, 256, 2, 4, true, false>(a, st);
    if (const int rc = launch_tile<256, 256, 2, 4, true, false>(a, st, 0, whole)) return rc;
    return launch_tile<128, 256, 2, 4, true, false>(a, st, whole);
  }
  const Fp8Cost* table = a.out_f32 ? wide : narrow;
  const int kinds = a.out_f32 ? 3 : 4;
  auto cheapest = [&](int64_t rows, double& least) {
    int best = -1;
    for (int i = 0; i < kinds; ++i) {
      const double c = fp8_cost(rows, a.N, a.Kb, table[i]);
      if (best < 0 || c < least) { best = i; least = c; }
    }
    return best;
  };
#define FP8_TILE(BM, BN, WM, WN, WIDE) launch_tile<BM, BN, WM, WN, false, WIDE>(a, st, row0, rows)
  auto run = [&](int kind, int row0, int rows) {
    switch (table[kind].BM + table[kind].BN) {
      case 128: return a.out_f32 ? FP8_TILE(64, 64, 2, 2, true) : FP8_TILE(64, 64, 2, 2, false);
      case 256: return a.out_f32 ? FP8_TILE(128, 128, 2, 2, true) : FP8_TILE(128, 128, 2, 2, false);
      case 384: return FP8_TILE(128, 256, 2, 4, false);
      default:
        return a.out_f32 ? FP8_TILE(256, 256, 2, 4, true) : FP8_TILE(256, 256, 2, 4, false);
    }
  };
#undef FP8_TILE
  double least = 0., tail = 0.;
  const int best = cheapest(a.M, least);
  const double s16 = fp8_stream_cost(a, 16), s32 = fp8_stream_cost(a, 32);
  if (s16 <= s32 && s16 < least) return a.out_f32 ? launch_stream<1, 1, true, void>(a, st) : launch_stream<1, 1, false, void>(a, st);
  if (s32 < least) return a.out_f32 ? launch_stream<2, 2, true, void>(a, st) : launch_stream<2, 2, false, void>(a, st);
  const int whole = fp8_whole(a.M, a.N);
  if (whole && whole < a.M) {
    const int kind = cheapest(a.M - whole, tail);
    if (kind != kinds - 1 && fp8_cost(whole, a.N, a.Kb, table[kinds - 1]) + FP8_LAUNCH + tail < least) {
      if (const int rc = run(kinds - 1, 0, whole)) return rc;
      return run(kind, whole, 0);
    }
  }
  return run(best, 0, 0);
}
