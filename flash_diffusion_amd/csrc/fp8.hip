// Matrix products of 8-bit floating-point codes with a scale for each block of 128 along the contraction (gfx950).
//
//   y[m][n] = sum_b 2^(ex[m][b] + ew[n/128][b]) * sum_{k in block b} qx[m][k] * qw[n][k]        qx, qw: e4m3 codes
//
// The scales are powers of two (e8m0 bytes): 2^e is the smallest power with amax <= 448 2^e over the block, so a code never saturates,
// scaling is exact and the only rounding of the format is the one to e4m3 (round to nearest even).  CDNA4's scaled matrix instruction
// takes such a scale per lane and 32 contraction steps: a block of 128 hands the same byte to its steps, and the scales cost no
// arithmetic of their own.  Sums are fp32 in the accumulators.  An infinity or NaN of the input becomes the NaN code (e4m3 has no
// infinity, and a saturated code would hide the overflow) and the block's scale comes from its finite values.
//
// Codes lie in tiles of 16 rows x 64 columns, 1 KiB each: [row tile][column tile][chunk of 16 columns][row][16 bytes].  One wave's load, store or
// LDS transfer moves whole tiles (row-major codes fill LDS at two thirds of that rate: 128 x 128 tiles of an 8192^3 product in 627 against
// 499 us), a matrix fragment is one 16-byte read per lane and tile, and the 16 lanes that LDS serves at once read 256 consecutive bytes.
// Scale bytes of activations: [block of 128 columns][rows padded to 16]; of weights: [block][groups of 32 rows, padded to four groups].
#include "fp8.h"
#include "gemm.h"

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

// eight consecutive elements of a row from column k on; columns >= K read as zero.  vec: rows start 16-byte aligned
template <typename T>
__device__ __forceinline__ void load8(const T* p, int k, int K, bool vec, float v[8]) {
  if (vec && k + 8 <= K) {
    if constexpr (sizeof(T) == 2) {
      const u16x8 t = *(const u16x8*)(p + k);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = bf2f(t[i]);
    } else {
      const float4 a = *(const float4*)(p + k), b = *(const float4*)(p + k + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
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
__device__ __forceinline__ void load16(const T* p, int k, int K, bool vec, float v[16]) {
  load8(p, k, K, vec, v);
  load8(p, k + 8, K, vec, v + 8);
}
__device__ __forceinline__ uint4 codes16(const float v[16], float up) {
  return make_uint4(codes4(v[0], v[1], v[2], v[3], up), codes4(v[4], v[5], v[6], v[7], up), codes4(v[8], v[9], v[10], v[11], up),
                    codes4(v[12], v[13], v[14], v[15], up));
}

// ---- rows of activations -------------------------------------------------------------------------------------------------------------
// Four rows per workgroup; a wave takes 256 columns at a time, 16 per lane (four neighbouring lanes hold the four rows of one chunk and write
// 64 consecutive bytes).  NORM: y = x * rsqrt(mean(x^2) + eps) * w in fp32 first, each wave summing one row's squares.
template <typename T, bool NORM>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* x, int64_t ldx, const float* w, float eps, uint8_t* q, uint8_t* s, int64_t M,
                                                         int64_t Mp, int K, int Kb, bool vec, bool wvec) {
  __shared__ float rs[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m0 = (int64_t)blockIdx.x * 4;
  if constexpr (NORM) {
    const T* row = x + (m0 + wave < M ? m0 + wave : M - 1) * ldx;
    float ss = 0.f, v[8];
    for (int k = lane * 8; k < K; k += 512) {
      load8(row, k, K, vec, v);
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
  const int first = NORM ? wave * 256 : (blockIdx.y * 4 + wave) * 256, step = NORM ? 1024 : Kb * 128;
  for (int k0 = first; k0 < Kb * 128; k0 += step) {
    const int k = k0 + c * 16;
    float v[16], g[16];
    load16(row, k, m < M ? K : 0, vec, v);
    if constexpr (NORM) {
      load16(w, k, K, wvec, g);
      const float rr = rs[r];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = v[i] * rr * g[i];
    }
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) a = fmaxf(a, finite_abs(v[i]));
#pragma unroll
    for (int o = 4; o <= 16; o <<= 1) a = fmaxf(a, __shfl_xor(a, o, 64));   // the eight chunks of a block of 128
    const int byte = scale_byte(a);
    if (k < Kb * 128) {
      *(uint4*)(q + ((m >> 4) * Kb * 2 + (k >> 6)) * 1024 + (c & 3) * 256 + (m & 15) * 16) = codes16(v, scale_up(byte));
      if ((c & 7) == 0) s[(k >> 7) * Mp + m] = (uint8_t)byte;
    }
  }
}

// ---- weights: one workgroup per 128 x 128 block, codes in both orders (once per weight) --------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(const T* w, int64_t ldw, int N, int K, uint8_t* q, uint8_t* s, uint8_t* qt, uint8_t* st) {
  __shared__ uint8_t tile[128][132];
  __shared__ float part[4];
  const int nb = blockIdx.y, kb = blockIdx.x, Nb = gridDim.y, Kb = gridDim.x;
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
    s[(int64_t)kb * (Nb * 4) + nb * 4 + threadIdx.x] = (uint8_t)byte;
    if (st) st[(int64_t)nb * (Kb * 4) + kb * 4 + threadIdx.x] = (uint8_t)byte;
  }
  __syncthreads();
  // 16-byte chunk i of the block's 16 tiles: row r, columns 16 c ..
  for (int i = threadIdx.x; i < 1024; i += 256) {
    const int r = i & 127, c = i >> 7;
    union { uint4 v; uint8_t b[16]; } u;
    const int rt = nb * 8 + (r >> 4);
    if (rt * 16 < N) {
#pragma unroll
      for (int e = 0; e < 16; ++e) u.b[e] = tile[r][c * 16 + e];
      *(uint4*)(q + ((int64_t)rt * Kb * 2 + kb * 2 + (c >> 2)) * 1024 + (c & 3) * 256 + (r & 15) * 16) = u.v;
    }
    const int ct = kb * 8 + (r >> 4);
    if (qt && ct * 16 < K) {
#pragma unroll
      for (int e = 0; e < 16; ++e) u.b[e] = tile[c * 16 + e][r];
      *(uint4*)(qt + ((int64_t)ct * Nb * 2 + nb * 2 + (c >> 2)) * 1024 + (c & 3) * 256 + (r & 15) * 16) = u.v;
    }
  }
}

// ---- which matrix pipe ------------------------------------------------------------------------------------------------------------
// The 8-bit pipe adds the products of eight consecutive contraction steps aligned to the largest of them and drops what lies 2^-13 below it
// (measured on crafted operands; between such groups the sums are fp32): 1e-4 of a typical result.  A bf16 result has 1.7e-3 of rounding
// and takes that pipe; a result that is kept in fp32 takes the bf16 pipe (half the rate; codes convert exactly, their scale rides in the
// conversion's exponent, products and sums are fp32).
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

// eight consecutive columns of one row: + bias + residual, activation, 16-byte stores.  Rows of C, the residual and the bias are aligned
__device__ __forceinline__ void store8(const Fp8GemmArgs& a, int m, int n, float v[8]) {
  if (a.bias) {
    const float4 p = *(const float4*)(a.bias + n), q = *(const float4*)(a.bias + n + 4);
    v[0] += p.x; v[1] += p.y; v[2] += p.z; v[3] += p.w; v[4] += q.x; v[5] += q.y; v[6] += q.z; v[7] += q.w;
  }
  if (a.act) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_of(a.act, v[i]);
  }
  if (a.out_f32) {
    float* c = (float*)a.C + (int64_t)m * a.ldc + n;
    if (a.residual) {
      const float* r = (const float*)a.residual + (int64_t)m * a.ldr + n;
      const float4 p = *(const float4*)r, q = *(const float4*)(r + 4);
      v[0] += p.x; v[1] += p.y; v[2] += p.z; v[3] += p.w; v[4] += q.x; v[5] += q.y; v[6] += q.z; v[7] += q.w;
    }
    *(float4*)c = make_float4(v[0], v[1], v[2], v[3]);
    *(float4*)(c + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    bf16_t* c = (bf16_t*)a.C + (int64_t)m * a.ldc + n;
    if (a.residual) {
      const u16x8 t = *(const u16x8*)((const bf16_t*)a.residual + (int64_t)m * a.ldr + n);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += bf2f(t[i]);
    }
    *(uint4*)c = make_uint4(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7]));
  }
}
__device__ __forceinline__ void store1(const Fp8GemmArgs& a, int m, int n, float v) {
  if (m >= a.M || n >= a.N) return;
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
// runs of four columns).  Rows past M or N repeat the last one; their results are not stored.
//
// A stage is 64 contraction steps: 64 bytes of every row, in a ring of four LDS slots filled by LDS-DMA up to three stages ahead (an
// operand that another XCD has not touched yet comes from memory: about 2000 clocks, more than a stage's products).  A stage is MF
// steps (32 rows of X, NF products each); the fragments of step s + AHEAD are read while step s is multiplied.  Where that reading
// crosses into the next stage the waves hand over: the stage behind has been read by all, the next one has landed, and the slot behind
// is refilled by pieces spread over the following steps (in one burst they would block the wave until the address unit, 64 B a
// clock, has taken them).  The scale bytes of up to SEG blocks lie beside the ring from the start; longer contractions run in segments.
constexpr int SEG = 96;                                              // blocks of 128 per segment
constexpr int fp8_scale_bytes(int BM, int BN, int kb) { return kb * (BM + 8); }   // [block][BM rows of X | 8 groups of W]
constexpr int fp8_smem(int BM, int BN, int kb) { return 4 * (BM + BN) * 64 + fp8_scale_bytes(BM, BN, kb < SEG ? kb : SEG) + 256; }   // (the last transfer of scales may be whole)

template <int BM, int BN, int WM, int WN, bool GATED, bool WIDE>
__global__ __launch_bounds__(WM * WN * 64) void fp8_tile_kernel(const Fp8GemmArgs a, int tilesN, bool vec) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int NW = WM * WN, MF = BM / WM / 32, NF = BN / WN / 32, STAGE = (BM + BN) * 64;
  constexpr int AP = BM / 16 / NW, WP = BN / 16 / NW, PIECES = AP + WP;   // 1 KiB pieces (16 rows) per wave and stage
  constexpr int AHEAD = MF >= 2 ? 2 : 1, RING = 2 * MF >= 4 ? 4 : 2, BURST = (PIECES + MF - 1) / MF, LATE = AHEAD * BURST < PIECES ? AHEAD * BURST : PIECES;
  static_assert(AP >= 1 && WP >= 1 && (!GATED || (NF == 2 && BN == 256)), "tile shape");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  // block b runs on XCD b % 8: give each XCD a contiguous range of tiles of a column-first walk through bands of eight tile rows (the
  // tiles in flight on an XCD share eight panels of X and a few of W)
  const int total = gridDim.x, b = blockIdx.x, xcd = b & 7, qd = total >> 3, rem = total & 7;
  const int t = (xcd < rem ? xcd * (qd + 1) : rem * (qd + 1) + (xcd - rem) * qd) + (b >> 3);
  const int tilesM = total / tilesN, band = t / (8 * tilesN), rows = tilesM - band * 8 < 8 ? tilesM - band * 8 : 8, in = t - band * 8 * tilesN;
  const int m0 = (band * 8 + in % rows) * BM, n0 = (in / rows) * BN;

  const unsigned panel = (unsigned)a.Kb * 2048;                       // bytes of one row tile
  const int Mt = (a.M + 15) >> 4, Nt = (a.N + 15) >> 4;
  unsigned xoff[AP], woff[WP];
  const uint8_t* wbase[WP];
  const uint8_t* xbase = a.X + (int64_t)(m0 >> 4) * panel;
#pragma unroll
  for (int p = 0; p < AP; ++p) {
    const int r = p * NW + wave;
    xoff[p] = (unsigned)((m0 >> 4) + r < Mt ? r : Mt - 1 - (m0 >> 4)) * panel + lane * 16;
  }
#pragma unroll
  for (int p = 0; p < WP; ++p) {
    const int r = p * NW + wave;
    if (GATED) {   // tile rows alternate between 32 of W and the same 32 features of W2
      const int f0 = n0 >> 5, f = (r >> 2) * 2 + (r & 1);
      wbase[p] = ((r >> 1) & 1 ? a.W2 : a.W) + (int64_t)f0 * panel;
      woff[p] = (unsigned)(f0 + f < Nt ? f : Nt - 1 - f0) * panel + lane * 16;
    } else {
      wbase[p] = a.W + (int64_t)(n0 >> 4) * panel;
      woff[p] = (unsigned)((n0 >> 4) + r < Nt ? r : Nt - 1 - (n0 >> 4)) * panel + lane * 16;
    }
  }
  const unsigned lds0 = (unsigned)(uintptr_t)((__attribute__((address_space(3))) char*)smem);
  const int stages = a.Kb * 2;
  // piece p of stage h.  A stage past the end repeats the last one (the count of transfers in flight stays the same; nothing reads it)
  auto piece = [&](int h, int p) {
    const unsigned to = (unsigned)__builtin_amdgcn_readfirstlane(lds0 + (h & 3) * STAGE + wave * 1024);
    const int64_t k = (int64_t)(h < stages ? h : stages - 1) * 1024;
    if (p < AP) dma16(xbase + k, xoff[p < AP ? p : 0], to + p * NW * 1024);
    else dma16(wbase[p < AP ? 0 : p - AP] + k, woff[p < AP ? 0 : p - AP], to + BM * 64 + (p - AP) * NW * 1024);
  };

  const int half = lane >> 5, j = lane & 31;
  f32x16 acc[NF][MF];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int k = 0; k < MF; ++k) acc[i][k] = (f32x16){};
  i32x8 x[RING], w[2][NF];
  mfma_b8 wide[WIDE ? NF : 1][4];
  int sx[MF], sw[NF], nsx[MF], nsw[NF];
  auto frag = [&](int h, int row) {               // rows row + (0 .. 31), columns 32 half + (0 .. 31) of stage h
    const char* r = smem + (h & 3) * STAGE + row * 64 + (j >> 4) * 1024 + half * 512 + (j & 15) * 16;
    return join(*(const uint4*)r, *(const uint4*)(r + 256));
  };
  auto read_step = [&](int kb, int s) {          // s counts through the two stages of block kb (and on into the next block)
    const int h = 2 * kb + s / MF;
    if (s % MF == 0) {
#pragma unroll
      for (int i = 0; i < NF; ++i) w[s / MF & 1][i] = frag(h, BM + wn * (BN / WN) + i * 32);
    }
    x[s % RING] = frag(h, wm * (BM / WM) + (s % MF) * 32);
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
  // scale bytes of block kb of this segment.  W's eight bytes: four 32-row groups from its first operand, four from the next four groups
  // or, gated, from W2 (a 64-row tile finds its two groups at the place they have among four)
  const char* sbase = smem + 4 * STAGE;
  auto read_scales = [&](int kb) {
    const char* q = sbase + kb * (BM + 8);
#pragma unroll
    for (int i = 0; i < MF; ++i) nsx[i] = *(const uint8_t*)(q + wm * (BM / WM) + i * 32 + j);
#pragma unroll
    for (int i = 0; i < NF; ++i) nsw[i] = *(const uint8_t*)(q + BM + (GATED ? i * 4 + wn : (BN < 128 ? (n0 >> 5) & 3 : 0) + wn * NF + i));
  };

  for (int seg = 0; seg < a.Kb; seg += SEG) {
    const int end = seg + SEG < a.Kb ? seg + SEG : a.Kb;
    if (seg) {                                    // the ring and the scales of the segment behind are free
      dma_wait<0>();
      __builtin_amdgcn_s_barrier();
    }
    const int per = BM / 4 + 2, count = (end - seg) * per;                      // four bytes per lane, 64 lanes per transfer
    const int64_t Mp = (int64_t)Mt * 16, Ng = (int64_t)((a.N + 127) >> 7) * 4;
    for (int e0 = wave * 64; e0 < count; e0 += NW * 64) {
      const int e = e0 + lane < count ? e0 + lane : count - 1, kb = e / per, r = e - kb * per;
      const uint8_t* src;
      if (r < BM / 4) src = a.sx + (seg + kb) * Mp + (m0 + r * 4 < Mp ? m0 + r * 4 : Mp - 4);
      else {
        const int64_t g = GATED ? (n0 >> 8) * 4 : (n0 >> 7) * 4 + (r - BM / 4) * 4;
        src = (GATED && r > BM / 4 ? a.sw2 : a.sw) + (seg + kb) * Ng + (g < Ng ? g : Ng - 4);
      }
      dma4(src, (unsigned)__builtin_amdgcn_readfirstlane(lds0 + 4 * STAGE + e0 * 4));
    }
    const int h0 = 2 * seg;
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int p = 0; p < (h < 3 ? PIECES : LATE); ++p) piece(h0 + h, p);   // (the loop's first steps issue the rest of the fourth)
    dma_wait<2 * PIECES + LATE>();                                          // (the scales are older: landed too)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read_scales(0);
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) read_step(seg, s);
    for (int kb = seg; kb < end; ++kb) {          // (no branch in this body: the compiler would sink the products past it)
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
        read_step(kb, s + AHEAD);
        if (s == 0) read_scales((kb + 1 < end ? kb + 1 : kb) - seg);
        __builtin_amdgcn_sched_barrier(0);
        multiply(s);
        __builtin_amdgcn_sched_barrier(0);
        const int u = (s + AHEAD) % MF, h = 2 * kb + (s + AHEAD) / MF + 3;   // burst u since the hand-over to stage h - 3
#pragma unroll
        for (int p = u * BURST; p < (u + 1) * BURST && p < PIECES; ++p) piece(h, p);
      }
    }
  }

  if constexpr (!GATED) {
    const int mw = m0 + wm * (BM / WM), nw = n0 + wn * (BN / WN);
    if (vec && nw + NF * 32 <= a.N) {
      // lanes l and l + 32 hold alternating runs of four columns: exchange so that each has eight consecutive ones
#pragma unroll
      for (int k = 0; k < MF; ++k)
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
            if (mw + k * 32 + j < a.M) store8(a, mw + k * 32 + j, nw + i * 32 + r * 16 + half * 8, v);
          }
    } else {
      // ragged or unaligned: each wave turns 32 rows at a time round in LDS and stores single columns
      dma_wait<0>();
      __syncthreads();
      constexpr int LD = NF * 32 + 1;
      float* turn = (float*)smem + wave * 32 * LD;
#pragma unroll
      for (int k = 0; k < MF; ++k) {
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) turn[j * LD + i * 32 + 8 * (r >> 2) + 4 * half + (r & 3)] = acc[i][k][r];
        for (int e = lane; e < 32 * NF * 32; e += 64) store1(a, mw + k * 32 + e / (NF * 32), nw + e % (NF * 32), turn[e / (NF * 32) * LD + e % (NF * 32)]);
      }
    }
  } else {
    // the tile's 128 features are one block of the next product's contraction: amax per row over the four waves of a row group
    float* red = (float*)smem;                                        // [BM][WN]
    dma_wait<0>();
    __syncthreads();
    float h[MF][16];
#pragma unroll
    for (int k = 0; k < MF; ++k) {
      float m = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int f = n0 / 2 + wn * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
        h[k][r] = f < a.N ? gelu_tanh_fast(acc[0][k][r]) * acc[1][k][r] : 0.f;
        m = fmaxf(m, finite_abs(h[k][r]));
      }
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      if (half == 0) red[(wm * (BM / WM) + k * 32 + j) * WN + wn] = m;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < MF; ++k) {
      const int row = wm * (BM / WM) + k * 32 + j, m = m0 + row;
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
      if (m < a.M) {
        const int nb = (a.N + 127) >> 7, blk = n0 >> 8;
        *(uint4*)(a.H + ((int64_t)(m >> 4) * nb * 2 + blk * 2 + (wn >> 1)) * 1024 + ((wn & 1) * 2 + half) * 256 + (m & 15) * 16) =
            make_uint4(e0[0], e0[1], e1[0], e1[1]);
        if (half == 0 && wn == 0) a.sh[(int64_t)blk * Mt * 16 + m] = (uint8_t)byte;
      }
    }
  }
}

template <int BM, int BN, int WM, int WN, bool GATED, bool WIDE>
int launch_tile(const Fp8GemmArgs& a, bool vec, hipStream_t st) {
  constexpr int most = fp8_smem(BM, BN, SEG);
  static_assert(most <= 160 * 1024, "LDS");
  FDMI_HIP(hipFuncSetAttribute((const void*)fp8_tile_kernel<BM, BN, WM, WN, GATED, WIDE>, hipFuncAttributeMaxDynamicSharedMemorySize, most));
  const int smem = fp8_smem(BM, BN, a.Kb);
  const int64_t tilesM = ((int64_t)a.M + BM - 1) / BM, tilesN = ((int64_t)a.N * (GATED ? 2 : 1) + BN - 1) / BN;
  FDMI_CHECK(tilesM * tilesN < (1ll << 31), "gemm_fp8: too many tiles");
  hipLaunchKernelGGL((fp8_tile_kernel<BM, BN, WM, WN, GATED, WIDE>), dim3((unsigned)(tilesM * tilesN)), dim3(WM * WN * 64), smem, st, a, (int)tilesN,
                     vec);
  FDMI_HIP(hipGetLastError());
  return 0;
}

bool aligned(const void* p, int64_t ld_bytes, int to) { return ((uintptr_t)p % to) == 0 && (ld_bytes % to) == 0; }

}  // namespace

int launch_quant_fp8(const void* x, int x_f32, int64_t ldx, const float* norm, float eps, uint8_t* q, uint8_t* s, int64_t M, int K,
                     hipStream_t st) {
  if (M == 0) return 0;
  const bool vec = aligned(x, ldx * (x_f32 ? 4 : 2), 16), wvec = ((uintptr_t)norm % 16) == 0;
  const int Kb = cdiv(K, 128);
  const int64_t Mp = (M + 15) / 16 * 16, rows4 = (M + 3) / 4;
  FDMI_CHECK(rows4 < (1ll << 31) && cdiv(Kb, 8) < 65536, "quant_fp8: too many rows or columns");
  const dim3 grid((unsigned)rows4, norm ? 1 : cdiv(Kb, 8));
#define FP8_QUANT(T, NORM) hipLaunchKernelGGL((quant_rows_kernel<T, NORM>), grid, dim3(256), 0, st, (const T*)x, ldx, norm, eps, q, s, M, Mp, K, Kb, vec, wvec)
  if (norm) { if (x_f32) FP8_QUANT(float, true); else FP8_QUANT(bf16_t, true); }
  else { if (x_f32) FP8_QUANT(float, false); else FP8_QUANT(bf16_t, false); }
#undef FP8_QUANT
  FDMI_HIP(hipGetLastError());
  return 0;
}

int launch_pack_fp8(const void* w, int w_f32, int64_t ldw, int N, int K, uint8_t* q, uint8_t* s, uint8_t* qt, uint8_t* st, hipStream_t stream) {
  const dim3 grid(cdiv(K, 128), cdiv(N, 128));
  if (w_f32) hipLaunchKernelGGL(pack_kernel<float>, grid, dim3(256), 0, stream, (const float*)w, ldw, N, K, q, s, qt, st);
  else hipLaunchKernelGGL(pack_kernel<bf16_t>, grid, dim3(256), 0, stream, (const bf16_t*)w, ldw, N, K, q, s, qt, st);
  FDMI_HIP(hipGetLastError());
  return 0;
}

int launch_gemm_fp8(const Fp8GemmArgs& a, hipStream_t st) {
  if (a.M == 0) return 0;
  const int es = a.out_f32 ? 4 : 2;
  const bool vec = a.H || (aligned(a.C, a.ldc * es, 16) && (!a.residual || aligned(a.residual, a.ldr * es, 16)) && ((uintptr_t)a.bias & 15) == 0);
  if (a.H) return a.M <= 64 ? launch_tile<64, 256, 1, 4, true, false>(a, vec, st) : launch_tile<128, 256, 2, 4, true, false>(a, vec, st);
  const int64_t big = ((int64_t)a.M + 127) / 128 * ((a.N + 127) / 128);
  if (a.out_f32) return big < 256 ? launch_tile<64, 64, 2, 2, false, true>(a, vec, st) : launch_tile<128, 128, 2, 2, false, true>(a, vec, st);
  if (big < 256) return launch_tile<64, 64, 2, 2, false, false>(a, vec, st);
  if (big < 2048) return launch_tile<128, 128, 2, 2, false, false>(a, vec, st);
  return launch_tile<256, 256, 2, 4, false, false>(a, vec, st);
}
