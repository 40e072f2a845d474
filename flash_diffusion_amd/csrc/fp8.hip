// Matrix products of 8-bit floating-point codes with a scale for each block of 128 along the contraction (gfx950).
//
//   y[m][n] = sum_b 2^(ex[m][b] + ew[n/128][b]) * sum_{k in block b} qx[m][k] * qw[n][k]        qx, qw: e4m3 codes
//
// The scales are powers of two (e8m0 bytes): 2^e is the smallest power with amax <= 448 2^e over the block, so a code never saturates,
// scaling is exact and the only rounding of the format is the one to e4m3 (round to nearest even).  CDNA4's scaled matrix instruction
// takes such a scale per lane and 32 contraction steps: a block of 128 hands the same byte to its steps, and the scales cost no
// arithmetic of their own.  Sums are fp32 in the accumulators.  An infinity or NaN of the input becomes the NaN code (e4m3 has no
// infinity, and a saturated code would hide the overflow) and the block's scale comes from its finite values.
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

// quantises the 8 values of each lane; 16 consecutive lanes hold one block of 128.  Returns the block's scale byte
__device__ __forceinline__ int quant8(const float v[8], uint2& q) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_abs(v[i]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
  const int byte = scale_byte(a);
  const float up = scale_up(byte);
  q.x = codes4(v[0], v[1], v[2], v[3], up);
  q.y = codes4(v[4], v[5], v[6], v[7], up);
  return byte;
}
// the four scale bytes of a wave's 512 columns as one word (valid in every lane)
__device__ __forceinline__ uint32_t word_of(int byte) {
  return (uint32_t)__builtin_amdgcn_readlane(byte, 0) | (uint32_t)__builtin_amdgcn_readlane(byte, 16) << 8 |
         (uint32_t)__builtin_amdgcn_readlane(byte, 32) << 16 | (uint32_t)__builtin_amdgcn_readlane(byte, 48) << 24;
}

// ---- rows of activations: one wave takes 512 columns of one row ----------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* x, int64_t ldx, uint8_t* q, int64_t ldq, uint8_t* s, int64_t lds, int64_t M,
                                                         int K, bool vec) {
  const int lane = threadIdx.x & 63;
  const int per = (int)(lds >> 2);                                  // 512-column pieces of a row
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= M * per) return;
  const int64_t m = unit / per;
  const int u = (int)(unit - m * per), k = u * 512 + lane * 8;
  float v[8];
  load8(x + m * ldx, k, K, vec, v);
  uint2 c;
  const uint32_t word = word_of(quant8(v, c));
  if (k < ldq) *(uint2*)(q + m * ldq + k) = c;
  if (lane == 0) *(uint32_t*)(s + m * lds + u * 4) = word;
}

// ---- the same behind a root-mean-square norm: y = x * rsqrt(mean(x^2) + eps) * w in fp32, one block per row ----------------------------
template <typename T>
__global__ __launch_bounds__(256) void quant_norm_kernel(const T* x, int64_t ldx, const float* w, float eps, uint8_t* q, int64_t ldq,
                                                         uint8_t* s, int64_t lds, int K, bool vec, bool wvec) {
  __shared__ float part[4];
  const int64_t m = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T* row = x + m * ldx;
  float ss = 0.f, v[8];
  for (int k = threadIdx.x * 8; k < K; k += 2048) {
    load8(row, k, K, vec, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
  }
  ss = wave_sum(ss);
  if (lane == 0) part[wave] = ss;
  __syncthreads();
  const float r = 1.f / sqrtf((part[0] + part[1] + part[2] + part[3]) / (float)K + eps);
  const int per = (int)(lds >> 2);
  for (int u = wave; u < per; u += 4) {
    const int k = u * 512 + lane * 8;
    float g[8];
    load8(row, k, K, vec, v);
    load8(w, k, K, wvec, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * r * g[i];
    uint2 c;
    const uint32_t word = word_of(quant8(v, c));
    if (k < ldq) *(uint2*)(q + m * ldq + k) = c;
    if (lane == 0) *(uint32_t*)(s + m * lds + u * 4) = word;
  }
}

// ---- weights: one block per 128 x 128 tile, codes in both orders (once per weight) ------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(const T* w, int64_t ldw, int N, int K, uint8_t* q, int64_t ldq, uint8_t* s, int64_t lds,
                                                   uint8_t* qt, int64_t ldqt, uint8_t* st, int64_t ldst) {
  __shared__ uint8_t tile[128][132];
  __shared__ float part[4];
  const int nb = blockIdx.y, kb = blockIdx.x;
  float amax = 0.f;
  for (int i = threadIdx.x; i < 128 * 128; i += 256) {
    const int n = nb * 128 + (i >> 7), k = kb * 128 + (i & 127);
    float v = 0.f;
    if (n < N && k < K) {
      if constexpr (sizeof(T) == 2) v = bf2f(w[(int64_t)n * ldw + k]);
      else v = w[(int64_t)n * ldw + k];
    }
    amax = fmaxf(amax, finite_abs(v));
  }
  amax = wave_max(amax);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = amax;
  __syncthreads();
  const int byte = scale_byte(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
  const float up = scale_up(byte);
  for (int i = threadIdx.x; i < 128 * 32; i += 256) {
    const int r = i >> 5, c = (i & 31) * 4, n = nb * 128 + r;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = kb * 128 + c + j;
      v[j] = 0.f;
      if (n < N && k < K) {
        if constexpr (sizeof(T) == 2) v[j] = bf2f(w[(int64_t)n * ldw + k]);
        else v[j] = w[(int64_t)n * ldw + k];
      }
    }
    const uint32_t p = codes4(v[0], v[1], v[2], v[3], up);
    if (n < N) *(uint32_t*)(q + (int64_t)n * ldq + kb * 128 + c) = p;
#pragma unroll
    for (int j = 0; j < 4; ++j) tile[r][c + j] = (uint8_t)(p >> (8 * j));
  }
  if (threadIdx.x == 0) {
    s[(int64_t)nb * lds + kb] = (uint8_t)byte;
    if (st) st[(int64_t)kb * ldst + nb] = (uint8_t)byte;
  }
  if (!qt) return;
  __syncthreads();
  for (int i = threadIdx.x; i < 128 * 32; i += 256) {
    const int r = i >> 5, c = (i & 31) * 4, k = kb * 128 + r;
    if (k < K)
      *(uint32_t*)(qt + (int64_t)k * ldqt + nb * 128 + c) =
          tile[c][r] | tile[c + 1][r] << 8 | tile[c + 2][r] << 16 | (uint32_t)tile[c + 3][r] << 24;
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
// global -> LDS without a register: lane i of the wave fetches 16 bytes from base + off and they land at lds + 16 i
__device__ __forceinline__ void dma16(const void* base, unsigned off, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "v"(off), "s"(base), "s"(lds));
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
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

// four consecutive columns of one row: + bias + residual, activation, store.  vec: rows of C (and the residual) are aligned for it
__device__ __forceinline__ void store4(const Fp8GemmArgs& a, int m, int n, const float* acc, bool vec) {
  if (m >= a.M || n >= a.N) return;
  const bool whole = n + 4 <= a.N;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = acc[i];
    if (a.bias && n + i < a.N) v[i] += a.bias[n + i];
  }
  if (a.out_f32) {
    float* c = (float*)a.C + (int64_t)m * a.ldc + n;
    const float* r = a.residual ? (const float*)a.residual + (int64_t)m * a.ldr + n : nullptr;
    if (vec && whole) {
      if (r) { const float4 t = *(const float4*)r; v[0] += t.x; v[1] += t.y; v[2] += t.z; v[3] += t.w; }
      *(float4*)c = make_float4(act_of(a.act, v[0]), act_of(a.act, v[1]), act_of(a.act, v[2]), act_of(a.act, v[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.N) c[i] = act_of(a.act, v[i] + (r ? r[i] : 0.f));
    }
  } else {
    bf16_t* c = (bf16_t*)a.C + (int64_t)m * a.ldc + n;
    const bf16_t* r = a.residual ? (const bf16_t*)a.residual + (int64_t)m * a.ldr + n : nullptr;
    if (vec && whole) {
      if (r) {
        const u16x4 t = *(const u16x4*)r;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += bf2f(t[i]);
      }
      uint2 p;
      p.x = pack2bf(act_of(a.act, v[0]), act_of(a.act, v[1]));
      p.y = pack2bf(act_of(a.act, v[2]), act_of(a.act, v[3]));
      *(uint2*)c = p;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.N) c[i] = f2bf(act_of(a.act, v[i] + (r ? bf2f(r[i]) : 0.f)));
    }
  }
}

// BM x BN output tile, WM x WN waves, v_mfma_scale_f32_32x32x64 with W's rows as the first operand (lane l then holds output row l & 31 and
// runs of four columns).  One LDS stage is 128 contraction steps = 128 bytes of every row; two stages, the next one landing while this one
// is multiplied.  16-byte chunk c of row r sits at c ^ ((r >> 1) & 7): the 16 lanes that a ds_read_b128 serves at once touch 16 chunks of
// different banks.  Rows past M or N repeat the last one; their results are not stored.
template <int BM, int BN, int WM, int WN, bool GATED, bool WIDE>
__global__ __launch_bounds__(WM * WN * 64) void fp8_tile_kernel(const Fp8GemmArgs a, int tilesN, bool vec) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int NW = WM * WN, MF = BM / WM / 32, NF = BN / WN / 32, STAGE = (BM + BN) * 128;
  constexpr int AP = BM / 8 / NW, WP = BN / 8 / NW;                  // 1 KiB pieces (8 rows) per wave and stage
  static_assert(NW % 2 == 0 && AP >= 1 && WP >= 1 && (!GATED || (NF == 2 && BN == 256)), "tile shape");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  // block b runs on XCD b % 8: give each XCD a contiguous range of tiles
  const int total = gridDim.x, b = blockIdx.x, xcd = b & 7, qd = total >> 3, rem = total & 7;
  const int t = (xcd < rem ? xcd * (qd + 1) : rem * (qd + 1) + (xcd - rem) * qd) + (b >> 3);
  const int m0 = (t / tilesN) * BM, n0 = (t % tilesN) * BN;

  const int lr = lane >> 3, chunk = (lane & 7) ^ ((wave & 1) * 4 + (lr >> 1));
  unsigned xoff[AP], woff[WP];
  const uint8_t* wbase[WP];
  const uint8_t* xb = a.X + (int64_t)m0 * a.ldx;
#pragma unroll
  for (int p = 0; p < AP; ++p) {
    const int r = (p * NW + wave) * 8 + lr;
    xoff[p] = (unsigned)((m0 + r < a.M ? r : a.M - 1 - m0) * a.ldx + chunk * 16);
  }
#pragma unroll
  for (int p = 0; p < WP; ++p) {
    const int r0 = (p * NW + wave) * 8, r = r0 + lr;
    if (GATED) {   // tile rows alternate between 32 of W and the same 32 features of W2
      const int f0 = n0 / 2, f = (r >> 6) * 32 + (r & 31);
      wbase[p] = ((r0 >> 5) & 1 ? a.W2 : a.W) + (int64_t)f0 * a.ldw;
      woff[p] = (unsigned)((f0 + f < a.N ? f : a.N - 1 - f0) * a.ldw + chunk * 16);
    } else {
      wbase[p] = a.W + (int64_t)n0 * a.ldw;
      woff[p] = (unsigned)((n0 + r < a.N ? r : a.N - 1 - n0) * a.ldw + chunk * 16);
    }
  }
  const unsigned lds0 = (unsigned)(uintptr_t)((__attribute__((address_space(3))) char*)smem) + wave * 1024;
  auto issue = [&](int kb, int slot) {
    const unsigned to = (unsigned)__builtin_amdgcn_readfirstlane(lds0 + slot * STAGE);
#pragma unroll
    for (int p = 0; p < AP; ++p) dma16(xb + (int64_t)kb * 128, xoff[p], to + p * NW * 1024);
#pragma unroll
    for (int p = 0; p < WP; ++p) dma16(wbase[p] + (int64_t)kb * 128, woff[p], to + BM * 128 + p * NW * 1024);
  };

  // scale rows: four blocks' bytes per word
  const int half = lane >> 5, j = lane & 31;
  const uint32_t* sxp[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    int m = m0 + wm * (BM / WM) + i * 32 + j;
    sxp[i] = (const uint32_t*)(a.sx + (int64_t)(m < a.M ? m : a.M - 1) * a.ldsx);
  }
  const uint32_t* swp[NF];
#pragma unroll
  for (int i = 0; i < NF; ++i) {
    int n = GATED ? n0 / 2 + wn * 32 : n0 + wn * (BN / WN) + i * 32;
    n = n < a.N ? n : a.N - 1;
    swp[i] = (const uint32_t*)((GATED && i ? a.sw2 : a.sw) + (int64_t)(n >> 7) * a.ldsw);
  }

  f32x16 acc[NF][MF];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int k = 0; k < MF; ++k) acc[i][k] = (f32x16){};
  uint32_t sx[MF], sw[NF];
  const int sz = (j >> 1) & 7;
  issue(0, 0);
  for (int kb = 0; kb < a.Kb; ++kb) {
    if ((kb & 3) == 0) {
#pragma unroll
      for (int i = 0; i < MF; ++i) sx[i] = sxp[i][kb >> 2];
#pragma unroll
      for (int i = 0; i < NF; ++i) sw[i] = swp[i][kb >> 2];
    }
    dma_wait();                        // this wave's pieces have landed and its reads of the other slot are done
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (kb + 1 < a.Kb) issue(kb + 1, (kb + 1) & 1);
    const char* st = smem + (kb & 1) * STAGE;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int p = ((ks * 4 + half * 2) ^ sz) * 16;
      i32x8 x[MF], w[NF];
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        const char* r = st + (BM + wn * (BN / WN) + i * 32 + j) * 128;
        w[i] = join(*(const uint4*)(r + p), *(const uint4*)(r + (p ^ 16)));
      }
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        const char* r = st + (wm * (BM / WM) + i * 32 + j) * 128;
        x[i] = join(*(const uint4*)(r + p), *(const uint4*)(r + (p ^ 16)));
      }
      if constexpr (!WIDE) {
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
          for (int k = 0; k < MF; ++k)
            acc[i][k] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[i], x[k], acc[i][k], 0, 0, 0, (int)sw[i], 0, (int)sx[k]);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          mfma_b8 xb[MF], wb[NF];
#pragma unroll
          for (int i = 0; i < NF; ++i) wb[i] = widen8(w[i][2 * q], w[i][2 * q + 1], scale_of(sw[i]));
#pragma unroll
          for (int k = 0; k < MF; ++k) xb[k] = widen8(x[k][2 * q], x[k][2 * q + 1], scale_of(sx[k]));
#pragma unroll
          for (int i = 0; i < NF; ++i)
#pragma unroll
            for (int k = 0; k < MF; ++k) acc[i][k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[i], xb[k], acc[i][k], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < MF; ++i) sx[i] >>= 8;
#pragma unroll
    for (int i = 0; i < NF; ++i) sw[i] >>= 8;
  }

  if constexpr (!GATED) {
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int k = 0; k < MF; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float v[4] = {acc[i][k][4 * r], acc[i][k][4 * r + 1], acc[i][k][4 * r + 2], acc[i][k][4 * r + 3]};
          store4(a, m0 + wm * (BM / WM) + k * 32 + j, n0 + wn * (BN / WN) + i * 32 + 8 * r + 4 * half, v, vec);
        }
  } else {
    // the tile's 128 features are one block of the next product's contraction: amax per row over the four waves of a row group
    float* red = (float*)smem;                                        // [BM][WN]
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
        *(uint4*)(a.H + (int64_t)m * a.ldh + n0 / 2 + wn * 32 + half * 16) = make_uint4(e0[0], e0[1], e1[0], e1[1]);
        if (half == 0 && wn == 0) a.sh[(int64_t)m * a.ldsh + (n0 >> 8)] = (uint8_t)byte;
      }
    }
  }
}

template <int BM, int BN, int WM, int WN, bool GATED, bool WIDE>
int launch_tile(const Fp8GemmArgs& a, bool vec, hipStream_t st) {
  constexpr int smem = 2 * (BM + BN) * 128;
  FDMI_HIP(hipFuncSetAttribute((const void*)fp8_tile_kernel<BM, BN, WM, WN, GATED, WIDE>, hipFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int64_t tilesM = ((int64_t)a.M + BM - 1) / BM, tilesN = ((int64_t)a.N * (GATED ? 2 : 1) + BN - 1) / BN;
  FDMI_CHECK(tilesM * tilesN < (1ll << 31), "gemm_fp8: too many tiles");
  hipLaunchKernelGGL((fp8_tile_kernel<BM, BN, WM, WN, GATED, WIDE>), dim3((unsigned)(tilesM * tilesN)), dim3(WM * WN * 64), smem, st, a, (int)tilesN,
                     vec);
  FDMI_HIP(hipGetLastError());
  return 0;
}

bool aligned(const void* p, int64_t ld_bytes, int to) { return ((uintptr_t)p % to) == 0 && (ld_bytes % to) == 0; }

}  // namespace

int launch_quant_fp8(const void* x, int x_f32, int64_t ldx, const float* norm, float eps, uint8_t* q, int64_t ldq, uint8_t* s, int64_t lds,
                     int64_t M, int K, hipStream_t st) {
  if (M == 0) return 0;
  const bool vec = aligned(x, ldx * (x_f32 ? 4 : 2), 16);
  if (norm) {
    const bool wvec = ((uintptr_t)norm % 16) == 0;
    if (x_f32) hipLaunchKernelGGL(quant_norm_kernel<float>, dim3((unsigned)M), dim3(256), 0, st, (const float*)x, ldx, norm, eps, q, ldq, s, lds, K, vec, wvec);
    else hipLaunchKernelGGL(quant_norm_kernel<bf16_t>, dim3((unsigned)M), dim3(256), 0, st, (const bf16_t*)x, ldx, norm, eps, q, ldq, s, lds, K, vec, wvec);
  } else {
    const int64_t blocks = (M * (lds >> 2) + 3) / 4;
    FDMI_CHECK(blocks < (1ll << 31), "quant_fp8: too many rows");
    if (x_f32) hipLaunchKernelGGL(quant_rows_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, st, (const float*)x, ldx, q, ldq, s, lds, M, K, vec);
    else hipLaunchKernelGGL(quant_rows_kernel<bf16_t>, dim3((unsigned)blocks), dim3(256), 0, st, (const bf16_t*)x, ldx, q, ldq, s, lds, M, K, vec);
  }
  FDMI_HIP(hipGetLastError());
  return 0;
}

int launch_pack_fp8(const void* w, int w_f32, int64_t ldw, int N, int K, uint8_t* q, int64_t ldq, uint8_t* s, int64_t lds, uint8_t* qt,
                    int64_t ldqt, uint8_t* st, int64_t ldst, hipStream_t stream) {
  const dim3 grid(cdiv(K, 128), cdiv(N, 128));
  if (w_f32) hipLaunchKernelGGL(pack_kernel<float>, grid, dim3(256), 0, stream, (const float*)w, ldw, N, K, q, ldq, s, lds, qt, ldqt, st, ldst);
  else hipLaunchKernelGGL(pack_kernel<bf16_t>, grid, dim3(256), 0, stream, (const bf16_t*)w, ldw, N, K, q, ldq, s, lds, qt, ldqt, st, ldst);
  FDMI_HIP(hipGetLastError());
  return 0;
}

int launch_gemm_fp8(const Fp8GemmArgs& a, hipStream_t st) {
  if (a.M == 0) return 0;
  const int es = a.out_f32 ? 4 : 2;
  const bool vec = a.H || (aligned(a.C, a.ldc * es, 4 * es) && (!a.residual || aligned(a.residual, a.ldr * es, 4 * es)));
  if (a.H) return a.M <= 64 ? launch_tile<64, 256, 2, 4, true, false>(a, vec, st) : launch_tile<128, 256, 2, 4, true, false>(a, vec, st);
  const int64_t big = ((int64_t)a.M + 127) / 128 * ((a.N + 127) / 128);
  if (a.out_f32) return big < 256 ? launch_tile<64, 64, 2, 2, false, true>(a, vec, st) : launch_tile<128, 128, 2, 2, false, true>(a, vec, st);
  if (big < 256) return launch_tile<64, 64, 2, 2, false, false>(a, vec, st);
  if (big < 2048) return launch_tile<128, 128, 2, 2, false, false>(a, vec, st);
  return launch_tile<256, 256, 2, 4, false, false>(a, vec, st);
}
