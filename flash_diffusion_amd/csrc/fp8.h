// 8-bit matrix products with a power-of-two scale for each block of 128 (fp8.hip), and the token-embedding lookup (embed.hip).
#pragma once
#include "common.h"

// threads of one launch along a grid's first dimension: HIP refuses 2^32 and more
constexpr int64_t FDMI_LAUNCH_THREADS = 0xffffffffll;

// One product  C[M][N] = act(X W^T + bias + residual)  of e4m3 codes in tiles (fp8.hip); Kb blocks of 128 along the contraction.  gated:
// W2 is a second weight of the same form and the result gelu_tanh(X W^T) * (X W2^T) leaves as codes H with scales sh instead of C.
struct Fp8GemmArgs {
  const uint8_t* X = nullptr; const uint8_t* sx = nullptr;
  const uint8_t* W = nullptr; const uint8_t* sw = nullptr;
  const uint8_t* W2 = nullptr; const uint8_t* sw2 = nullptr;
  int M = 0, N = 0, Kb = 0;
  const void* x = nullptr; int64_t ldxr = 0; int x_f32 = 0, K = 0;   // unquantised rows in X's place (fp8_fused problems)
  const float* bias = nullptr;
  const void* residual = nullptr; int64_t ldr = 0;             // of C's type
  void* C = nullptr; int64_t ldc = 0; int out_f32 = 0;
  int act = 0;
  uint8_t* H = nullptr; uint8_t* sh = nullptr;
};
bool fp8_fused(int64_t M, int K);
int launch_gemm_fp8(const Fp8GemmArgs& a, hipStream_t st);
int launch_quant_fp8(const void* x, int x_f32, int64_t ldx, const float* norm, float eps, uint8_t* q, uint8_t* s, int64_t M, int K,
                     hipStream_t st);
int launch_pack_fp8(const void* w, int w_f32, int64_t ldw, int N, int K, uint8_t* q, uint8_t* s, uint8_t* qt, uint8_t* st, hipStream_t stream);

// ---- embed.hip ----
int launch_embed_fwd(const void* table, int table_f32, int64_t V, int D, int64_t ldt, const void* ids, int ids64, int64_t n, float scale,
                     const float* pos, int64_t pos_rows, int64_t ldp, void* out, int out_f32, hipStream_t st);
int64_t embed_bwd_ws_bytes(int64_t n, int D);
int launch_embed_bwd(const void* dy, int dy_f32, int64_t lddy, const void* ids, int ids64, int64_t n, int64_t V, int D, float scale,
                     int accumulate, float* grad, int64_t ldg, void* ws, hipStream_t st);
