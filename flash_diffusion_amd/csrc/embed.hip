// Token-embedding lookup and the gradient of its table (gfx950).
//
//   forward    out[i][:] = scale * table[ids[i]][:] + pos[i mod pos_rows][:]
//   gradient   grad[v][:] = scale * sum over { i : ids[i] = v } of dy[i][:]
//
// Both are bound by HBM.  The gradient adds in a fixed order (no atomics): positions are ranked by (id, position), a chunk of the sorted
// list is summed by one group of lanes, and runs of one token that cross a chunk's edge leave partial rows that a second pass adds in order.
// An id outside the table reads as a row of NaN (a gather cannot raise on the device) and its gradient is dropped.
#include "fp8.h"

namespace {

constexpr int EMB_CHUNK = 32;          // sorted positions summed by one group of lanes

__device__ __forceinline__ int64_t id_at(const void* ids, int ids64, int64_t i) {
  return ids64 ? ((const int64_t*)ids)[i] : (int64_t)((const int32_t*)ids)[i];
}

// VEC columns of one token per thread
template <typename T, typename O, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const T* table, int64_t V, int D, int64_t ldt, const void* ids, int ids64, int64_t n,
                                                        float scale, const float* pos, int64_t pos_rows, int64_t ldp, O* out) {
  const int per = D / VEC;
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= n * per) return;
  const int64_t i = u / per;
  const int c = (int)(u - i * per) * VEC;
  const int64_t id = id_at(ids, ids64, i);
  const bool ok = id >= 0 && id < V;
  const T* row = table + (ok ? id : 0) * ldt + c;
  const float* pr = pos ? pos + (i % pos_rows) * ldp + c : nullptr;
  float v[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    float t;
    if constexpr (sizeof(T) == 2) t = bf2f(row[k]);
    else t = row[k];
    v[k] = ok ? fmaf(scale, t, pr ? pr[k] : 0.f) : __uint_as_float(0x7fc00000u);
  }
  O* o = out + i * D + c;
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    if constexpr (sizeof(O) == 2) o[k] = f2bf(v[k]);
    else o[k] = v[k];
  }
}

// position of i in the list sorted by (id, i); ids outside the table sort behind all others
__global__ __launch_bounds__(256) void rank_kernel(const void* ids, int ids64, int64_t n, int64_t V, int32_t* sid, int32_t* spos) {
  __shared__ int32_t key[256];
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  auto key_of = [&](int64_t p) {
    const int64_t id = id_at(ids, ids64, p);
    return id >= 0 && id < V ? (int32_t)id : 0x7fffffff;
  };
  const int32_t mine = i < n ? key_of(i) : 0;
  int64_t rank = 0;
  for (int64_t j0 = 0; j0 < n; j0 += 256) {
    __syncthreads();
    key[threadIdx.x] = j0 + threadIdx.x < n ? key_of(j0 + threadIdx.x) : 0x7fffffff;
    __syncthreads();
    const int lim = (int)(n - j0 < 256 ? n - j0 : 256);
    for (int j = 0; j < lim; ++j) rank += key[j] < mine || (key[j] == mine && j0 + j < i);
  }
  if (i < n) {
    sid[rank] = mine;
    spos[rank] = (int32_t)i;
  }
}

__global__ __launch_bounds__(256) void fill_rows_kernel(float* g, int64_t V, int D, int64_t ldg) {
  const int64_t total = V * D;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += (int64_t)gridDim.x * 256) g[u / D * ldg + u % D] = 0.f;
}

// one chunk of the sorted list, one column per thread.  part[c][0]: the run that came in over the chunk's left edge (the whole chunk, if it
// also leaves over the right one); part[c][1]: the run that begins here and leaves over the right edge
template <typename T>
__global__ __launch_bounds__(256) void run_sum_kernel(const T* dy, int64_t lddy, const int32_t* sid, const int32_t* spos, int64_t n, int D,
                                                      float scale, int accumulate, float* g, int64_t ldg, float* part) {
  const int64_t p0 = (int64_t)blockIdx.x * EMB_CHUNK, p1 = p0 + EMB_CHUNK < n ? p0 + EMB_CHUNK : n;
  const int col = blockIdx.y * 256 + threadIdx.x;
  if (col >= D) return;
  const int32_t before = p0 > 0 ? sid[p0 - 1] : -1, after = p1 < n ? sid[p1] : -1;
  float sum = 0.f;
  for (int64_t p = p0; p < p1; ++p) {
    const int32_t id = sid[p];
    const T* row = dy + (int64_t)spos[p] * lddy + col;
    if constexpr (sizeof(T) == 2) sum += bf2f(*row);
    else sum += *row;
    const int32_t next = p + 1 < p1 ? sid[p + 1] : -2;
    if (next == id) continue;
    if (id != 0x7fffffff) {
      if (id == before) part[((int64_t)blockIdx.x * 2) * D + col] = sum;
      else if (next == -2 && id == after) part[((int64_t)blockIdx.x * 2 + 1) * D + col] = sum;
      else {
        float* o = g + (int64_t)id * ldg + col;
        *o = accumulate ? fmaf(scale, sum, *o) : scale * sum;
      }
    }
    sum = 0.f;
  }
}

// runs that cross chunk edges: the block of the chunk where a run begins adds its partial rows in order
__global__ __launch_bounds__(256) void run_join_kernel(const int32_t* sid, int64_t n, int D, float scale, int accumulate, float* g, int64_t ldg,
                                                       const float* part) {
  const int64_t c = blockIdx.x, p0 = c * EMB_CHUNK, p1 = p0 + EMB_CHUNK;
  const int col = blockIdx.y * 256 + threadIdx.x;
  if (col >= D || p1 >= n) return;
  const int32_t id = sid[p1 - 1];
  if (id == 0x7fffffff || sid[p1] != id || (p0 > 0 && sid[p0 - 1] == id)) return;
  float sum = part[(c * 2 + 1) * D + col];
  for (int64_t k = c + 1; k * EMB_CHUNK < n && sid[k * EMB_CHUNK] == id; ++k) sum += part[(k * 2) * D + col];
  float* o = g + (int64_t)id * ldg + col;
  *o = accumulate ? fmaf(scale, sum, *o) : scale * sum;
}

}  // namespace

int launch_embed_fwd(const void* table, int table_f32, int64_t V, int D, int64_t ldt, const void* ids, int ids64, int64_t n, float scale,
                     const float* pos, int64_t pos_rows, int64_t ldp, void* out, int out_f32, hipStream_t st) {
  if (n == 0) return 0;
  const int64_t blocks = (n * D + 255) / 256;
  FDMI_CHECK(blocks < (1ll << 31), "embed_fwd: too many tokens");
#define EMB_FWD(T, O) hipLaunchKernelGGL((embed_fwd_kernel<T, O, 1>), dim3((unsigned)blocks), dim3(256), 0, st, (const T*)table, V, D, ldt, ids, \
                                         ids64, n, scale, pos, pos_rows, ldp, (O*)out)
  if (table_f32) { if (out_f32) EMB_FWD(float, float); else EMB_FWD(float, bf16_t); }
  else { if (out_f32) EMB_FWD(bf16_t, float); else EMB_FWD(bf16_t, bf16_t); }
#undef EMB_FWD
  FDMI_HIP(hipGetLastError());
  return 0;
}

int64_t embed_bwd_ws_bytes(int64_t n, int D) {
  return (n * 2 * 4 + 255) / 256 * 256 + (n + EMB_CHUNK - 1) / EMB_CHUNK * 2 * (int64_t)D * 4;
}
int launch_embed_bwd(const void* dy, int dy_f32, int64_t lddy, const void* ids, int ids64, int64_t n, int64_t V, int D, float scale,
                     int accumulate, float* grad, int64_t ldg, void* ws, hipStream_t st) {
  if (!accumulate) hipLaunchKernelGGL(fill_rows_kernel, dim3(4096), dim3(256), 0, st, grad, V, D, ldg);
  if (n > 0) {
    int32_t* sid = (int32_t*)ws;
    int32_t* spos = sid + n;
    float* part = (float*)((char*)ws + (n * 2 * 4 + 255) / 256 * 256);
    const dim3 grid(cdiv(n, EMB_CHUNK), cdiv(D, 256));
    hipLaunchKernelGGL(rank_kernel, dim3(cdiv(n, 256)), dim3(256), 0, st, ids, ids64, n, V, sid, spos);
    if (dy_f32) hipLaunchKernelGGL(run_sum_kernel<float>, grid, dim3(256), 0, st, (const float*)dy, lddy, sid, spos, n, D, scale, accumulate, grad, ldg, part);
    else hipLaunchKernelGGL(run_sum_kernel<bf16_t>, grid, dim3(256), 0, st, (const bf16_t*)dy, lddy, sid, spos, n, D, scale, accumulate, grad, ldg, part);
    hipLaunchKernelGGL(run_join_kernel, grid, dim3(256), 0, st, sid, n, D, scale, accumulate, grad, ldg, part);
  }
  FDMI_HIP(hipGetLastError());
  return 0;
}
