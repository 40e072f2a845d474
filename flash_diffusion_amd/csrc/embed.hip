// Token-embedding lookup and the gradient of its table (gfx950).
//
//   forward    out[i][:] = scale * table[ids[i]][:] + pos[i mod pos_rows][:]
//   gradient   grad[v][:] = scale * sum over { i : ids[i] = v } of dy[i][:]
//
// Both are bound by HBM.  The gradient adds in a fixed order (no atomics): positions are ranked by (id, position), a workgroup sums a chunk
// of the sorted list, and runs of one token that cross a chunk's edge leave partial rows that a last launch adds in order.  Three
// launches: the ranking, chunk sums together with the zeros, joins; one more before them where the list is long, one alone where it is
// short.  16384 bf16 rows of 4096 columns into 32128 fp32 rows, half of them padding: 156 us, 130 of them in the second of these launches
// for 725 MB (5.6 TB/s; a copy reaches 4.9, a fill 6.8); 1232 fp32 rows of 768 into 49408: 35 us, 24 of them (6.5 TB/s).
// An id outside the table reads as a row of NaN (a gather cannot raise on the device) and its gradient is dropped.
#include "fp8.h"

namespace {

constexpr int ROWS = 16, CHUNK = 64;   // sorted positions summed by one wave (its rows are in flight together) and by a workgroup
constexpr int32_t NONE = 0x7fffffff;   // key of an id outside the table: behind all others

__device__ __forceinline__ int64_t id_at(const void* ids, int ids64, int64_t i) {
  return ids64 & 1 ? ((const int64_t*)ids)[i] : (int64_t)((const int32_t*)ids)[i];
}
// VEC columns with 16-byte accesses at any address that an element may have.  A lane whose columns would pass the end
// of a row of D >= VEC takes the row's last VEC columns instead, and shares some of them with its neighbour
typedef uint16_t u16x8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
template <typename T, int VEC>
__device__ __forceinline__ void load_cols(const T* p, float v[VEC]) {
  if constexpr (VEC == 1) {
    if constexpr (sizeof(T) == 2) v[0] = bf2f(*p);
    else v[0] = *p;
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
      const f32x4_any t = *(const f32x4_any*)(p + k);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k + e] = t[e];
    }
  } else {
    const u16x8_any t = *(const u16x8_any*)p;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = bf2f(t[k]);
  }
}

// ---- lookup: one wave per token, VEC columns per lane and turn -------------------------------------------------------------------------
template <typename T, typename O, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const T* table, int64_t V, int D, int64_t ldt, const void* ids, int ids64, int64_t i0, int64_t n,
                                                        float scale, const float* pos, int64_t pos_rows, int64_t ldp, O* out) {
  const int64_t i = i0 + (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= n) return;
  int64_t id = id_at(ids, ids64, i);
  if (ids64 & 2) id += id < 0 ? V : 0;           // counted from the end, as in indexing
  const bool ok = id >= 0 && id < V;
  const T* row = table + (ok ? id : 0) * ldt;
  const float* pr = pos ? pos + (i % pos_rows) * ldp : nullptr;
  O* o = out + i * D;
  for (int c0 = (threadIdx.x & 63) * VEC; c0 < D; c0 += 64 * VEC) {
    const int c = c0 + VEC <= D ? c0 : D - VEC;
    float v[VEC], q[VEC];
    load_cols<T, VEC>(row + c, v);
#pragma unroll
    for (int k = 0; k < VEC; ++k) q[k] = 0.f;
    if (pr) load_cols<float, VEC>(pr + c, q);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = ok ? fmaf(scale, v[k], q[k]) : __uint_as_float(0x7fc00000u);
    if constexpr (VEC == 1) {
      if constexpr (sizeof(O) == 2) o[c] = f2bf(v[0]);
      else o[c] = v[0];
    } else if constexpr (sizeof(O) == 2) {
      *(u32x4_any*)(o + c) = (u32x4_any){pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7])};
    } else {
      *(f32x4_any*)(o + c) = (f32x4_any){v[0], v[1], v[2], v[3]};
      *(f32x4_any*)(o + c + 4) = (f32x4_any){v[4], v[5], v[6], v[7]};
    }
  }
}

// ---- gradient: the order ---------------------------------------------------------------------------------------------------------------
// A position's place in the list sorted by (id, position) is the number of keys below its own.  Up to DIRECT positions they are counted
// one by one (quadratic, but one launch: 4.6 us at 257 positions, 7.4 at 1232, 10.1 at 2048, 18 at 4096, 58 at 16384).  Longer lists are
// first sorted in parts of 256; the other parts' counts are then binary searches (two launches: 9.1 us at 1232, 9.2 at 2048, 9.7 at 4096,
// 17.5 at 16384, 98 at 131072; between two launches lies a microsecond).
// Each part is searched by every other one, so a call of more than SLICE positions (as many parts as run at once) adds up slice after slice:
// 2^20 positions of 512 bf16 columns take 1.2 ms (as one list the order alone would: 92 us at 2^17, and it grows with the square).
constexpr int DIRECT = 2048, PART = 256, SLICE = 512 * PART;
constexpr int TILE = 4096;             // keys in LDS at a time

__device__ __forceinline__ uint32_t key_of(const void* ids, int ids64, int64_t V, int64_t p) {
  const int64_t id = id_at(ids, ids64, p);
  return (uint32_t)(id >= 0 && id < V ? (int32_t)id : NONE);
}
// how many of 64 keys in LDS are below lim
__device__ __forceinline__ int below64(const uint32_t* key, uint32_t lim) {
  int r = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint4 k = ((const uint4*)key)[e];
    r += (k.x < lim) + (k.y < lim) + (k.z < lim) + (k.w < lim);
  }
  return r;
}
// the same for the 64 keys of a wave's own positions: equal keys of earlier lanes come first
__device__ __forceinline__ int below_own(const uint32_t* key, uint32_t mine, int lane) {
  int r = 0;
#pragma unroll
  for (int e = 0; e < 64; ++e) r += key[e] < mine + (e < lane ? 1u : 0u);
  return r;
}

// the place of this thread's key among those of its workgroup of PART (in LDS); threads without one (`real`) keep their own
__device__ __forceinline__ int rank_in_part(uint32_t* key, uint32_t mine, bool real) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  key[threadIdx.x] = mine;
  __syncthreads();
  int r = below_own(key + wave * 64, mine, lane);
  for (int q = 0; q < PART / 64; ++q)
    if (q != wave) r += below64(key + q * 64, mine + (q < wave && real ? 1u : 0u));
  return real ? r : threadIdx.x;
}

__global__ __launch_bounds__(PART) void part_sort_kernel(const void* ids, int ids64, int64_t n, int64_t V, uint32_t* pkey, int32_t* ppos) {
  __shared__ __attribute__((aligned(16))) uint32_t key[PART];
  const int64_t p0 = (int64_t)blockIdx.x * PART, p = p0 + threadIdx.x;
  const uint32_t mine = p < n ? key_of(ids, ids64, V, p) : 0xffffffffu;   // (behind everything; counted nowhere)
  const int r = rank_in_part(key, mine, p < n);
  pkey[p0 + r] = mine;
  ppos[p0 + r] = (int32_t)p;
}

template <bool PARTS>
__global__ __launch_bounds__(PARTS ? 1024 : 256) void order_kernel(const void* ids, int ids64, int64_t n, int64_t V, const uint32_t* pkey, const int32_t* ppos,
                                                    int32_t* sid, int32_t* spos) {
  __shared__ __attribute__((aligned(16))) uint32_t key[TILE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if constexpr (!PARTS) {                        // 64 positions per block, the list shared out over its waves
    __shared__ int32_t part[4][64];
    const int64_t i0 = (int64_t)blockIdx.x * 64, i = i0 + lane;
    const uint32_t mine = i < n ? key_of(ids, ids64, V, i) : 0;
    const int groups = (int)((n + 63) >> 6);     // (n <= DIRECT <= TILE: one tile)
    for (int p = threadIdx.x; p < groups * 64; p += 256) key[p] = p < n ? key_of(ids, ids64, V, p) : 0xffffffffu;
    __syncthreads();
    int r = 0;
    for (int q = wave; q < groups; q += 4)
      r += q * 64 != i0 ? below64(key + q * 64, mine + (q * 64 < i0 ? 1u : 0u)) : below_own(key + q * 64, mine, lane);
    part[wave][lane] = r;
    __syncthreads();
    if (wave == 0 && i < n) {
      const int at = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
      sid[at] = (int32_t)mine;
      spos[at] = (int32_t)i;
    }
  } else {                                       // one sorted part per block; each quarter of it searches every fourth part
    __shared__ int32_t found[3][PART];
    const int quarter = threadIdx.x / PART, t = threadIdx.x % PART;
    const int64_t p = (int64_t)blockIdx.x * PART + t;
    const uint32_t mine = pkey[p];
    const int32_t pos = ppos[p];
    const int parts = (int)((n + PART - 1) / PART);
    int32_t below = 0;
    for (int c0 = 0; c0 < parts; c0 += TILE / PART) {
      const int here = parts - c0 < TILE / PART ? parts - c0 : TILE / PART;
      __syncthreads();
      for (int q = threadIdx.x; q < here * PART; q += 1024) key[q] = pkey[(int64_t)c0 * PART + q];
      __syncthreads();
#pragma unroll 4
      for (int c = quarter; c < here; c += 4) {
        const uint32_t lim = mine + (c0 + c < (int)blockIdx.x ? 1u : 0u);   // equal keys of earlier parts come first
        const uint32_t* k = key + c * PART;
        int lo = 0;
#pragma unroll
        for (int step = PART / 2; step > 0; step >>= 1) lo += k[lo + step - 1] < lim ? step : 0;
        lo += k[lo] < lim;
        below += c0 + c == (int)blockIdx.x ? 0 : lo;
      }
    }
    if (quarter) found[quarter - 1][t] = below;
    __syncthreads();
    if (quarter == 0 && pos < n) {
      const int64_t at = (int64_t)t + below + found[0][t] + found[1][t] + found[2][t];
      sid[at] = (int32_t)mine;
      spos[at] = pos;
    }
  }
}

// a lane's VEC columns of a row of D, from `col` on as load_cols takes them (v: of the row's last VEC, if fewer are left)
template <int VEC>
__device__ __forceinline__ void put_row(float* row, int col, int D, const float v[VEC], float scale, int accumulate) {
  float* o = row + col;
  if (VEC == 1) {
    *o = accumulate ? fmaf(scale, v[0], *o) : scale * v[0];
  } else if (col + VEC <= D) {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
      f32x4_any t = {scale * v[k], scale * v[k + 1], scale * v[k + 2], scale * v[k + 3]};
      if (accumulate) {
        const f32x4_any b = *(const f32x4_any*)(o + k);
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = fmaf(scale, v[k + e], b[e]);
      }
      *(f32x4_any*)(o + k) = t;
    }
  } else {                                       // its own columns only (added to once), from the last on
    float w[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) w[k] = v[k];
#pragma unroll 1
    for (int c = D - 1; c >= col; --c) {
      row[c] = accumulate ? fmaf(scale, w[VEC - 1], row[c]) : scale * w[VEC - 1];
#pragma unroll
      for (int k = VEC - 1; k > 0; --k) w[k] = w[k - 1];
    }
  }
}

// ---- second launch: one workgroup per chunk of the sorted list and 64 VEC columns ---------------------------------------------------------
// Each wave sums the runs among its 16 positions.  Those that cross from wave to wave are joined through LDS, those that cross a chunk's
// edge leave part[c][0]: the run that came in over the chunk's left edge (the whole chunk, if it also leaves over the right one), and
// part[c][1]: the run that begins here and leaves over the right edge.
//
// The workgroups behind those of the sums write the zeros, the bulk of the bytes: ZROWS rows of the table each, but for the rows of tokens
// that occur (looked up in the sorted list; each is written once, by its run).
constexpr int ZROWS = 16;
// SMALL: at most PART positions and no other launch.  Every workgroup of the sums sorts the ids for itself and follows its runs over the
// chunk's right edge to their ends, those of the zeros look through the ids (256 positions: 8.7 us where three launches take 12.7 for 500
// rows of 256, 21.5 against 28.7 for 49408 of 768; lists of two to eight parts sorted so take longer than with the launches, 17 against 13 us
// and 63 against 19 for 500 rows, and following a run costs 3 us for 64 positions).
template <int VEC, bool SMALL>
__device__ __forceinline__ void zero_rows(int64_t v0, int64_t V, const void* ids, int ids64, const int32_t* sid, int64_t n, int D, float* g, int64_t ldg) {
  const int lane = threadIdx.x & 63;
  const int64_t v = v0 + (lane & (ZROWS - 1));
  uint32_t todo;
  if constexpr (SMALL) {
    __shared__ uint32_t taken;
    if (threadIdx.x == 0) taken = 0;
    __syncthreads();
    const int64_t d = threadIdx.x < n ? id_at(ids, ids64, threadIdx.x) - v0 : -1;
    if (d >= 0 && d < ZROWS) atomicOr(&taken, 1u << d);
    __syncthreads();
    todo = (uint32_t)__ballot(v < V) & ((1u << ZROWS) - 1) & ~taken;
  } else {
    int64_t lo = 0, hi = n;                                   // the first position whose key is not below v
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (sid[mid] < v) lo = mid + 1;
      else hi = mid;
    }
    const bool empty = v < V && !(lo < n && sid[lo] == v);
    todo = (uint32_t)__ballot(empty) & ((1u << ZROWS) - 1);
  }
  for (; todo; todo &= todo - 1) {
    float* row = g + (v0 + __ffs(todo) - 1) * ldg;
    for (int c = threadIdx.x * VEC; c < D; c += 256 * VEC) {
      if constexpr (VEC == 1) row[c] = 0.f;
      else *(f32x4_any*)(row + (c + VEC <= D ? c : D - VEC)) = (f32x4_any){0.f, 0.f, 0.f, 0.f};
    }
  }
}

template <typename T, int VEC, bool SMALL>
__global__ __launch_bounds__(256, VEC == 8 || SMALL ? 4 : 5) void run_sum_kernel(const T* dy, int64_t lddy, const void* ids, int ids64, const int32_t* gsid,
                                                      const int32_t* gspos, int64_t n, int D, int col_groups, float scale, int accumulate, float* g, int64_t ldg, float* part, int summers,
                                                      int64_t v0, int64_t V) {
  if ((int)blockIdx.x >= summers) return zero_rows<(VEC > 1 ? 4 : 1), SMALL>(v0 + ((int64_t)blockIdx.x - summers) * ZROWS, V, ids, ids64, gsid, n, D, g, ldg);
  __shared__ __attribute__((aligned(16))) uint32_t key[SMALL ? PART : 4];
  __shared__ int32_t lsid[SMALL ? PART : 1], lspos[SMALL ? PART : 1];
  if constexpr (SMALL) {
    const bool real = threadIdx.x < n;
    const uint32_t k = real ? key_of(ids, ids64, V, threadIdx.x) : 0xffffffffu;
    const int r = rank_in_part(key, k, real);
    lsid[r] = (int32_t)k;
    lspos[r] = threadIdx.x;
    __syncthreads();
  }
  auto sid = [&](int64_t p) { return SMALL ? lsid[SMALL ? p : 0] : gsid[p]; };
  auto spos = [&](int64_t p) { return SMALL ? lspos[SMALL ? p : 0] : gspos[p]; };
  __shared__ float head[4][64 * VEC];            // per wave: its share of the run that came in over its left edge
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t c = blockIdx.x / col_groups, p0 = c * CHUNK + wave * ROWS;
  const int col = ((int)(blockIdx.x - c * col_groups) * 64 + lane) * VEC, mine = col + VEC <= D ? col : D - VEC;
  const int count = (int)(p0 + ROWS < n ? ROWS : p0 < n ? n - p0 : 0);
  int32_t edge[5];                               // the key at each wave's left edge, and behind the chunk
#pragma unroll
  for (int q = 0; q < 5; ++q) edge[q] = c * CHUNK + q * ROWS < n ? sid(c * CHUNK + q * ROWS) : -1;
  const int32_t before = p0 > 0 && count ? sid(p0 - 1) : -1, after = p0 + ROWS < n ? sid(p0 + ROWS) : -1;
  float v[ROWS][VEC];
  int32_t id[ROWS];
#pragma unroll
  for (int q = 0; q < ROWS; ++q) {
    const int64_t p = q < count ? p0 + q : n - 1;
    id[q] = sid(p);
    load_cols<T, VEC>(dy + (int64_t)spos(p) * lddy + mine, v[q]);
  }
  float sum[VEC], out[VEC];
  int32_t leaves = NONE;                         // the run that begins in this wave and leaves it
#pragma unroll
  for (int k = 0; k < VEC; ++k) sum[k] = out[k] = 0.f;
#pragma unroll
  for (int q = 0; q < ROWS; ++q) {
    const bool here = q < count, last = q + 1 == count, ends = here && (last || id[q + 1 < ROWS ? q + 1 : q] != id[q]);
#pragma unroll
    for (int k = 0; k < VEC; ++k) sum[k] = here ? sum[k] + v[q][k] : sum[k];
    if (ends) {
      if (id[q] != NONE) {
        if (id[q] == before) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) head[wave][k * 64 + lane] = sum[k];
        } else if (last && id[q] == after) {
          leaves = id[q];
#pragma unroll
          for (int k = 0; k < VEC; ++k) out[k] = sum[k];
        } else if (col < D) {
          put_row<VEC>(g + (int64_t)id[q] * ldg, col, D, sum, scale, accumulate);
        }
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) sum[k] = 0.f;
    }
  }
  __syncthreads();
  auto add_heads = [&](int from, int32_t run, float s[VEC]) {          // of the waves from `from` on that begin with the run
#pragma unroll
    for (int u = 1; u < 4; ++u)
      if (u >= from && edge[u] == run)
#pragma unroll
        for (int k = 0; k < VEC; ++k) s[k] += head[u][k * 64 + lane];
  };
  if constexpr (SMALL) {
    if (leaves != NONE) add_heads(wave + 1, leaves, out);
    const int64_t e = (c + 1) * CHUNK;           // the run that begins in this chunk and leaves it: summed to its end
    const bool on = e < n && edge[4] != NONE && sid(e - 1) == edge[4] && (c == 0 || sid(c * CHUNK - 1) != edge[4]);
    if (on) {
      float more[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) more[k] = 0.f;
      for (int64_t p = e + wave * ROWS; p < n && sid(p) == edge[4]; p += CHUNK) {
#pragma unroll
        for (int q = 0; q < ROWS; ++q) load_cols<T, VEC>(dy + (int64_t)spos(p + q < n ? p + q : n - 1) * lddy + mine, v[q]);
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
          const bool here = p + q < n && sid(p + q) == edge[4];
#pragma unroll
          for (int k = 0; k < VEC; ++k) more[k] = here ? more[k] + v[q][k] : more[k];
        }
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < VEC; ++k) head[wave][k * 64 + lane] = more[k];
      __syncthreads();
      if (leaves == edge[4]) {
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int k = 0; k < VEC; ++k) out[k] += head[u][k * 64 + lane];
      }
    }
    if (leaves != NONE && col < D) put_row<VEC>(g + (int64_t)leaves * ldg, col, D, out, scale, accumulate);
    return;
  }
  if (leaves != NONE) {
    add_heads(wave + 1, leaves, out);
    if (col < D) {
      if (edge[4] == leaves) put_row<VEC>(part + (c * 2 + 1) * D, col, D, out, 1.f, 0);
      else put_row<VEC>(g + (int64_t)leaves * ldg, col, D, out, scale, accumulate);
    }
  }
  if (wave == 0 && before == edge[0] && before != NONE) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) out[k] = head[0][k * 64 + lane];
    add_heads(1, before, out);
    if (col < D) put_row<VEC>(part + (c * 2) * D, col, D, out, 1.f, 0);
  }
}

// ---- third launch: runs that cross chunk edges --------------------------------------------------------------------------------------------
// A workgroup looks after the runs that begin in 16 chunks, for 64 VEC columns.  Runs over at most SHORT further chunks go to one wave
// each; longer ones (padding) are shared out over the waves in contiguous parts that are added in order.
constexpr int SHORT = 16, JOINERS = 16;
template <int VEC>
__global__ __launch_bounds__(JOINERS * 64) void run_join_kernel(const int32_t* sid, int64_t n, int D, float scale, int accumulate, float* g,
                                                                   int64_t ldg, const float* part) {
  __shared__ float share[JOINERS][64 * VEC];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = (blockIdx.y * 64 + lane) * VEC, at = col + VEC <= D ? col : D - VEC;
  const int64_t chunks = (n + CHUNK - 1) / CHUNK, k0 = (int64_t)blockIdx.x * JOINERS, c = k0 + (lane & (JOINERS - 1));
  auto key = [&](int64_t p) { return sid[p < n ? p : n - 1]; };         // (all asked for at once)
  const int32_t before = c > 0 ? key(c * CHUNK - 1) : -1, last = key((c + 1) * CHUNK - 1), next = key((c + 1) * CHUNK);
  const int32_t beyond = key((c + 1 + SHORT) * CHUNK);
  const bool mine = lane < JOINERS && (c + 1) * CHUNK < n && last != NONE && next == last && before != last;
  const bool far = mine && c + 1 + SHORT < chunks && beyond == last;
  uint64_t longs = __ballot(far), near = __ballot(mine) & ~longs;
  if (!(longs | near)) return;
  auto add_rows = [&](int64_t from, int64_t to, float s[VEC]) {        // part[k][0], from <= k < to
    constexpr int DEEP = 8;                                            // in flight together
    for (int64_t k = from; k < to; k += DEEP) {
      float v[DEEP][VEC];
#pragma unroll
      for (int q = 0; q < DEEP; ++q) load_cols<float, VEC>(part + ((k + q < to ? k + q : to - 1) * 2) * D + at, v[q]);
#pragma unroll
      for (int q = 0; q < DEEP; ++q)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] = k + q < to ? s[e] + v[q][e] : s[e];
    }
  };
  auto end_of = [&](int64_t first, int32_t id, int64_t step) {         // the first chunk from `first` on that does not begin with id
    for (; ; step = 1) {                                               // by 64 at a time, then one by one
      while (true) {
        const int64_t k = first + (int64_t)lane * step;
        const uint64_t no = __ballot(!(k < chunks && sid[k * CHUNK] == id));
        if (no) {
          const int b = __ffsll((long long)no) - 1;
          if (step == 1) return first + b;
          first += b ? (b - 1) * step + 1 : 0;
          break;
        }
        first += 64 * step;
      }
    }
  };
  for (int turn = 0; near; ++turn) {
    const int b = __ffsll((long long)near) - 1;
    near &= near - 1;
    if (turn % JOINERS != wave) continue;
    const int64_t k = k0 + b;
    const int32_t id = __shfl(last, b, 64);
    const int64_t end = end_of(k + 1, id, 1);
    if (col < D) {
      float s[VEC];
      load_cols<float, VEC>(part + (k * 2 + 1) * D + at, s);
      add_rows(k + 1, end, s);
      put_row<VEC>(g + (int64_t)id * ldg, col, D, s, scale, accumulate);
    }
  }
  while (longs) {
    const int b = __ffsll((long long)longs) - 1;
    longs &= longs - 1;
    const int64_t k = k0 + b;
    const int32_t id = __shfl(last, b, 64);
    const int64_t end = end_of(k + 1, id, 64), each = (end - (k + 1) + JOINERS - 1) / JOINERS;
    const int64_t from = k + 1 + wave * each, to = from + each < end ? from + each : end;
    float s[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[e] = 0.f;
    if (col < D) {
      if (wave == 0) load_cols<float, VEC>(part + (k * 2 + 1) * D + at, s);
      add_rows(from, to, s);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) share[wave][lane * VEC + e] = s[e];
    __syncthreads();
    if (wave == 0 && col < D) {
      for (int q = 1; q < JOINERS; ++q)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] += share[q][lane * VEC + e];
      put_row<VEC>(g + (int64_t)id * ldg, col, D, s, scale, accumulate);
    }
    __syncthreads();
  }
}

}  // namespace

int launch_embed_fwd(const void* table, int table_f32, int64_t V, int D, int64_t ldt, const void* ids, int ids64, int64_t n, float scale,
                     const float* pos, int64_t pos_rows, int64_t ldp, void* out, int out_f32, hipStream_t st) {
  if (n == 0) return 0;
  const bool vec = D >= 8;
  constexpr int64_t TOKENS = 1ll << 25;            // of one launch (256 threads for four of them)
  for (int64_t i0 = 0; i0 < n; i0 += TOKENS) {
    const unsigned blocks = (unsigned)(((n - i0 < TOKENS ? n - i0 : TOKENS) + 3) / 4);
#define EMB_FWD(T, O, VEC) hipLaunchKernelGGL((embed_fwd_kernel<T, O, VEC>), dim3(blocks), dim3(256), 0, st, (const T*)table, V, D, ldt, \
                                              ids, ids64, i0, n, scale, pos, pos_rows, ldp, (O*)out)
    if (table_f32) { if (out_f32) { if (vec) EMB_FWD(float, float, 8); else EMB_FWD(float, float, 1); }
                     else { if (vec) EMB_FWD(float, bf16_t, 8); else EMB_FWD(float, bf16_t, 1); } }
    else { if (out_f32) { if (vec) EMB_FWD(bf16_t, float, 8); else EMB_FWD(bf16_t, float, 1); }
           else { if (vec) EMB_FWD(bf16_t, bf16_t, 8); else EMB_FWD(bf16_t, bf16_t, 1); } }
#undef EMB_FWD
    FDMI_HIP(hipGetLastError());
  }
  return 0;
}

// scratch: the sorted list's keys and positions, those of the sorted parts, and two partial rows per chunk
static int64_t list_bytes(int64_t n) { return ((n > DIRECT ? n + (n + PART - 1) / PART * PART : n) * 2 * 4 + 255) / 256 * 256; }
int64_t embed_bwd_ws_bytes(int64_t n, int D) {
  if (n > SLICE) n = SLICE;
  return list_bytes(n) + (n + CHUNK - 1) / CHUNK * 2 * (int64_t)D * 4;
}
static int launch_slice(const void* dy, int dy_f32, int64_t lddy, const void* ids, int ids64, int64_t n, int64_t V, int D, float scale,
                     int accumulate, float* grad, int64_t ldg, void* ws, hipStream_t st) {
  const bool parts = n > DIRECT, small = n <= PART;
  const int np = cdiv(n, PART);
  int32_t* sid = (int32_t*)ws;
  int32_t* spos = sid + n;
  uint32_t* pkey = (uint32_t*)(spos + n);
  int32_t* ppos = (int32_t*)pkey + (int64_t)np * PART;
  float* part = (float*)((char*)ws + list_bytes(n));
  if (parts) {
    hipLaunchKernelGGL(part_sort_kernel, dim3(np), dim3(PART), 0, st, ids, ids64, n, V, pkey, ppos);
    hipLaunchKernelGGL(order_kernel<true>, dim3(np), dim3(1024), 0, st, ids, ids64, n, V, pkey, ppos, sid, spos);
  } else if (!small) {
    hipLaunchKernelGGL(order_kernel<false>, dim3(cdiv(n, 64)), dim3(256), 0, st, ids, ids64, n, V, nullptr, nullptr, sid, spos);
  }
  const bool vec = D >= 8, vec8 = vec && !dy_f32;                                        // (16 bytes of a row per lane)
  const int groups = cdiv(D, vec8 ? 512 : vec ? 256 : 64);
  const int64_t chunks = (n + CHUNK - 1) / CHUNK, summers = chunks * groups, blocks = summers + (accumulate ? 0 : (V + ZROWS - 1) / ZROWS);
  constexpr int64_t MOST = FDMI_LAUNCH_THREADS / 256;       // workgroups of one launch
  if (blocks == 0) return 0;
  const dim3 join((unsigned)((chunks + JOINERS - 1) / JOINERS), cdiv(D, vec ? 256 : 64));
  // (the zeros of a table of more than about 2^28 rows take a second launch)
#define EMB_SUM(T, VEC) \
  for (int64_t b0 = 0; b0 < blocks; b0 += MOST) { if (small) EMB_SUM_OF(T, VEC, true); else EMB_SUM_OF(T, VEC, false); }
#define EMB_SUM_OF(T, VEC, SMALL) hipLaunchKernelGGL((run_sum_kernel<T, VEC, SMALL>), dim3((unsigned)(blocks - b0 < MOST ? blocks - b0 : MOST)), dim3(256), 0, st, \
                                           (const T*)dy, lddy, ids, ids64, sid, spos, n, D, groups, scale, accumulate, grad, ldg, part, (int)(b0 ? 0 : summers), \
                                           b0 ? (b0 - summers) * ZROWS : 0, V)
  if (vec) {
    if (dy_f32) { EMB_SUM(float, 4); } else { EMB_SUM(bf16_t, 8); }
    if (!small) hipLaunchKernelGGL(run_join_kernel<4>, join, dim3(JOINERS * 64), 0, st, sid, n, D, scale, accumulate, grad, ldg, part);
  } else {
    if (dy_f32) { EMB_SUM(float, 1); } else { EMB_SUM(bf16_t, 1); }
    if (!small) hipLaunchKernelGGL(run_join_kernel<1>, join, dim3(JOINERS * 64), 0, st, sid, n, D, scale, accumulate, grad, ldg, part);
  }
#undef EMB_SUM
#undef EMB_SUM_OF
  FDMI_HIP(hipGetLastError());
  return 0;
}

int launch_embed_bwd(const void* dy, int dy_f32, int64_t lddy, const void* ids, int ids64, int64_t n, int64_t V, int D, float scale,
                     int accumulate, float* grad, int64_t ldg, void* ws, hipStream_t st) {
  const int64_t groups = ((int64_t)D + (D < 8 ? 63 : dy_f32 ? 255 : 511)) / (D < 8 ? 64 : dy_f32 ? 256 : 512);
  FDMI_CHECK(D <= 65535 * 256 && ((n < SLICE ? n : SLICE) + CHUNK - 1) / CHUNK * groups <= FDMI_LAUNCH_THREADS / 256, "embed_bwd: too many columns");
  int64_t at = 0;
  do {
    const int64_t now = n - at < SLICE ? n - at : SLICE;
    if (const int rc = launch_slice((const char*)dy + at * lddy * (dy_f32 ? 4 : 2), dy_f32, lddy, (const char*)ids + at * (ids64 ? 8 : 4), ids64, now, V, D,
                                    scale, accumulate || at > 0, grad, ldg, ws, st)) return rc;
    at += now;
  } while (at < n);
  return 0;
}
