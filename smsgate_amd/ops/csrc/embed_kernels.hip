// smsgate_amd — token embedding of the training step and its gradient (gfx950).
//
//   x[i]  = scale * (E[ids[i]] + (add[i] >= 0 ? E[add[i]] : 0))          fp32, rounded once
//   dE[v] = scale * sum over { i : ids[i] = v } and { i : add[i] = v } of dx[i]
//
// E is [V, H] in fp32, bf16 or fp16; x, dx and dE have its type.  The sums run in fp32 in
// an order that the ids alone fix: by position, no atomics on floats, so a step's gradient
// is the same bits every time.  An id outside [0, V) reads nothing: its row of x is NaN and
// it has no part in dE (add: negative = none).
//
// Both directions are bound by memory: the rows read, x / dx, and dE written once whole.
//   * up to EG_SMALL entries (one message): ONE launch; every block scans all the ids for
//     its 16 rows of dE.  A launch costs more than the work (45 positions of 256 over 8192
//     ids, fp32: 2.5 us forward, 4.8 us gradient, of which 8.4 MB of dE take 2).
//   * else the entries are sorted by id (stable, so each id's positions stay in order), in
//     one launch up to EG_RANGE entries, else in three launches a pass of 8 bits; then one
//     wave a row of dE sums its positions (rows of no entry are zeroed there, so dE is
//     written once).  An id of many entries (a separator, the shared prompt) would leave
//     one wave with thousands of rows: runs of EG_CHUNK sorted entries of one id are summed
//     beforehand, and rows of over EG_COOP terms are shared by the block's 4 waves.
// Measured: 7808 positions with second rows, 576 fp32 over 8576 ids: 7 us forward (2.6 TB/s
// with the rows from L2), 18 sort, 5 chunks, 14 rows.  130999 positions, 960 bf16 over 49152
// ids: 75 us forward (4.6 TB/s, a large copy's 4.8), 41 sort, 42 chunks, 72 rows.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "train_ops.hpp"

namespace {

constexpr int EG_SMALL = 256;    // entries that the one-launch gradient takes
// Entries, and ids, that the one-launch sort takes.  Its blocks each read every id: 18 us at
// 15616 entries, where the passes need seven launches (about 30 us); a form of it that reads
// more than the registers hold took 192 us at 130999, the passes 41.
constexpr int EG_RANGE = 1 << 14;
constexpr int EG_RANGE_V = 1 << 18;
constexpr int EG_CHUNK = 32;     // sorted entries of one id summed beforehand
constexpr int EG_COOP = 16;      // terms of a row that one wave sums alone
constexpr int EG_TILE = 2048;    // entries of one block of a radix pass

template <typename T>
__device__ __forceinline__ float eg_f(T v) {
  return (float)v;
}

// VEC elements of T (16 bytes, or one element where H or a pointer is not a multiple of 16 bytes)
template <typename T, int VEC>
struct __attribute__((aligned(sizeof(T) * VEC))) EgVec {
  T v[VEC];
};

__device__ __forceinline__ long eg_id(const void* ids, int is64, long i) {
  return is64 ? reinterpret_cast<const long*>(ids)[i] : (long)reinterpret_cast<const int*>(ids)[i];
}

// Entry e < n is ids[e], entry n + i is add[i]; an id of no row becomes the key V.
__device__ __forceinline__ uint32_t eg_key(const void* ids, const void* add, int is64, int n, int e, int V) {
  const long id = e < n ? eg_id(ids, is64, e) : eg_id(add, is64, e - n);
  return id >= 0 && id < V ? (uint32_t)id : (uint32_t)V;
}

// One row per 2^lp lanes, chunks of VEC elements.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const void* __restrict__ ids, const void* __restrict__ add,
                                                        int is64, const T* __restrict__ table, T* __restrict__ x,
                                                        int n, int V, int H, int lp, float scale) {
  typedef EgVec<T, VEC> vec;
  const int nch = H / VEC, lane = threadIdx.x & ((1 << lp) - 1);
  const long row = (long)blockIdx.x * (256 >> lp) + (threadIdx.x >> lp);
  if (row >= n) return;
  const long a = eg_id(ids, is64, row), b = add != nullptr ? eg_id(add, is64, row) : -1;
  const bool bad = a < 0 || a >= V || b >= V;
  const vec* ra = reinterpret_cast<const vec*>(table + (size_t)(bad ? 0 : a) * H);
  const vec* rb = reinterpret_cast<const vec*>(table + (size_t)(bad || b < 0 ? 0 : b) * H);
  vec* out = reinterpret_cast<vec*>(x + (size_t)row * H);
  for (int c = lane; c < nch; c += 1 << lp) {
    vec va = ra[c], o;
    if (b >= 0) {
      const vec vb = rb[c];
#pragma unroll
      for (int k = 0; k < VEC; ++k) o.v[k] = (T)((eg_f(va.v[k]) + eg_f(vb.v[k])) * scale);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) o.v[k] = (T)(eg_f(va.v[k]) * scale);
    }
    if (bad) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) o.v[k] = (T)__builtin_nanf("");
    }
    out[c] = o;
  }
}

// dE in one launch for at most EG_SMALL entries: block b owns rows [16 b, 16 b + 16).
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_grad_small_kernel(const void* __restrict__ ids,
                                                               const void* __restrict__ add, int is64,
                                                               const T* __restrict__ dx, T* __restrict__ dt, int n,
                                                               int n2, int V, int H, float scale) {
  typedef EgVec<T, VEC> vec;
  __shared__ int list[EG_SMALL];  // (row in the block) << 16 | entry, by entry
  __shared__ int cnt[4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int v0 = blockIdx.x * 16;
  const uint32_t key = tid < n2 ? eg_key(ids, add, is64, n, tid, V) : (uint32_t)V;
  const bool mine = key < (uint32_t)V && key >= (uint32_t)v0 && key < (uint32_t)(v0 + 16);
  const unsigned long long m = __ballot(mine);
  if (lane == 0) cnt[wave] = __popcll(m);
  __syncthreads();
  int at = __popcll(m & ((1ull << lane) - 1));
  for (int w = 0; w < wave; ++w) at += cnt[w];
  const int total = cnt[0] + cnt[1] + cnt[2] + cnt[3];
  if (mine) list[at] = ((int)(key - v0) << 16) | tid;
  __syncthreads();
  const int nch = H / VEC;
  for (int r = wave; r < 16 && v0 + r < V; r += 4) {
    vec* out = reinterpret_cast<vec*>(dt + (size_t)(v0 + r) * H);
    for (int c = lane; c < nch; c += 64) {
      float acc[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
      for (int j = 0; j < total; ++j) {
        const int u = list[j];
        if ((u >> 16) != r) continue;
        const int e = u & 0xffff, row = e < n ? e : e - n;
        const vec d = reinterpret_cast<const vec*>(dx + (size_t)row * H)[c];
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += eg_f(d.v[k]);
      }
      vec o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) o.v[k] = (T)(acc[k] * scale);
      out[c] = o;
    }
  }
}

// ---- stable radix sort of (key, entry) ----------------------------------------------
// Lanes of the wave with the same 8-bit digit (the wave's active lanes only).
__device__ __forceinline__ unsigned long long eg_peers(uint32_t digit, bool on) {
  unsigned long long m = __ballot(on);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const unsigned long long s = __ballot((digit >> b) & 1);
    m &= (digit >> b) & 1 ? s : ~s;
  }
  return m;
}

// One stable step of a wave's entries, 64 at a time: `cnt` (this wave's 256 counters) holds
// each digit's next place.  (Counting alone needs no order: LDS additions of whole numbers.)
template <typename F>
__device__ __forceinline__ void eg_wave_step(volatile int* cnt, uint32_t digit, bool on, int lane, F place) {
  const unsigned long long peers = eg_peers(digit, on);
  const int rank = __popcll(peers & ((1ull << lane) - 1));
  if (on) {
    place(cnt[digit] + rank);
    __builtin_amdgcn_wave_barrier();
    if (rank == 0) cnt[digit] = cnt[digit] + __popcll(peers);
    __builtin_amdgcn_wave_barrier();
  }
}

// Sorts up to EG_RANGE entries in one launch: block b places the entries of the 256 ids
// [256 b, 256 b + 256) by itself.  It reads every id (from L2: 8 n2 bytes a block), counts its
// own and the entries of lower ids, which is where its own begin, and places them; a wave
// owns a run of entries, so places keep their order.  Writes seg of its ids.
__global__ void __launch_bounds__(1024) embed_range_sort_kernel(const void* __restrict__ ids,
                                                                const void* __restrict__ add, int is64, int n, int n2,
                                                                int V, uint32_t* __restrict__ keys,
                                                                int* __restrict__ ents, int2* __restrict__ seg) {
  __shared__ int cnt[16 * 256];  // [wave][id]
  __shared__ int sum[256], low[16];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const uint32_t v0 = blockIdx.x * 256;
  const int per = ((n2 + 15) / 16 + 63) & ~63;
  const int w0 = wave * per, w1 = min(n2, w0 + per);
  volatile int* mine = cnt + wave * 256;
  for (int i = tid; i < 16 * 256; i += 1024) cnt[i] = 0;
  __syncthreads();
  // the wave's entries stay in registers: f(entry, key, in range)
  constexpr int R = EG_RANGE / 16 / 64;
  uint32_t key[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int e = w0 + 64 * r + lane;
    key[r] = e < w1 ? eg_key(ids, add, is64, n, e, V) : (uint32_t)V;
  }
  auto walk = [&](auto f) {
#pragma unroll
    for (int r = 0; r < R; ++r) f(w0 + 64 * r + lane, key[r], key[r] - v0 < 256u && key[r] < (uint32_t)V);
  };
  int below = 0;
  walk([&](int, uint32_t k, bool on) {
    below += k < v0;  // (an id of no row is V: in no range and below none)
    if (on) atomicAdd(&cnt[wave * 256 + (k - v0)], 1);
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o, 64);
  if (lane == 0) low[wave] = below;
  __syncthreads();
  if (tid < 256) {  // places of an id's entries within it, wave by wave
    int c = 0;
    for (int w = 0; w < 16; ++w) {
      const int x = cnt[w * 256 + tid];
      cnt[w * 256 + tid] = c;
      c += x;
    }
    sum[tid] = c;
  }
  __syncthreads();
  if (tid < 64) {  // where each id begins: the lower ids' entries, then the range's in order
    int base = 0;
    for (int w = 0; w < 16; ++w) base += low[w];
    int a[4], s = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      a[k] = s;
      s += sum[4 * tid + k];
    }
    int inc = s;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(inc, o, 64);
      if (lane >= o) inc += t;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int x = base + inc - s + a[k], y = sum[4 * tid + k];
      if (v0 + 4 * tid + k < (uint32_t)V) seg[v0 + 4 * tid + k] = make_int2(x, x + y);
      sum[4 * tid + k] = x;
    }
  }
  __syncthreads();
  for (int i = tid; i < 16 * 256; i += 1024) cnt[i] += sum[i & 255];
  __syncthreads();
  walk([&](int e, uint32_t k, bool on) {
    if (__any(on))
      eg_wave_step(mine, (k - v0) & 255u, on, lane, [&](int at) {
        keys[at] = k;
        ents[at] = e;
      });
  });
}

// Radix pass over tiles of EG_TILE entries.  The first pass reads the ids themselves.
__device__ __forceinline__ uint32_t eg_load(const uint32_t* keys, const void* ids, const void* add, int is64, int n,
                                            int e, int V) {
  return keys != nullptr ? keys[e] : eg_key(ids, add, is64, n, e, V);
}

// hist[digit][tile]; zeroes seg on the way (grid-stride).
__global__ void __launch_bounds__(256) embed_hist_kernel(const uint32_t* __restrict__ keys,
                                                         const void* __restrict__ ids, const void* __restrict__ add,
                                                         int is64, int n, int n2, int V, int sh,
                                                         int* __restrict__ hist, int2* __restrict__ seg) {
  __shared__ int h[256];
  const int tid = threadIdx.x;
  h[tid] = 0;
  __syncthreads();
  const int e0 = blockIdx.x * EG_TILE;
  for (int i = tid; i < EG_TILE && e0 + i < n2; i += 256)
    atomicAdd(&h[(eg_load(keys, ids, add, is64, n, e0 + i, V) >> sh) & 255u], 1);
  __syncthreads();
  hist[(size_t)tid * gridDim.x + blockIdx.x] = h[tid];
  if (seg != nullptr)
    for (long v = (long)blockIdx.x * 256 + tid; v < V; v += (long)gridDim.x * 256) seg[v] = make_int2(0, 0);
}

// Exclusive sums over the tiles of a digit in place, a wave a digit, and the digit's total
// behind all of them (the scatter adds the lower digits' totals).
__global__ void __launch_bounds__(256) embed_scan_kernel(int* __restrict__ hist, int tiles) {
  const int digit = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  int* row = hist + (size_t)digit * tiles;
  int base = 0;
  for (int t0 = 0; t0 < tiles; t0 += 64) {
    const int x = t0 + lane < tiles ? row[t0 + lane] : 0;
    int inc = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(inc, o, 64);
      if (lane >= o) inc += t;
    }
    if (t0 + lane < tiles) row[t0 + lane] = base + inc - x;
    base += __shfl(inc, 63, 64);
  }
  if (lane == 0) hist[(size_t)256 * tiles + digit] = base;
}

__global__ void __launch_bounds__(256) embed_scatter_kernel(const uint32_t* __restrict__ keys,
                                                            const int* __restrict__ ents,
                                                            const void* __restrict__ ids,
                                                            const void* __restrict__ add, int is64, int n, int n2,
                                                            int V, int sh, const int* __restrict__ hist,
                                                            uint32_t* __restrict__ keys_out,
                                                            int* __restrict__ ents_out) {
  __shared__ int cnt[4 * 256], low[256];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int w0 = blockIdx.x * EG_TILE + wave * (EG_TILE / 4), w1 = min(n2, w0 + EG_TILE / 4);
  volatile int* mine = cnt + wave * 256;
  uint32_t key[EG_TILE / 256];
  for (int i = tid; i < 1024; i += 256) cnt[i] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < EG_TILE / 256; ++r) {
    const int e = w0 + 64 * r + lane;
    key[r] = e < w1 ? eg_load(keys, ids, add, is64, n, e, V) : 0u;
    if (e < w1) atomicAdd(&cnt[wave * 256 + ((key[r] >> sh) & 255u)], 1);
  }
  if (wave == 0) {  // exclusive sums of the digits' totals, 4 a lane
    const int* total = hist + (size_t)256 * gridDim.x + 4 * lane;
    int a[4], s = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      a[k] = s;
      s += total[k];
    }
    int inc = s;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(inc, o, 64);
      if (lane >= o) inc += t;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) low[4 * lane + k] = inc - s + a[k];
  }
  __syncthreads();
  {
    int s = low[tid] + hist[(size_t)tid * gridDim.x + blockIdx.x];
    for (int w = 0; w < 4; ++w) {
      const int c = cnt[w * 256 + tid];
      cnt[w * 256 + tid] = s;
      s += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < EG_TILE / 256; ++r) {
    const int e = w0 + 64 * r + lane;
    const int ent = keys != nullptr && e < w1 ? ents[e] : e;
    eg_wave_step(mine, (key[r] >> sh) & 255u, e < w1, lane, [&](int at) {
      keys_out[at] = key[r];
      ents_out[at] = ent;
    });
  }
}

__global__ void __launch_bounds__(256) embed_bounds_kernel(const uint32_t* __restrict__ keys, int n2, int V,
                                                           int2* __restrict__ seg) {
  const int e = blockIdx.x * 256 + threadIdx.x;
  if (e >= n2) return;
  const uint32_t k = keys[e];
  if (k >= (uint32_t)V) return;
  if (e == 0 || keys[e - 1] != k) seg[k].x = e;
  if (e + 1 == n2 || keys[e + 1] != k) seg[k].y = e + 1;
}

// ---- sums ----------------------------------------------------------------------------
// acc += the dx rows of sorted entries [e0, e1), in order, FLY rows in flight.
template <typename T, int VEC, int FLY = 8>
__device__ __forceinline__ void eg_sum_entries(float (&acc)[VEC], const int* __restrict__ ents,
                                               const T* __restrict__ dx, int n, int H, int c, int e0, int e1) {
  typedef EgVec<T, VEC> vec;
  for (int e = e0; e < e1; e += FLY) {
    vec d[FLY];
#pragma unroll
    for (int k = 0; k < FLY; ++k) {
      const int en = ents[min(e + k, e1 - 1)], row = en < n ? en : en - n;
      d[k] = reinterpret_cast<const vec*>(dx + (size_t)row * H)[c];
    }
#pragma unroll
    for (int k = 0; k < FLY; ++k)
      if (e + k < e1) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += eg_f(d[k].v[j]);
      }
  }
}

// Partial sums of the chunks whose EG_CHUNK entries share one id (else nothing).  Behind the
// last entry of an id of a row, keys holds anything: seg tells.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_chunk_kernel(const uint32_t* __restrict__ keys,
                                                          const int2* __restrict__ seg,
                                                          const int* __restrict__ ents, const T* __restrict__ dx,
                                                          float* __restrict__ part, int n, int n2, int V, int H) {
  const int ch = blockIdx.x * 4 + (threadIdx.x >> 6), e0 = ch * EG_CHUNK;
  if (e0 + EG_CHUNK > n2) return;
  const uint32_t k = keys[e0];
  if (k >= (uint32_t)V) return;
  const int2 s = seg[k];
  if (s.x > e0 || s.y < e0 + EG_CHUNK) return;
  const int c = blockIdx.y * 64 + (threadIdx.x & 63);
  if (c >= H / VEC) return;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  eg_sum_entries<T, VEC, EG_CHUNK>(acc, ents, dx, n, H, c, e0, e0 + EG_CHUNK);
#pragma unroll
  for (int j = 0; j < VEC; ++j) part[(size_t)ch * H + (size_t)c * VEC + j] = acc[j];
}

// dE: of B blocks, block b owns the rows b + i B, i = 0..3 (ids of many entries are often
// neighbours), x chunks [64 y, 64 y + 64).  A row's terms are its entries up to a chunk
// border, the sums of its whole chunks, and the entries behind.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_rows_kernel(const int2* __restrict__ seg, const int* __restrict__ ents,
                                                         const T* __restrict__ dx, const float* __restrict__ part,
                                                         T* __restrict__ dt, int n, int V, int H, float scale) {
  typedef EgVec<T, VEC> vec;
  __shared__ float red[4][64][VEC];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int c = blockIdx.y * 64 + lane;
  const bool on = c < H / VEC;
  auto terms = [](int2 s, int& a, int& b) {  // whole chunks [a, b); the number of terms
    a = (s.x + EG_CHUNK - 1) / EG_CHUNK;
    b = s.y / EG_CHUNK;
    if (b <= a) {
      a = b = 0;
      return s.y - s.x;
    }
    return (a * EG_CHUNK - s.x) + (b - a) + (s.y - b * EG_CHUNK);
  };
  // terms [t0, t1) of a row, in order
  auto sum = [&](float (&acc)[VEC], int2 s, int a, int b, int t0, int t1) {
    if (a == b) {
      eg_sum_entries<T, VEC>(acc, ents, dx, n, H, c, s.x + t0, s.x + t1);
      return;
    }
    const int n1 = a * EG_CHUNK - s.x, nb = b - a;
    if (t0 < n1) eg_sum_entries<T, VEC>(acc, ents, dx, n, H, c, s.x + t0, s.x + min(t1, n1));
    for (int t = max(t0, n1); t < min(t1, n1 + nb); t += 4) {
      float d[4][VEC];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int ch = a + min(t + k, n1 + nb - 1) - n1;
#pragma unroll
        for (int j = 0; j < VEC; ++j) d[k][j] = part[(size_t)ch * H + (size_t)c * VEC + j];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (t + k < min(t1, n1 + nb)) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += d[k][j];
        }
    }
    if (t1 > n1 + nb) {
      const int e = b * EG_CHUNK - (n1 + nb);
      eg_sum_entries<T, VEC>(acc, ents, dx, n, H, c, e + max(t0, n1 + nb), e + t1);
    }
  };
  auto store = [&](int v, const float (&acc)[VEC]) {
    vec o;
#pragma unroll
    for (int j = 0; j < VEC; ++j) o.v[j] = (T)(acc[j] * scale);
    reinterpret_cast<vec*>(dt + (size_t)v * H)[c] = o;
  };
  const int nb = gridDim.x, mine = blockIdx.x + wave * nb;
  int a, b;
  if (mine < V) {
    const int2 s = seg[mine];
    const int nt = terms(s, a, b);
    if (nt <= EG_COOP && on) {
      float acc[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
      sum(acc, s, a, b, 0, nt);
      store(mine, acc);
    }
  }
  for (int v = blockIdx.x; v < V; v += nb) {  // at most 4; the same for every wave: seg decides
    const int2 s = seg[v];
    const int nt = terms(s, a, b);
    if (nt <= EG_COOP) continue;
    const int per = (nt + 3) / 4;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    if (on) sum(acc, s, a, b, min(nt, wave * per), min(nt, wave * per + per));
#pragma unroll
    for (int j = 0; j < VEC; ++j) red[wave][lane][j] = acc[j];
    __syncthreads();
    if (wave == 0 && on) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] = (red[0][lane][j] + red[1][lane][j]) + (red[2][lane][j] + red[3][lane][j]);
      store(v, acc);
    }
    __syncthreads();
  }
}

template <typename T, int VEC>
int eg_forward(const void* ids, const void* add, int is64, const void* table, void* x, int n, int V, int H,
               float scale, hipStream_t st) {
  int lp = 0;
  while (lp < 6 && (1 << lp) < H / VEC) ++lp;
  const long rows = 256 >> lp;
  embed_fwd_kernel<T, VEC><<<dim3((unsigned)((n + rows - 1) / rows)), dim3(256), 0, st>>>(
      ids, add, is64, (const T*)table, (T*)x, n, V, H, lp, scale);
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

template <typename T, int VEC>
int eg_backward(const void* ids, const void* add, int is64, const void* dx, void* dt, int n, int n2, int V, int H,
                float scale, const uint32_t* keys, const int* ents, const int2* seg, float* part, hipStream_t st) {
  const int ncb = (H / VEC + 63) / 64;
  if (n2 <= EG_SMALL) {
    embed_grad_small_kernel<T, VEC><<<dim3((V + 15) / 16), dim3(256), 0, st>>>(ids, add, is64, (const T*)dx, (T*)dt, n,
                                                                               n2, V, H, scale);
    return hipGetLastError() == hipSuccess ? 0 : 2;
  }
  const int nchunk = n2 / EG_CHUNK;
  embed_chunk_kernel<T, VEC><<<dim3((nchunk + 3) / 4, ncb), dim3(256), 0, st>>>(keys, seg, ents, (const T*)dx, part, n,
                                                                                n2, V, H);
  embed_rows_kernel<T, VEC><<<dim3((V + 3) / 4, ncb), dim3(256), 0, st>>>(seg, ents, (const T*)dx, part, (T*)dt, n, V,
                                                                          H, scale);
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

// (64 threads a row of x and a row of dE, 256 a block, and a grid holds 2^32 - 1)
constexpr int EG_MOST = (1 << 26) - 4;
bool eg_bad(int n, int V, int H, int dtype, int vec) {
  return n <= 0 || n > EG_MOST || V <= 0 || V > EG_MOST || H <= 0 || H > (1 << 20) || dtype < 0 || dtype > 2 ||
         (vec && H % (dtype == 0 ? 4 : 8));
}

}  // namespace

extern "C" {

// dtype 0 fp32, 1 bf16, 2 fp16; vec: every pointer and row is a multiple of 16 bytes
int sg_embed_fwd(const void* ids, const void* add, int is64, const void* table, void* x, int n, int V, int H,
                 float scale, int dtype, int vec, hipStream_t st) {
  if (eg_bad(n, V, H, dtype, vec)) return 1;
  if (dtype == 0)
    return vec ? eg_forward<float, 4>(ids, add, is64, table, x, n, V, H, scale, st)
               : eg_forward<float, 1>(ids, add, is64, table, x, n, V, H, scale, st);
  if (dtype == 1)
    return vec ? eg_forward<__bf16, 8>(ids, add, is64, table, x, n, V, H, scale, st)
               : eg_forward<__bf16, 1>(ids, add, is64, table, x, n, V, H, scale, st);
  return vec ? eg_forward<_Float16, 8>(ids, add, is64, table, x, n, V, H, scale, st)
             : eg_forward<_Float16, 1>(ids, add, is64, table, x, n, V, H, scale, st);
}

// Workspace that sg_embed_grad needs for n2 entries, in units of 256 bytes (0: none).
int sg_embed_grad_ws(int n2, int V, int H) {
  if (n2 <= EG_SMALL) return 0;
  const long tiles = (n2 + EG_TILE - 1) / EG_TILE;
  return (int)((2L * V + 4L * n2 + 256 * (tiles + 1) + (long)(n2 / EG_CHUNK) * H + 63) / 64);
}

int sg_embed_grad(const void* ids, const void* add, int is64, const void* dx, void* dt, int n, int V, int H,
                  float scale, int dtype, int vec, void* ws, int ws_units, hipStream_t st) {
  if (eg_bad(n, V, H, dtype, vec)) return 1;
  const int n2 = add != nullptr ? 2 * n : n;
  uint32_t* keys = nullptr;
  int* ents = nullptr;
  int2* seg = nullptr;
  float* part = nullptr;
  if (n2 > EG_SMALL) {
    if (ws == nullptr || ws_units < sg_embed_grad_ws(n2, V, H)) return 3;
    const long tiles = (n2 + EG_TILE - 1) / EG_TILE;
    int* w = (int*)ws;
    seg = (int2*)w;
    w += 2L * V;
    uint32_t* kb[2] = {(uint32_t*)w, (uint32_t*)w + n2};
    w += 2L * n2;
    int* eb[2] = {w, w + n2};
    w += 2L * n2;
    int* hist = w;
    w += 256 * (tiles + 1);
    part = (float*)w;
    int passes = 1;
    while (passes < 4 && (V >> (8 * passes)) != 0) ++passes;
    if (n2 <= EG_RANGE && V <= EG_RANGE_V) {
      keys = kb[0];
      ents = eb[0];
      embed_range_sort_kernel<<<dim3((V + 255) / 256), dim3(1024), 0, st>>>(ids, add, is64, n, n2, V, keys, ents, seg);
    } else {
      const uint32_t* ksrc = nullptr;
      const int* esrc = nullptr;
      for (int p = 0; p < passes; ++p) {
        embed_hist_kernel<<<dim3((unsigned)tiles), dim3(256), 0, st>>>(ksrc, ids, add, is64, n, n2, V, 8 * p, hist,
                                                                       p == 0 ? seg : nullptr);
        embed_scan_kernel<<<dim3(64), dim3(256), 0, st>>>(hist, (int)tiles);
        embed_scatter_kernel<<<dim3((unsigned)tiles), dim3(256), 0, st>>>(ksrc, esrc, ids, add, is64, n, n2, V, 8 * p,
                                                                          hist, kb[p & 1], eb[p & 1]);
        ksrc = kb[p & 1];
        esrc = eb[p & 1];
      }
      keys = const_cast<uint32_t*>(ksrc);
      ents = const_cast<int*>(esrc);
      embed_bounds_kernel<<<dim3((n2 + 255) / 256), dim3(256), 0, st>>>(keys, n2, V, seg);
    }
    if (hipGetLastError() != hipSuccess) return 2;
  }
  if (dtype == 0)
    return vec ? eg_backward<float, 4>(ids, add, is64, dx, dt, n, n2, V, H, scale, keys, ents, seg, part, st)
               : eg_backward<float, 1>(ids, add, is64, dx, dt, n, n2, V, H, scale, keys, ents, seg, part, st);
  if (dtype == 1)
    return vec ? eg_backward<__bf16, 8>(ids, add, is64, dx, dt, n, n2, V, H, scale, keys, ents, seg, part, st)
               : eg_backward<__bf16, 1>(ids, add, is64, dx, dt, n, n2, V, H, scale, keys, ents, seg, part, st);
  return vec ? eg_backward<_Float16, 8>(ids, add, is64, dx, dt, n, n2, V, H, scale, keys, ents, seg, part, st)
             : eg_backward<_Float16, 1>(ids, add, is64, dx, dt, n, n2, V, H, scale, keys, ents, seg, part, st);
}

}  // extern "C"
