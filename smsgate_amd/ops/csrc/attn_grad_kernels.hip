// smsgate_amd — attention of the training step over whole sequences, and its gradients,
// in matrix instructions (gfx950).
//
//   S = c q k^T (c = scale),  L = logsumexp S,  P = exp(S - L),  o = P v
//   dP = do v^T,  D = rowsum(do * o),  dS = P (dP - D),  dq = c dS k,  dk = c dS^T q,
//   dv = P^T do;  dk and dv sum over the query heads that share a key head
//
// q [B, nh, T, D], k / v [B, nkv, T, D] (rows of D contiguous, any other strides), bf16 or
// fp16, D 64 or 128; o and do [B, T, nh * D].  Query i sees keys j < len[b] (causal: j <= i
// too); rows at or behind len[b] are written as zeros, in o and in every gradient, and what
// they hold in q, k, v and do is never multiplied.
//
// Nothing of size T x T is stored: the forward keeps each row's L, and the backward
// recomputes P from it, once for the rows' gradient (attn_dq) and once for the keys'
// (attn_dkv), so that every sum has one owner and a fixed order: no float atomics.
//
// All products are v_mfma_f32_32x32x16.  Its result holds, in lane l, column l & 31 and
// rows (r & 3) + 8 (r >> 2) + 4 (l >> 5), r = 0..15; its operands hold row l & 31, k-values
// 8 (l >> 5) + 0..7.  The k-order is free as long as both operands agree, so a result's
// registers 8t..8t+7 are used as they are for the 16 k-values of the next product (P and
// dS never leave registers), and the other operand is read from LDS in that order: k-value
// j of lane half h is row 16 t + 8 (j >> 2) + 4 h + (j & 3) of the tile: two transposing reads
// (ds_read_b64_tr_b16: 4 rows x 16 columns, each lane gets a column's 4 values).
//   forward:  S^T = K Q^T  (keys in registers, a query a lane),  O^T = V^T P^T
//   attn_dq:  S^T, dP^T = V dO^T,  dQ^T = K^T dS^T
//   attn_dkv: S = Q K^T (queries in registers, a key a lane), dP = dO V^T,
//             dV^T = dO^T P,  dK^T = Q^T dS
// The operand of the wave's own 32 rows stays in registers; the tiles that are walked are
// copied into LDS by the DMA path (global_load_lds), two buffers, one barrier a tile.  A
// tile's 16-byte chunks are XORed by row, so that neither row nor transposing reads meet on
// a bank.
//
// Sums, L, D and the running maximum are fp32.  The forward keeps what rounding took from o
// (another value of the type), so that D is taken from 16 more bits of o: from the rounded o
// alone its error was a third of dq's and dk's (2.8e-3 instead of 2.3e-3 of their norm at
// 61 rows, bf16).  P and dS are rounded to the inputs' type as operands (at most 2^-8 relative
// in bf16, as the inputs themselves are; see at_mma_p).  fp16 holds no value under 2^-24: there
// P is scaled by 2^8 (by 2^7 forward) and dS by a power of two that the longest rows of the
// sequence's do and v set (and nothing in another sequence).
//
// What bounds it: the waves' own chains (product, exp2, rounding, product): at 16384 rows the
// matrix units work a third of the time, the vector units half, and neither copies (10 % less
// time without them) nor exp2 (8 %) nor LDS (no bank conflicts, a quarter of its time) alone
// hold it up.  4 waves a block: 2 took 404 -> 525 us forward, 700 -> 770 in attn_dkv (copies
// are shared by fewer), 8 took 436 and 726 (one barrier holds more).  Measured, bf16, causal,
// 9 / 3 heads of 64, 16384 rows: forward 404 us (766 TFLOP/s of the products that the mask
// leaves), attn_dq 500, attn_dkv 700 (S and dP are each taken twice); 128 sequences of up to 61
// rows: 15 + 16 + 12 us, 48 MB.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "train_ops.hpp"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* at_lds_t;
typedef __attribute__((address_space(3))) s16x4* at_tr_t;

constexpr float AT_LOG2E = 1.4426950408889634f;
constexpr float AT_LN2 = 0.6931471805599453f;
constexpr int AT_FP16_P = 8;    // fp16: log2 of the factor on P in attn_dkv
constexpr int AT_MAXPARTS = 256;  // fp16: blocks of each maximum over the batch, but one a sequence at least

__device__ const uint4 at_zero = {0, 0, 0, 0};  // what rows outside a sequence are read as

struct AtArgs {
  const uint16_t *q, *k, *v, *o, *dout;
  uint16_t *out, *olo, *dq, *dk, *dv;  // olo: what rounding took from o, or null (no backward)
  float *lse, *dsum, *part;   // [B, nh, Tp]: -L in log2, -D; [B, nh, T, D] x 2: dk, dv by query head
  float* omax;                // fp16: [B][2][parts] maxima of |do|^2 and of |v|^2
  const int* lens;            // [B] or null
  long qb, qh, qt, kb, kh, kt, vb, vh, vt;  // strides in elements
  int B, T, Tp, nh, nkv, causal, split, parts;
  float scale;
};

template <bool BF>
__device__ __forceinline__ f32x16 at_mma(u16x8 a, u16x8 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

template <bool BF>
__device__ __forceinline__ uint16_t at_round(float x) {
  if constexpr (BF) {
    const __bf16 b = (__bf16)x;
    return __builtin_bit_cast(uint16_t, b);
  } else {
    const _Float16 b = (_Float16)x;
    return __builtin_bit_cast(uint16_t, b);
  }
}

template <bool BF>
__device__ __forceinline__ float at_float(uint16_t x) {
  if constexpr (BF)
    return __uint_as_float((uint32_t)x << 16);
  else
    return (float)__builtin_bit_cast(_Float16, x);
}

// the values of both lane halves l and l ^ 32
__device__ __forceinline__ float at_max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float at_sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// What is XORed into the 16-byte chunk index of row `row` of a tile.  LDS serves 256 bytes a
// cycle over 64 banks: 16 lanes of a row read (16 rows, one chunk) or 32 of a transposing
// read (4 rows, 4 chunks); either way the chunks differ modulo 256 bytes.
template <int D>
__device__ __forceinline__ int at_swz(int row) {
  if constexpr (D == 64)  // 128-byte rows: row & 1 is half of the banks already
    return ((row >> 1) & 1) << 2 | ((row >> 2) & 1) | ((row >> 3) & 1) << 1;
  else
    return (row & 3) << 2 | ((row >> 2) & 3);
}

// Rows [r0, r0 + ROWS) of a [.., D] matrix into LDS, rows at or behind `end` as zeros.
template <int D, int ROWS, int NW>
__device__ __forceinline__ void at_stage(const uint16_t* src, long ld, int r0, int end, uint16_t* dst, int wave,
                                         int lane) {
  constexpr int CPR = D / 8, RPI = 64 / CPR;  // chunks a row, rows a DMA instruction
  constexpr int N = ROWS / RPI;
  const int rr = lane / CPR, p = lane % CPR;
#pragma unroll
  for (int i = 0; i < (N + NW - 1) / NW; ++i) {
    const int g = wave + NW * i;
    if (N % NW != 0 && g >= N) break;
    const int row = RPI * g + rr;
    const uint16_t* gp = src + (long)(r0 + row) * ld + ((p ^ at_swz<D>(row)) << 3);
    if (r0 + row >= end) gp = reinterpret_cast<const uint16_t*>(&at_zero);
    __builtin_amdgcn_global_load_lds((const void*)gp, (at_lds_t)(dst + g * RPI * D), 16, 0, 0);
  }
}

// Row operand: row `row` of the tile, k-values 16 s + 8 h + 0..7.
template <int D>
__device__ __forceinline__ u16x8 at_row(const uint16_t* tile, int row, int s, int h) {
  return *reinterpret_cast<const u16x8*>(tile + row * D + (((2 * s + h) ^ at_swz<D>(row)) << 3));
}

// Column operand: column 32 dt + (lane & 31), k-values = rows r0 + 8 (j >> 2) + 4 h + (j & 3).
template <int D>
__device__ __forceinline__ u16x8 at_col(const uint16_t* tile, int r0, int dt, int lane) {
  const int i = lane & 15, ch = 4 * dt + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
  const int row = r0 + 4 * (lane >> 5) + (i >> 2);
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (at_tr_t)(tile + row * D + ((ch ^ at_swz<D>(row)) << 3) + ((i & 1) << 2)));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (at_tr_t)(tile + (row + 8) * D + ((ch ^ at_swz<D>(row + 8)) << 3) + ((i & 1) << 2)));
  const s16x4 both[2] = {lo, hi};
  u16x8 r;
  __builtin_memcpy(&r, both, 16);
  return r;
}

// The wave's own rows as an operand: row r (zeros when !on), k-values 16 s + 8 h + 0..7.
template <int D>
__device__ __forceinline__ void at_own(u16x8 (&f)[D / 16], const uint16_t* row, bool on, int h) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    f[s] = (u16x8)(uint16_t)0;
    if (on) f[s] = *reinterpret_cast<const u16x8*>(row + 16 * s + 8 * h);
  }
}

template <bool BF>
__device__ __forceinline__ u16x8 at_pack(const float* p) {
  u16x8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = at_round<BF>(p[j]);
  return r;
}

// Eight values of P or dS as operands: rounded, and (FINE) what rounding took as a second
// product.  A result carries its terms' roundings besides its own: 2.4e-3 of its norm off in
// bf16 for 1.7e-3, and where few rows are summed 2.7e-3.  FINE is for those, dS up to 64 rows
// (dq and dk 1.9e-3; 128 x 61 rows take 41.7 us with it for 40.1), P up to 32 (out and dv as
// near as their type allows; up to 64 rows it takes 1.4 us more, and they stay under 2.3e-3).
template <bool BF, bool FINE, int DT>
__device__ __forceinline__ void at_mma_p(f32x16 (&o)[DT], const u16x8 (&col)[DT], const float* p) {
  const u16x8 hi = at_pack<BF>(p);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = at_mma<BF>(col[dt], hi, o[dt]);
  if constexpr (FINE) {
    float r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = p[j] - at_float<BF>(hi[j]);
    const u16x8 lo = at_pack<BF>(r);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = at_mma<BF>(col[dt], lo, o[dt]);
  }
}

__device__ __forceinline__ void at_wait() {
  // this wave's DMAs have landed and its reads of the other buffer are done ...
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();  // ... and every wave's
  asm volatile("" ::: "memory");
}

// 16 values of a [.., D]-row (zeros when !on): columns 32 dt + 8 g + 4 h + 0..3, g = 0..3
template <bool BF>
__device__ __forceinline__ void at_store(uint16_t* row, const f32x16& x, float f, bool on, int dt, int h) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    uint16_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = on ? at_round<BF>(x[4 * g + e] * f) : (uint16_t)0;
    *reinterpret_cast<uint2*>(row + 32 * dt + 8 * g + 4 * h) =
        make_uint2((uint32_t)w[0] | ((uint32_t)w[1] << 16), (uint32_t)w[2] | ((uint32_t)w[3] << 16));
  }
}

constexpr int AT_KT = 64;  // rows of a walked tile

// Blocks of the long rows of a causal batch start first: block -> (tile, batch x head).
__device__ __forceinline__ void at_tile_of(int tiles, int pairs, bool heavy_last, int& tile, int& pair) {
  const int t = blockIdx.x / pairs;
  pair = blockIdx.x - t * pairs;
  tile = heavy_last ? tiles - 1 - t : t;
}

template <bool BF, int D, int NW>
__global__ void __launch_bounds__(NW * 64) attn_fwd_kernel(AtArgs a) {
  constexpr int TILE = AT_KT * D;
  __shared__ __attribute__((aligned(16))) uint16_t sm[4 * TILE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  int qi, bh;
  at_tile_of((a.Tp + 32 * NW - 1) / (32 * NW), a.B * a.nh, a.causal, qi, bh);
  const int b = bh / a.nh, hq = bh - b * a.nh, g = hq / (a.nh / a.nkv);
  const int len = a.lens != nullptr ? min(max(a.lens[b], 0), a.T) : a.T;
  const int q0 = qi * 32 * NW, qw = q0 + 32 * wave, qr = qw + (lane & 31);
  const uint16_t* kp = a.k + b * a.kb + g * a.kh;
  const uint16_t* vp = a.v + b * a.vb + g * a.vh;
  const int kend = q0 < len ? (a.causal ? min(len, q0 + 32 * NW) : len) : 0;  // keys of the block
  const int kw = qw < len ? (a.causal ? min(len, qw + 32) : len) : 0;         // ... of the wave
  const int lim = a.causal ? min(len, qr + 1) : len;                          // ... of the lane
  const int nt = (kend + AT_KT - 1) / AT_KT;
  u16x8 qf[D / 16];
  at_own<D>(qf, a.q + b * a.qb + hq * a.qh + qr * a.qt, qr < len, h);
  f32x16 o[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) o[dt] = (f32x16)0.f;
  float m = -INFINITY, ref = 0.f, l = 0.f;  // ref: m, or 0 while every S is -infinity
  const float c = a.scale * AT_LOG2E;
  auto stage = [&](int t) {
    uint16_t* dst = sm + (t & 1) * 2 * TILE;
    at_stage<D, AT_KT, NW>(kp, a.kt, t * AT_KT, len, dst, wave, lane);
    at_stage<D, AT_KT, NW>(vp, a.vt, t * AT_KT, len, dst + TILE, wave, lane);
  };
  if (nt > 0) stage(0);
  for (int t = 0; t < nt; ++t) {
    at_wait();
    if (t + 1 < nt) stage(t + 1);
    const int k0 = t * AT_KT;
    if (k0 >= kw) continue;
    const uint16_t *ks = sm + (t & 1) * 2 * TILE, *vs = ks + TILE;
    f32x16 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = (f32x16)0.f;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) s[u] = at_mma<BF>(at_row<D>(ks, 32 * u + (lane & 31), e, h), qf[e], s[u]);
    }
    if (k0 + AT_KT > (a.causal ? min(len, qw + 1) : len)) {  // some lane's border is in this tile
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + 32 * u + (r & 3) + 8 * (r >> 2) + 4 * h >= lim) s[u][r] = -INFINITY;
    }
    // (NaN passes: then m, l and o are NaN too)
    float top = __builtin_elementwise_maximum(s[0][0], s[1][0]);
#pragma unroll
    for (int r = 1; r < 16; ++r)
      top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, s[0][r]), s[1][r]);
    top = at_max_halves(top) * c;
    // any reference value serves the softmax: m follows the maximum only when it rises by
    // over 2^8, so most tiles skip the rescaling of o.  fp16: the reference lies 2^7 below,
    // so that P (at most 2^15) loses less under fp16's 2^-24
    constexpr float LOW = BF ? 0.f : 7.f;
    if (__any(top > m + (8.f + LOW))) {
      const float was = m;
      m = fmaxf(m, top - LOW);
      ref = m == -INFINITY ? 0.f : m;
      const float f = __builtin_amdgcn_exp2f(was - ref);
      l *= f;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= f;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], c, -ref));
        l += p[r];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        u16x8 vc[D / 32];
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) vc[dt] = at_col<D>(vs, 32 * u + 16 * e, dt, lane);
        at_mma_p<BF, NW == 1, D / 32>(o, vc, p + 8 * e);
      }
    }
  }
  l = at_sum_halves(l);
  const bool on = qr < len;
  const float inv = 1.f / l;
  if (qr < a.T) {
    uint16_t* row = a.out + ((size_t)b * a.T + qr) * a.nh * D + hq * D;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      at_store<BF>(row, o[dt], inv, on, dt, h);
      if (a.olo != nullptr) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float x = o[dt][r] * inv;
          o[dt][r] = x - at_float<BF>(at_round<BF>(x));
        }
        at_store<BF>(a.olo + (row - a.out), o[dt], 1.f, on, dt, h);
      }
    }
  }
  if (h == 0 && qr < a.Tp) a.lse[(size_t)bh * a.Tp + qr] = on ? -(m + __log2f(l)) : -INFINITY;
}

// fp16: the factor on dS.  dS = P (dP - D) where D is the mean of dP, so |dS| is at most half
// of the largest |dP|, and that at most |do| |v| over the longest finite rows of both in the
// sequence: the factor takes this bound to 2^15, under fp16's 65504.
__device__ __forceinline__ float at_ds_factor(const AtArgs& a, int b, int lane) {
  const float* m = a.omax + (size_t)b * 2 * a.parts;
  float x = 0.f, y = 0.f;
  for (int i = lane; i < a.parts; i += 64) {
    x = fmaxf(x, m[i]);
    y = fmaxf(y, m[a.parts + i]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    x = fmaxf(x, __shfl_xor(x, o, 64));
    y = fmaxf(y, __shfl_xor(y, o, 64));
  }
  x *= y;
  if (!(x > 0.f && x < 1e30f)) return 1.f;
  const int e = (int)(__float_as_uint(x) >> 23) - 127;  // |do| |v| < 2^(e / 2 rounded down + 1)
  return __uint_as_float((uint32_t)(127 + 15 - (e >> 1)) << 23);
}

// The largest squared length of do's (y = 0) and v's (y = 1) finite rows of a head, sequence by
// sequence: neither what lies behind a sequence, nor another one, nor an infinity (a matter of
// the rows that meet it) moves the factor.  D / 8 lanes a row; block part of `parts`.
template <int D>
__global__ void __launch_bounds__(1024) attn_omax_kernel(AtArgs a) {
  __shared__ float red[16];
  const bool isv = blockIdx.y == 1;
  const int b = blockIdx.x / a.parts, part = blockIdx.x - b * a.parts;
  const int len = a.lens != nullptr ? min(max(a.lens[b], 0), a.T) : a.T;
  const uint16_t* src = isv ? a.v + b * a.vb : a.dout + (size_t)b * a.T * a.nh * D;
  const long n = (long)len * (isv ? a.nkv : a.nh) * (D / 8);
  float m = 0.f;
  for (long i = (long)part * 1024 + threadIdx.x; i < n; i += (long)a.parts * 1024) {
    const long r = i / (D / 8);
    const int c = (int)(i % (D / 8)) * 8;
    const uint16_t* p = src + r * D + c;
    if (isv) {  // (64-bit divisions cost most of the kernel; almost every batch does without)
      const long g = n >> 32 ? r / len : (long)((uint32_t)r / (uint32_t)len);
      p = src + g * a.vh + (r - g * len) * a.vt + c;
    }
    const f16x8 v = *reinterpret_cast<const f16x8*>(p);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s = fmaf((float)v[k], (float)v[k], s);
#pragma unroll
    for (int o = 1; o < D / 8; o <<= 1) s += __shfl_xor(s, o, 64);
    if (s < INFINITY) m = fmaxf(m, s);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) m = fmaxf(m, red[w]);
    a.omax[((size_t)b * 2 + blockIdx.y) * a.parts + part] = m;
  }
}

template <bool BF, int D, int NW>
__global__ void __launch_bounds__(NW * 64) attn_dq_kernel(AtArgs a) {
  constexpr int TILE = AT_KT * D;
  __shared__ __attribute__((aligned(16))) uint16_t sm[4 * TILE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  int qi, bh;
  at_tile_of((a.Tp + 32 * NW - 1) / (32 * NW), a.B * a.nh, a.causal, qi, bh);
  const int b = bh / a.nh, hq = bh - b * a.nh, g = hq / (a.nh / a.nkv);
  const int len = a.lens != nullptr ? min(max(a.lens[b], 0), a.T) : a.T;
  const int q0 = qi * 32 * NW, qw = q0 + 32 * wave, qr = qw + (lane & 31);
  const uint16_t* kp = a.k + b * a.kb + g * a.kh;
  const uint16_t* vp = a.v + b * a.vb + g * a.vh;
  const int kend = q0 < len ? (a.causal ? min(len, q0 + 32 * NW) : len) : 0;
  const int kw = qw < len ? (a.causal ? min(len, qw + 32) : len) : 0;
  const int lim = a.causal ? min(len, qr + 1) : len;
  const int nt = (kend + AT_KT - 1) / AT_KT;
  auto stage = [&](int t) {
    uint16_t* dst = sm + (t & 1) * 2 * TILE;
    at_stage<D, AT_KT, NW>(kp, a.kt, t * AT_KT, len, dst, wave, lane);
    at_stage<D, AT_KT, NW>(vp, a.vt, t * AT_KT, len, dst + TILE, wave, lane);
  };
  if (nt > 0) stage(0);
  const bool on = qr < len;
  u16x8 qf[D / 16], df[D / 16];
  at_own<D>(qf, a.q + b * a.qb + hq * a.qh + qr * a.qt, on, h);
  const size_t orow = ((size_t)b * a.T + qr) * a.nh * D + hq * D;
  at_own<D>(df, a.dout + orow, on, h);
  float dsum = 0.f;  // D of the lane's row, half of its columns
  {
    u16x8 of[D / 16], lo[D / 16];
    at_own<D>(of, a.o + orow, on, h);
    at_own<D>(lo, a.olo + orow, on, h);
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        dsum = fmaf(at_float<BF>(of[s][j]) + at_float<BF>(lo[s][j]), at_float<BF>(df[s][j]), dsum);
  }
  dsum = at_sum_halves(dsum);
  if (h == 0 && qr < a.Tp) a.dsum[(size_t)bh * a.Tp + qr] = -dsum;
  const float lse = on ? a.lse[(size_t)bh * a.Tp + qr] : -INFINITY;  // -L
  const float c = a.scale * AT_LOG2E;
  float dsf = 1.f;
  if constexpr (!BF) dsf = at_ds_factor(a, b, lane);
  f32x16 dq[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) dq[dt] = (f32x16)0.f;
  // BORDER: some lane's border of keys is in the tile
  auto tile = [&](const uint16_t* ks, int k0, auto border) {
    const uint16_t* vs = ks + TILE;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x16 s = (f32x16)0.f, dp = (f32x16)(-dsum);
#pragma unroll
      for (int e = 0; e < D / 16; ++e) s = at_mma<BF>(at_row<D>(ks, 32 * u + (lane & 31), e, h), qf[e], s);
#pragma unroll
      for (int e = 0; e < D / 16; ++e) dp = at_mma<BF>(at_row<D>(vs, 32 * u + (lane & 31), e, h), df[e], dp);
      float ds[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float p = __builtin_amdgcn_exp2f(fmaf(s[r], c, lse));
        // (a row of one key has P = 1 and dS = 0, not the rounding of dP - D)
        if (border.value && (k0 + 32 * u + (r & 3) + 8 * (r >> 2) + 4 * h >= lim || lim == 1)) p = 0.f;
        ds[r] = BF ? p * dp[r] : p * dp[r] * dsf;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        u16x8 kc[D / 32];
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) kc[dt] = at_col<D>(ks, 32 * u + 16 * e, dt, lane);
        at_mma_p<BF, NW <= 2, D / 32>(dq, kc, ds + 8 * e);
      }
    }
  };
  const int whole = a.causal ? min(len, qw + 1) : len;  // keys that every lane of the wave sees
  for (int t = 0; t < nt; ++t) {
    at_wait();
    if (t + 1 < nt) stage(t + 1);
    const int k0 = t * AT_KT;
    const uint16_t* ks = sm + (t & 1) * 2 * TILE;
    if (k0 + AT_KT <= whole)
      tile(ks, k0, std::false_type());
    else if (k0 < kw)
      tile(ks, k0, std::true_type());
  }
  if (qr < a.T) {
    uint16_t* row = a.dq + ((size_t)bh * a.T + qr) * D;
    const float f = a.scale / dsf;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) at_store<BF>(row, dq[dt], f, on, dt, h);
  }
}

// dk, dv of 32 NW keys: a key head's own (split 0: its query heads one after the other) or
// one query head's (split 1: fp32 into part, attn_join sums the heads).
template <bool BF, int D, int NW>
__global__ void __launch_bounds__(NW * 64) attn_dkv_kernel(AtArgs a) {
  constexpr int TILE = AT_KT * D;
  constexpr int STAGE = 2 * TILE + 4 * AT_KT;  // Q, dO and the rows' L and D (fp32)
  __shared__ __attribute__((aligned(16))) uint16_t sm[2 * STAGE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int rep = a.nh / a.nkv, heads = a.split ? a.nh : a.nkv;
  int ki, bh;
  at_tile_of((a.T + 32 * NW - 1) / (32 * NW), a.B * heads, false, ki, bh);
  const int b = bh / heads, hx = bh - b * heads;
  const int g = a.split ? hx / rep : hx, h0 = a.split ? hx : hx * rep, nrep = a.split ? 1 : rep;
  const int len = a.lens != nullptr ? min(max(a.lens[b], 0), a.T) : a.T;
  const int k0 = ki * 32 * NW, kw = k0 + 32 * wave, kr = kw + (lane & 31);
  const bool on = kr < len;
  const int t0 = a.causal ? k0 / AT_KT : 0;
  const int per = k0 < len ? (len + AT_KT - 1) / AT_KT - t0 : 0;  // query tiles of a head
  const int nt = per * nrep;
  auto stage = [&](int i) {
    const int r = i / per, q0 = (t0 + i - r * per) * AT_KT, hq = h0 + r;
    uint16_t* dst = sm + (i & 1) * STAGE;
    at_stage<D, AT_KT, NW>(a.q + b * a.qb + hq * a.qh, a.qt, q0, len, dst, wave, lane);
    at_stage<D, AT_KT, NW>(a.dout + ((size_t)b * a.T) * a.nh * D + hq * D, (long)a.nh * D, q0, len, dst + TILE, wave,
                           lane);
    const size_t at = ((size_t)b * a.nh + hq) * a.Tp + q0 + lane;
    if (wave == 0)
      __builtin_amdgcn_global_load_lds((const void*)(a.lse + at), (at_lds_t)(dst + 2 * TILE), 4, 0, 0);
    if (wave == NW - 1)
      __builtin_amdgcn_global_load_lds((const void*)(a.dsum + at), (at_lds_t)(dst + 2 * TILE + 2 * AT_KT), 4, 0, 0);
  };
  if (nt > 0) stage(0);
  u16x8 kf[D / 16], vf[D / 16];
  at_own<D>(kf, a.k + b * a.kb + g * a.kh + kr * a.kt, on, h);
  at_own<D>(vf, a.v + b * a.vb + g * a.vh + kr * a.vt, on, h);
  const float c = a.scale * AT_LOG2E;
  float dsf = 1.f;
  if constexpr (!BF) dsf = at_ds_factor(a, b, lane) * (1.f / (1 << AT_FP16_P));
  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) dk[dt] = dv[dt] = (f32x16)0.f;
  // BORDER: the tile holds queries before some lane's key
  auto tile = [&](const uint16_t* qs, int q0, auto border) {
    const uint16_t* os = qs + TILE;
    const float* ls = reinterpret_cast<const float*>(os + TILE);  // -L, -D
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x16 s = (f32x16)0.f, dp;
      float lq[16];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 x = *reinterpret_cast<const float4*>(ls + 32 * u + 8 * e + 4 * h);
        const float4 y = *reinterpret_cast<const float4*>(ls + AT_KT + 32 * u + 8 * e + 4 * h);
        lq[4 * e] = x.x, lq[4 * e + 1] = x.y, lq[4 * e + 2] = x.z, lq[4 * e + 3] = x.w;
        dp[4 * e] = y.x, dp[4 * e + 1] = y.y, dp[4 * e + 2] = y.z, dp[4 * e + 3] = y.w;
      }
#pragma unroll
      for (int e = 0; e < D / 16; ++e) s = at_mma<BF>(at_row<D>(qs, 32 * u + (lane & 31), e, h), kf[e], s);
#pragma unroll
      for (int e = 0; e < D / 16; ++e) dp = at_mma<BF>(at_row<D>(os, 32 * u + (lane & 31), e, h), vf[e], dp);
      float p[16], ds[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, BF ? lq[r] : lq[r] + (float)AT_FP16_P));
        if (border.value && q0 + 32 * u + (r & 3) + 8 * (r >> 2) + 4 * h < kr) p[r] = 0.f;
        ds[r] = BF ? p[r] * dp[r] : p[r] * dp[r] * dsf;
      }
      if (border.value && q0 == 0 && u == 0 && h == 0) ds[0] = 0.f;  // query 0 has one key: dS = 0
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        u16x8 oc[D / 32], qc[D / 32];
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) {
          oc[dt] = at_col<D>(os, 32 * u + 16 * e, dt, lane);
          qc[dt] = at_col<D>(qs, 32 * u + 16 * e, dt, lane);
        }
        at_mma_p<BF, NW == 1, D / 32>(dv, oc, p + 8 * e);
        at_mma_p<BF, NW <= 2, D / 32>(dk, qc, ds + 8 * e);
      }
    }
  };
  for (int i = 0; i < nt; ++i) {
    at_wait();
    if (i + 1 < nt) stage(i + 1);
    const int q0 = (t0 + i % per) * AT_KT;
    const uint16_t* qs = sm + (i & 1) * STAGE;
    if (kw >= len) continue;
    if (!a.causal || q0 >= kw + 31)
      tile(qs, q0, std::false_type());
    else if (q0 + AT_KT > kw)
      tile(qs, q0, std::true_type());
  }
  if (kr >= a.T) return;
  const float fk = BF ? a.scale : a.scale / (dsf * (1 << AT_FP16_P));
  const float fv = BF ? 1.f : 1.f / (1 << AT_FP16_P);
  const bool dkon = on && len > 1;  // (one key: dS = 0)
  const size_t row = ((size_t)bh * a.T + kr) * D;
  if (a.split) {
    float* pk = a.part + row;
    float* pv = pk + (size_t)a.B * a.nh * a.T * D;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 32 * dt + 8 * e + 4 * h;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
        if (dkon)
          x = make_float4(dk[dt][4 * e] * fk, dk[dt][4 * e + 1] * fk, dk[dt][4 * e + 2] * fk, dk[dt][4 * e + 3] * fk);
        if (on)
          y = make_float4(dv[dt][4 * e] * fv, dv[dt][4 * e + 1] * fv, dv[dt][4 * e + 2] * fv, dv[dt][4 * e + 3] * fv);
        *reinterpret_cast<float4*>(pk + d) = x;
        *reinterpret_cast<float4*>(pv + d) = y;
      }
  } else {
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      at_store<BF>(a.dk + row, dk[dt], fk, dkon, dt, h);
      at_store<BF>(a.dv + row, dv[dt], fv, on, dt, h);
    }
  }
}

// dk, dv [B, nkv, T * D] = the sums of `part` [2][B, nh, T * D] over each key head's query
// heads, in their order; 4 elements a thread.
template <bool BF>
__global__ void __launch_bounds__(256) attn_join_kernel(const float* __restrict__ part, uint16_t* __restrict__ dk,
                                                        uint16_t* __restrict__ dv, long pairs, long td, int rep) {
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4, n = pairs * td;  // pairs = B nkv
  if (i >= n) return;
  const long pr = i / td, e = i - pr * td;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const float* src = part + (w ? n * rep : 0) + pr * rep * td + e;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r = 0; r < rep; ++r) {
      const float4 x = *reinterpret_cast<const float4*>(src + r * td);
      s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
    }
    *reinterpret_cast<uint2*>((w ? dv : dk) + i) =
        make_uint2((uint32_t)at_round<BF>(s.x) | ((uint32_t)at_round<BF>(s.y) << 16),
                   (uint32_t)at_round<BF>(s.z) | ((uint32_t)at_round<BF>(s.w) << 16));
  }
}

bool at_bad(int B, int T, int nh, int nkv, int D) {
  return B <= 0 || T <= 0 || T > (1 << 24) || nkv <= 0 || nh <= 0 || nh % nkv != 0 || (D != 64 && D != 128) ||
         (long)B * nh > (1 << 20) || ((long)T + 127) / 128 * B * nh >= 1 << 24;  // (a grid holds 2^32 threads)
}

int at_parts(int B) {
  int p = AT_MAXPARTS;
  while (p > 1 && p * B > AT_MAXPARTS) p >>= 1;
  return p;
}

template <bool BF, int D>
void at_launch_fwd(const AtArgs& a, hipStream_t st) {
  const int pairs = a.B * a.nh;
  if (a.T <= 32)
    attn_fwd_kernel<BF, D, 1><<<dim3((a.Tp + 31) / 32 * pairs), dim3(64), 0, st>>>(a);
  else if (a.T <= 64)
    attn_fwd_kernel<BF, D, 2><<<dim3((a.Tp + 63) / 64 * pairs), dim3(128), 0, st>>>(a);
  else
    attn_fwd_kernel<BF, D, 4><<<dim3((a.Tp + 127) / 128 * pairs), dim3(256), 0, st>>>(a);
}

template <bool BF, int D>
void at_launch_bwd(const AtArgs& a, hipStream_t st) {
  const int pairs = a.B * a.nh, kpairs = a.B * (a.split ? a.nh : a.nkv);
  if constexpr (!BF) attn_omax_kernel<D><<<dim3(a.B * a.parts, 2), dim3(1024), 0, st>>>(a);
  if (a.T <= 32) {
    attn_dq_kernel<BF, D, 1><<<dim3((a.Tp + 31) / 32 * pairs), dim3(64), 0, st>>>(a);
    attn_dkv_kernel<BF, D, 1><<<dim3((a.T + 31) / 32 * kpairs), dim3(64), 0, st>>>(a);
  } else if (a.T <= 64) {
    attn_dq_kernel<BF, D, 2><<<dim3((a.Tp + 63) / 64 * pairs), dim3(128), 0, st>>>(a);
    attn_dkv_kernel<BF, D, 2><<<dim3((a.T + 63) / 64 * kpairs), dim3(128), 0, st>>>(a);
  } else {
    attn_dq_kernel<BF, D, 4><<<dim3((a.Tp + 127) / 128 * pairs), dim3(256), 0, st>>>(a);
    attn_dkv_kernel<BF, D, 4><<<dim3((a.T + 127) / 128 * kpairs), dim3(256), 0, st>>>(a);
  }
  if (a.split)
    attn_join_kernel<BF><<<dim3((unsigned)(((long)a.B * a.nkv * a.T * D / 4 + 255) / 256)), dim3(256), 0, st>>>(
        a.part, a.dk, a.dv, (long)a.B * a.nkv, (long)a.T * D, a.nh / a.nkv);
}

}  // namespace

extern "C" {

// Row count of the fp32 row statistics (lse, dsum: [B, nh, rows]).
int sg_attn_rows(int T) { return (T + AT_KT - 1) / AT_KT * AT_KT; }

// Whether the keys' gradient is taken per query head and joined: with few key heads and
// rows a block per key head leaves most of the card idle (B nkv T / 128 blocks on 256 CUs,
// and under a causal mask the first keys' blocks run twice the mean).
int sg_attn_split(int B, int T, int nh, int nkv) {
  return nh != nkv && (long)B * nkv * ((T + 127) / 128) < 1024 && T > 128 ? 1 : 0;
}

// fp16: floats of the maxima that the factors on dS come from.
int sg_attn_maxima(int B) { return (2 * B * at_parts(B) + 63) / 64 * 64; }

int sg_attn_fwd(const void* q, const void* k, const void* v, const void* lens, void* out, void* olo, void* lse,
                const void* strides,
                int B, int T, int nh, int nkv, int D, int causal, int fp16, float scale, hipStream_t st) {
  if (at_bad(B, T, nh, nkv, D)) return 1;
  const long* s = (const long*)strides;
  AtArgs a = {};
  a.q = (const uint16_t*)q, a.k = (const uint16_t*)k, a.v = (const uint16_t*)v, a.lens = (const int*)lens;
  a.out = (uint16_t*)out, a.olo = (uint16_t*)olo, a.lse = (float*)lse;
  a.qb = s[0], a.qh = s[1], a.qt = s[2], a.kb = s[3], a.kh = s[4], a.kt = s[5], a.vb = s[6], a.vh = s[7], a.vt = s[8];
  a.B = B, a.T = T, a.Tp = sg_attn_rows(T), a.nh = nh, a.nkv = nkv, a.causal = causal, a.scale = scale;
  if (fp16)
    D == 64 ? at_launch_fwd<false, 64>(a, st) : at_launch_fwd<false, 128>(a, st);
  else
    D == 64 ? at_launch_fwd<true, 64>(a, st) : at_launch_fwd<true, 128>(a, st);
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

// ws: fp32 [B nh rows] (D), then sg_attn_maxima (fp16 only), then [2][B, nh, T, D] where sg_attn_split
int sg_attn_bwd(const void* q, const void* k, const void* v, const void* lens, const void* out, const void* olo,
                const void* lse, const void* dout, void* dq, void* dk, void* dv, void* ws, const void* strides, int B, int T, int nh,
                int nkv, int D, int causal, int fp16, float scale, hipStream_t st) {
  if (at_bad(B, T, nh, nkv, D)) return 1;
  const long* s = (const long*)strides;
  AtArgs a = {};
  a.q = (const uint16_t*)q, a.k = (const uint16_t*)k, a.v = (const uint16_t*)v, a.lens = (const int*)lens;
  a.o = (const uint16_t*)out, a.olo = (uint16_t*)const_cast<void*>(olo), a.lse = (float*)const_cast<void*>(lse), a.dout = (const uint16_t*)dout;
  a.dq = (uint16_t*)dq, a.dk = (uint16_t*)dk, a.dv = (uint16_t*)dv;
  a.qb = s[0], a.qh = s[1], a.qt = s[2], a.kb = s[3], a.kh = s[4], a.kt = s[5], a.vb = s[6], a.vh = s[7], a.vt = s[8];
  a.B = B, a.T = T, a.Tp = sg_attn_rows(T), a.nh = nh, a.nkv = nkv, a.causal = causal, a.scale = scale;
  a.split = sg_attn_split(B, T, nh, nkv);
  a.dsum = (float*)ws;
  float* w = a.dsum + (size_t)B * nh * a.Tp;
  if (fp16) {
    a.omax = w;
    a.parts = at_parts(B);
    w += sg_attn_maxima(B);
  }
  a.part = w;
  if (fp16)
    D == 64 ? at_launch_bwd<false, 64>(a, st) : at_launch_bwd<false, 128>(a, st);
  else
    D == 64 ? at_launch_bwd<true, 64>(a, st) : at_launch_bwd<true, 128>(a, st);
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

}  // extern "C"
