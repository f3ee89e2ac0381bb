// smsgate_amd — softmax cross entropy of hidden states over the rows of the embedding, and
// the gradients of both, without a [rows, vocabulary] matrix of logits (gfx950).
//
//   z = h E^T,  L_i = logsumexp z_i,  loss_i = L_i - z_i[y_i]
//   d_i[v] = w_i (exp(z_i[v] - L_i) - [v = y_i]),  dh = f d E,  dE = f d^T h
//
// h [N, H] and E [V, H] in bf16 or fp16, H a multiple of 8, any N and V.  Rows whose label
// is ignore_index are left out before any product: loss_rows lists the others, loss_hidden
// copies them together, and every later block reads the count from the device and ends at
// once behind it (an SMS batch labels about a third of its positions).
//
//   forward   loss_logits<0>: a tile's logits stay in the accumulators; each row's maximum
//             and sum of exponentials over the tile's ids but the label go out (8 bytes a row and
//             tile), the label's logit from the tile that has it;
//             loss_join: L, loss and its mean or sum
//   backward  per piece of the vocabulary: loss_logits<1> recomputes the tile's logits and
//             writes d in the inputs' type; loss_grad: the piece's rows of dE, and dh's
//             shares, fp32, the piece's columns split over blocks; loss_dh sums the shares in
//             order and puts the rows back (ignored: zeros)
//
// Four products of 2 n V H flops where keeping the logits would need three: z is needed in
// fp32 (its rounding to 16 bits would put errors of per cents into exp), and storing it
// costs more memory time at H = 576 than multiplying again.  d is rounded to the inputs'
// type as an operand (as the gradient of such logits is under autocast; up to 128 rows what
// rounding took is a second operand); fp16 holds
// nothing under 2^-24, so there d is scaled by 2^10 (|d| <= 1) and f takes it out.  Every
// other sum, L and dh's shares are fp32; no float atomics, every sum has a fixed order.
//
// A trained model is nearly sure of most labels, and at logits of hundreds 1 - p is far below
// L's last bit.  So L is kept in two parts, the largest logit and the logarithm of the sum over
// it; and with t = the others' sum over the label's exponential, loss = log(1 + t) and the
// label's d = -t / (1 + t): as exact as t, where exp(z - L) - 1 would be rounding alone.
//
// Products: v_mfma_f32_32x32x16, result in lane l: column l & 31 (the "lane" side: a hidden
// row, or a vocabulary row for dE), rows (r & 3) + 8 (r >> 2) + 4 (l >> 5) (the "register"
// side).  h, E and d lie in panels of 32 columns (h's rows and E are copied once a
// call); a tile comes by DMA (global_load_lds) into two buffers, one barrier a 32-wide step.
// Operands whose k runs along a panel's rows are read from LDS as rows, others by transposing
// reads (ds_read_b64_tr_b16), so no transposed copy exists.
//
// What bounds it: the operands' way from L2 (11 TB/s in loss_logits at 8192 rows; a third
// less time with the copies left out, none with LDS reads or exp left out), and that a block's
// waves wait together: three blocks a CU of 128 x 256 (165 registers) beat two of them with
// deeper buffers (467 us against 491) and one of 256 x 256 (518).  Measured at 8192 rows, 49152
// ids, 576 columns, bf16: logits 467 to 483 us (993 to 960 TFLOP/s), d 525 to 538, both
// gradients 1057 to 1086 (878 to 854 TFLOP/s); the library's single products of these shapes
// take 539, 604 and 750.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "train_ops.hpp"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lk_lds_t;
typedef __attribute__((address_space(3))) s16x4* lk_tr_t;

constexpr float LK_LOG2E = 1.4426950408889634f;
constexpr int LK_K = 64;         // hc's columns and dh's splits are whole multiples
constexpr int LK_PAD = 256;      // rows and pieces are padded to whole tiles
constexpr float LK_FP16 = 1024.f;  // factor on d in fp16

struct LossArgs {
  const uint16_t *h, *table;
  const void* labels;
  uint16_t *hc, *ec, *d, *dh, *dtable;  // hc, ec, d: panels
  long lo;                          // few rows: what rounding took from d lies so far behind it, else 0
  int *pos, *rows, *lab, *cnt;      // [N] place or -1; [Mp] row of a place; [Mp] label; rows, blocks done, splits
  float *top, *ls2;                 // [Mp] x 2: L = top + ls2 ln 2
  float *rl;                        // [Mp] label's logit, from the join on its 1 - p
  float *loss, *w;                  // out; [Mp] row weights or null
  float2* part;                     // [v tiles][Mp] (maximum, sum of exp(z - maximum)) without the label
  float* share;                     // [splits][Mp][Hp]
  const float *g, *gmax;            // incoming gradient; none: its largest magnitude
  long ignore;
  int N, V, H, Mp, Hp, Vp, is64, mode;  // mode 0 mean, 1 sum, 2 none
  int v0, vn;                       // piece: first row, rows (of them < V - v0 real)
  int splits, want, most, first;    // dh: shares of Mp rows in the workspace; the card's places; splits at most
  int bl, nr;                       // dh: rows of a tile, tiles over H
  int t2;                           // blocks of dE, a multiple of 8
};

template <bool BF>
__device__ __forceinline__ f32x16 lk_mma(u16x8 a, u16x8 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

template <bool BF>
__device__ __forceinline__ uint16_t lk_round(float x) {
  if constexpr (BF) {
    const __bf16 b = (__bf16)x;
    return __builtin_bit_cast(uint16_t, b);
  } else {
    const _Float16 b = (_Float16)x;
    return __builtin_bit_cast(uint16_t, b);
  }
}

// x without what rounding to the type keeps of it
template <bool BF>
__device__ __forceinline__ float lk_rest(float x) {
  if constexpr (BF)
    return x - (float)(__bf16)x;
  else
    return x - (float)(_Float16)x;
}

template <bool BF>
__device__ __forceinline__ uint2 lk_pack4(float a, float b, float c, float d) {
  return make_uint2((uint32_t)lk_round<BF>(a) | ((uint32_t)lk_round<BF>(b) << 16),
                    (uint32_t)lk_round<BF>(c) | ((uint32_t)lk_round<BF>(d) << 16));
}

// Eight values 8 e + 4 h + 0..3 (e: a pair of groups) of a row held by lanes l and l ^ 32:
// the halves trade, so that each lane writes 16 bytes (half 0 group e, half 1 group e + 1).
template <bool BF>
__device__ __forceinline__ uint4 lk_trade(float4 x, float4 y) {
  const uint2 p = lk_pack4<BF>(x.x, x.y, x.z, x.w), q = lk_pack4<BF>(y.x, y.y, y.z, y.w);
  const auto a = __builtin_amdgcn_permlane32_swap(p.x, q.x, false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(p.y, q.y, false, false);
  return make_uint4(a[0], b[0], a[1], b[1]);
}

__device__ __forceinline__ float lk_max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float lk_sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float lk_exp(float x) { return __builtin_amdgcn_exp2f(x * LK_LOG2E); }
// e^x without the rounding of x log2(e), which costs |x| 2^-24.  The small tiles' sums and the
// joins take it, as a loss of few rows shows that where a mean over many does not; the large
// tiles' epilogues would take 8 % longer with it (63 us for 58, 4773 rows of 8192 x 576).
__device__ __forceinline__ float lk_exp_fine(float x) {
  const float t = x * LK_LOG2E, lo = fmaf(x, 1.92596303e-8f, fmaf(x, LK_LOG2E, -t));
  const float e = __builtin_amdgcn_exp2f(t);
  return x < -150.f ? 0.f : fmaf(e, lo * 0.693147181f, e);  // (-infinity would give NaN)
}

__device__ __forceinline__ float4 lk_four(const f32x16& x, int e, float f) {
  return make_float4(x[4 * e] * f, x[4 * e + 1] * f, x[4 * e + 2] * f, x[4 * e + 3] * f);
}

// ---- rows with a label, operands in panels ------------------------------------------------
// Every operand of the products lies in panels of LK_PANEL columns, [panel][rows][LK_PANEL]:
// a tile is runs of memory of 1 KB and more whichever way it is read, nothing of it is out of
// bounds, and its copies need no address but a wave's own.  (Tiles of the matrices as they
// come, 64 bytes a row, kept the copies waiting for twice as many memory requests.)
constexpr int LK_PANEL = 32;
__device__ __forceinline__ size_t lk_at(long rows, long row, int c) {  // 16-byte chunk c of a row
  return ((c >> 2) * rows + row) * LK_PANEL + (c & 3) * 8;
}

// 16-byte chunk i of ec = E in panels, zeros behind its rows and columns
__device__ __forceinline__ void lk_lay_table(const LossArgs& a, long i) {
  const int nch = a.Hp / 8;
  const long r = i / nch;
  const int c = (int)(i - r * nch);
  if (r >= a.Vp) return;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (r < a.V && 8 * c < a.H) v = *reinterpret_cast<const uint4*>(a.table + (size_t)r * a.H + 8 * c);
  *reinterpret_cast<uint4*>(a.ec + lk_at(a.Vp, r, c)) = v;
}

// ... of hc = h[rows], zeros behind the last row up to a whole tile
__device__ __forceinline__ void lk_lay_hidden(const LossArgs& a, long i, int cnt, const int* rows) {
  const int nch = a.Hp / 8, m = (int)(i / nch), c = (int)(i - (long)m * nch);
  if (m >= (cnt + LK_PAD - 1) / LK_PAD * LK_PAD || m >= a.Mp) return;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (m < cnt && 8 * c < a.H) v = *reinterpret_cast<const uint4*>(a.h + (size_t)rows[m] * a.H + 8 * c);
  *reinterpret_cast<uint4*>(a.hc + lk_at(a.Mp, m, c)) = v;
}

__device__ __forceinline__ long lk_label(const LossArgs& a, int i) {
  return i >= a.N     ? a.ignore
         : a.is64 ? reinterpret_cast<const long*>(a.labels)[i]
                  : (long)reinterpret_cast<const int*>(a.labels)[i];
}

// What is known of row i: its place (or none).  A label outside [0, V) becomes -2 (its loss
// and gradients are NaN).
__device__ __forceinline__ void lk_put(const LossArgs& a, int i, long y, int place) {
  if (i >= a.N) return;
  const bool on = y != a.ignore;
  a.pos[i] = on ? place : -1;
  if (on) {
    a.rows[place] = i;
    a.lab[place] = y >= 0 && y < a.V ? (int)y : -2;
  } else if (a.mode == 2) {
    a.loss[i] = 0.f;
  }
}

constexpr int LK_SMALL = 1024;  // rows that a block numbers by itself

// The table in panels (the blocks from nb on), and the places of the labelled rows, in order.
// SMALL (up to LK_SMALL rows): every hidden block numbers the rows by itself and copies its
// part of them, so that one launch does all; else block 0 numbers them beside the table's
// copy, and loss_hidden follows.
template <bool SMALL>
__global__ void __launch_bounds__(1024) loss_rows_kernel(LossArgs a, int nb) {
  __shared__ int part[16], list[SMALL ? LK_SMALL : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if ((int)blockIdx.x >= nb) {
    lk_lay_table(a, (long)(blockIdx.x - nb) * 1024 + tid);
    return;
  }
  const unsigned long long before = (1ull << lane) - 1;
  int cnt = 0;
  if constexpr (SMALL) {
    const long y = lk_label(a, tid);
    const unsigned long long m = __ballot(y != a.ignore);
    if (lane == 0) part[wave] = __popcll(m);
    __syncthreads();
    int at = __popcll(m & before);
    for (int w = 0; w < 16; ++w) {
      if (w < wave) at += part[w];
      cnt += part[w];
    }
    if (y != a.ignore) list[at] = tid;
    if (blockIdx.x == 0) lk_put(a, tid, y, at);
    __syncthreads();
    lk_lay_hidden(a, (long)blockIdx.x * 1024 + tid, cnt, list);
  } else {
    for (int i0 = 0; i0 < a.N; i0 += 16384) {  // a wave owns 1024 labels, 64 at a time
      const int w0 = i0 + 1024 * wave + lane;
      long y[16];
      int n = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k) y[k] = lk_label(a, w0 + 64 * k);
#pragma unroll
      for (int k = 0; k < 16; ++k) n += __popcll(__ballot(y[k] != a.ignore));
      if (lane == 0) part[wave] = n;
      __syncthreads();
      int at = cnt;
      for (int w = 0; w < 16; ++w) {
        if (w < wave) at += part[w];
        cnt += part[w];
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const unsigned long long m = __ballot(y[k] != a.ignore);
        lk_put(a, w0 + 64 * k, y[k], at + __popcll(m & before));
        at += __popcll(m);
      }
      __syncthreads();
    }
  }
  if (blockIdx.x == 0 && tid == 0) a.cnt[0] = cnt, a.cnt[1] = 0;
}

__global__ void __launch_bounds__(256) loss_hidden_kernel(LossArgs a) {
  lk_lay_hidden(a, (long)blockIdx.x * 256 + threadIdx.x, a.cnt[0], a.rows);
}

// ---- products --------------------------------------------------------------------------
// A tile in LDS is [panel][rows][32] too, each 16-byte chunk XORed by its row: LDS serves 256
// bytes a cycle over 64 banks, and neither 16 lanes of a row read (16 rows, one chunk) nor
// 32 of a transposing read (4 rows, 4 chunks) meet on a bank.
__device__ __forceinline__ int lk_swz(int row) { return (row >> 2) & 3; }

// Row operand: row `row`, k-values (columns of the tile's panel) 16 s + 8 h + 0..7.
__device__ __forceinline__ u16x8 lk_row(const uint16_t* tile, int row, int s, int h) {
  return *reinterpret_cast<const u16x8*>(tile + row * LK_PANEL + (((2 * s + h) ^ lk_swz(row)) << 3));
}

// Column operand: column lane & 31 of a panel, the same k-values (its 32 rows).
__device__ __forceinline__ u16x8 lk_col(const uint16_t* panel, int s, int lane) {
  const int i = lane & 15, ch = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
  const int row = 16 * s + 8 * (lane >> 5) + (i >> 2);
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lk_tr_t)(panel + row * LK_PANEL + ((ch ^ lk_swz(row)) << 3) + ((i & 1) << 2)));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lk_tr_t)(panel + (row + 4) * LK_PANEL + ((ch ^ lk_swz(row + 4)) << 3) + ((i & 1) << 2)));
  const s16x4 both[2] = {lo, hi};
  u16x8 r;
  __builtin_memcpy(&r, both, 16);
  return r;
}

// Copies a tile by DMA, 16 rows of a panel an instruction.  !COL: SIDE rows of one panel;
// COL: 32 rows of SIDE / 32 panels, `stride` elements apart (panels behind the last repeat
// it: their results are not stored).  src: the tile's first row and panel.
template <int SIDE, int NW, bool COL>
__device__ __forceinline__ void lk_stage(const uint16_t* src, long stride, int panels, uint16_t* dst, int wave,
                                         uint32_t lane_off) {
  static_assert(SIDE / 16 % NW == 0, "whole instructions a wave");
#pragma unroll
  for (int i = 0; i < SIDE / 16 / NW; ++i) {
    const int g = wave + NW * i;
    const uint16_t* p = src + (COL ? min(g >> 1, panels - 1) * stride + (g & 1) * 512 : g * 512);
    __builtin_amdgcn_global_load_lds((const void*)(reinterpret_cast<const char*>(p) + lane_off),
                                     (lk_lds_t)(dst + g * 512), 16, 0, 0);
  }
}

// Splits of the piece's columns that dh's shares are taken in (the same for every piece, so
// that later pieces add to the shares of the first), chosen once for the count of rows by the
// 64 lanes of a wave, one candidate each: the end of the launch if its blocks go to the card's
// places in turn, dE's first, and the shares' memory time.  Steps of the blocks that end last
// count 0.73 us each (a block among others; with all places full a step's work adds 0.68 us
// whatever the split), a share's float 1.7e-6 us, written and read; over 1 to 11 splits of
// three large calls the sum is within 8 % of what was measured, but for launches that leave
// most places empty.  (8192 rows, 16384 of the ids, 576 columns: 2 splits 362 us, 3 432, 4 376,
// 5 433; a fixed number of blocks picked 4.)  The 64 x 64 tiles take the same numbers, though
// five of their blocks fit a CU and their steps are shorter: there they only keep any block from
// being much longer than the others.
__device__ int lk_choose(const LossArgs& a, int cnt, int lane) {
  const int nl = (cnt + a.bl - 1) / a.bl, nh = nl * a.nr, s = lane + 1;
  if (nh == 0) return 1;
  const int fit = min(a.most, (int)((long)a.splits * a.Mp / ((long)nl * a.bl)));
  const int ne = a.vn / a.bl * a.nr, e = (cnt + 31) / 32 + 4, r = ne % a.want;  // 4: a block's start and end
  const int l = ((a.vn / LK_K + s - 1) / s * LK_K) / 32 + 4;
  const float t0 = (float)(ne / a.want) * e, b = (float)nh * s;
  // after t0 steps: want - r places free, r more e steps later
  auto done = [&](float t) { return (a.want - r) * floorf(t / l) + r * floorf(fmaxf(t - e, 0.f) / l); };
  const float x = (b * l + (float)r * e) / a.want;  // were blocks divisible
  float end = INFINITY;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float p = (ceilf(x / l) + k) * l, q = e + (ceilf(fmaxf(x - e, 0.f) / l) + k) * l;
    if (done(p) >= b) end = fminf(end, p);
    if (done(q) >= b) end = fminf(end, q);
  }
  if (end == INFINITY) end = x + l;
  end = t0 + fmaxf(end, r ? (float)e : 0.f);
  float cost = s <= max(fit, 1) ? 0.73f * end + 1.7e-6f * s * cnt * a.Hp : INFINITY;
  int best = s;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float c = __shfl_xor(cost, o, 64);
    const int n = __shfl_xor(best, o, 64);
    if (c < cost || (c == cost && n < best)) cost = c, best = n;
  }
  return best;
}

// MODE 0 / 1: lane side = hidden rows, register side = vocabulary rows, k = H.
// MODE 2: lane = the piece's vocabulary rows, register = H, k = hidden rows.
// MODE 3: lane = hidden rows, register = H, k = a split of the piece.
// 32 k-values a step, ST buffers: the copies of the next ST - 1 steps are in flight.
// FINE: d is two operands, its rounding and what that took, a tile of each in every step.
template <bool BF, int MODE, int BL, int BR, int WL, int WR, int ST, bool FINE>
struct LkTile {
  static constexpr int NW = WL * WR, TL = BL / WL, TR = BR / WR, FL = TL / 32, FR = TR / 32;
  static constexpr int LT = FINE && MODE >= 2 ? 2 : 1;  // lane-side tiles a step
  static constexpr int BK = LK_PANEL, STAGE = (LT * BL + BR) * BK, NI = (LT * BL + BR) / 16 / NW;
  static_assert(ST * STAGE * 2 <= 160 * 1024 && BL % (32 * WL) == 0 && BR % (32 * WR) == 0, "tile");
  static __device__ __forceinline__ void run(const LossArgs& a, int block, uint16_t* sm);
};

template <bool BF, int MODE, int BL, int BR, int WL, int WR, int ST, bool FINE>
__device__ __forceinline__ void LkTile<BF, MODE, BL, BR, WL, WR, ST, FINE>::run(const LossArgs& a, int block,
                                                                                uint16_t* sm) {
  constexpr bool LCOL = MODE == 2, RCOL = MODE >= 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int wl = wave / WR, wr = wave % WR;
  const int cnt = a.cnt[0];
  const int nl = MODE == 2 ? a.vn / BL : (cnt + BL - 1) / BL;
  const int nr = MODE >= 2 ? (a.H + BR - 1) / BR : a.vn / BR;
  const int splits = MODE == 3 ? a.cnt[2] : 1;
  // blocks go round the 8 XCDs: each gets a run of tiles, walked in bands of 8 lane-side
  // tiles, so that what an XCD has in flight shares its L2.  Runs of the labelled rows'
  // tiles only (the grid holds all rows'): else a few XCDs would have all the work
  int t, z = 0;
  {
    const int T = nl * nr * splits, x = block & 7, q = T >> 3, r = T & 7, i = block >> 3;
    if (i >= q + (x < r)) return;
    t = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + i;
  }
  if constexpr (MODE == 3) {
    z = t / (nl * nr);
    t -= z * nl * nr;
  }
  const int band = t / (8 * nr), bl = t - band * 8 * nr, bw = min(8, nl - 8 * band);
  const int l0 = (8 * band + bl % bw) * BL, r0 = (bl / bw) * BR;
  int kb = 0, ke = (a.H + BK - 1) / BK * BK;  // (a step wholly behind either matrix would add zeros)
  if constexpr (MODE == 2) ke = (cnt + BK - 1) / BK * BK;
  if constexpr (MODE == 3) {
    const int per = (a.vn / LK_K + splits - 1) / splits * LK_K;
    const int end = (min(a.vn, a.V - a.v0) + BK - 1) / BK * BK;
    kb = min(end, z * per);
    ke = min(end, kb + per);
  }
  const uint32_t lane_off = (lane >> 2) * 64 + (((lane & 3) ^ lk_swz(lane >> 2)) << 4);
  const long mpan = (long)a.Mp * LK_PANEL, vpan = (long)a.Vp * LK_PANEL;  // a panel of hc or d, of ec
  auto stage = [&](int k0, int buf) {
    uint16_t *ls = sm + buf * STAGE, *rs = ls + LT * BL * BK;
    const int kp = k0 / LK_PANEL;
    if constexpr (MODE <= 1) {
      lk_stage<BL, NW, false>(a.hc + kp * mpan + (long)l0 * LK_PANEL, 0, 0, ls, wave, lane_off);
      lk_stage<BR, NW, false>(a.ec + kp * vpan + (long)(a.v0 + r0) * LK_PANEL, 0, 0, rs, wave, lane_off);
    } else if constexpr (MODE == 2) {
      const uint16_t* d = a.d + l0 / LK_PANEL * mpan + (long)k0 * LK_PANEL;
#pragma unroll
      for (int t = 0; t < LT; ++t) lk_stage<BL, NW, true>(d + t * a.lo, mpan, BL / 32, ls + t * BL * BK, wave, lane_off);
      lk_stage<BR, NW, true>(a.hc + r0 / LK_PANEL * mpan + (long)k0 * LK_PANEL, mpan, (a.Hp - r0) / LK_PANEL, rs, wave,
                             lane_off);
    } else {
      const uint16_t* d = a.d + kp * mpan + (long)l0 * LK_PANEL;
#pragma unroll
      for (int t = 0; t < LT; ++t) lk_stage<BL, NW, false>(d + t * a.lo, 0, 0, ls + t * BL * BK, wave, lane_off);
      lk_stage<BR, NW, true>(a.ec + r0 / LK_PANEL * vpan + (long)(a.v0 + k0) * LK_PANEL, vpan, (a.Hp - r0) / LK_PANEL,
                             rs, wave, lane_off);
    }
  };
  f32x16 acc[FR][FL];
#pragma unroll
  for (int i = 0; i < FR; ++i)
#pragma unroll
    for (int j = 0; j < FL; ++j) acc[i][j] = (f32x16)0.f;
#pragma unroll
  for (int i = 0; i < ST - 1; ++i)
    if (kb + i * BK < ke) stage(kb + i * BK, i);
  int buf = 0;
  for (int k0 = kb; k0 < ke; k0 += BK) {
    // this wave's copies for this step have landed (those of the ST - 2 steps behind may be
    // under way) and its reads of the buffer before are done; then every wave's
    if (k0 + (ST - 2) * BK < ke)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(NI * (ST - 2)) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (k0 + (ST - 1) * BK < ke) stage(k0 + (ST - 1) * BK, buf == 0 ? ST - 1 : buf - 1);
    const uint16_t *ls = sm + buf * STAGE, *rs = ls + LT * BL * BK;
    buf = buf + 1 == ST ? 0 : buf + 1;
    // the operands of the next 16 k-values are read while these are multiplied
    u16x8 lf[2][LT][FL], rf[2][FR];
    auto read = [&](int s) {
#pragma unroll
      for (int t = 0; t < LT; ++t)
#pragma unroll
        for (int j = 0; j < FL; ++j)
          lf[s & 1][t][j] = LCOL ? lk_col(ls + t * BL * BK + (wl * FL + j) * 32 * LK_PANEL, s, lane)
                                 : lk_row(ls + t * BL * BK, wl * TL + 32 * j + (lane & 31), s, h);
#pragma unroll
      for (int i = 0; i < FR; ++i)
        rf[s & 1][i] = RCOL ? lk_col(rs + (wr * FR + i) * 32 * LK_PANEL, s, lane)
                            : lk_row(rs, wr * TR + 32 * i + (lane & 31), s, h);
    };
    read(0);
#pragma unroll
    for (int s = 0; s < BK / 16; ++s) {
      if (s + 1 < BK / 16) read(s + 1);
#pragma unroll
      for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int j = 0; j < FL; ++j)
#pragma unroll
          for (int t = 0; t < LT; ++t) acc[i][j] = lk_mma<BF>(rf[s & 1][i], lf[s & 1][t][j], acc[i][j]);
    }
  }
  // register r of acc[i][j]: register-side index r0 + wr TR + 32 i + 8 (r >> 2) + 4 h + (r & 3)
  const int ln = l0 + wl * TL + (lane & 31), rn = r0 + wr * TR + 4 * h;
  if constexpr (MODE == 0) {
    float2* red = reinterpret_cast<float2*>(sm);  // [WR][BL]
    __syncthreads();
    const int vend = a.V - a.v0;
#pragma unroll
    for (int j = 0; j < FL; ++j) {
      // the label's logit, where this lane holds it, goes out and takes no part in the sum
      const int n = ln + 32 * j, y = (n < cnt ? a.lab[n] : -1) - a.v0 - rn;
      if (__any(y >= 0 && y < TR)) {
        float zy = 0.f;
#pragma unroll
        for (int i = 0; i < FR; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const bool it = y == 32 * i + 8 * (r >> 2) + (r & 3);
            zy = it ? acc[i][j][r] : zy;
            acc[i][j][r] = it ? -INFINITY : acc[i][j][r];
          }
        if (y >= 0 && y < TR && !(y & 4)) a.rl[n] = zy;
      }
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (r0 + BR > vend && rn + 32 * i + 8 * (r >> 2) + (r & 3) >= vend) acc[i][j][r] = -INFINITY;
          top = fmaxf(top, acc[i][j][r]);
        }
      top = lk_max_halves(top);
      // z - top first: a loss near 0 is a difference of large logits
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          sum += BL == 64 ? lk_exp_fine(acc[i][j][r] - ref) : lk_exp(acc[i][j][r] - ref);
      sum = lk_sum_halves(sum);
      if (h == 0) red[wr * BL + wl * TL + 32 * j + lane] = make_float2(top, sum);
    }
    __syncthreads();
    for (int n = threadIdx.x; n < BL; n += NW * 64) {
      float2 x = red[n];
#pragma unroll
      for (int w = 1; w < WR; ++w) {
        const float2 y = red[w * BL + n];
        const float m = fmaxf(x.x, y.x), ref = m == -INFINITY ? 0.f : m;
        x = make_float2(m, x.y * lk_exp_fine(x.x - ref) + y.y * lk_exp_fine(y.x - ref));
      }
      a.part[(size_t)(r0 / BR) * a.Mp + l0 + n] = x;
    }
  } else if constexpr (MODE == 1) {
    const int vend = a.V - a.v0;
#pragma unroll
    for (int j = 0; j < FL; ++j) {
      const int n = ln + 32 * j;
      const float top = n < cnt ? a.top[n] : INFINITY, ls2 = n < cnt ? a.ls2[n] : 0.f;
      const float w = (a.w != nullptr && n < cnt ? a.w[n] : 1.f) * (BF ? 1.f : LK_FP16);
      const int y = (n < cnt ? a.lab[n] : -1) - a.v0 - rn;  // its place in this lane's registers
      const bool here = y >= 0 && y < TR;
      uint16_t* row = a.d + (r0 + wr * TR) / LK_PANEL * mpan + (size_t)n * LK_PANEL;
#pragma unroll
      for (int i = 0; i < FR; ++i) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          acc[i][j][r] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][r] - top, LK_LOG2E, -ls2));
        if (__any(here)) {
          const float miss = here ? a.rl[n] : 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (y == 32 * i + 8 * (r >> 2) + (r & 3)) acc[i][j][r] = -miss;
        }
        if (r0 + BR > vend) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (rn + 32 * i + 8 * (r >> 2) + (r & 3) >= vend) acc[i][j][r] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          float4 x = lk_four(acc[i][j], e, w), y = lk_four(acc[i][j], e + 1, w);
          uint16_t* at = row + i * mpan + 8 * (e + h);
          *reinterpret_cast<uint4*>(at) = lk_trade<BF>(x, y);
          if constexpr (FINE) {
            x = make_float4(lk_rest<BF>(x.x), lk_rest<BF>(x.y), lk_rest<BF>(x.z), lk_rest<BF>(x.w));
            y = make_float4(lk_rest<BF>(y.x), lk_rest<BF>(y.y), lk_rest<BF>(y.z), lk_rest<BF>(y.w));
            *reinterpret_cast<uint4*>(at + a.lo) = lk_trade<BF>(x, y);
          }
        }
      }
    }
  } else {
    const float f = MODE == 3 ? 1.f
                              : (a.mode == 2 ? a.gmax[0] : a.mode == 1 ? a.g[0] : a.g[0] / (float)max(cnt, 1)) *
                                    (BF ? 1.f : 1.f / LK_FP16);
#pragma unroll
    for (int j = 0; j < FL; ++j) {
      const int n = ln + 32 * j;
#pragma unroll
      for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = rn + 32 * i + 8 * e;
          if constexpr (MODE == 2) {
            if (e & 1) continue;
            const uint4 x = lk_trade<BF>(lk_four(acc[i][j], e, f), lk_four(acc[i][j], e + 1, f));
            const int c8 = c + 4 * h;  // group e, in half 1 group e + 1
            if (a.v0 + n < a.V && c8 < a.H)
              *reinterpret_cast<uint4*>(a.dtable + (size_t)(a.v0 + n) * a.H + c8) = x;
          } else if (c < a.H) {
            float4* p = reinterpret_cast<float4*>(a.share + ((size_t)z * nl * BL + n) * a.Hp + c);
            float4 x = make_float4(acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]);
            if (!a.first) {
              const float4 y = *p;
              x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
            }
            *p = x;
          }
        }
    }
  }
}

template <bool BF, int MODE, int BL, int BR, int WL, int WR, int ST, bool FINE>
__global__ void __launch_bounds__(WL * WR * 64, FINE ? 2 : 3) loss_logits_kernel(LossArgs a) {
  typedef LkTile<BF, MODE, BL, BR, WL, WR, ST, FINE> Tile;
  __shared__ __attribute__((aligned(16))) uint16_t sm[ST * Tile::STAGE];
  Tile::run(a, blockIdx.x, sm);
}

// dE's tiles (the first a.t2 blocks), then dh's: one launch, because neither fills the card
// by itself (16384 ids and 576 columns: 384 tiles for 768 places) and dh's, split as finely
// as one likes, fill the places that dE's leave.
template <bool BF, int BL, int BR, int WL, int WR, int ST, bool FINE>
__global__ void __launch_bounds__(WL * WR * 64, 3) loss_grad_kernel(LossArgs a) {
  typedef LkTile<BF, 2, BL, BR, WL, WR, ST, FINE> Table;
  typedef LkTile<BF, 3, BL, BR, WL, WR, ST, FINE> Hidden;
  __shared__ __attribute__((aligned(16))) uint16_t sm[ST * Table::STAGE];
  if ((int)blockIdx.x < a.t2)
    Table::run(a, blockIdx.x, sm);
  else
    Hidden::run(a, blockIdx.x - a.t2, sm);
}

// ---- joins -----------------------------------------------------------------------------
// The loss from the join's sums (of block b over its own rows' first tile in part, 32 b), in
// their order; mean: no labelled row gives 0 / 0, as the mean of nothing.  One block of 256.
__device__ __forceinline__ void lk_total(const LossArgs& a, int blocks, float* red) {
  const float* sums = reinterpret_cast<const float*>(a.part);
  float s = 0.f;
  for (int b0 = threadIdx.x; b0 < blocks; b0 += 1024) {
    float x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[k] = 0.f;
      if (b0 + 256 * k < blocks)
        x[k] = __hip_atomic_load(sums + 32 * (size_t)(b0 + 256 * k), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    s += (x[0] + x[1]) + (x[2] + x[3]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = (red[0] + red[1]) + (red[2] + red[3]);
    a.loss[0] = a.mode == 0 ? s / (float)a.cnt[0] : s;
  }
}

__device__ __forceinline__ int lk_join_blocks(int cnt) { return max(1, (cnt + 15) / 16); }

__global__ void __launch_bounds__(256) loss_sum_kernel(LossArgs a) {
  __shared__ float red[4];
  lk_total(a, lk_join_blocks(a.cnt[0]), red);
}

// 16 rows a block: L from the tiles' (maximum, sum) and the label's logit, the loss.  TOTAL: the
// block that ends last, whichever it is, takes the total too.  That saves a small call a
// launch (5.0 us for 4.2 + 3.5), but every block's sum has to reach the others' caches: 300
// blocks take 14.1 us with it for 4.4 + 4.3.
template <bool TOTAL>
__global__ void __launch_bounds__(256) loss_join_kernel(LossArgs a, int tiles) {
  __shared__ float2 red[16][16];
  __shared__ bool last;
  const int m0 = blockIdx.x * 16, cnt = a.cnt[0], blocks = lk_join_blocks(cnt);
  if (blockIdx.x == gridDim.x - 1) {  // a block more: the backward's splits
    if (threadIdx.x >= 64) return;
    const int splits = lk_choose(a, cnt, threadIdx.x);
    if (threadIdx.x == 0) a.cnt[2] = splits;
    return;
  }
  if ((int)blockIdx.x >= blocks) return;
  const int r = threadIdx.x & 15, g = threadIdx.x >> 4;  // row, share of the tiles
  float2 x = make_float2(-INFINITY, 0.f);
  for (int t = g; t < tiles; t += 64) {
    float2 y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      y[k] = make_float2(-INFINITY, 0.f);
      if (t + 16 * k < tiles) y[k] = a.part[(size_t)(t + 16 * k) * a.Mp + m0 + r];
    }
    float top = x.x;
#pragma unroll
    for (int k = 0; k < 4; ++k) top = fmaxf(top, y[k].x);
    const float ref = top == -INFINITY ? 0.f : top;
    float s = x.y * lk_exp_fine(x.x - ref);
#pragma unroll
    for (int k = 0; k < 4; ++k) s += y[k].y * lk_exp_fine(y[k].x - ref);
    x = make_float2(top, s);
  }
  red[g][r] = x;
  __syncthreads();
  const int m = m0 + threadIdx.x;
  float loss = 0.f;
  if (threadIdx.x < 16 && m < cnt) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 16; ++w) top = fmaxf(top, red[w][threadIdx.x].x);
    const float ref = top == -INFINITY ? 0.f : top;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += red[w][threadIdx.x].y * lk_exp_fine(red[w][threadIdx.x].x - ref);
    // the label joins: over the larger of both logits, e is its exponential, s the others' sum
    // (the library's logarithms: the hardware's is off by more than an ulp near 1)
    const float zy = a.lab[m] == -2 ? __builtin_nanf("") : a.rl[m];
    const bool first = !(top > zy);
    const float over = first ? zy : top, e = lk_exp_fine(zy - over);
    if (first) s *= lk_exp_fine(top - over);
    const float ls = first ? log1pf(s) : logf(s + e);
    loss = (over - zy) + ls;
    a.top[m] = over;
    a.ls2[m] = ls * LK_LOG2E;
    a.rl[m] = s / (s + e);
    if (a.mode == 2) a.loss[a.rows[m]] = loss;
  }
  if (a.mode == 2) return;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) loss += __shfl_xor(loss, o, 64);
  if (threadIdx.x == 0) reinterpret_cast<float*>(a.part)[2 * (size_t)m0] = loss;
  if constexpr (TOTAL) {
    if (threadIdx.x == 0) {
      __threadfence();
      last = atomicAdd(&a.cnt[1], 1) == blocks - 1;
      __threadfence();
    }
    __syncthreads();
    if (last) lk_total(a, blocks, reinterpret_cast<float*>(red));
  }
}

// none: gmax = the largest finite |g|, w = g / gmax (in [-1, 1])
__global__ void __launch_bounds__(1024) loss_weights_kernel(LossArgs a, float* gmax) {
  __shared__ float red[16];
  const int cnt = a.cnt[0], lane = threadIdx.x & 63;
  float t = 0.f;
  for (int m = threadIdx.x; m < cnt; m += 1024) {
    const float x = fabsf(a.g[a.rows[m]]);
    if (x < INFINITY) t = fmaxf(t, x);  // (an infinite or NaN g is its own row's matter)
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor(t, o, 64));
  if (lane == 0) red[threadIdx.x >> 6] = t;
  __syncthreads();
  for (int w = 0; w < 16; ++w) t = fmaxf(t, red[w]);
  for (int m = threadIdx.x; m < cnt; m += 1024) {
    const float g = a.g[a.rows[m]];
    a.w[m] = t > 0.f ? g / t : g;
  }
  if (threadIdx.x == 0) gmax[0] = t;
}

// dh: the shares' sum, in order, for labelled rows; zeros for the others.  4 columns a thread.
template <bool BF>
__global__ void __launch_bounds__(256) loss_dh_kernel(LossArgs a) {
  const int nch = a.H / 4;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)a.N * nch) return;
  const int row = (int)(i / nch), c = (int)(i - (long)row * nch) * 4, m = a.pos[row];
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (m >= 0) {
    const int rows = (a.cnt[0] + a.bl - 1) / a.bl * a.bl;
    const int splits = a.cnt[2];
    for (int z0 = 0; z0 < splits; z0 += 8) {
      float4 x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        x[k] = *reinterpret_cast<const float4*>(a.share + ((size_t)min(z0 + k, splits - 1) * rows + m) * a.Hp + c);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (z0 + k < splits) s.x += x[k].x, s.y += x[k].y, s.z += x[k].z, s.w += x[k].w;
    }
    const float f = (a.mode == 2 ? a.gmax[0] : a.mode == 1 ? a.g[0] : a.g[0] / (float)a.cnt[0]) *
                    (BF ? 1.f : 1.f / LK_FP16);
    s.x *= f, s.y *= f, s.z *= f, s.w *= f;
  }
  *reinterpret_cast<uint2*>(a.dh + (size_t)row * a.H + c) = lk_pack4<BF>(s.x, s.y, s.z, s.w);
}

// ---- plan ------------------------------------------------------------------------------
// Big tiles, 128 x 256 for the logits and 128 x 192 for the gradients; a few hundred rows, or
// few ids, leave most of the card without one (fewer than 256 squares of 256), so there 64 x 64
// tiles run instead.  All have 4 waves.
//
// The gradients' tile is 192 of H's columns wide whatever H is.  At 576 and 960 columns that is
// whole tiles (8192 rows of 49152 ids: 1080 and 1928 us, where 128 wide takes 1440 and 2275); at
// 128, 256 and 384 a third, a third and nothing of the products is padding (775, 862 and 852 us
// for 715, 735 and 818; 4773 rows of 8192 ids 122, 123 and 125 us for 104, 104 and 113).
struct LossPlan {
  int Mp, Hp, small, fine, vtiles, piece, splits, want, most;
};

// Rows up to which d is two operands.  Its rounding adds to the gradients' own (sqrt 2 of it
// over many rows); of few rows, each with its label's term, one rounding shows as it is: 1.5 to
// 2.2 of the gradient's own for a third of the calls of one row, a tenth of those of 5 and a
// thirtieth of those of 64, none of 120 from 128 rows on.  The gradients of 61 rows, 8192 x 256,
// take 8.1 us for 7.6, a whole call of 128 rows, 49152 x 576, 139 us for 125.
constexpr int LK_FINE = 128;

constexpr int LK_BL = 128;  // lane side of the gradients' big tiles
constexpr long LK_PIECE = 1L << 27;  // elements of d (256 MB: what the last-level cache holds)

LossPlan lk_plan(int N, int V, int H) {
  LossPlan p;
  p.Mp = (N + LK_PAD - 1) / LK_PAD * LK_PAD;
  p.Hp = (H + LK_K - 1) / LK_K * LK_K;
  const long vp = ((long)V + LK_PAD - 1) / LK_PAD * LK_PAD;
  p.fine = N <= LK_FINE;
  p.small = (p.Mp / 256) * (vp / 256) < 256;
  p.vtiles = (int)(vp / (p.small ? 64 : 256));
  long piece = LK_PIECE / (1 + p.fine) / p.Mp / LK_PAD * LK_PAD;
  if (piece < 4 * LK_PAD) piece = 4 * LK_PAD;
  p.piece = (int)(piece < vp ? piece : vp);
  // dh: blocks over the card, each with at least 4 steps of k
  const int bl = p.small ? 64 : LK_BL, br = p.small ? 64 : 192;
  const int tiles = p.Mp / bl * ((H + br - 1) / br);
  p.want = 768;
  p.most = p.piece / (4 * LK_K) < 64 ? p.piece / (4 * LK_K) : 64;
  const int s = (p.want + tiles - 1) / tiles;
  p.splits = s < p.most ? s : p.most;
  return p;
}

template <bool BF, int MODE>
void lk_logits(const LossArgs& a, const LossPlan& p, hipStream_t st) {
  const dim3 grid = p.small ? a.Mp / 64 * (a.vn / 64) : a.Mp / 128 * (a.vn / 256);
  constexpr bool FINE = MODE == 1;
  if (p.small && p.fine && FINE)
    loss_logits_kernel<BF, MODE, 64, 64, 2, 2, 4, FINE><<<grid, dim3(256), 0, st>>>(a);
  else if (p.small)
    loss_logits_kernel<BF, MODE, 64, 64, 2, 2, 4, false><<<grid, dim3(256), 0, st>>>(a);
  else if (p.fine && FINE)
    loss_logits_kernel<BF, MODE, 128, 256, 1, 4, 2, FINE><<<grid, dim3(256), 0, st>>>(a);
  else
    loss_logits_kernel<BF, MODE, 128, 256, 1, 4, 2, false><<<grid, dim3(256), 0, st>>>(a);
}

// dh has as many blocks as any count of rows may want (its tiles' rows x splits are at most the
// workspace's shares).
template <bool BF>
void lk_grads(LossArgs a, const LossPlan& p, hipStream_t st) {
  a.t2 = a.dtable != nullptr ? (a.vn / a.bl * a.nr + 7) / 8 * 8 : 0;
  long t3 = 0;
  if (a.dh != nullptr) {
    t3 = (long)a.Mp / a.bl * a.nr * a.splits;
  }
  if (a.t2 + t3 == 0) return;
  const dim3 grid((unsigned)(a.t2 + t3));
  if (p.small && p.fine)
    loss_grad_kernel<BF, 64, 64, 2, 2, 4, true><<<grid, dim3(256), 0, st>>>(a);
  else if (p.fine)
    loss_grad_kernel<BF, LK_BL, 192, 4, 1, 2, true><<<grid, dim3(256), 0, st>>>(a);
  else if (p.small)
    loss_grad_kernel<BF, 64, 64, 2, 2, 4, false><<<grid, dim3(256), 0, st>>>(a);
  else
    loss_grad_kernel<BF, LK_BL, 192, 4, 1, 2, false><<<grid, dim3(256), 0, st>>>(a);
}

template <bool BF>
void lk_forward(LossArgs a, const LossPlan& p, hipStream_t st) {
  const long nch = p.Hp / 8, hidden = (p.Mp * nch + 1023) / 1024, table = (a.Vp * nch + 1023) / 1024;
  if (a.N <= LK_SMALL) {
    loss_rows_kernel<true><<<dim3((unsigned)(hidden + table)), dim3(1024), 0, st>>>(a, (int)hidden);
  } else {
    loss_rows_kernel<false><<<dim3((unsigned)(1 + table)), dim3(1024), 0, st>>>(a, 1);
    loss_hidden_kernel<<<dim3((unsigned)((p.Mp * nch + 255) / 256)), dim3(256), 0, st>>>(a);
  }
  a.v0 = 0;
  a.vn = p.vtiles * (p.small ? 64 : 256);
  lk_logits<BF, 0>(a, p, st);
  a.vn = a.vn < p.piece ? a.vn : p.piece;  // (for the choice of the backward's splits)
  if (a.N <= LK_SMALL && a.mode != 2) {
    loss_join_kernel<true><<<dim3(p.Mp / 16 + 1), dim3(256), 0, st>>>(a, p.vtiles);
    return;
  }
  loss_join_kernel<false><<<dim3(p.Mp / 16 + 1), dim3(256), 0, st>>>(a, p.vtiles);
  if (a.mode != 2) loss_sum_kernel<<<dim3(1), dim3(256), 0, st>>>(a);
}

template <bool BF>
void lk_backward(LossArgs a, const LossPlan& p, hipStream_t st) {
  if (a.mode == 2) loss_weights_kernel<<<dim3(1), dim3(1024), 0, st>>>(a, const_cast<float*>(a.gmax));
  const int vp = p.vtiles * (p.small ? 64 : 256);
  for (int v0 = 0; v0 < vp; v0 += p.piece) {
    a.v0 = v0;
    a.vn = vp - v0 < p.piece ? vp - v0 : p.piece;
    a.first = v0 == 0;
    lk_logits<BF, 1>(a, p, st);
    lk_grads<BF>(a, p, st);
  }
  if (a.dh != nullptr)
    loss_dh_kernel<BF><<<dim3((unsigned)(((long)a.N * (a.H / 4) + 255) / 256)), dim3(256), 0, st>>>(a);
}

bool lk_bad(int N, int V, int H, int mode) {
  return N <= 0 || N > (1 << 24) || V <= 0 || V > (1 << 24) || H <= 0 || H % 8 != 0 || H > (1 << 14) || mode < 0 ||
         // a grid holds 2^32 threads: 256 a tile of 128 x 256, one for 16 bytes of hc, ec or dh
         mode > 2 || ((long)N + 255) / 128 * (((long)V + 255) / 256) >= 1 << 24 || ((long)N + V + 512) * (H + 63) >= 1L << 34;
}

// state: ints cnt[64], rows[Mp], lab[Mp]; floats top[Mp], ls2[Mp], rl[Mp]; ints pos[N]
void lk_state(LossArgs& a, const LossPlan& p, void* state) {
  int* s = (int*)state;
  a.cnt = s;
  a.rows = s + 64;
  a.lab = a.rows + p.Mp;
  a.top = (float*)(a.lab + p.Mp);
  a.ls2 = a.top + p.Mp;
  a.rl = a.ls2 + p.Mp;
  a.pos = (int*)(a.rl + p.Mp);
  a.Mp = p.Mp, a.Hp = p.Hp, a.Vp = p.vtiles * (p.small ? 64 : 256);
  a.splits = p.splits, a.want = p.want, a.most = p.most;
  a.lo = p.fine ? (long)p.Mp * p.piece : 0;
  a.bl = p.small ? 64 : LK_BL, a.nr = p.small ? (a.H + 63) / 64 : (a.H + 191) / 192;
}

}  // namespace

extern "C" {

// out[0..5]: rows and columns of hc, rows of ec (as many columns); state and the forward's and
// the backward's workspace, in units of 256 bytes
int sg_loss_plan(int N, int V, int H, void* out) {
  if (lk_bad(N, V, H, 0)) return 1;
  const LossPlan p = lk_plan(N, V, H);
  int* o = (int*)out;
  o[0] = p.Mp;
  o[1] = p.Hp;
  o[2] = p.vtiles * (p.small ? 64 : 256);
  o[3] = (64 + 5 * p.Mp + N + 63) / 64;
  o[4] = (int)((2L * p.vtiles * p.Mp + 63) / 64);
  o[5] = (int)((64 + p.Mp + (long)p.Mp * p.piece / 2 * (1 + p.fine) + (long)p.splits * p.Mp * p.Hp + 63) / 64);
  return 0;
}

// mode: 0 mean, 1 sum (loss [1]), 2 none (loss [N])
int sg_loss_fwd(const void* h, const void* table, const void* labels, int is64, int ignore, void* hc, void* ec,
                void* state, void* ws, void* loss, int N, int V, int H, int mode, int fp16, hipStream_t st) {
  if (lk_bad(N, V, H, mode)) return 1;
  const LossPlan p = lk_plan(N, V, H);
  LossArgs a = {};
  a.h = (const uint16_t*)h, a.table = (const uint16_t*)table, a.labels = labels, a.is64 = is64, a.ignore = ignore;
  a.hc = (uint16_t*)hc, a.ec = (uint16_t*)ec, a.loss = (float*)loss, a.part = (float2*)ws;
  a.N = N, a.V = V, a.H = H, a.mode = mode;
  lk_state(a, p, state);
  fp16 ? lk_forward<false>(a, p, st) : lk_forward<true>(a, p, st);
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

// g: the gradient of loss ([1], none: [N]); dh or dtable may be null (not wanted)
int sg_loss_bwd(const void* hc, const void* ec, void* state, const void* g, void* ws, void* dh, void* dtable, int N,
                int V, int H, int mode, int fp16, hipStream_t st) {
  if (lk_bad(N, V, H, mode)) return 1;
  const LossPlan p = lk_plan(N, V, H);
  LossArgs a = {};
  a.hc = (uint16_t*)const_cast<void*>(hc), a.ec = (uint16_t*)const_cast<void*>(ec), a.g = (const float*)g;
  a.dh = (uint16_t*)dh, a.dtable = (uint16_t*)dtable;
  a.N = N, a.V = V, a.H = H, a.mode = mode;
  lk_state(a, p, state);
  float* w = (float*)ws;
  a.gmax = w;
  a.w = mode == 2 ? w + 64 : nullptr;
  a.d = (uint16_t*)(w + 64 + p.Mp);
  a.share = w + 64 + p.Mp + (size_t)p.Mp * p.piece / 2 * (1 + p.fine);
  fp16 ? lk_backward<false>(a, p, st) : lk_backward<true>(a, p, st);
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

}  // extern "C"
