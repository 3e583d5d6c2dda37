#pragma once
// kvq_paged_cols.cuh — attention of a few query rows per sequence over the
// pages: single-token decode, drafted tokens, and ragged steps of few rows a
// sequence on average.
//
// Mathematics.  A unit is one (sequence, kv head) and up to 8 * NT of its
// query columns (column c is token c / rep, head c % rep of the group), so a
// K or V byte serves every query head that shares it.  With codes c, scales
// s and biases z of a group:
//   q . (s c + z) = s (q . c) + z sum(q);   sum_j p_j (s_j c_j + z_j) =
//   sum_j (p_j s_j) c_j + sum_j p_j z_j,
// so codes enter the tensor cores as integers and nothing of K is rounded: a
// code is the fp16 subnormal c 2^-24 (its bits in the low mantissa bits; 4-bit
// codes of odd nibbles are taken unshifted as 16 c and the 16 is divided out
// of q or of the output).  q is scaled by the power of two that brings its
// largest element into [2^13, 2^14), so bf16 queries between 2^-87 and 2^113 and
// the divided ones keep all their bits in fp16.  p_j s_j is rounded to fp16 (an
// error of at most 2^-11 of it, times c); softmax statistics and all sums are
// f32.  For fp16 outputs that error is centred: with x_j the rounded p_j s_j
// and h the middle code,
//   sum_j x_j c_j - h sum_j x_j + sum_j p_j (z_j + h s_j),
// so it multiplies c - h (half the range, 0 in the middle) instead of c; the
// sum of x_j comes from one more MMA with ones.
//
// Keeping p_j s_j in fp16's normal range, whatever the scales: the softmax
// reference m of a column is a running maximum, over the keys it sees, of logit +
// floor(log2(largest |s| of the key's row)) - kRaise rather than of the logit, so
// p_j s_j reaches 2^15 and is normal down to 2^-24 of the terms that matter; and a
// group whose scales lie below the others' is brought up to them by a power of
// two of its own, in p_j s_j and its sums, divided out at the end.  Both are worked
// out when a term passes the reference by more than 2^kLazy (always on the first
// keys), from the keys at hand: a key that a column does not see has no say in
// its reference, however large or not finite its scale.  Biases count by 2^-64 of
// their size, which keeps sum p z in f32's range next to tiny scales.  The powers
// are the same for all columns and at most 2^20 (kMaxUp): a group 2^39 below the
// reference's, or left 2^20 behind by the powers of columns that see more, still
// has its largest term at 2^-5, 2^20 above fp16's last bit.  fp16 scales span 2^37;
// bf16 ones of groups of neighbouring keys may lie 2^39 apart.  Measured against a
// reference by the lane's rows as a whole and without powers: 0 to 3 % of the
// time of the forms of up to 8 columns, 1 to 12 % of those of 16.
//
// Bound: HBM.  4 bits, D 128, group 64: 144 B per key and kv head; at the
// measured copy rate an SM gets 23 B per clock, one 16-key tile per 100
// clocks, in which its four schedulers can issue 400 warp instructions.  With
// up to 4 columns (ST = 2) half of the MMA's 8 columns would idle: two tiles
// go through side by side, tile i in columns 4 i.. of the same registers, so
// the softmax, scale and bias work of two tiles costs that of one.
//
// Work split: the 16-key tiles of all units, laid end to end, are cut into one
// equal run per warp (one CTA per SM), whatever the lengths in the batch.  A
// warp streams its run through a ring of its own (one bulk copy per tile, no
// barrier shared with another warp).  A unit inside one run is finished by its
// warp; the pieces of a cut unit meet in shared memory when its warps share a
// CTA, and otherwise in the merge kernel, always in order of the keys.
//
// Measured (B200): 64 ragged sequences of 1,024 to 32,768 keys, 8 kv heads, D
// 128, 4 bits (1,050 MB): 197 us, 5.3 TB/s; 8 sequences of 8,193 keys: 26.7 us;
// one of 2,048 keys in 8 bits: 11.5 us, all of it latency.
#include <mutex>
#include <set>

#include "kvq_attn_impl.cuh"
#include "kvq_paged.cuh"

namespace kvq {
namespace paged {

using attn::ex2;
using attn::kNeg;
using attn::mma16816;
using attn::movmatrix_t;
using attn::pack_h2;
using attn::prmt;

constexpr float kLazy = 4.0f;       // m moves when a term would exceed 2^4
constexpr float kMinScale = 8.673617379884035e-19f;  // 2^-60: the smallest that a reference goes by
constexpr float kRaise = 10.0f;     // terms are at most 2^(kLazy + 1 + kRaise) = 2^15
constexpr int kMaxUp = 20;          // most that a group is brought up, log2 (half of what fp16 scales span)
constexpr float kBiasShare = 5.421010862427522e-20f;  // 2^-64: p z stays in f32's range too
constexpr int kPlanMax = 512;       // sequences and column blocks whose plan fits in shared memory

// ------------------------------------------------------------- the plan --

// Column blocks of every sequence, and the tiles of every column block.
struct Plan {
  const int* gpre;           // [B + 1] first block of each sequence (with cu)
  const long long* tpre;     // [NG + 1] tiles of one kv head before each block
  int NG;
};

// One column block: keys it sees, as a list of 16-key tiles.
struct Block {
  int b, row0, col0, cols;   // first token row of the sequence, columns col0..col0 + cols
  int p0;                    // position of the sequence's first row
  int pmin, pmax;            // query positions of the block's columns
  int nsink, lo, nt;         // tiles [0, nsink) and [lo, lo + nt - nsink)
};

__device__ __forceinline__ int tile_of(const Block& k, int i) {
  return i < k.nsink ? i : k.lo + i - k.nsink;
}

// Rows of sequence b, checked: n = 0 when cu_rows or the length make no sense.
__device__ __forceinline__ void checked_rows(const View& v, int b, int& row0, int& n, int& len,
                                             bool report) {
  seq_rows(v, b, row0, n, len);
  if (n < 0 || row0 < 0 || (int64_t)row0 + n > v.rows) {
    if (report) raise(v);
    n = 0;
  }
  if (len < 0 || len > ((int64_t)v.max_pages << v.page_shift)) {
    if (report) raise(v);
    len = 0;
  }
}

// KS: log2 of the keys in a list entry (16 here, 128 in the chunk kernel).
template <int KS>
__device__ __forceinline__ void block_keys(Block& k, const AttnArgs& a, int len, int n) {
  k.p0 = len - n;
  k.pmin = k.p0 + k.col0 / a.rep;
  k.pmax = k.p0 + (k.col0 + k.cols - 1) / a.rep;
  const int hi = len == 0 || k.pmax < 0 ? 0 : (k.pmax >> KS) + 1;
  k.nsink = k.lo = 0;
  if (a.window > 0) {
    const int first = max(0, k.pmin - a.window + 1);
    k.lo = min(first >> KS, hi);
    k.nsink = (int)(((int64_t)min(a.sinks, first) + (1 << KS) - 1) >> KS);
    if (k.nsink >= k.lo) k.nsink = k.lo = 0;
  }
  k.nt = k.nsink + hi - k.lo;
}

template <int NC, int KS = 4>
__device__ __forceinline__ Block get_block(const AttnArgs& a, const Plan& P, int gi) {
  Block k;
  int cb;
  if (a.v.cu) {
    int x = 0, y = a.v.B;  // gpre[x] <= gi < gpre[y]
    while (y - x > 1) {
      const int m = (x + y) >> 1;
      if (P.gpre[m] <= gi) x = m;
      else y = m;
    }
    k.b = x;
    cb = gi - P.gpre[x];
  } else {
    const int per = (a.rep + NC - 1) / NC;
    k.b = gi / per;
    cb = gi - k.b * per;
  }
  int n, len;
  checked_rows(a.v, k.b, k.row0, n, len, false);
  k.col0 = cb * NC;
  k.cols = max(0, min(NC, n * a.rep - k.col0));
  block_keys<KS>(k, a, len, n);
  return k;
}

// Exclusive scan over the block's threads; returns the total too.  `tmp` holds
// 33 values.  Every thread calls it.
__device__ __forceinline__ long long block_scan(long long x, long long* tmp, long long& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  long long s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  __syncthreads();
  if (lane == 31) tmp[w] = s;
  __syncthreads();
  if (w == 0) {
    long long y = lane < nw ? tmp[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    tmp[lane] = y;
  }
  __syncthreads();
  total = tmp[nw - 1];
  return s - x + (w ? tmp[w - 1] : 0);
}

// Fill gpre / tpre (room for B + 1 and max_blocks + 1) and return the number of
// column blocks.  Blocks beyond max_blocks (overlapping cu_rows) are dropped.
template <int NC, int KS = 4>
__device__ __forceinline__ int build_plan(const AttnArgs& a, int* gpre, long long* tpre,
                                          int max_blocks, long long* tmp, bool report) {
  const View& v = a.v;
  int NG;
  long long total;
  if (v.cu) {
    long long base = 0;
    for (int b0 = 0; b0 < v.B; b0 += blockDim.x) {
      const int b = b0 + threadIdx.x;
      int row0, n = 0, len;
      if (b < v.B) checked_rows(v, b, row0, n, len, report);
      const long long e = base + block_scan(((long long)n * a.rep + NC - 1) / NC, tmp, total);
      if (b < v.B) gpre[b] = (int)min(e, (long long)max_blocks);
      base += total;
    }
    if (base > max_blocks && threadIdx.x == 0 && report) raise(v);
    NG = (int)min(base, (long long)max_blocks);
    if (threadIdx.x == 0) gpre[v.B] = NG;
  } else {
    NG = v.B * ((a.rep + NC - 1) / NC);
    if (report)
      for (int b = threadIdx.x; b < v.B; b += blockDim.x) {
        int row0, n, len;
        checked_rows(v, b, row0, n, len, true);
      }
  }
  __syncthreads();
  long long base = 0;
  const Plan P{gpre, tpre, NG};
  for (int g0 = 0; g0 < NG; g0 += blockDim.x) {
    const int gi = g0 + threadIdx.x;
    const int nt = gi < NG ? get_block<NC, KS>(a, P, gi).nt : 0;
    const long long e = base + block_scan(nt, tmp, total);
    if (gi < NG) tpre[gi] = e;
    base += total;
  }
  if (threadIdx.x == 0) tpre[NG] = base;
  __syncthreads();
  return NG;
}

// ------------------------------------------------------------- geometry --

// NT: column tiles of 8; ST: key streams that share one (NT = 1 when ST = 2).
template <int BITS, int D, int GS, int NT, int ST>
struct Cfg {
  using G = attn::Geo<BITS, D, GS>;
  static constexpr int NC = 8 * NT / ST;            // columns of a block
  static constexpr int CRB = D * BITS / 8;
  static constexpr int PRB = D / GS * 4;
  static constexpr int HALF = kTileRows * (CRB + PRB);
  static constexpr int TILE = 2 * HALF;
  static constexpr int TPS = ST == 2 || TILE <= 2560 ? 2 : 1;  // tiles per ring stage
  static constexpr int STAGE = TPS * TILE;
  static constexpr int FR = D / 16 * NT;            // float4 fragments per lane of an output
  static constexpr int PIECE = 16 * NT + FR * 128;  // floats of a piece: m, l, O fragments
  // ring depth: a few KB in flight per warp; two stages of the large tiles
  static constexpr int STAGES = STAGE <= 5120 ? 3 : (STAGE <= 9216 && TPS == 1 ? 3 : 2);
  // warps: what the registers allow (168 or 255 a thread), then shared memory.
  // Four groups in 4 bits at one column a lane spill at 168 (8 columns, 32
  // sequences of 8,000 to 16,000 keys: 118 us with 8 warps, 135 with 12; in 8
  // bits 149 and 137)
  static constexpr int W_REG = D * NT > 128 || (BITS == 4 && D / GS >= 4 && ST == 1) ? 8 : 12;
  static constexpr int W_MEM = 224000 / (STAGES * STAGE + PIECE * 4);
  static constexpr int W = W_REG < W_MEM ? W_REG : W_MEM;
  static constexpr int PLAN_BYTES = (kPlanMax + 1) * 12 + 4;
  static constexpr int O_PIECE = W * STAGES * STAGE;
  static constexpr int O_PLAN = O_PIECE + W * PIECE * 4;
  static constexpr int O_TMP = (O_PLAN + PLAN_BYTES + 15) / 16 * 16;
  static constexpr int O_BAR = O_TMP + 33 * 8 + 8;
  static constexpr int O_META = O_BAR + W * STAGES * 8;
  static constexpr int O_INFO = (O_META + W * STAGES * TPS * 4 + 15) / 16 * 16;
  static constexpr int O_UP = O_INFO + W * 2 * 16;
  static constexpr int SMEM = O_UP + W * (D / GS) * 4 + 128;
  static_assert(PIECE * 4 <= STAGES * STAGE, "a warp's last piece lies in its ring");
  static_assert(SMEM <= 232448, "shared memory");
  static_assert(ST == 1 || (ST == 2 && NT == 1), "two streams share one column tile");
};

struct Work {
  float* slots;     // [2 * CTAs][PIECE]
  int4* meta;       // [CTAs]: unit of slot 1 (or -1); slot 0 (0 none, 1 goes on, 2 ends) +
                    // columns of slot 1's block << 8; its first token row and column
  int* gpre;        // plan in global memory (nullable: built in shared memory)
  long long* tpre;
  int* ng;
  int max_blocks;
  int vec;          // q rows are 16-byte aligned
};

// Physical row of MMA row i (0..7; + 8 for the upper half): neighbouring
// columns of a lane group's V rows then start in different bank halves.
__device__ __forceinline__ int row_of(int i) { return (i >> 1) + (i & 1) * 4; }

template <int BITS, int D, int GS, int NT>
struct State {
  using G = attn::Geo<BITS, D, GS>;
  uint32_t q[G::KSTEPS][NT][2];
  float qs[NT][G::NG][2];    // sum of the scaled q per group, times 2^-24
  float fac[NT][2];          // logit units to log2 units
  int qp[NT][2];             // query position of the lane's columns
  float m[NT][2], l[NT][2], pz[NT][G::NG][2];
  float x1[NT][G::NG][4];    // sum of x per group (fp16 outputs)
  // powers of two in x, o and x1 of each group, the same in all lanes; beyond two
  // groups in shared memory, to spare registers
  static constexpr bool kUpsHere = G::NG <= 2;
  float up[kUpsHere ? G::NG : 1];
  float o[G::MT][NT][4];

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        m[n][c] = kNeg;
        l[n][c] = 0.0f;
#pragma unroll
        for (int g = 0; g < G::NG; g++) pz[n][g][c] = x1[n][g][c] = x1[n][g][c + 2] = 0.0f;
      }
#pragma unroll
    for (int i = 0; i < G::MT; i++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int c = 0; c < 4; c++) o[i][n][c] = 0.0f;
  }
};

// The lane's query fragments: column n * 8 + g at the elements its K fragments
// pair with (8 consecutive ones per 4-bit word, 4 per 8-bit word).
template <int BITS, int D, int GS, int NT, int ST, bool BF>
__device__ __forceinline__ void load_q(State<BITS, D, GS, NT>& S, const AttnArgs& a, const Block& k,
                                       int h, bool vec, int g, int t) {
  using G = attn::Geo<BITS, D, GS>;
  constexpr int PW = 32 / BITS;
  constexpr float kUnit = 5.9604644775390625e-8f;  // 2^-24
#pragma unroll
  for (int n = 0; n < NT; n++) {
    const int c = ST == 2 ? g & 3 : n * 8 + g;
    const bool ok = c < k.cols;
    const int col = k.col0 + (ok ? c : 0);
    const int tok = col / a.rep, hh = col - tok * a.rep;
    const uint16_t* row =
        a.q + (int64_t)(k.row0 + tok) * a.q_row + (int64_t)(h * a.rep + hh) * a.q_head;
    float x[G::NG][G::KW][PW];
    float big = 0.0f;
#pragma unroll
    for (int gr = 0; gr < G::NG; gr++)
#pragma unroll
      for (int w = 0; w < G::KW; w++) {
        const uint16_t* p = row + gr * GS + t * (GS / 4) + w * PW;
        uint16_t e[PW];
        if (vec) {
          uint32_t u[PW / 2];
          if constexpr (PW == 8) {
            const uint4 y = *reinterpret_cast<const uint4*>(p);
            u[0] = y.x, u[1] = y.y, u[2] = y.z, u[3] = y.w;
          } else {
            const uint2 y = *reinterpret_cast<const uint2*>(p);
            u[0] = y.x, u[1] = y.y;
          }
#pragma unroll
          for (int i = 0; i < PW; i++) e[i] = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
        } else {
#pragma unroll
          for (int i = 0; i < PW; i++) e[i] = p[i];
        }
#pragma unroll
        for (int i = 0; i < PW; i++) {
          x[gr][w][i] = ok ? attn::dt_to_f<BF>(e[i]) : 0.0f;
          big = fmaxf(big, fabsf(x[gr][w][i]));
        }
      }
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    // 2^e brings the largest element into [2^13, 2^14)
    int e = 13 - (((__float_as_int(big) >> 23) & 255) - 127);
    e = big > 0.0f ? max(-100, min(100, e)) : 0;
    const float up = __int_as_float((127 + e) << 23);
#pragma unroll
    for (int gr = 0; gr < G::NG; gr++) {
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < G::KW; w++)
#pragma unroll
        for (int i = 0; i < PW; i++) sum = fmaf(x[gr][w][i], up, sum);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum *= kUnit;
      S.qs[n][gr][0] = __shfl_sync(0xffffffffu, sum, (2 * t) << 2);
      S.qs[n][gr][1] = __shfl_sync(0xffffffffu, sum, (2 * t + 1) << 2);
#pragma unroll
      for (int kin = 0; kin < G::MTG; kin++)
#pragma unroll
        for (int w2 = 0; w2 < 2; w2++) {
          const int v = 2 * kin + w2;
          float y0, y1;
          if constexpr (BITS == 4) {
            const float f = (v & 1) ? up * 0.0625f : up;
            y0 = x[gr][v / 4][v % 4] * f;
            y1 = x[gr][v / 4][v % 4 + 4] * f;
          } else {
            y0 = x[gr][v / 2][2 * (v % 2)] * up;
            y1 = x[gr][v / 2][2 * (v % 2) + 1] * up;
          }
          S.q[gr * G::MTG + kin][n][w2] = pack_h2(y0, y1);
        }
    }
    const float f = a.scale * attn::kLog2e * __int_as_float((127 - e) << 23) * attn::kCodeUnitInv;
    S.fac[n][0] = __shfl_sync(0xffffffffu, f, (2 * t) << 2);
    S.fac[n][1] = __shfl_sync(0xffffffffu, f, (2 * t + 1) << 2);
#pragma unroll
    for (int c2 = 0; c2 < 2; c2++) {
      const int cc = ST == 2 ? 2 * (t & 1) + c2 : n * 8 + 2 * t + c2;
      S.qp[n][c2] = cc < k.cols ? k.p0 + (k.col0 + cc) / a.rep : -1;
    }
  }
}

template <int NG, bool BF>
__device__ __forceinline__ void load_pairs(float (&s)[NG], float (&z)[NG], const uint8_t* p) {
  uint32_t w[NG];
  attn::lds_words<NG * 4>(w, p);
#pragma unroll
  for (int i = 0; i < NG; i++) {
    if constexpr (BF) {
      s[i] = __uint_as_float(w[i] << 16);
      z[i] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const __half2 h = *reinterpret_cast<const __half2*>(&w[i]);
      s[i] = __low2float(h);
      z[i] = __high2float(h);
    }
  }
}

// 1 / x of a power of two
__device__ __forceinline__ float pow2_inv(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }

// T tiles of a stage: keys j0[i]..j0[i] + 15.  MASK: some of them are not seen
// by some column (or, j0 < 0, the tile was not there to be read): their
// logits, scales and biases, whatever they hold, are replaced.
template <int BITS, int D, int GS, int NT, int ST, bool BF, int T, bool MASK>
__device__ __forceinline__ void process(State<BITS, D, GS, NT>& S, float* s_ups, const uint8_t* st,
                                        const int (&j0)[T], int window, int sinks, int g, int t) {
  using C = Cfg<BITS, D, GS, NT, ST>;
  using G = attn::Geo<BITS, D, GS>;
  constexpr int NG = G::NG;
  constexpr int VT = ST == 2 ? 1 : T;  // sets of logits a lane holds
  constexpr float kMid = (float)((1 << BITS) - 1) * 0.5f;
  static_assert(ST == 1 || T == 2, "two streams take two tiles");
  float* ups = State<BITS, D, GS, NT>::kUpsHere ? S.up : s_ups;
  const int ra = row_of(g);
  const bool up_stream = t >= 2;       // ST = 2: this lane's columns belong to tile 1
  float val[VT][NT][4];
  bool see[VT][NT][4];
#pragma unroll
  for (int i = 0; i < VT; i++) {
    float acc[NG][NT][4];
#pragma unroll
    for (int i2 = 0; i2 < ST; i2++) {
      const uint8_t* kt = st + (i + i2) * C::TILE;
#pragma unroll
      for (int gr = 0; gr < NG; gr++) {
        uint32_t wa[G::KW], wb[G::KW];
        attn::lds_words<G::KB>(wa, kt + ra * C::CRB + gr * G::GB + t * G::KB);
        attn::lds_words<G::KB>(wb, kt + (ra + 8) * C::CRB + gr * G::GB + t * G::KB);
        float x[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int c = 0; c < 4; c++) x[n][c] = 0.0f;
#pragma unroll
        for (int kin = 0; kin < G::MTG; kin++) {
          constexpr int XW = BITS == 4 ? 4 : 2;  // fragment registers per word
          const int v0 = 2 * kin, v1 = 2 * kin + 1;
          const uint32_t af[4] = {attn::k_extract<BITS>(wa[v0 / XW], v0 % XW),
                                  attn::k_extract<BITS>(wb[v0 / XW], v0 % XW),
                                  attn::k_extract<BITS>(wa[v1 / XW], v1 % XW),
                                  attn::k_extract<BITS>(wb[v1 / XW], v1 % XW)};
#pragma unroll
          for (int n = 0; n < NT; n++)
            mma16816(x[n], af, S.q[gr * G::MTG + kin][n][0], S.q[gr * G::MTG + kin][n][1]);
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int c = 0; c < 4; c++) acc[gr][n][c] = i2 == 0 || up_stream ? x[n][c] : acc[gr][n][c];
      }
    }
    const uint8_t* kp = st + (ST == 2 ? (up_stream ? C::TILE : 0) : i * C::TILE) + kTileRows * C::CRB;
    float sa[NG], za[NG], sb[NG], zb[NG];
    load_pairs<NG, BF>(sa, za, kp + ra * C::PRB);
    load_pairs<NG, BF>(sb, zb, kp + (ra + 8) * C::PRB);
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int c = 0; c < 4; c++) {
        float x = 0.0f;
#pragma unroll
        for (int gr = 0; gr < NG; gr++)
          x = fmaf(c < 2 ? sa[gr] : sb[gr], acc[gr][n][c],
                   fmaf(c < 2 ? za[gr] : zb[gr], S.qs[n][gr][c & 1], x));
        val[i][n][c] = x * S.fac[n][c & 1];
        if constexpr (MASK) {
          const int first = ST == 2 ? (up_stream ? j0[T - 1] : j0[0]) : j0[i];
          const int j = first + ra + (c >> 1) * 8, p = S.qp[n][c & 1];
          see[i][n][c] = first >= 0 && j <= p && (window == 0 || j > p - window || j < sinks);
          if (!see[i][n][c]) val[i][n][c] = kNeg;
        }
      }
    }
  }
  // V's scales (times the groups' powers) and biases.  A row counts towards the
  // reference by the exponent of its largest scale, less kRaise; here the
  // largest of all of the lane's rows stands for each
  const uint8_t* vp = st + (ST == 2 && up_stream ? C::TILE : 0) + C::HALF + kTileRows * C::CRB + ra * C::PRB;
  float vs[VT][2][NG], vz[VT][2][NG];
  auto load_v = [&]() {
#pragma unroll
    for (int i = 0; i < VT; i++)
#pragma unroll
      for (int r = 0; r < 2; r++) {
        load_pairs<NG, BF>(vs[i][r], vz[i][r], vp + i * C::TILE + 8 * r * C::PRB);
#pragma unroll
        for (int gr = 0; gr < NG; gr++) {
          if constexpr (!BF) vz[i][r][gr] = fmaf(kMid, vs[i][r][gr], vz[i][r][gr]);
          vs[i][r][gr] *= ups[gr];
        }
      }
  };
  auto any_sees = [&](int i, int r) {
    bool any = !MASK;
    if constexpr (MASK) {
#pragma unroll
      for (int n = 0; n < NT; n++) any = any || see[i][n][2 * r] || see[i][n][2 * r + 1];
    }
    return any;
  };
  // 2^23 + the exponent field, by its bits
  auto exponent = [&](float x) {
    return __uint_as_float(__funnelshift_r(__float_as_uint(x), 0x4b000000u >> 9, 23)) - (8388608.0f + 127.0f + kRaise);
  };
  load_v();
  float big = kMinScale, big_z = 0.0f;
#pragma unroll
  for (int i = 0; i < VT; i++)
#pragma unroll
    for (int r = 0; r < 2; r++) {
      if (!any_sees(i, r)) continue;  // (whatever lies there must not change a bit)
#pragma unroll
      for (int gr = 0; gr < NG; gr++) {
        big = fmaxf(big, fabsf(vs[i][r][gr]));
        if constexpr (BF) big_z = fmaxf(big_z, fabsf(vz[i][r][gr]));
      }
    }
  const float most_exp = exponent(BF ? fmaxf(big, big_z * kBiasShare) : big);
  bool up = false;
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int c = 0; c < 2; c++) {
      float x = fmaxf(val[0][n][c], val[0][n][c + 2]);
#pragma unroll
      for (int i = 1; i < VT; i++) x = fmaxf(x, fmaxf(val[i][n][c], val[i][n][c + 2]));
      up = up || x + most_exp > S.m[n][c] + kLazy;
    }
  if (__any_sync(0xffffffffu, up)) {
    // the groups' powers anew: each brings its largest scale in the rows that
    // are seen up to the largest of all.  What is not finite has no say.  (Pairs
    // are read again one at a time: held over this, they cost spills.)
    asm volatile("" ::: "memory");
    auto pair = [&](int i, int r, int gr) {
      return *reinterpret_cast<const uint32_t*>(vp + i * C::TILE + 8 * r * C::PRB + 4 * gr);
    };
    uint32_t most[NG], all = 0;
    float grow[NG], row_exp[VT][2];
#pragma unroll
    for (int gr = 0; gr < NG; gr++) {
      uint32_t e = 0;
#pragma unroll
      for (int i = 0; i < VT; i++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
          const uint32_t x = __float_as_uint(fabsf(attn::dt_to_f<BF>((uint16_t)pair(i, r, gr))));
          if (any_sees(i, r) && x < 0x7f800000u) e = max(e, x);
        }
      most[gr] = __reduce_max_sync(0xffffffffu, e) >> 23;
      all = max(all, most[gr]);
      grow[gr] = pow2_inv(ups[gr]);
    }
    __syncwarp();  // every lane has read them
#pragma unroll
    for (int gr = 0; gr < NG; gr++) {
      const float now = __uint_as_float((127u + min(all - most[gr], (uint32_t)kMaxUp)) << 23);
      grow[gr] *= now;
      ups[gr] = now;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < VT; i++)
#pragma unroll
      for (int r = 0; r < 2; r++) {
        float x = kMinScale;
#pragma unroll
        for (int gr = 0; gr < NG; gr++) {
          const uint32_t w = pair(i, r, gr);
          const float y = fabsf(attn::dt_to_f<BF>((uint16_t)w)) * ups[gr];
          const float z = BF ? fabsf(attn::dt_to_f<BF>((uint16_t)(w >> 16))) * kBiasShare : 0.0f;
          x = fmaxf(x, fmaxf(y < INFINITY ? y : 0.0f, z < INFINITY ? z : 0.0f));
        }
        row_exp[i][r] = exponent(x);
      }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        float x = fmaxf(val[0][n][c] + row_exp[0][0], val[0][n][c + 2] + row_exp[0][1]);
#pragma unroll
        for (int i = 1; i < VT; i++)
          x = fmaxf(x, fmaxf(val[i][n][c] + row_exp[i][0], val[i][n][c + 2] + row_exp[i][1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        // only where its own keys pass it: what moved another column stays there
        x = x > S.m[n][c] + kLazy ? x : S.m[n][c];
        const float f = ex2(S.m[n][c] - x);
        S.m[n][c] = x;
        S.l[n][c] *= f;
#pragma unroll
        for (int gr = 0; gr < NG; gr++) {
          const float fg = f * grow[gr];
          S.pz[n][gr][c] *= f;
          if constexpr (!BF) S.x1[n][gr][c] *= fg;
#pragma unroll
          for (int k = gr * G::MTG; k < (gr + 1) * G::MTG; k++) {
            S.o[k][n][c] *= fg;
            S.o[k][n][c + 2] *= fg;
          }
        }
      }
    asm volatile("" ::: "memory");
    load_v();
  }
#pragma unroll
  for (int i = 0; i < VT; i++) {
    float p[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int c = 0; c < 4; c++) {
        p[n][c] = ex2(val[i][n][c] - S.m[n][c & 1]);
        if constexpr (MASK)
          if (!see[i][n][c]) p[n][c] = 0.0f;
        S.l[n][c & 1] += p[n][c];
      }
#pragma unroll
    for (int gr = 0; gr < NG; gr++) {
      uint32_t b0[NT], b1[NT];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float x[4];
#pragma unroll
        for (int c = 0; c < 4; c++) {
          x[c] = p[n][c] * vs[i][c >> 1][gr];
          if constexpr (MASK) {
            if (!see[i][n][c]) x[c] = 0.0f;
            S.pz[n][gr][c & 1] += see[i][n][c] ? p[n][c] * vz[i][c >> 1][gr] : 0.0f;
          } else {
            S.pz[n][gr][c & 1] = fmaf(p[n][c], vz[i][c >> 1][gr], S.pz[n][gr][c & 1]);
          }
        }
        b0[n] = movmatrix_t(pack_h2(x[0], x[1]));
        b1[n] = movmatrix_t(pack_h2(x[2], x[3]));
        if constexpr (!BF) {
          constexpr uint32_t kOnes = 0x3c003c00u;
          const uint32_t ones[4] = {kOnes, kOnes, kOnes, kOnes};
          mma16816(S.x1[n][gr], ones, b0[n], b1[n]);
        }
      }
#pragma unroll
      for (int i2 = 0; i2 < ST; i2++) {
        const uint8_t* vt = st + (i + i2) * C::TILE + C::HALF;
        uint32_t c0[NT], c1[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const bool keep = ST == 1 || (g >> 2) == i2;  // the other stream's columns get nothing
          c0[n] = keep ? b0[n] : 0u;
          c1[n] = keep ? b1[n] : 0u;
        }
        uint32_t w[4][G::VW];
#pragma unroll
        for (int r = 0; r < 4; r++)
          attn::lds_words<G::VB>(w[r], vt + (t + 4 * r) * C::CRB + gr * G::GB + g * G::VB);
        constexpr int E = G::E;  // elements per 16-bit chunk
#pragma unroll
        for (int ci = 0; ci < G::C; ci++) {
          const uint32_t sel = (ci & 1) ? 0x7632u : 0x5410u;
          const uint32_t x = prmt(w[0][ci / 2], w[1][ci / 2], sel);
          const uint32_t y = prmt(w[2][ci / 2], w[3][ci / 2], sel);
#pragma unroll
          for (int j = 0; j < E; j += 2) {
            const uint32_t af[4] = {attn::v_extract<BITS>(x, j), attn::v_extract<BITS>(x, j + 1),
                                    attn::v_extract<BITS>(y, j), attn::v_extract<BITS>(y, j + 1)};
            const int mt = gr * G::MTG + (ci * E + j) / 2;
#pragma unroll
            for (int n = 0; n < NT; n++) mma16816(S.o[mt][n], af, c0[n], c1[n]);
          }
        }
      }
    }
  }
}

// d of fragment (mt, row g); row g + 8 is d + 1
template <int BITS, int D, int GS>
__device__ __forceinline__ int frag_d(int mt, int g) {
  using G = attn::Geo<BITS, D, GS>;
  const int gr = mt / G::MTG, e = (mt % G::MTG) * 2;  // element of the lane's list
  return gr * GS + (g * G::C) * G::E + e;
}

// Two output values d, d + 1 of column c of block k
template <int NT, bool BF>
__device__ __forceinline__ void store_out(const AttnArgs& a, const Block& k, int h, int c, int d,
                                          float x, float y) {
  if (c >= k.cols) return;
  const int col = k.col0 + c, tok = col / a.rep, hh = col - tok * a.rep;
  uint16_t* dst = a.out + ((int64_t)(k.row0 + tok) * a.Hq + h * a.rep + hh) * a.v.D + d;
  const uint16_t lo = attn::f_to_dt<BF>(x), hi = attn::f_to_dt<BF>(y);
  if (a.out_align) {
    *reinterpret_cast<uint32_t*>(dst) = (uint32_t)lo | ((uint32_t)hi << 16);
  } else {  // a view that starts at an odd element
    dst[0] = lo;
    dst[1] = hi;
  }
}

// Close a segment: sums over the lanes of a column, outputs in natural units,
// the two streams joined.
template <int BITS, int D, int GS, int NT, int ST, bool BF>
__device__ __forceinline__ void close(State<BITS, D, GS, NT>& S, const float* s_ups) {
  const float* ups = State<BITS, D, GS, NT>::kUpsHere ? S.up : s_ups;
  using G = attn::Geo<BITS, D, GS>;
  constexpr float kMid = (float)((1 << BITS) - 1) * 0.5f;
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int c = 0; c < 2; c++) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        S.l[n][c] += __shfl_xor_sync(0xffffffffu, S.l[n][c], o);
#pragma unroll
        for (int gr = 0; gr < G::NG; gr++)
          S.pz[n][gr][c] += __shfl_xor_sync(0xffffffffu, S.pz[n][gr][c], o);
      }
#pragma unroll
      for (int k = 0; k < G::MT; k++) {
        const float down = pow2_inv(ups[k / G::MTG]), unit = attn::kCodeUnitInv * down;
        const float odd = BITS == 4 ? unit * 0.0625f : unit;
        float add = S.pz[n][k / G::MTG][c];
        if constexpr (!BF) add = fmaf(-kMid * down, S.x1[n][k / G::MTG][c], add);
        S.o[k][n][c] = fmaf(S.o[k][n][c], unit, add);
        S.o[k][n][c + 2] = fmaf(S.o[k][n][c + 2], odd, add);
      }
      if constexpr (ST == 2) {
        const float other = __shfl_xor_sync(0xffffffffu, S.m[n][c], 2);
        const float x = fmaxf(S.m[n][c], other), f = ex2(S.m[n][c] - x);
        S.m[n][c] = x;
        S.l[n][c] *= f;
        S.l[n][c] += __shfl_xor_sync(0xffffffffu, S.l[n][c], 2);
#pragma unroll
        for (int k = 0; k < G::MT; k++)
#pragma unroll
          for (int e = c; e < 4; e += 2) {
            S.o[k][n][e] *= f;
            S.o[k][n][e] += __shfl_xor_sync(0xffffffffu, S.o[k][n][e], 2);
          }
      }
    }
}

struct __align__(16) PieceInfo {
  int unit;        // -1: none
  int flags;       // 1: begins the unit, 2: ends it; columns << 8
  int row0, col0;  // of the unit's block
};

template <int BITS, int D, int GS, int NT, int ST, bool BF>
__global__ void __launch_bounds__(Cfg<BITS, D, GS, NT, ST>::W * 32, 1)
    cols_kernel(const AttnArgs a, const Work ws) {
  using C = Cfg<BITS, D, GS, NT, ST>;
  using G = attn::Geo<BITS, D, GS>;
  constexpr int W = C::W, NC = C::NC, TPS = C::TPS, STAGES = C::STAGES;
  extern __shared__ __align__(128) uint8_t smem[];
  const View& v = a.v;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + w * STAGES * C::STAGE;
  float* piece_a = reinterpret_cast<float*>(smem + C::O_PIECE) + w * C::PIECE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::O_BAR) + w * STAGES;
  int* meta = reinterpret_cast<int*>(smem + C::O_META) + w * STAGES * TPS;
  PieceInfo* info = reinterpret_cast<PieceInfo*>(smem + C::O_INFO);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (lane == 0)
    for (int s = 0; s < STAGES; s++) attn::mbar_init(bars + s, 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  if (lane < 2) info[2 * w + lane] = PieceInfo{-1, 0, 0, 0};
  asm volatile("griddepcontrol.wait;" ::: "memory");

  Plan P;
  const int fixed = v.B * ((a.rep + NC - 1) / NC);  // column blocks of a decode
  if (!v.cu && fixed <= 32) {
    // few sequences: every warp makes the plan with its lanes and writes the
    // same values, so no barrier stands before the first copy
    long long* tpre = reinterpret_cast<long long*>(smem + C::O_PLAN);
    P = Plan{nullptr, tpre, fixed};
    int n = lane < fixed ? get_block<NC>(a, P, lane).nt : 0;
    long long e = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, e, o);
      if (lane >= o) e += y;
    }
    if (lane < fixed) tpre[lane + 1] = e;
    if (lane == 0) tpre[0] = 0;
    if (blockIdx.x == 0 && w == 0 && lane < v.B) {
      int row0, rn, len;
      checked_rows(v, lane, row0, rn, len, true);
    }
    __syncwarp();
  } else if (ws.tpre) {
    P = Plan{ws.gpre, ws.tpre, *ws.ng};
    __syncthreads();
  } else {
    long long* tpre = reinterpret_cast<long long*>(smem + C::O_PLAN);
    int* gpre = reinterpret_cast<int*>(tpre + kPlanMax + 1);
    const int NG = build_plan<NC>(a, gpre, tpre, ws.max_blocks,
                                  reinterpret_cast<long long*>(smem + C::O_TMP), blockIdx.x == 0);
    P = Plan{gpre, tpre, NG};
  }
  const long long RT = P.tpre[P.NG] * v.Hkv;
  const long long all = (long long)gridDim.x * W, gw = (long long)blockIdx.x * W + w;
  // at least one stage per warp
  const long long act = max(1ll, min(all, RT / TPS));
  const long long t0 = gw < act ? gw * RT / act : RT, t1 = gw < act ? (gw + 1) * RT / act : RT;

  // column blocks that see no key: zero rows
  for (long long gi = gw; gi < P.NG; gi += all) {
    if (P.tpre[gi + 1] != P.tpre[gi]) continue;
    const Block k = get_block<NC>(a, P, (int)gi);
    for (int h = 0; h < v.Hkv; h++)
      for (int c = 0; c < k.cols; c++)
        for (int d = lane * 2; d < D; d += 64) store_out<NT, BF>(a, k, h, c, d, 0.0f, 0.0f);
  }

  if (t0 < t1) {
    // block holding tile t0
    int x = 0, y = P.NG;  // tpre[x] * Hkv <= t0 < tpre[y] * Hkv
    while (y - x > 1) {
      const int mid = (x + y) >> 1;
      if (P.tpre[mid] * v.Hkv <= t0) x = mid;
      else y = mid;
    }
    // a block without tiles shares its successor's start: take the last
    int gi = x;
    Block kc = get_block<NC>(a, P, gi);
    long long rel = t0 - P.tpre[gi] * v.Hkv;
    int hc = (int)(rel / kc.nt), ic = (int)(rel - (long long)hc * kc.nt);
    int left = (int)(t1 - t0);  // tiles to consume, this segment's included

    // The issue side runs ahead.  Lane i holds the source of tile ibase + i of
    // its unit and issues that tile's copy itself; the page numbers of the 32
    // tiles after those are already on their way.
    const int32_t* itable;
    int insink, ilo, int_, gii = gi, ih = hc, ii = ic, ibase, iwin, iend, irest = left;
    int next_page, my_j0, my_bytes;
    const uint8_t* my_src;
    int istage = 0;
    auto tile_at = [&](int i) { return i < insink ? i : ilo + i - insink; };
    auto fetch = [&](int i) { return i < int_ ? __ldg(itable + (tile_at(i) >> v.tiles_shift)) : -1; };
    auto place = [&](int page) {  // tiles ii.. of the unit, lane's in `page`
      ibase = ii;
      iwin = min(iend, ibase + 32);
      const int tt = tile_at(ibase + lane);
      const bool in = ibase + lane < iwin, ok = in && page >= 0 && page < v.num_pages;
      if (in && !ok) raise(v);
      my_src = tile_ptr(v, ok ? page : 0, ih, tt & ((1 << v.tiles_shift) - 1));
      my_j0 = ok ? tt << 4 : -1;
      // bytes of the stage that starts with the lane's tile; -1: no such tile
      const unsigned have = __ballot_sync(0xffffffffu, ok);
      my_bytes = in ? __popc((have >> lane) & ((1 << TPS) - 1)) * C::TILE : -1;
      next_page = fetch(ibase + 32 + lane);
    };
    auto set_unit = [&](const Block& k) {
      itable = v.table + (int64_t)k.b * v.table_stride;
      insink = k.nsink;
      ilo = k.lo;
      int_ = k.nt;
      iend = min(int_, ii + irest);
      irest -= iend - ii;
      place(fetch(ii + lane));
    };
    set_unit(kc);
    auto issue = [&]() {
      if (ii == iwin) {
        if (ii < iend) {
          place(next_page);
        } else {
          if (irest == 0) return;
          if (++ih == v.Hkv) {
            ih = 0;
            do {
              gii++;
            } while (P.tpre[gii + 1] == P.tpre[gii]);
          }
          ii = 0;
          set_unit(get_block<NC>(a, P, gii));
        }
      }
      const int off = lane - (ii - ibase);
      if ((unsigned)off < (unsigned)TPS && my_bytes >= 0) {
        if (off == 0) attn::mbar_expect_tx(bars + istage, my_bytes);
        meta[istage * TPS + off] = my_j0;
        if (my_j0 >= 0)
          attn::bulk_g2s(ring + istage * C::STAGE + off * C::TILE, my_src, C::TILE, bars + istage);
      }
      ii = min(ii + TPS, iwin);
      istage = istage + 1 == STAGES ? 0 : istage + 1;
    };
#pragma unroll 1
    for (int s = 0; s < STAGES; s++) issue();

    State<BITS, D, GS, NT> S;
    float* ups = reinterpret_cast<float*>(smem + C::O_UP) + w * G::NG;
    auto start_ups = [&]() {
      __syncwarp();
      if (lane < G::NG) ups[lane] = 1.0f;
#pragma unroll
      for (float& x : S.up) x = 1.0f;
      __syncwarp();
    };
    S.reset();
    start_ups();
    load_q<BITS, D, GS, NT, ST, BF>(S, a, kc, hc, ws.vec, g, t);
    bool begun = ic == 0;  // this segment holds the unit's first tile
    int stage = 0;
    uint32_t phase = 0;
    while (left > 0) {
      // list indices [fa, fb): tiles that every column sees whole
      const int e = min(kc.nt, ic + left);
      const int fa = a.window == 0 ? 0
                                   : kc.nsink + max(0, ((kc.pmax - a.window + 16) >> 4) - kc.lo);
      const int fb = min(e, kc.nsink + ((kc.pmin - 15) >> 4) - kc.lo + 1);
      left -= e - ic;
#pragma unroll 1
      while (ic < e) {
        __syncwarp();
        if (!attn::mbar_wait(bars + stage, phase)) {
          // give up: wait (bounded) for the copies still in flight, then leave
          if (lane == 0) gave_up(v);
          for (int s = 1; s < STAGES; s++) attn::mbar_wait(bars + (stage + s) % STAGES, (stage + s) / STAGES ^ phase);
          left = 0;
          break;
        }
        const uint8_t* st = ring + stage * C::STAGE;
        int j0[TPS], bad = 0;
#pragma unroll
        for (int i = 0; i < TPS; i++) {
          j0[i] = meta[stage * TPS + i];
          bad |= j0[i];
        }
        if (ic >= fa && ic + TPS <= fb && bad >= 0) {
          process<BITS, D, GS, NT, ST, BF, TPS, false>(S, ups, st, j0, a.window, a.sinks, g, t);
        } else {
          if (TPS == 2 && ic + 1 == e) j0[TPS - 1] = -1;
          process<BITS, D, GS, NT, ST, BF, TPS, true>(S, ups, st, j0, a.window, a.sinks, g, t);
        }
        __syncwarp();
        issue();
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
        ic += TPS;
      }
      ic = e;

      // the segment ends: the unit is done, or the warp's run is
      close<BITS, D, GS, NT, ST, BF>(S, ups);
      const bool ended = ic == kc.nt;
      const int unit = gi * v.Hkv + hc;
      if (begun && ended) {
#pragma unroll
        for (int nn = 0; nn < NT; nn++)
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const float inv = S.l[nn][c] != 0.0f ? 1.0f / S.l[nn][c] : 0.0f;
#pragma unroll
            for (int k = 0; k < G::MT; k++)
              store_out<NT, BF>(a, kc, hc, nn * 8 + 2 * t + c, frag_d<BITS, D, GS>(k, g),
                                S.o[k][nn][c] * inv, S.o[k][nn][c + 2] * inv);
          }
      } else {
        // the first piece waits in its own area, a last one in the idle ring
        float* dst = begun ? reinterpret_cast<float*>(ring) : piece_a;
#pragma unroll
        for (int nn = 0; nn < NT; nn++) {
          if (g == 0) {
#pragma unroll
            for (int c = 0; c < 2; c++) {
              dst[nn * 8 + 2 * t + c] = S.m[nn][c];
              dst[8 * NT + nn * 8 + 2 * t + c] = S.l[nn][c];
            }
          }
#pragma unroll
          for (int k = 0; k < G::MT; k++)
            *reinterpret_cast<float4*>(dst + 16 * NT + ((k * NT + nn) * 32 + lane) * 4) =
                make_float4(S.o[k][nn][0], S.o[k][nn][1], S.o[k][nn][2], S.o[k][nn][3]);
        }
        if (lane == 0)
          info[2 * w + (begun ? 1 : 0)] =
              PieceInfo{unit, (begun ? 1 : 0) | (ended ? 2 : 0) | (kc.cols << 8), kc.row0, kc.col0};
      }
      if (left > 0) {
        ic = 0;
        if (++hc == v.Hkv) {
          hc = 0;
          do {
            gi++;
          } while (P.tpre[gi + 1] == P.tpre[gi]);
          kc = get_block<NC>(a, P, gi);
        }
        S.reset();
        start_ups();
        load_q<BITS, D, GS, NT, ST, BF>(S, a, kc, hc, ws.vec, g, t);
        begun = true;
      }
    }
  }
  __syncthreads();

  // combine the CTA's pieces, unit by unit in key order; warp w takes the
  // fragments w, w + W, ..., four pieces' loads at a time
  static_assert(2 * W <= 32, "a lane per piece");
  const PieceInfo mine = lane < 2 * W ? info[lane] : PieceInfo{-1, 0, 0, 0};
  int4 mt = make_int4(-1, 0, 0, 0);  // slot 1's unit, slot 0's state + columns << 8, row, column
  for (unsigned rest = __ballot_sync(0xffffffffu, mine.unit >= 0); rest;) {
    const int p0 = __ffs(rest) - 1, unit = __shfl_sync(0xffffffffu, mine.unit, p0);
    const unsigned chain = __ballot_sync(0xffffffffu, mine.unit == unit);
    const int flags = __reduce_or_sync(0xffffffffu, mine.unit == unit ? mine.flags & 3 : 0);
    Block k;
    k.cols = __shfl_sync(0xffffffffu, mine.flags, p0) >> 8;
    k.row0 = __shfl_sync(0xffffffffu, mine.row0, p0);
    k.col0 = __shfl_sync(0xffffffffu, mine.col0, p0);
    rest &= ~chain;
    auto piece = [&](int p) -> const float* {
      return (p & 1) ? reinterpret_cast<const float*>(smem + (p >> 1) * STAGES * C::STAGE)
                     : reinterpret_cast<const float*>(smem + C::O_PIECE) + (p >> 1) * C::PIECE;
    };
    const bool whole = flags == 3;
    float* out_slot = ws.slots + (size_t)(2 * blockIdx.x + ((flags & 1) ? 1 : 0)) * C::PIECE;
    for (int f = w; f < C::FR; f += W) {
      const int nn = f % NT, c0 = nn * 8 + 2 * t;
      float m0 = kNeg, m1 = kNeg, l0 = 0.0f, l1 = 0.0f;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (unsigned todo = chain; todo;) {
        float2 x[4], l[4];
        float4 z[4];
        float n0 = m0, n1 = m1;
        int n = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float* q = piece(todo ? __ffs(todo) - 1 : p0);
          const bool there = todo != 0;
          todo &= todo - 1;
          n += there;
          x[i] = *reinterpret_cast<const float2*>(q + c0);
          l[i] = *reinterpret_cast<const float2*>(q + 8 * NT + c0);
          z[i] = *reinterpret_cast<const float4*>(q + 16 * NT + (f * 32 + lane) * 4);
          if (there) {
            n0 = fmaxf(n0, x[i].x);
            n1 = fmaxf(n1, x[i].y);
          }
        }
        const float r0 = ex2(m0 - n0), r1 = ex2(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= r0;
        l1 *= r1;
        o = make_float4(o.x * r0, o.y * r1, o.z * r0, o.w * r1);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if (i >= n) break;
          const float e0 = ex2(x[i].x - m0), e1 = ex2(x[i].y - m1);
          l0 = fmaf(e0, l[i].x, l0);
          l1 = fmaf(e1, l[i].y, l1);
          o.x = fmaf(e0, z[i].x, o.x);
          o.y = fmaf(e1, z[i].y, o.y);
          o.z = fmaf(e0, z[i].z, o.z);
          o.w = fmaf(e1, z[i].w, o.w);
        }
      }
      if (whole) {
        const float i0 = l0 != 0.0f ? 1.0f / l0 : 0.0f, i1 = l1 != 0.0f ? 1.0f / l1 : 0.0f;
        const int d = frag_d<BITS, D, GS>(f / NT, g), h = unit % v.Hkv;
        store_out<NT, BF>(a, k, h, c0, d, o.x * i0, o.z * i0);
        store_out<NT, BF>(a, k, h, c0 + 1, d, o.y * i1, o.w * i1);
      } else {
        *reinterpret_cast<float4*>(out_slot + 16 * NT + (f * 32 + lane) * 4) = o;
        if (f < NT && g == 0) {
          *reinterpret_cast<float2*>(out_slot + c0) = make_float2(m0, m1);
          *reinterpret_cast<float2*>(out_slot + 8 * NT + c0) = make_float2(l0, l1);
        }
      }
    }
    if (!whole) {
      if (flags & 1) mt = make_int4(unit, mt.y | (k.cols << 8), k.row0, k.col0);
      else mt.y |= (flags & 2) ? 2 : 1;
    }
  }
  if (tid == 0) ws.meta[blockIdx.x] = mt;
}

// Block (c, f): the unit that begins in CTA c and goes on, fragment f; its
// pieces are slot 1 of c and slot 0 of the CTAs after it up to the one that
// ends it.  Warps take the pieces in turn; their sums meet in warp order.
constexpr int kMergeWarps = 4;
template <int BITS, int D, int GS, int NT, int ST, bool BF>
__global__ void __launch_bounds__(kMergeWarps * 32) cols_merge_kernel(const AttnArgs a, const Work ws) {
  using C = Cfg<BITS, D, GS, NT, ST>;
  __shared__ float sm[kMergeWarps][32][2], sl[kMergeWarps][32][2];
  __shared__ float4 so[kMergeWarps][32];
  __shared__ int s_end;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const View& v = a.v;
  const int c = blockIdx.x, n = gridDim.x, f = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
  const int4 where = ws.meta[c];
  int end = n - 1;  // the CTA that ends the unit: the first after c that ends one
  for (int i = c + 1 + tid; i < n; i += kMergeWarps * 32)
    if ((ws.meta[i].y & 255) == 2) {
      end = i;
      break;
    }
  const int unit = where.x;
  if (unit < 0) return;
  if (tid == 0) s_end = n - 1;
  __syncthreads();
  if (end < n - 1) atomicMin(&s_end, end);
  __syncthreads();
  const int last = s_end;
  auto piece = [&](int i) -> const float* {
    return ws.slots + (size_t)(i == c ? 2 * c + 1 : 2 * i) * C::PIECE;
  };
  const int nn = f % NT, c0 = nn * 8 + 2 * t;
  float m0 = kNeg, m1 = kNeg, l0 = 0.0f, l1 = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = c + w; i <= last; i += kMergeWarps) {
    const float* q = piece(i);
    const float2 x = *reinterpret_cast<const float2*>(q + c0);
    const float2 l = *reinterpret_cast<const float2*>(q + 8 * NT + c0);
    const float4 z = *reinterpret_cast<const float4*>(q + 16 * NT + (f * 32 + lane) * 4);
    const float n0 = fmaxf(m0, x.x), n1 = fmaxf(m1, x.y);
    const float r0 = ex2(m0 - n0), r1 = ex2(m1 - n1), e0 = ex2(x.x - n0), e1 = ex2(x.y - n1);
    m0 = n0;
    m1 = n1;
    l0 = fmaf(e0, l.x, l0 * r0);
    l1 = fmaf(e1, l.y, l1 * r1);
    o.x = fmaf(e0, z.x, o.x * r0);
    o.y = fmaf(e1, z.y, o.y * r1);
    o.z = fmaf(e0, z.z, o.z * r0);
    o.w = fmaf(e1, z.w, o.w * r1);
  }
  sm[w][lane][0] = m0, sm[w][lane][1] = m1, sl[w][lane][0] = l0, sl[w][lane][1] = l1;
  so[w][lane] = o;
  __syncthreads();
  if (w) return;
  for (int i = 1; i < kMergeWarps; i++) {
    m0 = fmaxf(m0, sm[i][lane][0]);
    m1 = fmaxf(m1, sm[i][lane][1]);
  }
  l0 = l1 = 0.0f;
  o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i = 0; i < kMergeWarps; i++) {
    const float e0 = ex2(sm[i][lane][0] - m0), e1 = ex2(sm[i][lane][1] - m1);
    const float4 z = so[i][lane];
    l0 = fmaf(e0, sl[i][lane][0], l0);
    l1 = fmaf(e1, sl[i][lane][1], l1);
    o.x = fmaf(e0, z.x, o.x);
    o.y = fmaf(e1, z.y, o.y);
    o.z = fmaf(e0, z.z, o.z);
    o.w = fmaf(e1, z.w, o.w);
  }
  const float i0 = l0 != 0.0f ? 1.0f / l0 : 0.0f, i1 = l1 != 0.0f ? 1.0f / l1 : 0.0f;
  Block k;
  k.cols = where.y >> 8;
  k.row0 = where.z;
  k.col0 = where.w;
  const int d = frag_d<BITS, D, GS>(f / NT, g), h = unit % v.Hkv;
  store_out<NT, BF>(a, k, h, c0, d, o.x * i0, o.z * i0);
  store_out<NT, BF>(a, k, h, c0 + 1, d, o.y * i1, o.w * i1);
}

template <int NC, int KS>
__global__ void __launch_bounds__(1024) plan_kernel(const AttnArgs a, const Work ws) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ long long tmp[33];
  const int NG = build_plan<NC, KS>(a, ws.gpre, ws.tpre, ws.max_blocks, tmp, true);
  if (threadIdx.x == 0) *ws.ng = NG;
}

// The merge keeps the column kernel's split of the SM's memory, so that it can
// become resident without waiting for the SM to empty.
inline int32_t kernel_carveout(const void* kern, int dev) {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> done;
  std::lock_guard<std::mutex> lk(mu);
  if (done.count({kern, dev})) return KVQ_OK;
  KVQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout,
                                    cudaSharedmemCarveoutMaxShared));
  done.insert({kern, dev});
  return KVQ_OK;
}

template <int BITS, int D, int GS, int NT, int ST, bool BF>
int32_t launch_cols_one(const AttnArgs& a, const Work& ws, int ctas, int dev, cudaStream_t st) {
  using C = Cfg<BITS, D, GS, NT, ST>;
  auto kern = cols_kernel<BITS, D, GS, NT, ST, BF>;
  const int32_t rc = kernel_setup(reinterpret_cast<const void*>(kern), C::W * 32, C::SMEM, dev, nullptr);
  if (rc) return rc;
  if (ws.tpre) KVQ_CUDA_TRY(launch_pdl(plan_kernel<C::NC, 4>, dim3(1), dim3(1024), 0, st, a, ws));
  KVQ_CUDA_TRY(launch_pdl(kern, dim3((unsigned)ctas), dim3(C::W * 32), C::SMEM, st, a, ws));
  auto merge = cols_merge_kernel<BITS, D, GS, NT, ST, BF>;
  const int32_t rm = kernel_carveout(reinterpret_cast<const void*>(merge), dev);
  if (rm) return rm;
  KVQ_CUDA_TRY(launch_pdl(merge, dim3((unsigned)ctas, C::FR), dim3(kMergeWarps * 32), 0, st, a, ws));
  return KVQ_OK;
}

// Defined for each (bits, dtype) in its own file.  NC: columns of a block, 4, 8
// or 16 (D up to 128).
template <int BITS, bool BF>
int32_t launch_cols(const AttnArgs& a, const Work& ws, int NC, int ctas, int dev, cudaStream_t st);

template <int BITS, bool BF>
int32_t launch_cols_impl(const AttnArgs& a, const Work& ws, int NC, int ctas, int dev, cudaStream_t st) {
#define KVQ_COLS(DD, GG)                                                                       \
  if (a.v.D == DD && a.v.gs == GG) {                                                           \
    if (NC == 4) return launch_cols_one<BITS, DD, GG, 1, 2, BF>(a, ws, ctas, dev, st);         \
    if (NC == 8) return launch_cols_one<BITS, DD, GG, 1, 1, BF>(a, ws, ctas, dev, st);         \
    return launch_cols_one<BITS, DD, GG, DD == 256 ? 1 : 2, 1, BF>(a, ws, ctas, dev, st);      \
  }
  KVQ_COLS(64, 32)
  KVQ_COLS(64, 64)
  KVQ_COLS(128, 32)
  KVQ_COLS(128, 64)
  KVQ_COLS(128, 128)
  KVQ_COLS(256, 32)
  KVQ_COLS(256, 64)
  KVQ_COLS(256, 128)
#undef KVQ_COLS
  return fail(KVQ_ERR_ARG, "paged: unsupported head_dim / group_size");
}

}  // namespace paged
}  // namespace kvq
