#pragma once
// kvq_paged_chunk.cuh — attention of many query rows per sequence over the
// pages (prompt chunks) on the tcgen05 tensor cores.
//
// A unit is one (sequence, kv head) and MR query rows (row c is token c / rep,
// head c % rep: every query head of the group shares the tile's K and V).  Its
// 128-key tiles (D 256: 64) are dequantized once, to the dtype, into 128-byte-swizzled
// shared tiles and serve all MR rows: S = Q K^T into TMEM, softmax from TMEM
// to P in the same columns, O += P V with A from TMEM.
//   * D 64 / 128: MR 256, two row tiles of 128 (TMEM lanes) in turn: the tensor
//     core works on one while the softmax warps have the other.
//   * D 256: MR 128 (its O takes 256 TMEM columns), two S buffers instead.
// Warps: 8 per row tile for the softmax (two threads share a row, half of the keys each;
// one exchange of the maximum per tile), 7 that dequantize (a thread owns a key
// row of K or of V; the 32-row blocks of K and V of each tile go round), 1
// that issues the MMAs.  All hand-offs are mbarriers with bounded waits.  A wait
// tells two neighbouring phases apart only, so a barrier whose waiter may be more
// releases behind comes in several, taken in turn.
//
// Roundings: K, V (as a dense cache of the dtype holds them) and the
// probabilities go through the tensor core in the dtype (what exact codes would
// cost: a product for every group, and as many columns of S); logits, statistics
// and O are f32.  RMS error against 64 bits 5.5e-4 (fp16) and 3.4e-3 (bf16) of
// the output's, of which its own rounding is 2.1e-4 and 1.7e-3.  O is rescaled only when a row's maximum has grown by more
// than 2^8 since the last time.  fp16 probabilities stand for 2^-7 of their value
// (kLift: at most 2^15 with that growth), so that a key far below the row's
// maximum keeps 2^-32 of it before it is lost: behind a first token that takes
// the softmax, thousands of such keys are the output.
//
// Bound: per 128 keys and 256 rows at D 128 the tensor core needs 2048 clocks
// (8192 dense flops a clock) and so do the exponentials (16 a clock per SM).
//
// Work split: the tiles of all units laid end to end, one equal run per SM;
// the pieces of a cut unit (m, l, O in f32) meet in the merge kernel in order.
//
// Measured (B200): 512 rows over 16,896 keys, 32 query and 8 kv heads, D 128, 8
// bits (139.6 GFLOP): 184 us, 759 TFLOP/s, about 5,000 clocks a tile.  D 256, two
// chunks of up to 1,024 rows, window 1,024, 8 bits: 110 us; one K / V buffer of 128
// keys instead of two of 64 took 133.
#include "kvq_paged_cols.cuh"
#include "kvq_tc.cuh"

namespace kvq {
namespace paged {

template <int BITS, int D, int GS>
struct Chunk {
  static constexpr int QT = D == 256 ? 1 : 2;   // row tiles of 128
  static constexpr int MR = 128 * QT;
  static constexpr int KL = D == 256 ? 6 : 7, KT = 1 << KL;  // keys per tile: 64 or 128
  static constexpr int NBK = KT / 32, BL = KL - 4;  // 32-row blocks of K; log2 of K's and V's
  static constexpr int KB = 2;                  // K (and V) buffers, taken by a tile's parity
  static constexpr int QPANEL = 128 * 128;      // bytes: 128 rows of 64 elements
  static constexpr int QTILE = D / 64 * QPANEL;
  static constexpr int PANEL = KT * 128;        // the same of a K or V tile
  static constexpr int TILE = D / 64 * PANEL;
  static constexpr int CRB = D * BITS / 8;
  static constexpr int PRB = D / GS * 4;
  static constexpr int HALF = kTileRows * (CRB + PRB);
  static constexpr int O_Q = 0;
  static constexpr int O_K = QT * QTILE;
  static constexpr int O_V = O_K + KB * TILE;
  static constexpr int O_PLAN = O_V + KB * TILE;
  static constexpr int O_TMP = (O_PLAN + (kPlanMax + 1) * 12 + 4 + 15) / 16 * 16;
  static constexpr int O_BAR = O_TMP + 34 * 8;
  static constexpr int O_MISC = O_BAR + 40 * 8;  // TMEM address, bad tiles [4][4]
  static constexpr int O_WALK = O_MISC + 64;         // the softmax warps' place in the tile list
  static constexpr int O_MAX = O_WALK + 16 * 256;    // f32 [2 tiles][QT][2 halves][128]
  static constexpr int SMEM = O_MAX + 2 * QT * 2 * 128 * 4 + 1024;  // + alignment of the tiles
  static constexpr int kSoftWarps = 8 * QT;
  static constexpr int kDequantWarps = 7;
  static constexpr int kMmaWarp = kSoftWarps + kDequantWarps;
  static constexpr int kThreads = (kMmaWarp + 1) * 32;  // 24 warps of 80 registers, or 16 of 128
  static constexpr int TM_O = 256;              // TMEM columns: S at 0 and 128, O from 256
  static constexpr int PIECE = MR * (D + 2);    // floats: m [MR], l [MR], O [D / 4][MR][4]
  static_assert(SMEM <= 232448, "shared memory");
};

// log2 of what a probability is multiplied by before it is rounded; the sums
// above and below the line carry it alike.  bf16 has exponents to spare the other
// way: 2^31 keys of V's largest value stay in range of the f32 sums.
template <bool BF>
constexpr float kLift = BF ? -40.0f : 7.0f;

struct ChunkBars {
  uint64_t q_full[2], s_full[2], p_full[2], o_done[2];
  uint64_t k_full[2], v_full[2], k_empty[4], v_empty[4];
  uint64_t x[2][4][2];  // the exchange of two warps with the same rows, alternating
};

// The segments (runs of tiles inside one unit) of a CTA, walked by each role.
template <int BITS, int D, int GS>
struct Walk {
  using C = Chunk<BITS, D, GS>;
  Plan P;
  int gi, h, i0, i1;   // tiles [i0, i1) of the unit's list
  long long left;
  Block k;

  __device__ __forceinline__ void start(const AttnArgs& a, const Plan& plan, long long t0, long long t1) {
    P = plan;
    left = t1 - t0;
    if (left <= 0) return;
    const int Hkv = a.v.Hkv;
    int x = 0, y = P.NG;
    while (y - x > 1) {
      const int mid = (x + y) >> 1;
      if (P.tpre[mid] * Hkv <= t0) x = mid;
      else y = mid;
    }
    gi = x;
    k = get_block<C::MR, C::KL>(a, P, gi);
    const long long rel = t0 - P.tpre[gi] * Hkv;
    h = (int)(rel / k.nt);
    i0 = (int)(rel - (long long)h * k.nt);
    i1 = (int)min((long long)k.nt, i0 + left);
  }
  __device__ __forceinline__ bool valid() const { return left > 0; }
  __device__ __forceinline__ void next(const AttnArgs& a) {
    left -= i1 - i0;
    if (left <= 0) return;
    if (++h == a.v.Hkv) {
      h = 0;
      do {
        gi++;
      } while (P.tpre[gi + 1] == P.tpre[gi]);
      k = get_block<C::MR, C::KL>(a, P, gi);
    }
    i0 = 0;
    i1 = (int)min((long long)k.nt, left);
  }
};

// 8 codes to 8 dtype values code * s + z, one rounding.  4-bit words give them
// in the order 0 4 1 5 2 6 3 7 (Q is laid out alike, and O's columns are put
// back when they are written), 8-bit words in their own.
template <int BITS, bool BF>
struct Dequant {
  uint32_t s2, z2;  // scale and bias, twice
  float sf, zf;
  __device__ __forceinline__ explicit Dequant(uint32_t pair) {
    s2 = prmt(pair, 0u, 0x1010u);
    z2 = prmt(pair, 0u, 0x3232u);
    sf = attn::dt_to_f<BF>((uint16_t)pair);
    zf = attn::dt_to_f<BF>((uint16_t)(pair >> 16));
  }
  static __device__ __forceinline__ uint32_t fma_h(uint32_t c, uint32_t s, uint32_t z) {
    const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&c), *reinterpret_cast<__half2*>(&s),
                              *reinterpret_cast<__half2*>(&z));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint32_t fma_b(uint32_t c, uint32_t s, uint32_t z) {
    const __nv_bfloat162 r =
        __hfma2(*reinterpret_cast<__nv_bfloat162*>(&c), *reinterpret_cast<__nv_bfloat162*>(&s),
                *reinterpret_cast<__nv_bfloat162*>(&z));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  // w: 1 word of 4-bit or 2 words of 8-bit codes
  __device__ __forceinline__ uint4 eight(const uint32_t* w) const {
    uint32_t r[4];
    if constexpr (BITS == 4) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (BF) {
          // 128 + c, minus 128
          const uint32_t x = ((w[0] >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
          r[i] = fma_b(fma_b(x, 0x3f803f80u, 0xc300c300u), s2, z2);
        } else {
          // 1024 + c minus 1024; odd nibbles (1024 + 16 c) / 16 - 64
          const uint32_t y = i >= 2 ? w[0] >> 8 : w[0];
          const uint32_t x = (y & ((i & 1) ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
          r[i] = fma_h((i & 1) ? fma_h(x, 0x2c002c00u, 0xd400d400u) : fma_h(x, 0x3c003c00u, 0xe400e400u),
                       s2, z2);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t u = w[i >> 1];
        if constexpr (BF) {
          // codes up to 255 have no bf16 form with a free offset: f32, rounded once
          float2 x = make_float2(__uint_as_float(prmt(u, 0x4b000000u, (i & 1) ? 0x7442u : 0x7440u)),
                                 __uint_as_float(prmt(u, 0x4b000000u, (i & 1) ? 0x7443u : 0x7441u)));
          x = __fadd2_rn(x, make_float2(-8388608.0f, -8388608.0f));  // from 2^23 + c
          x = __ffma2_rn(x, make_float2(sf, sf), make_float2(zf, zf));
          const __nv_bfloat162 t = __floats2bfloat162_rn(x.x, x.y);
          r[i] = *reinterpret_cast<const uint32_t*>(&t);
        } else {
          const uint32_t x = prmt(u, 0x64646464u, (i & 1) ? 0x4342u : 0x4140u);
          r[i] = fma_h(fma_h(x, 0x3c003c00u, 0xe400e400u), s2, z2);
        }
      }
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
};

// UMMA with the descriptors' low words (address, leading offset) in registers;
// the high word (8-row groups 1024 B apart, 128-byte swizzle) is a constant.
constexpr uint32_t kDescHi = 64u | (1u << 14) | (2u << 29);
__device__ __forceinline__ void umma_ss_lo(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n"
      " mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, {%6, %6, %6, %6}, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHi), "r"(0u));
}
__device__ __forceinline__ void umma_ts_lo(uint32_t d, uint32_t a_tmem, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, {%6, %6, %6, %6}, p;\n}\n" ::"r"(d),
      "r"(a_tmem), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHi), "r"(0u));
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

// Wait of at most 2 s; the hint lets the thread sleep in the hardware meanwhile.
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity) {
  const uint32_t addr = attn::smem_u32(b);
  uint64_t t0 = 0;
  for (long long i = 0; i < attn::kWaitLimit; i++) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(addr), "r"(parity), "r"(100000u)
        : "memory");
    if (ok) return true;
    if ((i & 63) == 0) {
      const uint64_t now = attn::global_ns();
      if (i == 0) t0 = now;
      else if (now - t0 > attn::kWaitNs) return false;
    }
  }
  return false;
}

// position of list element i of a 4-bit word's eight values
__device__ __forceinline__ constexpr int nib_pos(int i) { return (i >> 1) + (i & 1) * 4; }

__device__ __forceinline__ uint32_t idesc_for(bool bf, int M, int N, int b_mn_major) {
  return attn::tc::idesc_f16(M, N, b_mn_major) | (bf ? (1u << 7) | (1u << 10) : 0u);
}

// n columns of a finished row to an `out` whose rows start anywhere, by element:
// not inlined, since a branch in the usual loop costs the call 1 to 3 %.
template <int BITS, bool BF>
__device__ __noinline__ void store_any(uint32_t tO, uint16_t* dst, float inv, bool live, int n) {
#pragma unroll 1
  for (int d = 0; d < n; d += 8) {
    uint32_t o[8];
    attn::tc::tmem_ld8(tO + d, o);
    attn::tc::tmem_wait_ld();
    if (!live) continue;
#pragma unroll
    for (int e = 0; e < 8; e++)
      dst[d + (BITS == 4 ? nib_pos(e) : e)] = attn::f_to_dt<BF>(__uint_as_float(o[e]) * inv);
  }
}

// Values that are not finite.  A row that does not see a key has p = 0 for it,
// but 0 times an infinite V is not 0, so the tensor core gets finite ones only:
// V that is not finite becomes 0 or the dtype's largest, and the rows that do
// see such a pair are marked when they are written.  Finite pairs whose value
// passes the dtype's range (the rounded scale times the last code does, in a row
// of its largest values) count as the range's end, K and V alike.  A K pair that
// is not finite stays: its logits are masked where they are hidden.
template <bool BF>
struct Range {
  static constexpr uint32_t kInf = BF ? 0x7f80u : 0x7c00u;
};

// Whether a row's values are all finite and in range (bf16: below 2^127, to be
// sure of the 8-bit codes' two roundings).  The last code's tells: a value is
// monotone in its code, code 0 gives the bias, which is in range if it is finite,
// and no finite value comes of a pair that is not.
template <int BITS, int NG, bool BF>
__device__ __forceinline__ bool pairs_in_range(const uint32_t (&pr)[NG]) {
  constexpr uint32_t kLast = BF ? (BITS == 4 ? 0x41704170u : 0x437f437fu) : (BITS == 4 ? 0x4b804b80u : 0x5bf85bf8u);
  constexpr uint32_t kStep = BF ? 0x01000100u : 0x04000400u;  // carries those exponents into the sign
  uint32_t out = 0;
#pragma unroll
  for (int e = 0; e < NG; e += 2) {
    const uint32_t other = pr[e + 1 < NG ? e + 1 : e];
    const uint32_t s = prmt(pr[e], other, 0x5410u), z = prmt(pr[e], other, 0x7632u);
    const uint32_t end = BF ? Dequant<BITS, BF>::fma_b(kLast, s, z) : Dequant<BITS, BF>::fma_h(kLast, s, z);
    out |= (end & 0x7fff7fffu) + kStep;
  }
  return (out & 0x80008000u) == 0;
}

// One dequantized row in its swizzled panels, and its groups' pairs.  Not inlined:
// the check and this call cost 512 rows over 16,896 keys 181 -> 184 us, inlined 186.
template <int N>
struct Pairs {
  uint32_t w[N];
};
template <int D, int GS, int PANEL, bool BF>
__device__ __noinline__ void hold_range(uint8_t* row, int r7, Pairs<D / GS> pr, bool is_v) {
  uint32_t bad = 0;
#pragma unroll
  for (int e = 0; e < D / GS; e++)
    if ((pr.w[e] & 0x7fffu) >= Range<BF>::kInf || ((pr.w[e] >> 16) & 0x7fffu) >= Range<BF>::kInf) bad |= 1u << e;
  constexpr uint32_t kInf = Range<BF>::kInf;
#pragma unroll 1
  for (int e = 0; e < D / 8; e++) {
    if (!is_v && ((bad >> (e * 8 / GS)) & 1u)) continue;
    uint32_t* w = reinterpret_cast<uint32_t*>(row + (e >> 3) * PANEL + (((e & 7) ^ r7) << 4));
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t x = (w[i >> 1] >> (16 * (i & 1))) & 0xffffu, m = x & 0x7fffu;
      if (m < kInf) continue;
      const uint32_t y = m > kInf ? 0u : (x & 0x8000u) | (kInf - 1);
      w[i >> 1] = (w[i >> 1] & ~(0xffffu << (16 * (i & 1)))) | (y << (16 * (i & 1)));
    }
  }
}

// The row at position p (of this lane; -1: none): NaN in its half of O wherever a
// V pair that it sees in the segment is not finite.  A lane reads the pairs of
// one key, every row takes those it sees.
template <int BITS, int D, int GS, bool BF>
__device__ __noinline__ void mark_lost(const AttnArgs& a, const Walk<BITS, D, GS>& wk, int p,
                                       uint32_t tO, int half) {
  using C = Chunk<BITS, D, GS>;
  constexpr uint32_t kInf = Range<BF>::kInf;
  const View& v = a.v;
  const Block& k = wk.k;
  const int lane = threadIdx.x & 31, klo = a.window > 0 ? max(0, k.pmin - a.window + 1) : 0;
  const int32_t* table = v.table + (int64_t)k.b * v.table_stride;
  uint32_t lost = 0;
#pragma unroll 1
  for (int n = 0; n < (wk.i1 - wk.i0) * (C::KT / 32); n++) {
    const int j0 = (tile_of(k, wk.i0 + n / (C::KT / 32)) << C::KL) + n % (C::KT / 32) * 32, j = j0 + lane;
    uint32_t bad = 0;
    if (j <= k.pmax && (j >= klo || j < a.sinks)) {
      const int page = table[j >> v.page_shift];
      if (page >= 0 && page < v.num_pages) {
        const uint8_t* src = tile_ptr(v, page, wk.h, (j & v.page_mask) >> 4) + C::HALF + kTileRows * C::CRB + (j & 15) * C::PRB;
        for (int g = 0; g < D / GS; g++) {
          const uint32_t pair = reinterpret_cast<const uint32_t*>(src)[g];
          if ((pair & 0x7fffu) >= kInf || ((pair >> 16) & 0x7fffu) >= kInf) bad |= 1u << g;
        }
      }
    }
    for (uint32_t any = __ballot_sync(0xffffffffu, bad != 0); any; any &= any - 1) {
      const int s = __ffs(any) - 1, jj = j0 + s;
      const uint32_t x = __shfl_sync(0xffffffffu, bad, s);
      if (jj <= p && (a.window == 0 || jj > p - a.window || jj < a.sinks)) lost |= x;
    }
  }
#pragma unroll 1
  for (int d = half * (D / 2); d < (half + 1) * (D / 2); d += 32) {
    const bool hit = (lost >> (d / GS)) & 1u;
    if (!__any_sync(0xffffffffu, hit)) continue;
    uint32_t o[32];
    attn::tc::tmem_ld32(tO + d, o);
    attn::tc::tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 32; e++) o[e] = hit ? 0x7fc00000u : o[e];
    attn::tc::tmem_st32(tO + d, o);
    attn::tc::tmem_wait_st();
  }
}

template <int BITS, int D, int GS, bool BF>
__global__ void __launch_bounds__(Chunk<BITS, D, GS>::kThreads, 1)
    chunk_kernel(const __grid_constant__ AttnArgs a, const Work ws) {
  using C = Chunk<BITS, D, GS>;
  using namespace attn::tc;
  constexpr int QT = C::QT, NG = D / GS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024 - (attn::smem_u32(smem_raw) & 1023)) & 1023);
  const View& v = a.v;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  ChunkBars& bar = *reinterpret_cast<ChunkBars*>(sm + C::O_BAR);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(sm + C::O_MISC);
  volatile uint8_t* s_bad = sm + C::O_MISC + 16;  // [4 tiles in flight][4 warps]
  // [4]: what the MMA warp is to do with a tile (first / last of a segment)
  volatile int* s_what = reinterpret_cast<volatile int*>(sm + C::O_MISC + 32);
  volatile int* s_lost = reinterpret_cast<volatile int*>(sm + C::O_MISC + 48);  // a V pair was not finite
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      attn::mbar_init(&bar.q_full[i], 256);
      attn::mbar_init(&bar.s_full[i], 1);
      attn::mbar_init(&bar.p_full[i], 256);
      attn::mbar_init(&bar.o_done[i], 1);
      attn::mbar_init(&bar.k_full[i], C::KT);
      attn::mbar_init(&bar.v_full[i], C::KT);
      attn::mbar_init(&bar.k_empty[i], 1);
      attn::mbar_init(&bar.k_empty[i + 2], 1);
      attn::mbar_init(&bar.v_empty[i], 1);
      attn::mbar_init(&bar.v_empty[i + 2], 1);
      for (int w = 0; w < 8; w++) attn::mbar_init(&bar.x[w >> 2][w & 3][i], 64);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *s_lost = 0;
  }
  if (warp == C::kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     attn::smem_u32(s_tmem)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Plan P;
  if (ws.tpre) {
    P = Plan{ws.gpre, ws.tpre, *ws.ng};
  } else {
    long long* tpre = reinterpret_cast<long long*>(sm + C::O_PLAN);
    int* gpre = reinterpret_cast<int*>(tpre + kPlanMax + 1);
    const int NG_ = build_plan<C::MR, C::KL>(a, gpre, tpre, ws.max_blocks,
                                         reinterpret_cast<long long*>(sm + C::O_TMP), blockIdx.x == 0);
    P = Plan{gpre, tpre, NG_};
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = *s_tmem;
  const long long RT = P.tpre[P.NG] * v.Hkv;
  const long long act = max(1ll, min((long long)gridDim.x, RT / 2));
  const long long c = blockIdx.x;
  const long long t0 = c < act ? c * RT / act : RT, t1 = c < act ? (c + 1) * RT / act : RT;
  // column blocks that see no key: zero rows
  for (long long gi = c; gi < P.NG; gi += gridDim.x) {
    if (P.tpre[gi + 1] != P.tpre[gi]) continue;
    const Block k = get_block<C::MR, C::KL>(a, P, (int)gi);
    for (int64_t e = tid; e < (int64_t)v.Hkv * k.cols * (D / 2); e += C::kThreads) {
      const int d = (int)(e % (D / 2)) * 2, x = (int)(e / (D / 2));
      store_out<1, BF>(a, k, x / k.cols, x % k.cols, d, 0.0f, 0.0f);
    }
  }
  // Bounded; a role that gives up leaves its loop, and the others' waits run
  // out in turn.  All lanes together.
  auto wait_all = [&](uint64_t* b, int parity) -> bool {
    if (__all_sync(0xffffffffu, bar_wait(b, (uint32_t)parity))) return true;
    gave_up(v);
    return false;
  };
  if (warp < C::kSoftWarps) {
    // --------------------------------- softmax: half of a row's keys a thread
    constexpr int VW = C::KT / 64;  // 32-key words of a half
    const int q = warp >> 3, half = (warp >> 2) & 1, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    // in shared memory, to spare registers
    static_assert(sizeof(Walk<BITS, D, GS>) <= 128, "walk");
    // (two places: the segment at hand and the next one)
    auto place = [&](int u) -> Walk<BITS, D, GS>& {
      return *reinterpret_cast<Walk<BITS, D, GS>*>(sm + C::O_WALK + warp * 256 + (u & 1) * 128);
    };
    float* s_max = reinterpret_cast<float*>(sm + C::O_MAX) + q * 256 + r;  // [half] 128 apart
    int xc = 0;  // exchanges so far
    // the other half's value for this row; false: it did not come
    auto exchange = [&](float& x) -> bool {
      float* p = s_max + (xc & 1) * QT * 256;
      p[half * 128] = x;
      uint64_t* b = &bar.x[q][warp & 3][xc & 1];
      attn::mbar_arrive(b);
      const bool there = wait_all(b, (xc >> 1) & 1);
      xc++;
      x = p[(half ^ 1) * 128];
      return there;
    };
    if (lane == 0) place(0).start(a, P, t0, t1);
    __syncwarp();
    // this CTA's pieces: nothing yet
    if (tid == 0) ws.meta[c] = make_int4(-1, 0, 0, 0);
    const float c2 = fmaxf(fabsf(a.scale) * attn::kLog2e, 1e-30f);  // never 0: -inf stays -inf
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
    int tc = 0;  // tiles so far
    bool ok = true;
    const int row = q * 128 + r;
    // the thread's half of its Q row; returns the row's position
    auto load_q = [&](const Walk<BITS, D, GS>& w_) -> int {
      const Block& k = w_.k;
      const bool live = row < k.cols;
      const int col = k.col0 + (live ? row : 0), tok = col / a.rep;
      const int head = w_.h * a.rep + (col - tok * a.rep);
      const uint16_t* src = a.q + (int64_t)(k.row0 + tok) * a.q_row + (int64_t)head * a.q_head;
      uint8_t* dst = sm + C::O_Q + q * C::QTILE;
#pragma unroll 4
      for (int e = half * (D / 16); e < (half + 1) * (D / 16); e++) {
        uint16_t x[8];
        if (ws.vec) {
          const uint4 y = *reinterpret_cast<const uint4*>(src + e * 8);
          const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] = src[e * 8 + i];
        }
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint32_t lo = x[BITS == 4 ? nib_pos(2 * i) : 2 * i];
          const uint32_t hi = x[BITS == 4 ? nib_pos(2 * i + 1) : 2 * i + 1];
          w[i] = live ? (lo | (hi << 16)) ^ flip : 0u;
        }
        *reinterpret_cast<uint4*>(dst + (e >> 3) * C::QPANEL + sw128(r, (e & 7) * 8)) =
            make_uint4(w[0], w[1], w[2], w[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      attn::mbar_arrive(&bar.q_full[q]);
      return live ? k.p0 + tok : -1;
    };
    int p = -1;
    if (place(0).valid()) p = load_q(place(0));
    for (int u = 0; place(u).valid(); u++) {
      const Walk<BITS, D, GS>& wk = place(u);
      const Block& k = wk.k;
      // where the CTA goes next, worked out while the first S is on its way
      __syncwarp();
      if (lane == 0) {
        place(u + 1) = wk;
        place(u + 1).next(a);
      }
      __syncwarp();
      float m = kNeg, l = 0.0f;
      const int i1 = wk.i1;
      for (int i = wk.i0; i < i1; i++, tc++) {
        const int sb = QT == 2 ? q : tc & 1;
        const uint32_t tS = tm + lanes + sb * 128 + half * (C::KT / 2);  // its keys' columns
        if (!wait_all(&bar.s_full[sb], QT == 2 ? tc & 1 : (tc >> 1) & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int kb = (tile_of(k, i) << C::KL) + half * (C::KT / 2);
        // two bits for each 32 keys: 16-key tiles without a page
        uint32_t bad2 = s_bad[(tc & 3) * 4 + half * VW];
        if (VW == 2) bad2 |= (uint32_t)s_bad[(tc & 3) * 4 + half * VW + 1] << 8;
        const bool full = kb + C::KT / 2 - 1 <= k.pmin && bad2 == 0 &&
                          (a.window == 0 || kb > k.pmax - a.window || kb + C::KT / 2 - 1 < a.sinks);
        uint32_t vis[VW];
        if (!full) {
          // bits of the keys that this row sees
#pragma unroll
          for (int w = 0; w < VW; w++) {
            const int j0 = kb + 32 * w;
            auto upto = [](int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); };
            uint32_t x = upto(p + 1 - j0);
            if (a.window > 0) x &= ~upto(p - a.window + 1 - j0) | upto(a.sinks - j0);
            const uint32_t b2 = (bad2 >> (8 * w)) & 3u;
            x &= ~(((b2 & 1u) ? 0x0000ffffu : 0u) | ((b2 & 2u) ? 0xffff0000u : 0u));
            vis[w] = x;
          }
        }
        float mx = kNeg;
#pragma unroll
        for (int w = 0; w < VW; w++) {
          uint32_t s[32];
          tmem_ld32(tS + 32 * w, s);
          tmem_wait_ld();
          if (full) {
#pragma unroll
            for (int e = 0; e < 32; e += 2)
              mx = fmaxf(mx, fmaxf(__uint_as_float(s[e]), __uint_as_float(s[e + 1])));
          } else {
#pragma unroll
            for (int e = 0; e < 32; e++)
              if ((vis[w] >> e) & 1u) mx = fmaxf(mx, __uint_as_float(s[e]));
          }
        }
        float other = mx;
        if (!exchange(other)) {
          ok = false;
          break;
        }
        mx = fmaxf(mx, other);
        mx = mx > 0.5f * kNeg ? mx * c2 : kNeg;
        // the same for both halves; m is the reference, kLift below a maximum
        if (__any_sync(0xffffffffu, mx > m + (8.0f + kLift<BF>))) {
          const float mn = fmaxf(m, mx - kLift<BF>), f = ex2(m - mn);
          m = mn;
          l *= f;
          if (i > wk.i0) {
            // every earlier product of this unit must have landed in O
            if (!wait_all(&bar.o_done[QT == 2 ? q : (tc - 1) & 1], QT == 2 ? (tc - 1) & 1 : ((tc - 1) >> 1) & 1)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int d = half * (D / 2); d < (half + 1) * (D / 2); d += 32) {
              uint32_t o[32];
              const uint32_t tO = tm + lanes + C::TM_O + q * D + d;
              tmem_ld32(tO, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(tO, o);
            }
            tmem_wait_st();
          }
        }
        const float2 cc = make_float2(c2, c2), mm = make_float2(-m, -m);
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < VW; w++) {
          uint32_t s[32], pk[16];
          tmem_ld32(tS + 32 * w, s);
          tmem_wait_ld();
          if (!full) {
#pragma unroll
            for (int e = 0; e < 32; e++)
              if (!((vis[w] >> e) & 1u)) s[e] = 0xff800000u;  // -inf: p is 0
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), cc, mm);
            const float2 y = make_float2(ex2(x.x), ex2(x.y));
            sum = __fadd2_rn(sum, y);
            if constexpr (BF) {
              const __nv_bfloat162 t = __floats2bfloat162_rn(y.x, y.y);
              pk[e / 2] = *reinterpret_cast<const uint32_t*>(&t);
            } else {
              pk[e / 2] = pack_h2(y.x, y.y);
            }
          }
          // over columns of S that this thread has read already
          tmem_st16(tS + 16 * w, pk);
        }
        l += sum.x + sum.y;
        tmem_wait_st();
        tc_fence_before();
        attn::mbar_arrive(&bar.p_full[sb]);
      }
      // Q is free: this row tile's last S is there.  The next unit's, so that its
      // first S follows while O is written.
      int p_next = -1;
      if (ok && place(u + 1).valid()) p_next = load_q(place(u + 1));
      if (!ok || !wait_all(&bar.o_done[QT == 2 ? q : (tc - 1) & 1], QT == 2 ? (tc - 1) & 1 : ((tc - 1) >> 1) & 1)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float rest = l;
      if (!exchange(rest)) {
        ok = false;
        break;
      }
      l += rest;
      // of any unit of the CTA so far; set before that tile's P V was issued
      if (__any_sync(0xffffffffu, *s_lost))
        mark_lost<BITS, D, GS, BF>(a, wk, p, tm + lanes + C::TM_O + q * D, half);
      const bool begun = wk.i0 == 0, ended = wk.i1 == k.nt, whole = begun && ended;
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
      const bool live = row < k.cols;
      const int col = k.col0 + (live ? row : 0), tok = col / a.rep;
      uint16_t* dst = a.out + ((int64_t)(k.row0 + tok) * a.Hq + wk.h * a.rep + (col - tok * a.rep)) * D;
      float* slot = ws.slots + (size_t)(2 * c + (begun ? 1 : 0)) * C::PIECE;
      if (!whole) {
        if (half == 0) {
          slot[row] = m;
          slot[C::MR + row] = l;
        }
        if (tid == 0) {
          if (begun) {
            ws.meta[c].x = wk.gi * v.Hkv + wk.h;
            ws.meta[c].y |= k.cols << 8;
            ws.meta[c].z = k.row0;
            ws.meta[c].w = k.col0;
          } else {
            ws.meta[c].y |= ended ? 2 : 1;
          }
        }
      }
      const int d0 = half * (D / 2);
      const bool apart = whole && a.out_align < 2;
      if (apart) store_any<BITS, BF>(tm + lanes + C::TM_O + q * D + d0, dst + d0, inv, live, D / 2);
#pragma unroll 1
      for (int d = d0; d < (apart ? d0 : d0 + D / 2); d += 32) {
        uint32_t o[32];
        tmem_ld32(tm + lanes + C::TM_O + q * D + d, o);
        tmem_wait_ld();
        float x[32];
#pragma unroll
        for (int e = 0; e < 32; e++)
          x[BITS == 4 ? (e & ~7) + nib_pos(e & 7) : e] = __uint_as_float(o[e]);
        if (whole) {
          if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; i++)
                w[i] = (uint32_t)attn::f_to_dt<BF>(x[e + 2 * i] * inv) |
                       ((uint32_t)attn::f_to_dt<BF>(x[e + 2 * i + 1] * inv) << 16);
              *reinterpret_cast<uint4*>(dst + d + e) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<float4*>(slot + 2 * C::MR + ((size_t)((d + e) / 4) * C::MR + row) * 4) =
                make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
        }
      }
      tc_fence_before();
      p = p_next;
    }
  } else if (warp < C::kMmaWarp) {
    // ------------------------- dequantize: 32-row blocks of K, then of V, of each tile
    constexpr int RW = C::CRB / 16;  // 16-byte words of a code row
    Walk<BITS, D, GS> wk;
    wk.start(a, P, t0, t1);
    int first = 0;  // tiles of the CTA before the walk's segment
    const int total = (int)(t1 - t0);
    // where block n's row lies: list index of its tile, position, page
    auto seek = [&](int n) {
      while ((n >> C::BL) - first >= wk.i1 - wk.i0) {
        first += wk.i1 - wk.i0;
        wk.next(a);
      }
    };
    auto key_of = [&](int n) { return (tile_of(wk.k, wk.i0 + (n >> C::BL) - first) << C::KL) + (n & (C::NBK - 1)) * 32 + lane; };
    auto page_of = [&](int j) -> int {  // -1: nobody sees the row
      if ((j >> 4) > (wk.k.pmax >> 4)) return -1;
      return __ldg(v.table + (int64_t)wk.k.b * v.table_stride + (j >> v.page_shift));
    };
    int n = warp - C::kSoftWarps, j = 0, page = -1;
    if (n < total << C::BL) {
      seek(n);
      j = key_of(n);
      page = page_of(j);
    }
    while (n < total << C::BL) {
      const int tc = n >> C::BL, quarter = n & (C::NBK - 1);
      const bool is_v = n & C::NBK;
      const Block& k = wk.k;
      const int klo = a.window > 0 ? max(0, k.pmin - a.window + 1) : 0;
      const bool wanted = j <= k.pmax && (j >= klo || j < a.sinks);
      const bool here = (j >> 4) <= (k.pmax >> 4);
      const bool found = page >= 0 && page < v.num_pages;
      const int li = wk.i0 + tc - first;
      const int what = (li == wk.i0 ? 1 : 0) | (li + 1 == wk.i1 ? 2 : 0);
      uint4 raw[RW];
      uint32_t pr[NG];
      if (wanted && found) {
        const uint8_t* src = tile_ptr(v, page, wk.h, (j & v.page_mask) >> 4) + (is_v ? C::HALF : 0);
        const uint4* cw = reinterpret_cast<const uint4*>(src + (j & 15) * C::CRB);
#pragma unroll
        for (int e = 0; e < RW; e++) raw[e] = __ldg(cw + e);
#pragma unroll
        for (int e = 0; e < NG; e++)
          pr[e] = __ldg(reinterpret_cast<const uint32_t*>(src + kTileRows * C::CRB + (j & 15) * C::PRB) + e);
      } else {
#pragma unroll
        for (int e = 0; e < RW; e++) raw[e] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int e = 0; e < NG; e++) pr[e] = 0u;
      }
      const unsigned lost = __ballot_sync(0xffffffffu, here && wanted && !found);
      // the next block's page, on its way while this one is converted
      n += C::kDequantWarps;
      if (n < total << C::BL) {
        seek(n);
        j = key_of(n);
        page = page_of(j);
      }
      const bool in_range = pairs_in_range<BITS, NG, BF>(pr);
      const int buf = tc & 1;
      // the buffer's last reader was tile tc - 2.  Four barriers by that tile's
      // number: a warp that had no V block for some tiles may be several releases
      // behind, which fewer barriers' parities cannot tell apart.
      const int was = tc - C::KB;
      if (was >= 0 && !wait_all(is_v ? &bar.v_empty[was & 3] : &bar.k_empty[was & 3], (was >> 2) & 1)) break;
      const int r = quarter * 32 + lane;
      uint8_t* dst = sm + (is_v ? C::O_V : C::O_K) + buf * C::TILE + (r >> 3) * 1024 + (r & 7) * 128;
#pragma unroll
      for (int e = 0; e < D / 8; e++) {
        const Dequant<BITS, BF> dq(pr[e * 8 / GS]);
        const uint32_t* words = reinterpret_cast<const uint32_t*>(raw) + e * BITS / 4;
        *reinterpret_cast<uint4*>(dst + (e >> 3) * C::PANEL + (((e & 7) ^ (r & 7)) << 4)) = dq.eight(words);
      }
      if (!in_range) {
        Pairs<NG> all;
#pragma unroll
        for (int e = 0; e < NG; e++) all.w[e] = pr[e];
        if (is_v) *s_lost = 1;
        hold_range<D, GS, C::PANEL, BF>(dst, r & 7, all, is_v);
      }
      if (!is_v && lane == 0) {
        s_bad[(tc & 3) * 4 + quarter] = (uint8_t)(((lost & 0xffffu) ? 1 : 0) | ((lost >> 16) ? 2 : 0));
        if (lost) raise(v);
        if (quarter == 0) s_what[tc & 3] = what;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      attn::mbar_arrive(is_v ? &bar.v_full[buf] : &bar.k_full[buf]);
    }
  } else {
    // ------------------------------------------------------------ MMA issue
    const uint32_t iqk = idesc_for(BF, 128, C::KT, 0), ipv = idesc_for(BF, 128, D, 1);
    // low descriptor words; V's 64-element panels lie PANEL bytes apart
    const uint32_t dq0 = (attn::smem_u32(sm + C::O_Q) >> 4) | (1u << 16);
    const uint32_t dk0 = (attn::smem_u32(sm + C::O_K) >> 4) | (1u << 16);
    const uint32_t dv0 = (attn::smem_u32(sm + C::O_V) >> 4) | ((uint32_t)(C::PANEL >> 4) << 16);
    bool ok = true;
    // The whole warp runs this role, so that addresses and descriptors stay in
    // uniform registers; one elected lane issues.
    auto qk = [&](int q, int t) {  // S of row tile q, tile t
      const int buf = t & 1;
      const uint32_t dS = tm + (QT == 2 ? q : t & 1) * 128;
      if (!elect_one()) return;
#pragma unroll
      for (int ks = 0; ks < D / 16; ks++) {
        const uint32_t oq = (ks >> 2) * C::QPANEL + 32 * (ks & 3), ok_ = (ks >> 2) * C::PANEL + 32 * (ks & 3);
        umma_ss_lo(dS, dq0 + ((q * C::QTILE + oq) >> 4), dk0 + ((buf * C::TILE + ok_) >> 4), iqk, ks ? 1u : 0u);
      }
      umma_commit(&bar.s_full[QT == 2 ? q : t & 1]);
    };
    auto pv = [&](int q, int t, bool first) {
      const int buf = t & 1;
      const uint32_t tP = tm + (QT == 2 ? q : t & 1) * 128;
      if (!elect_one()) return;
#pragma unroll
      for (int ks = 0; ks < C::KT / 16; ks++)
        umma_ts_lo(tm + C::TM_O + q * D, tP + 8 * (ks % (C::KT / 32)) + C::KT / 2 * (ks / (C::KT / 32)), dv0 + ((buf * C::TILE + 2048 * ks) >> 4), ipv,
                (first && ks == 0) ? 0u : 1u);
      umma_commit(&bar.o_done[QT == 2 ? q : t & 1]);
    };
    auto commit = [&](uint64_t* b) {
      if (elect_one()) umma_commit(b);
    };
    auto kwait = [&](int t) { return wait_all(&bar.k_full[t & 1], (t >> 1) & 1); };
    auto vwait = [&](int t) { return wait_all(&bar.v_full[t & 1], (t >> 1) & 1); };
    // A tile's products S are issued before the turn of its predecessor's P V
    // ends; `what` says when that predecessor belongs to another unit.
    auto start = [&](int t, int u) {  // the first tile of a segment
      for (int q = 0; q < QT; q++)
        if (!wait_all(&bar.q_full[q], u & 1)) return false;
      tc_fence_after();
      for (int q = 0; q < QT; q++) qk(q, t);
      commit(&bar.k_empty[t & 3]);
      return true;
    };
    const int total = (int)(t1 - t0);
    int u = 0;
    for (int tc = 0; tc < total && ok; tc++) {
      if (tc == 0 && !(kwait(0) && start(0, 0))) break;
      const int what = s_what[tc & 3];
      const bool first = what & 1, more = !(what & 2);
      if constexpr (QT == 2) {
        // V and the next K are there early; a row tile's P is what it waits for
        ok = vwait(tc) && (!more || kwait(tc + 1)) && wait_all(&bar.p_full[0], tc & 1);
        if (!ok) break;
        tc_fence_after();
        pv(0, tc, first);
        if (more) qk(0, tc + 1);
        if (!(ok = wait_all(&bar.p_full[1], tc & 1))) break;
        tc_fence_after();
        pv(1, tc, first);
        commit(&bar.v_empty[tc & 3]);
        if (more) {
          qk(1, tc + 1);
          commit(&bar.k_empty[(tc + 1) & 3]);
        }
      } else {
        if (more) {
          if (!(ok = kwait(tc + 1))) break;
          tc_fence_after();
          qk(0, tc + 1);
          commit(&bar.k_empty[(tc + 1) & 3]);
        }
        ok = vwait(tc) && wait_all(&bar.p_full[tc & 1], (tc >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        pv(0, tc, first);
        commit(&bar.v_empty[tc & 3]);
      }
      if (!more && tc + 1 < total) ok = kwait(tc + 1) && start(tc + 1, ++u);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == C::kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512));
  }
}

// Block (c, y): 32 rows of the unit that begins in CTA c and goes on; its
// pieces are slot 1 of c and slot 0 of the CTAs after it, in that order.  Warp
// w takes D / 8 columns.
template <int BITS, int D, int GS, bool BF>
__global__ void __launch_bounds__(256) chunk_merge_kernel(const AttnArgs a, const Work ws) {
  using C = Chunk<BITS, D, GS>;
  constexpr int NV = D / 32;  // float4s a thread holds
  __shared__ int s_end;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x, n = gridDim.x, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int4 where = ws.meta[c];
  if (where.x < 0) return;
  if (tid == 0) s_end = n - 1;
  __syncthreads();
  for (int i = c + 1 + tid; i < n; i += 256)
    if ((ws.meta[i].y & 255) == 2) atomicMin(&s_end, i);
  __syncthreads();
  const int last = s_end;
  Block k;
  k.cols = where.y >> 8;
  k.row0 = where.z;
  k.col0 = where.w;
  const int row = blockIdx.y * 32 + lane;
  float m = kNeg, l = 0.0f;
  float4 o[NV];
#pragma unroll
  for (int i = 0; i < NV; i++) o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i = c; i <= last; i++) {
    const float* p = ws.slots + (size_t)(i == c ? 2 * c + 1 : 2 * i) * C::PIECE;
    const float pm = p[row], pl = p[C::MR + row];
    float4 z[NV];
#pragma unroll
    for (int e = 0; e < NV; e++)
      z[e] = *reinterpret_cast<const float4*>(p + 2 * C::MR + ((size_t)(w * NV + e) * C::MR + row) * 4);
    const float mn = fmaxf(m, pm), f = ex2(m - mn), g = ex2(pm - mn);
    m = mn;
    l = fmaf(g, pl, l * f);
#pragma unroll
    for (int e = 0; e < NV; e++) {
      o[e].x = fmaf(g, z[e].x, o[e].x * f);
      o[e].y = fmaf(g, z[e].y, o[e].y * f);
      o[e].z = fmaf(g, z[e].z, o[e].z * f);
      o[e].w = fmaf(g, z[e].w, o[e].w * f);
    }
  }
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  const int h = where.x % a.v.Hkv;
#pragma unroll
  for (int e = 0; e < NV; e++) {
    const int d = (w * NV + e) * 4;
    store_out<1, BF>(a, k, h, row, d, o[e].x * inv, o[e].y * inv);
    store_out<1, BF>(a, k, h, row, d + 2, o[e].z * inv, o[e].w * inv);
  }
}

template <int BITS, int D, int GS, bool BF>
int32_t launch_chunk_one(const AttnArgs& a, const Work& ws, int ctas, int dev, cudaStream_t st) {
  using C = Chunk<BITS, D, GS>;
  auto kern = chunk_kernel<BITS, D, GS, BF>;
  auto merge = chunk_merge_kernel<BITS, D, GS, BF>;
  int32_t rc = kernel_setup(reinterpret_cast<const void*>(kern), C::kThreads, C::SMEM, dev, nullptr);
  if (rc) return rc;
  if ((rc = kernel_carveout(reinterpret_cast<const void*>(merge), dev))) return rc;
  if (ws.tpre) KVQ_CUDA_TRY(launch_pdl(plan_kernel<C::MR, C::KL>, dim3(1), dim3(1024), 0, st, a, ws));
  KVQ_CUDA_TRY(launch_pdl(kern, dim3((unsigned)ctas), dim3(C::kThreads), C::SMEM, st, a, ws));
  KVQ_CUDA_TRY(launch_pdl(merge, dim3((unsigned)ctas, C::MR / 32), dim3(256), 0, st, a, ws));
  return KVQ_OK;
}

// Defined for each (bits, dtype) in its own file.
template <int BITS, bool BF>
int32_t launch_chunk(const AttnArgs& a, const Work& ws, int ctas, int dev, cudaStream_t st);

template <int BITS, bool BF>
int32_t launch_chunk_impl(const AttnArgs& a, const Work& ws, int ctas, int dev, cudaStream_t st) {
#define KVQ_CHUNK(DD, GG) \
  if (a.v.D == DD && a.v.gs == GG) return launch_chunk_one<BITS, DD, GG, BF>(a, ws, ctas, dev, st);
  KVQ_CHUNK(64, 32)
  KVQ_CHUNK(64, 64)
  KVQ_CHUNK(128, 32)
  KVQ_CHUNK(128, 64)
  KVQ_CHUNK(128, 128)
  KVQ_CHUNK(256, 32)
  KVQ_CHUNK(256, 64)
  KVQ_CHUNK(256, 128)
#undef KVQ_CHUNK
  return fail(KVQ_ERR_ARG, "paged: unsupported head_dim / group_size");
}

}  // namespace paged
}  // namespace kvq
