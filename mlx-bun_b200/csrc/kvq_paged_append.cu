// kvq_paged_append.cu — RoPE, quantize and write into pages, one launch.
//
// Per token row at position p: angle_i = (scale * p) * inv_freq_i and its
// cosine and sine in 64 bits, (x, y) -> (x cos - y sin, x sin + y cos) for K and
// Q to well beyond 32 bits, rounded to 32 bits and then to the dtype; K and V
// rows then go through the affine group rule of kvq_qrule.cuh into their page.
// A 32-bit angle at position 131,072 is off by up to 0.004 rad, more than a bf16
// step of the result; and with products this exact the rounded values, and so
// the codes, do not depend on how they are computed.
//
// The rotation itself is done on pairs of floats (cos = ch + cl, sin = sh + sl,
// x and y exact): products split by fma, one two-sum, the small terms added at
// the end, an error of about 2^-46 of the larger product.  64-bit arithmetic
// would need its conversions, which run at an eighth of the rate.
//
// A block takes one to four token rows (their cosines and sines are computed
// once, in shared memory) and a share of the rows' units; a unit is 8
// consecutive elements of a K or V row (quantized by the group's lanes with
// shuffles) or 8 elements and their 8 rotation partners of a Q row (so that q
// may be rotated in place).
#include "kvq_paged.cuh"
#include "kvq_qrule.cuh"

namespace kvq {
namespace paged {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;
constexpr int kMaxRows = 4;  // rows of a block
constexpr int kSms = 148;    // of a B200

template <bool BF>
__device__ __forceinline__ float to_f(uint16_t v) {
  if constexpr (BF) return __uint_as_float((uint32_t)v << 16);
  else return __half2float(__ushort_as_half(v));
}
template <bool BF>
__device__ __forceinline__ uint16_t to_bits(float f) {
  if constexpr (BF) return __bfloat16_as_ushort(__float2bfloat16_rn(f));
  else return __half_as_ushort(__float2half_rn(f));
}
template <bool BF>
__device__ __forceinline__ float2 to_f2(uint32_t w) {
  if constexpr (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF>
__device__ __forceinline__ uint32_t to_bits2(float2 f) {
  if constexpr (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// The angles of one row.  Pairs 2 j and 2 j + 1 share an entry: their cosines'
// high and low parts in `c`, their sines' in `s` (x, y high; z, w low).  Eight
// consecutive pairs are one unit's, so entry j sits at slot (j % 4) * stride + j
// / 4 and neighbouring lanes read neighbouring slots.
struct Angle2 {
  float4 c, s;
};
struct Table {
  const float4 *c, *s;
  int stride;
  __device__ __forceinline__ Angle2 at2(int j) const {
    const int k = (j & 3) * stride + (j >> 2);
    return Angle2{c[k], s[k]};
  }
};

// Two pairs at once: x cos + y sin, rounded to 32 bits and then to the dtype
template <bool BF>
__device__ __forceinline__ uint32_t turn2(float2 x, float2 y, const Angle2& a) {
  const float2 ch = make_float2(a.c.x, a.c.y), cl = make_float2(a.c.z, a.c.w);
  const float2 sh = make_float2(a.s.x, a.s.y), sl = make_float2(a.s.z, a.s.w);
  const float2 one = make_float2(-1.0f, -1.0f);
  const float2 p = __fmul2_rn(x, ch), q = __fmul2_rn(y, sh);
  const float2 pe = __ffma2_rn(x, ch, make_float2(-p.x, -p.y));
  const float2 qe = __ffma2_rn(y, sh, make_float2(-q.x, -q.y));
  const float2 hi = __fadd2_rn(p, q);
  const float2 b = __ffma2_rn(p, one, hi);    // hi - p
  const float2 bp = __ffma2_rn(b, one, hi);   // hi - b
  float2 lo = __fadd2_rn(__ffma2_rn(bp, one, p), __ffma2_rn(b, one, q));
  lo = __fadd2_rn(lo, __fadd2_rn(pe, qe));
  lo = __ffma2_rn(x, cl, __ffma2_rn(y, sl, lo));
  float2 r = __fadd2_rn(hi, lo);
  // infinite inputs leave no finite remainder
  if (lo.x != lo.x) r.x = hi.x;
  if (lo.y != lo.y) r.y = hi.y;
  return to_bits2<BF>(r);
}
// one pair i of the same table
template <bool BF>
__device__ __forceinline__ uint16_t turn1(float x, float y, const Table& T, int i) {
  const Angle2 a = T.at2(i >> 1);
  return (uint16_t)(turn2<BF>(make_float2(x, x), make_float2(y, y), a) >> (16 * (i & 1)));
}

// The 8 elements from e0 of a row after rotation; o: their rotation partners
// (not traditional).  All 8 rotate, in the same half.
template <bool BF>
__device__ __forceinline__ void rotate8(uint32_t (&y)[4], const uint32_t (&o)[4], int e0, const RopeArgs& r,
                                        const Table& T) {
  if (r.traditional) {
    // words are (x, y) pairs: regroup into two x and two y
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const float2 a = to_f2<BF>(y[i]), b = to_f2<BF>(y[i + 1]);
      const Angle2 t = T.at2((e0 >> 2) + (i >> 1));
      const float2 u = make_float2(a.x, b.x), v = make_float2(a.y, b.y);
      const uint32_t p = turn2<BF>(u, make_float2(-v.x, -v.y), t), q = turn2<BF>(v, u, t);
      y[i] = __byte_perm(p, q, 0x5410);
      y[i + 1] = __byte_perm(p, q, 0x7632);
    }
    return;
  }
  const bool lo = e0 < r.half;
  const int j = (lo ? e0 : e0 - r.half) >> 1;
  const uint32_t flip = lo ? 0x80008000u : 0u;
#pragma unroll
  for (int i = 0; i < 4; i++)
    y[i] = turn2<BF>(to_f2<BF>(y[i]), to_f2<BF>(o[i] ^ flip), T.at2(j + i));
}

// Quantize the 8 elements y of element e0.. of a K or V row; the group's
// gs / 8 lanes hold its other elements.
template <bool BF, int BITS, int GS>
__device__ __forceinline__ void quantize8(const uint32_t (&y)[4], int e0, uint8_t* codes, uint8_t* pairs) {
  constexpr float NB = (float)((1 << BITS) - 1);
  float w[8];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = to_f2<BF>(y[i]);
    w[2 * i] = f.x;
    w[2 * i + 1] = f.y;
  }
  float mn = w[0], mx = w[0];
#pragma unroll
  for (int i = 1; i < 8; i++) {
    mn = fminf(mn, w[i]);
    mx = fmaxf(mx, w[i]);
  }
  constexpr int lanes = GS >> 3;
  const int lane = threadIdx.x & 31;
  const unsigned mask = (0xffffffffu >> (32 - lanes)) << (lane & ~(lanes - 1));
#pragma unroll
  for (int o = 1; o < lanes; o <<= 1) {
    mn = fminf(mn, __shfl_xor_sync(mask, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(mask, mx, o));
  }
  float scale, bias;
  quant_params(mn, mx, NB, scale, bias);
  // The rule's code is round((w - bias) / scale), half away from zero, of the
  // IEEE quotient.  With r = 1 / scale the product (w - bias) r is within 2^-22
  // of the quotient relatively, 6.1e-5 for codes up to 255, so its nearest
  // integer is the code unless it lies within 1e-4 of a half; only then (ties
  // of short mantissas, mostly) is the division itself done.  Adding 1.5 2^23
  // leaves the integer in the low bits of the sum.
  const float rs = __frcp_rn(scale);
  constexpr float kMagic = 12582912.0f;
  constexpr uint32_t kMagicBits = 0x4b400000u;
  uint32_t word[BITS / 4] = {};
  unsigned near = fabsf(scale) < 1e30f ? 0u : 0xffu;  // elements to divide
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float q = fminf(fmaxf((w[i] - bias) * rs, 0.0f), NB);
    const float t = q + kMagic;
    if (fabsf(q - (t - kMagic)) > 0.4999f) near |= 1u << i;
    word[i * BITS / 32] += (__float_as_uint(t) - kMagicBits) << (i * BITS % 32);
  }
  while (near) {
    const int i = __ffs(near) - 1;
    near &= near - 1;
    const uint32_t yw = i < 4 ? (i < 2 ? y[0] : y[1]) : (i < 6 ? y[2] : y[3]);
    const uint32_t c = quant_code(to_f<BF>((uint16_t)(yw >> (16 * (i & 1)))), scale, bias, NB);
    const int sh = i * BITS % 32;
#pragma unroll
    for (int k = 0; k < BITS / 4; k++)
      if (i * BITS / 32 == k) word[k] = (word[k] & ~(((1u << BITS) - 1u) << sh)) | (c << sh);
  }
  uint8_t* dst = codes + e0 * BITS / 8;
  if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(dst) = word[0];
  else *reinterpret_cast<uint2*>(dst) = make_uint2(word[0], word[1]);
  if ((e0 & (GS - 1)) == 0)
    *reinterpret_cast<uint32_t*>(pairs + e0 / GS * 4) =
        (uint32_t)to_bits<BF>(scale) | ((uint32_t)to_bits<BF>(bias) << 16);
}

// What a block knows of its rows: positions, pages, angles.
struct Shared {
  float4 c[kMaxRows][kMaxHalf / 2], s[kMaxRows][kMaxHalf / 2];
  double inv[kMaxHalf];
  int pos[kMaxRows], page[kMaxRows];  // page: -2 no such row, -1 no page
};

// Each row's sequence, position and page by one warp, the frequencies by the
// others meanwhile; then the angles by all.  Returns the angles' slot stride.
__device__ __forceinline__ int place_rows(Shared& sh, const AppendArgs& a, int t0, int nr) {
  const View& v = a.v;
  const RopeArgs& r = a.rope;
  const int tid = threadIdx.x, lane = tid & 31;
  if (tid >> 5 < nr) {
    const int k = tid >> 5, t = t0 + k;
    int b = t;
    if (v.cu) {
      b = 0;
      for (int b0 = 0; b0 < v.B; b0 += 32)
        b += __popc(__ballot_sync(0xffffffffu, b0 + lane < v.B && v.cu[min(b0 + lane, v.B - 1) + 1] <= t));
    }
    if (lane == 0) {
      int pos = -1, page = -2;
      if (b < v.B) {
        int row0, n, len;
        seq_rows(v, b, row0, n, len);
        pos = len - n + (t - row0);
        if (t < row0 || n <= 0 || pos < 0 || (pos >> v.page_shift) >= v.max_pages) {
          if (blockIdx.y == 0) raise(v);
        } else {
          page = v.table[(int64_t)b * v.table_stride + (pos >> v.page_shift)];
          if (page < 0 || page >= v.num_pages) {
            page = -1;
            if (blockIdx.y == 0) raise(v);
          }
        }
      }
      sh.pos[k] = pos;
      sh.page[k] = page;
    }
  }
  for (int i = kThreads - 1 - tid; i < r.half; i += kThreads)
    sh.inv[i] = r.freqs ? 1.0 / (double)r.freqs[i] : pow(r.base, -2.0 * (double)i / (double)r.dims);
  __syncthreads();
  const int stride = (r.half + 7) >> 3;
  for (int i = tid; i < nr * r.half; i += kThreads) {
    const int k = i / r.half, e = i - k * r.half, j = e >> 1;
    double s, c;
    sincos((r.scale * (double)sh.pos[k]) * sh.inv[e], &s, &c);
    c *= r.pre;
    s *= r.pre;
    const float ch = (float)c, sn = (float)s;
    const int at = ((j & 3) * stride + (j >> 2)) * 4 + (e & 1);
    float* pc = reinterpret_cast<float*>(sh.c[k]) + at;
    float* ps = reinterpret_cast<float*>(sh.s[k]) + at;
    pc[0] = ch;
    pc[2] = (float)(c - (double)ch);
    ps[0] = sn;
    ps[2] = (float)(s - (double)sn);
  }
  __syncthreads();
  return stride;
}

__device__ __forceinline__ void unpack(uint32_t (&x)[4], const uint4& u) {
  x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
}

// grid (row groups, parts): a block takes R rows from R * blockIdx.x and the
// units part * kThreads + threadIdx.x, + parts * kThreads, ... of each.  A thread
// works a unit's place in the row out once, and the next row's loads are on
// their way while one is computed.  16-byte accesses, rotation halves that split
// into eights.
template <bool BF, int BITS, int GS, int R>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ Shared sh;
  const View& v = a.v;
  const RopeArgs& r = a.rope;
  const int t0 = blockIdx.x * R, tid = threadIdx.x, nr = min(R, v.rows - t0);
  const int stride = place_rows(sh, a, t0, nr);
  const int D = v.D, per_log2 = __ffs(D) - 4;  // units of 8 in a row
  const int kv_units = v.Hkv << per_log2;
  const int crb = code_row_bytes(D, BITS), prb = pair_row_bytes(D, v.gs);
  // Q units of a head: rotated ones, then the rest of the row
  const int q_rot = r.traditional ? r.dims >> 3 : r.half >> 3;
  const int q_head_units = a.q ? q_rot + ((D - r.dims) >> 3) : 0;
  const int units = 2 * kv_units + a.Hq * q_head_units;
  for (int x = blockIdx.y * kThreads + tid; x < units; x += gridDim.y * kThreads) {
    const bool is_q = x >= 2 * kv_units, is_v = !is_q && x >= kv_units;
    int h, e0, other;  // elements from e0, their partners from `other`
    const uint16_t* src;
    int64_t row;       // elements between rows
    bool rot;
    if (is_q) {
      const int k = x - 2 * kv_units;
      h = k / q_head_units;
      const int j = k - h * q_head_units;
      rot = j < q_rot;
      e0 = rot ? j << 3 : r.dims + ((j - q_rot) << 3);
      other = rot && !r.traditional ? e0 + r.half : e0;
      src = a.q + h * a.q_head;
      row = a.q_row;
    } else {
      const int k = is_v ? x - kv_units : x;
      h = k >> per_log2;
      e0 = (k - (h << per_log2)) << 3;
      rot = !is_v && e0 < r.dims;
      other = rot && !r.traditional ? (e0 < r.half ? e0 + r.half : e0 - r.half) : e0;
      src = is_v ? a.val + h * a.v_head : a.k + h * a.k_head;
      row = is_v ? a.v_row : a.k_row;
    }
    src += t0 * row;
    uint4 own = *reinterpret_cast<const uint4*>(src + e0);
    uint4 far = *reinterpret_cast<const uint4*>(src + other);
#pragma unroll 1
    for (int k = 0; k < nr; k++) {
      const int page = sh.page[k];
      const Table T{sh.c[k], sh.s[k], stride};
      uint32_t y[4], o[4];
      unpack(y, own);
      unpack(o, far);
      if (k + 1 < nr) {
        src += row;
        own = *reinterpret_cast<const uint4*>(src + e0);
        far = *reinterpret_cast<const uint4*>(src + other);
      }
      if (page == -2) continue;
      if (!is_q) {
        if (rot) rotate8<BF>(y, o, e0, r, T);
        if (page >= 0) {
          const int pos = sh.pos[k], pr = pos & (kTileRows - 1);
          uint8_t* tile = tile_ptr(v, page, h, (pos & v.page_mask) >> 4) + (is_v ? kTileRows * (crb + prb) : 0);
          quantize8<BF, BITS, GS>(y, e0, tile + pr * crb, tile + kTileRows * crb + pr * prb);
        }
        continue;
      }
      uint16_t* dst = a.q_out + ((int64_t)(t0 + k) * a.Hq + h) * D + e0;
      if (rot && !r.traditional) {
        uint32_t z[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const Angle2 t = T.at2((e0 >> 1) + i);
          const float2 p = to_f2<BF>(y[i]), q = to_f2<BF>(o[i]);
          z[i] = turn2<BF>(q, p, t);
          y[i] = turn2<BF>(p, make_float2(-q.x, -q.y), t);
        }
        *reinterpret_cast<uint4*>(dst + r.half) = make_uint4(z[0], z[1], z[2], z[3]);
      } else if (rot) {
        rotate8<BF>(y, y, e0, r, T);
      }
      *reinterpret_cast<uint4*>(dst) = make_uint4(y[0], y[1], y[2], y[3]);
    }
  }
}

// Any strides, alignments and rotation sizes: 8 K or V elements, or one Q pair
// or element, a thread, loaded one by one.  grid (rows, parts).
template <bool BF, int BITS, int GS>
__global__ void __launch_bounds__(kThreads) append_any_kernel(const AppendArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ Shared sh;
  const View& v = a.v;
  const RopeArgs& r = a.rope;
  const int t = blockIdx.x;
  const int stride = place_rows(sh, a, t, 1);
  const int page = sh.page[0], pos = sh.pos[0];
  if (page == -2) return;
  const Table T{sh.c[0], sh.s[0], stride};
  const int D = v.D, per_log2 = __ffs(D) - 4, kv_units = v.Hkv << per_log2;
  const int crb = code_row_bytes(D, BITS), prb = pair_row_bytes(D, v.gs);
  const int q_head = a.q ? D - r.half : 0;  // pairs, then the rest of the row
  const int units = 2 * kv_units + a.Hq * q_head;
  // element e of a row after rotation
  auto element = [&](const uint16_t* src, int e) -> uint16_t {
    if (e >= r.dims) return src[e];
    const bool first = r.traditional ? !(e & 1) : e < r.half;
    const int i = r.traditional ? e >> 1 : (first ? e : e - r.half);
    const float x = to_f<BF>(src[e]), y = to_f<BF>(src[r.traditional ? e ^ 1 : (first ? e + r.half : e - r.half)]);
    return turn1<BF>(x, first ? -y : y, T, i);
  };
  for (int x = blockIdx.y * kThreads + threadIdx.x; x < units; x += gridDim.y * kThreads) {
    if (x < 2 * kv_units) {
      const bool is_v = x >= kv_units;
      const int k = is_v ? x - kv_units : x, h = k >> per_log2, e0 = (k - (h << per_log2)) << 3;
      const uint16_t* src = is_v ? a.val + t * a.v_row + h * a.v_head : a.k + t * a.k_row + h * a.k_head;
      uint32_t y[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int e = e0 + 2 * i;
        y[i] = is_v ? (uint32_t)src[e] | ((uint32_t)src[e + 1] << 16)
                    : (uint32_t)element(src, e) | ((uint32_t)element(src, e + 1) << 16);
      }
      if (page >= 0) {
        const int pr = pos & (kTileRows - 1);
        uint8_t* tile = tile_ptr(v, page, h, (pos & v.page_mask) >> 4) + (is_v ? kTileRows * (crb + prb) : 0);
        quantize8<BF, BITS, GS>(y, e0, tile + pr * crb, tile + kTileRows * crb + pr * prb);
      }
      continue;
    }
    const int k = x - 2 * kv_units, h = k / q_head, j = k - h * q_head;
    const uint16_t* src = a.q + t * a.q_row + h * a.q_head;
    uint16_t* dst = a.q_out + ((int64_t)t * a.Hq + h) * D;
    if (j < r.half) {  // both of a pair before either is written: q_out may be q
      const int i0 = r.traditional ? 2 * j : j, i1 = r.traditional ? 2 * j + 1 : j + r.half;
      const uint16_t y0 = element(src, i0), y1 = element(src, i1);
      dst[i0] = y0;
      dst[i1] = y1;
    } else {
      const int e = j - r.half + r.dims;
      dst[e] = src[e];
    }
  }
}

bool vec_ok(const void* p, int64_t row, int64_t head) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row % 8 == 0 && head % 8 == 0;
}

template <bool BF, int BITS, int GS>
int32_t launch(bool vec, cudaStream_t st, const AppendArgs& a) {
  // Few rows: one unit per thread (up to two blocks an SM, 296), so that a step's
  // latency is one pass; many: four rows to a block, whose angles then keep all
  // its threads busy, from eight rows an SM (148) on.  us, three shapes (32 + 8
  // heads x 128 in 4 bits, 16 + 8 x 256 in 8, 8 + 2 x 64 in 4): 16 rows split /
  // not split 3.4 / 4.2, 4.1 / 5.9, 3.2 / 3.2; one row a block / four: 592 rows
  // 7.4 / 8.5, 10.4 / 13.9, 4.0 / 5.5; 1,184 rows 12.6 / 11.3, 19.1 / 22.2, 6.6 /
  // 6.0; 1,776 rows 18.1 / 14.8, 27.5 / 23.1, 9.4 / 6.2.
  const int units = (2 * a.v.Hkv + (a.q ? a.Hq : 0)) * a.v.D / 8;
  int parts = 1;
  while (parts < (units + kThreads - 1) / kThreads && (int64_t)a.v.rows * parts < 2 * kSms) parts++;
  const dim3 grid((unsigned)a.v.rows, (unsigned)parts), block(kThreads);
  if (!vec)
    KVQ_CUDA_TRY(launch_pdl(append_any_kernel<BF, BITS, GS>, grid, block, 0, st, a));
  else if (a.v.rows < 8 * kSms)
    KVQ_CUDA_TRY(launch_pdl(append_kernel<BF, BITS, GS, 1>, grid, block, 0, st, a));
  else
    KVQ_CUDA_TRY(launch_pdl(append_kernel<BF, BITS, GS, kMaxRows>,
                            dim3((unsigned)((a.v.rows + kMaxRows - 1) / kMaxRows)), block, 0, st, a));
  return KVQ_OK;
}

template <bool BF, int BITS>
int32_t dispatch(bool vec, cudaStream_t st, const AppendArgs& a) {
  switch (a.v.gs) {
    case 32: return launch<BF, BITS, 32>(vec, st, a);
    case 64: return launch<BF, BITS, 64>(vec, st, a);
    default: return launch<BF, BITS, 128>(vec, st, a);
  }
}

}  // namespace

int32_t launch_paged_append(const AppendArgs& a, cudaStream_t st) {
  bool vec = vec_ok(a.k, a.k_row, a.k_head) && vec_ok(a.val, a.v_row, a.v_head) && a.rope.half % 8 == 0;
  if (a.q) vec = vec && vec_ok(a.q, a.q_row, a.q_head) && vec_ok(a.q_out, 8, 8);
  if (a.v.bits == 4) return a.bf16 ? dispatch<true, 4>(vec, st, a) : dispatch<false, 4>(vec, st, a);
  return a.bf16 ? dispatch<true, 8>(vec, st, a) : dispatch<false, 8>(vec, st, a);
}

}  // namespace paged
}  // namespace kvq
