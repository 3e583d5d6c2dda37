// kvq_paged_append.cu — RoPE, quantize and write into pages, one launch.
//
// Per token row at position p: angle_i = (scale * p) * inv_freq_i and its
// cosine and sine in 64 bits, (x, y) -> (x cos - y sin, x sin + y cos) in 64
// bits for K and Q, rounded to 32 bits and then to the dtype; K and V rows
// then go through the affine group rule of kvq_qrule.cuh into their page.  A
// 32-bit angle at position 131,072 is off by up to 0.004 rad, more than a
// bf16 step of the result; and with 64-bit rotation the rounded values, and
// so the codes, do not depend on the order of operations.
//
// A block takes one token row (its cosines and sines are computed once, in
// shared memory) and a share of the row's units; a unit is 8 consecutive
// elements of a K or V row (quantized by the group's lanes with shuffles) or
// 8 elements and their 8 rotation partners of a Q row (so that q may be
// rotated in place).
#include "kvq_paged.cuh"
#include "kvq_qrule.cuh"

namespace kvq {
namespace paged {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;

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

template <bool VEC>
__device__ __forceinline__ void load8(uint16_t (&x)[8], const uint16_t* p) {
  if constexpr (VEC) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = p[i];
  }
}

template <bool VEC>
__device__ __forceinline__ void store8(uint16_t* p, const uint16_t (&x)[8]) {
  if constexpr (VEC) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = (uint32_t)x[2 * i] | ((uint32_t)x[2 * i + 1] << 16);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) p[i] = x[i];
  }
}

// cos / sin of pair i: 8 consecutive pairs are one unit's, so pair i sits at
// slot (i % 8) * stride + i / 8 and neighbouring lanes read neighbouring slots
struct Table {
  const double2* cs;
  int stride;
  __device__ __forceinline__ double2 at(int i) const { return cs[(i & 7) * stride + (i >> 3)]; }
};

template <bool BF>
__device__ __forceinline__ uint16_t round_out(double x) {
  return to_bits<BF>((float)x);
}

// Element e of a row after rotation, x its raw row
template <bool BF, bool VEC>
__device__ __forceinline__ void rotate8(uint16_t (&y)[8], const uint16_t* row, int e0,
                                        const RopeArgs& r, const Table& T) {
  load8<VEC>(y, row + e0);
  if (e0 >= r.dims) return;
  if (r.traditional) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if (e0 + i < r.dims) {
        const double2 c = T.at((e0 + i) >> 1);
        const double a = to_f<BF>(y[i]), b = to_f<BF>(y[i + 1]);
        y[i] = round_out<BF>(a * c.x - b * c.y);
        y[i + 1] = round_out<BF>(a * c.y + b * c.x);
      }
    }
    return;
  }
  uint16_t z[8];
  if ((r.half & 7) == 0) {
    load8<VEC>(z, row + (e0 < r.half ? e0 + r.half : e0 - r.half));
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int e = e0 + i;
      z[i] = e < r.dims ? row[e < r.half ? e + r.half : e - r.half] : (uint16_t)0;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int e = e0 + i;
    if (e < r.dims) {
      const bool lo = e < r.half;
      const double2 c = T.at(lo ? e : e - r.half);
      const double own = to_f<BF>(y[i]), other = to_f<BF>(z[i]);
      y[i] = round_out<BF>(lo ? own * c.x - other * c.y : other * c.y + own * c.x);
    }
  }
}

// Quantize the 8 elements y of element e0.. of a K or V row; the group's
// gs / 8 lanes hold its other elements.
template <bool BF, int BITS>
__device__ __forceinline__ void quantize8(const uint16_t (&y)[8], int e0, int gs, uint8_t* codes,
                                          uint8_t* pairs) {
  constexpr float NB = (float)((1 << BITS) - 1);
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; i++) w[i] = to_f<BF>(y[i]);
  float mn = w[0], mx = w[0];
#pragma unroll
  for (int i = 1; i < 8; i++) {
    mn = fminf(mn, w[i]);
    mx = fmaxf(mx, w[i]);
  }
  const int lanes = gs >> 3, lane = threadIdx.x & 31;
  const unsigned mask = (0xffffffffu >> (32 - lanes)) << (lane & ~(lanes - 1));
  for (int o = 1; o < lanes; o <<= 1) {
    mn = fminf(mn, __shfl_xor_sync(mask, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(mask, mx, o));
  }
  float scale, bias;
  quant_params(mn, mx, NB, scale, bias);
  uint32_t word[BITS / 4] = {};
#pragma unroll
  for (int i = 0; i < 8; i++)
    word[i * BITS / 32] |= quant_code(w[i], scale, bias, NB) << (i * BITS % 32);
  uint8_t* dst = codes + e0 * BITS / 8;
  if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(dst) = word[0];
  else *reinterpret_cast<uint2*>(dst) = make_uint2(word[0], word[1]);
  if ((e0 & (gs - 1)) == 0)
    *reinterpret_cast<uint32_t*>(pairs + e0 / gs * 4) =
        (uint32_t)to_bits<BF>(scale) | ((uint32_t)to_bits<BF>(bias) << 16);
}

// grid (rows, parts): block (t, part) takes the units part * kThreads +
// threadIdx.x, + parts * kThreads, ... of row t.
template <bool BF, int BITS, bool VEC>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ double2 cs[kMaxHalf];
  const View& v = a.v;
  const RopeArgs& r = a.rope;
  const int t = blockIdx.x, tid = threadIdx.x;
  const int b = block_find_seq(v, t);
  if (b >= v.B) return;  // padding
  int row0, n, len;
  seq_rows(v, b, row0, n, len);
  const int pos = len - n + (t - row0);
  const bool placed = t >= row0 && n > 0 && pos >= 0 && (pos >> v.page_shift) < v.max_pages;
  if (!placed) {
    if (tid == 0 && blockIdx.y == 0) raise(v);
    return;
  }
  const int page = v.table[(int64_t)b * v.table_stride + (pos >> v.page_shift)];
  const bool stored = page >= 0 && page < v.num_pages;
  if (!stored && tid == 0 && blockIdx.y == 0) raise(v);

  const Table T{cs, (r.half + 7) >> 3};
  for (int i = tid; i < r.half; i += kThreads) {
    const double inv =
        r.freqs ? 1.0 / (double)r.freqs[i] : pow(r.base, -2.0 * (double)i / (double)r.dims);
    double s, c;
    sincos((r.scale * (double)pos) * inv, &s, &c);
    cs[(i & 7) * T.stride + (i >> 3)] = make_double2(c * r.pre, s * r.pre);
  }
  __syncthreads();

  const int D = v.D, per = D >> 3;
  const int kv_units = v.Hkv * per;
  const int crb = code_row_bytes(D, BITS), prb = pair_row_bytes(D, v.gs);
  // Q units of a head: rotated ones (8 elements and their partners when not
  // traditional), then the rest of the row, 8 elements each; element by
  // element when the halves do not split into eights
  const bool q_vec = (r.half & 7) == 0;
  const int q_rot = q_vec ? (r.traditional ? r.dims >> 3 : r.half >> 3) : r.half;
  const int q_head_units = a.q ? q_rot + (q_vec ? (D - r.dims) >> 3 : D - r.dims) : 0;
  const int units = 2 * kv_units + a.Hq * q_head_units;
  for (int u = blockIdx.y * kThreads + tid; u < units; u += gridDim.y * kThreads) {
    if (u < 2 * kv_units) {
      const bool is_v = u >= kv_units;
      const int k = is_v ? u - kv_units : u;
      const int h = k / per, e0 = (k - h * per) << 3;
      uint16_t y[8];
      if (is_v)
        load8<VEC>(y, a.val + (int64_t)t * a.v_row + (int64_t)h * a.v_head + e0);
      else
        rotate8<BF, VEC>(y, a.k + (int64_t)t * a.k_row + (int64_t)h * a.k_head, e0, r, T);
      if (stored) {
        const int row = pos & (kTileRows - 1);
        uint8_t* tile = tile_ptr(v, page, h, (pos & v.page_mask) >> 4) +
                        (is_v ? kTileRows * (crb + prb) : 0);
        quantize8<BF, BITS>(y, e0, v.gs, tile + row * crb, tile + kTileRows * crb + row * prb);
      }
      continue;
    }
    const int k = u - 2 * kv_units;
    const int h = k / q_head_units, j = k - h * q_head_units;
    const uint16_t* src = a.q + (int64_t)t * a.q_row + (int64_t)h * a.q_head;
    uint16_t* dst = a.q_out + ((int64_t)t * a.Hq + h) * D;
    if (!q_vec) {
      if (j >= r.half) {
        dst[r.dims + j - r.half] = src[r.dims + j - r.half];
      } else {
        const int i0 = r.traditional ? 2 * j : j, i1 = r.traditional ? 2 * j + 1 : j + r.half;
        const double2 c = T.at(j);
        const double x = to_f<BF>(src[i0]), y = to_f<BF>(src[i1]);
        dst[i0] = round_out<BF>(x * c.x - y * c.y);
        dst[i1] = round_out<BF>(x * c.y + y * c.x);
      }
      continue;
    }
    uint16_t y[8];
    if (j >= q_rot) {
      const int e0 = r.dims + ((j - q_rot) << 3);
      load8<VEC>(y, src + e0);
      store8<VEC>(dst + e0, y);
    } else if (r.traditional) {
      rotate8<BF, VEC>(y, src, j << 3, r, T);
      store8<VEC>(dst + (j << 3), y);
    } else {
      uint16_t z[8];
      load8<VEC>(y, src + (j << 3));
      load8<VEC>(z, src + (j << 3) + r.half);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const double2 c = T.at((j << 3) + i);
        const double x = to_f<BF>(y[i]), w = to_f<BF>(z[i]);
        y[i] = round_out<BF>(x * c.x - w * c.y);
        z[i] = round_out<BF>(x * c.y + w * c.x);
      }
      store8<VEC>(dst + (j << 3), y);
      store8<VEC>(dst + (j << 3) + r.half, z);
    }
  }
}

bool vec_ok(const void* p, int64_t row, int64_t head) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row % 8 == 0 && head % 8 == 0;
}

template <bool BF, int BITS>
int32_t dispatch(bool vec, dim3 grid, cudaStream_t st, const AppendArgs& a) {
  if (vec) KVQ_CUDA_TRY(launch_pdl(append_kernel<BF, BITS, true>, grid, dim3(kThreads), 0, st, a));
  else KVQ_CUDA_TRY(launch_pdl(append_kernel<BF, BITS, false>, grid, dim3(kThreads), 0, st, a));
  return KVQ_OK;
}

}  // namespace

int32_t launch_paged_append(const AppendArgs& a, cudaStream_t st) {
  bool vec = vec_ok(a.k, a.k_row, a.k_head) && vec_ok(a.val, a.v_row, a.v_head);
  if (a.q) vec = vec && vec_ok(a.q, a.q_row, a.q_head) && vec_ok(a.q_out, 8, 8);
  const int units = (2 * a.v.Hkv + (a.q ? a.Hq : 0)) * a.v.D / 8;
  // few rows: one unit per thread, so that a step's latency is one pass
  int parts = 1;
  while (parts < (units + kThreads - 1) / kThreads && (int64_t)a.v.rows * parts < 296) parts++;
  const dim3 grid((unsigned)a.v.rows, (unsigned)parts);
  if (a.v.bits == 4)
    return a.bf16 ? dispatch<true, 4>(vec, grid, st, a) : dispatch<false, 4>(vec, grid, st, a);
  return a.bf16 ? dispatch<true, 8>(vec, grid, st, a) : dispatch<false, 8>(vec, grid, st, a);
}

}  // namespace paged
}  // namespace kvq
