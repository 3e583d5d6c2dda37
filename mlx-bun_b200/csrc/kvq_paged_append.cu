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

// One unit's raw elements: 8 consecutive ones, and 8 rotation partners of them.
struct Raw {
  uint4 own, other;
};
__device__ __forceinline__ void unpack(uint16_t (&x)[8], const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
}

// grid (row groups, parts): a block takes R rows from R * blockIdx.x and the
// units part * kThreads + threadIdx.x, + parts * kThreads, ... of their list.
// VEC: 16-byte loads, and rotation halves that split into eights; the next
// unit's loads are then on their way while one is computed.
template <bool BF, int BITS, bool VEC>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs a, const int R) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ double2 cs[kMaxRows * kMaxHalf];
  __shared__ double inv[kMaxHalf];
  __shared__ int s_pos[kMaxRows], s_page[kMaxRows];  // page: -2 no such row, -1 no page
  const View& v = a.v;
  const RopeArgs& r = a.rope;
  const int t0 = blockIdx.x * R, tid = threadIdx.x, lane = tid & 31;
  const int nr = min(R, v.rows - t0);

  // Each row's sequence, position and page by one warp, the frequencies by the
  // others meanwhile.
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
      s_pos[k] = pos;
      s_page[k] = page;
    }
  }
  for (int i = kThreads - 1 - tid; i < r.half; i += kThreads)
    inv[i] = r.freqs ? 1.0 / (double)r.freqs[i] : pow(r.base, -2.0 * (double)i / (double)r.dims);
  __syncthreads();
  const int stride = (r.half + 7) >> 3;
  for (int i = tid; i < nr * r.half; i += kThreads) {
    const int k = i / r.half, e = i - k * r.half;
    double s, c;
    sincos((r.scale * (double)s_pos[k]) * inv[e], &s, &c);
    cs[k * kMaxHalf + (e & 7) * stride + (e >> 3)] = make_double2(c * r.pre, s * r.pre);
  }
  __syncthreads();

  const int D = v.D, per_log2 = __ffs(D) - 4;  // units of 8 in a row
  const int kv_units = v.Hkv << per_log2;
  const int crb = code_row_bytes(D, BITS), prb = pair_row_bytes(D, v.gs);
  // Q units of a head: rotated ones (8 elements and their partners when not
  // traditional), then the rest of the row, 8 elements each; element by
  // element when the halves do not split into eights
  const bool q_vec = VEC || (r.half & 7) == 0;
  const int q_rot = q_vec ? (r.traditional ? r.dims >> 3 : r.half >> 3) : r.half;
  const int q_head_units = a.q ? q_rot + (q_vec ? (D - r.dims) >> 3 : D - r.dims) : 0;
  const int units = 2 * kv_units + a.Hq * q_head_units;
  const int padded = (units + 31) & ~31;  // rows start on a warp: groups keep their lanes
  const int step = gridDim.y * kThreads, end = nr * padded;

  // row k and unit x of list entry u; where its elements lie
  struct Unit {
    int k, x, h, e0;
    bool run;
    const uint16_t *own, *other;
  };
  auto find = [&](int u) {
    Unit z;
    z.k = u < end ? u / padded : 0;
    z.x = u < end ? u - z.k * padded : 0;
    z.run = u < end && z.x < units && s_page[z.k] != -2;
    const int64_t t = t0 + z.k;
    if (z.x < 2 * kv_units || z.x >= units) {
      const bool is_v = z.x >= kv_units;
      const int k = z.x >= units ? 0 : (is_v ? z.x - kv_units : z.x);
      z.h = k >> per_log2;
      z.e0 = (k - (z.h << per_log2)) << 3;
      const uint16_t* row = is_v ? a.val + t * a.v_row + z.h * a.v_head : a.k + t * a.k_row + z.h * a.k_head;
      z.own = row + z.e0;
      const bool turn = !is_v && !r.traditional && z.e0 < r.dims;
      z.other = turn ? row + (z.e0 < r.half ? z.e0 + r.half : z.e0 - r.half) : z.own;
    } else {
      const int k = z.x - 2 * kv_units;
      z.h = k / q_head_units;
      const int j = k - z.h * q_head_units;
      const uint16_t* row = a.q + t * a.q_row + z.h * a.q_head;
      z.e0 = j >= q_rot ? r.dims + ((j - q_rot) << 3) : j << 3;  // (q_vec)
      z.own = row + z.e0;
      z.other = j < q_rot && !r.traditional ? z.own + r.half : z.own;
      if (!q_vec) {
        z.e0 = j;
        z.own = z.other = row;
      }
    }
    return z;
  };
  auto fetch = [&](const Unit& z) {
    Raw w{};
    if constexpr (VEC) {
      w.own = *reinterpret_cast<const uint4*>(z.own);
      w.other = *reinterpret_cast<const uint4*>(z.other);
    }
    return w;
  };
  int u = blockIdx.y * kThreads + tid;
  Unit z = find(u);
  Raw raw = fetch(z);
  for (; u < end; u += step) {
    const Unit cur = z;
    const Raw w = raw;
    z = find(u + step);
    raw = fetch(z);
    if (!cur.run) continue;
    const Table T{cs + cur.k * kMaxHalf, stride};
    const int pos = s_pos[cur.k], page = s_page[cur.k];
    const int64_t t = t0 + cur.k;
    uint16_t y[8], o[8];
    if (cur.x < 2 * kv_units) {
      const bool is_v = cur.x >= kv_units;
      if constexpr (VEC) {
        unpack(y, w.own);
        if (!is_v && cur.e0 < r.dims) {
          unpack(o, w.other);
          if (r.traditional) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
              const double2 c = T.at((cur.e0 + i) >> 1);
              const double p = to_f<BF>(y[i]), q = to_f<BF>(y[i + 1]);
              y[i] = round_out<BF>(p * c.x - q * c.y);
              y[i + 1] = round_out<BF>(p * c.y + q * c.x);
            }
          } else {
            const bool lo = cur.e0 < r.half;
            const int i0 = lo ? cur.e0 : cur.e0 - r.half;
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const double2 c = T.at(i0 + i);
              const double own = to_f<BF>(y[i]), other = to_f<BF>(o[i]);
              y[i] = round_out<BF>(lo ? own * c.x - other * c.y : other * c.y + own * c.x);
            }
          }
        }
      } else {
        if (is_v) load8<false>(y, cur.own);
        else rotate8<BF, false>(y, cur.own - cur.e0, cur.e0, r, T);
      }
      if (page >= 0) {
        const int row = pos & (kTileRows - 1);
        uint8_t* tile = tile_ptr(v, page, cur.h, (pos & v.page_mask) >> 4) + (is_v ? kTileRows * (crb + prb) : 0);
        quantize8<BF, BITS>(y, cur.e0, v.gs, tile + row * crb, tile + kTileRows * crb + row * prb);
      }
      continue;
    }
    uint16_t* dst = a.q_out + (t * a.Hq + cur.h) * D;
    if (!q_vec) {
      const int j = cur.e0;
      const uint16_t* src = cur.own;
      if (j >= r.half) {
        dst[r.dims + j - r.half] = src[r.dims + j - r.half];
      } else {
        const int i0 = r.traditional ? 2 * j : j, i1 = r.traditional ? 2 * j + 1 : j + r.half;
        const double2 c = T.at(j);
        const double x = to_f<BF>(src[i0]), q = to_f<BF>(src[i1]);
        dst[i0] = round_out<BF>(x * c.x - q * c.y);
        dst[i1] = round_out<BF>(x * c.y + q * c.x);
      }
      continue;
    }
    if constexpr (VEC) unpack(y, w.own);
    else load8<false>(y, cur.own);
    if (cur.e0 >= r.dims) {
      store8<VEC>(dst + cur.e0, y);
    } else if (r.traditional) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const double2 c = T.at((cur.e0 + i) >> 1);
        const double p = to_f<BF>(y[i]), q = to_f<BF>(y[i + 1]);
        y[i] = round_out<BF>(p * c.x - q * c.y);
        y[i + 1] = round_out<BF>(p * c.y + q * c.x);
      }
      store8<VEC>(dst + cur.e0, y);
    } else {
      if constexpr (VEC) unpack(o, w.other);
      else load8<false>(o, cur.other);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const double2 c = T.at(cur.e0 + i);
        const double x = to_f<BF>(y[i]), q = to_f<BF>(o[i]);
        y[i] = round_out<BF>(x * c.x - q * c.y);
        o[i] = round_out<BF>(x * c.y + q * c.x);
      }
      store8<VEC>(dst + cur.e0, y);
      store8<VEC>(dst + cur.e0 + r.half, o);
    }
  }
}

bool vec_ok(const void* p, int64_t row, int64_t head) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row % 8 == 0 && head % 8 == 0;
}

template <bool BF, int BITS>
int32_t dispatch(bool vec, dim3 grid, cudaStream_t st, const AppendArgs& a, int R) {
  if (vec) KVQ_CUDA_TRY(launch_pdl(append_kernel<BF, BITS, true>, grid, dim3(kThreads), 0, st, a, R));
  else KVQ_CUDA_TRY(launch_pdl(append_kernel<BF, BITS, false>, grid, dim3(kThreads), 0, st, a, R));
  return KVQ_OK;
}

}  // namespace

int32_t launch_paged_append(const AppendArgs& a, cudaStream_t st) {
  bool vec = vec_ok(a.k, a.k_row, a.k_head) && vec_ok(a.val, a.v_row, a.v_head);
  if (a.q) vec = vec && vec_ok(a.q, a.q_row, a.q_head) && vec_ok(a.q_out, 8, 8);
  vec = vec && a.rope.half % 8 == 0;
  // few rows: one unit per thread, so that a step's latency is one pass; many:
  // four to a block, whose angles then keep all its threads busy
  const int units = (2 * a.v.Hkv + (a.q ? a.Hq : 0)) * a.v.D / 8;
  const int R = a.v.rows >= 148 * 8 ? kMaxRows : 1;
  int parts = 1;
  while (R == 1 && parts < (units + kThreads - 1) / kThreads && (int64_t)a.v.rows * parts < 296) parts++;
  const dim3 grid((unsigned)((a.v.rows + R - 1) / R), (unsigned)parts);
  if (a.v.bits == 4)
    return a.bf16 ? dispatch<true, 4>(vec, grid, st, a, R) : dispatch<false, 4>(vec, grid, st, a, R);
  return a.bf16 ? dispatch<true, 8>(vec, grid, st, a, R) : dispatch<false, 8>(vec, grid, st, a, R);
}

}  // namespace paged
}  // namespace kvq
