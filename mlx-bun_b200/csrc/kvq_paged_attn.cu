// kvq_paged_attn.cu — causal attention of ragged query rows over the pages
// (sliding window and sinks), the plain form: one block per (token row, query
// head), each warp takes every fourth visible key, lanes share the row.
#include "kvq_paged.cuh"

namespace kvq {
namespace paged {
namespace {

constexpr int kWarps = 4;
constexpr float kNegInf = -3.0e38f;

template <bool BF>
__device__ __forceinline__ float to_f(uint32_t v) {
  if constexpr (BF) return __uint_as_float(v << 16);
  else return __half2float(__ushort_as_half((uint16_t)v));
}

// This lane's PER elements of one K or V row
template <bool BF, int BITS, int PER>
__device__ __forceinline__ void row_values(float (&x)[PER], const uint8_t* half, int row, int e0,
                                           int crb, int gs, int prb) {
  const uint32_t pr = *reinterpret_cast<const uint32_t*>(half + kTileRows * crb + row * prb + e0 / gs * 4);
  const float s = to_f<BF>(pr & 0xffffu), z = to_f<BF>(pr >> 16);
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int bit = (e0 + i) * BITS;
    const uint8_t byte = half[row * crb + bit / 8];
    const int c = BITS == 8 ? byte : (byte >> (bit & 4)) & 15;
    x[i] = fmaf((float)c, s, z);
  }
}

template <bool BF, int BITS, int PER>
__global__ void __launch_bounds__(kWarps * 32) attn_rows_kernel(const AttnArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int D = 32 * PER;
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][D];
  const View& v = a.v;
  const int t = blockIdx.x, h = blockIdx.y, hk = h / a.rep;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, e0 = lane * PER;
  const int b = block_find_seq(v, t);
  if (b >= v.B) return;
  int row0, n, len;
  seq_rows(v, b, row0, n, len);
  int pos = len - n + (t - row0);
  if (t < row0 || len < 0 || len > (int64_t)v.max_pages << v.page_shift) {
    if (threadIdx.x == 0) raise(v);
    pos = -1;
  }
  int lo = 0, head = 0;
  if (a.window > 0) {
    lo = max(0, pos - a.window + 1);
    head = min(a.sinks, lo);
  }
  float q[PER], o[PER] = {};
  const uint16_t* qr = a.q + (int64_t)t * a.q_row + (int64_t)h * a.q_head + e0;
#pragma unroll
  for (int i = 0; i < PER; i++) q[i] = to_f<BF>(qr[i]) * a.scale;
  float m = kNegInf, l = 0.0f;
  const int crb = code_row_bytes(D, BITS), prb = pair_row_bytes(D, v.gs);
  const int keys = pos < 0 ? 0 : head + pos + 1 - lo;
  for (int i = w; i < keys; i += kWarps) {
    const int j = i < head ? i : lo + i - head;
    const int page = v.table[(int64_t)b * v.table_stride + (j >> v.page_shift)];
    if (page < 0 || page >= v.num_pages) {
      if (lane == 0) raise(v);
      continue;
    }
    const uint8_t* tile = tile_ptr(v, page, hk, (j & v.page_mask) >> 4);
    float x[PER];
    row_values<BF, BITS, PER>(x, tile, j & 15, e0, crb, v.gs, prb);
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < PER; k++) s = fmaf(q[k], x[k], s);
#pragma unroll
    for (int k = 16; k; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
    const float m2 = fmaxf(m, s), f = expf(m - m2), p = expf(s - m2);
    m = m2;
    l = l * f + p;
    row_values<BF, BITS, PER>(x, tile + kTileRows * (crb + prb), j & 15, e0, crb, v.gs, prb);
#pragma unroll
    for (int k = 0; k < PER; k++) o[k] = fmaf(p, x[k], o[k] * f);
  }
  if (lane == 0) sm[w] = m, sl[w] = l;
#pragma unroll
  for (int i = 0; i < PER; i++) so[w][e0 + i] = o[i];
  __syncthreads();
  float mx = sm[0];
  for (int i = 1; i < kWarps; i++) mx = fmaxf(mx, sm[i]);
  float lt = 0.0f;
  for (int i = 0; i < kWarps; i++) lt += sl[i] * expf(sm[i] - mx);
  for (int e = threadIdx.x; e < D; e += kWarps * 32) {
    float s = 0.0f;
    for (int i = 0; i < kWarps; i++) s += so[i][e] * expf(sm[i] - mx);
    s = lt > 0.0f ? s / lt : 0.0f;
    uint16_t r;
    if constexpr (BF) r = __bfloat16_as_ushort(__float2bfloat16_rn(s));
    else r = __half_as_ushort(__float2half_rn(s));
    a.out[((int64_t)t * a.Hq + h) * D + e] = r;
  }
}

template <bool BF, int BITS>
int32_t dispatch(const AttnArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)a.v.rows, (unsigned)a.Hq), block(kWarps * 32);
  switch (a.v.D) {
    case 64: KVQ_CUDA_TRY(launch_pdl(attn_rows_kernel<BF, BITS, 2>, grid, block, 0, st, a)); break;
    case 128: KVQ_CUDA_TRY(launch_pdl(attn_rows_kernel<BF, BITS, 4>, grid, block, 0, st, a)); break;
    default: KVQ_CUDA_TRY(launch_pdl(attn_rows_kernel<BF, BITS, 8>, grid, block, 0, st, a)); break;
  }
  return KVQ_OK;
}

}  // namespace

size_t paged_attn_workspace(const AttnArgs&) { return 0; }

int32_t launch_paged_attn(const AttnArgs& a, void*, size_t, cudaStream_t st) {
  if (a.v.bits == 4) return a.bf16 ? dispatch<true, 4>(a, st) : dispatch<false, 4>(a, st);
  return a.bf16 ? dispatch<true, 8>(a, st) : dispatch<false, 8>(a, st);
}

}  // namespace paged
}  // namespace kvq
