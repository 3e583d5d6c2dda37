// kvq_paged_attn.cu — host side of the attention over pages: which kernel, its
// workspace and its launches.
#include <algorithm>

#include "kvq_paged_chunk.cuh"

namespace kvq {
namespace paged {

template <>
int32_t launch_cols<4, false>(const AttnArgs&, const Work&, int, int, int, cudaStream_t);
template <>
int32_t launch_cols<4, true>(const AttnArgs&, const Work&, int, int, int, cudaStream_t);
template <>
int32_t launch_cols<8, false>(const AttnArgs&, const Work&, int, int, int, cudaStream_t);
template <>
int32_t launch_cols<8, true>(const AttnArgs&, const Work&, int, int, int, cudaStream_t);

template <>
int32_t launch_chunk<4, false>(const AttnArgs&, const Work&, int, int, cudaStream_t);
template <>
int32_t launch_chunk<4, true>(const AttnArgs&, const Work&, int, int, cudaStream_t);
template <>
int32_t launch_chunk<8, false>(const AttnArgs&, const Work&, int, int, cudaStream_t);
template <>
int32_t launch_chunk<8, true>(const AttnArgs&, const Work&, int, int, cudaStream_t);

namespace {

// Query rows (times heads of a group) per sequence above which a call goes to
// the chunk kernel: a mean over the call, since rows of single sequences are known
// on the GPU only.  The two cross between 32 and 130 (us at 32, 64, 128 columns,
// column kernel / chunk kernel): 16 sequences of 8,000 keys, D 128, 4
// bits: 107 / 164, 194 / 165, 366 / 169; one, 8 bits: 21 / 41, 27 / 42, 42 / 43; 4
// of 4,000, D 256, 8 bits: 58 / 61, 100 / 63, 183 / 66; 8 of 4,000, D 64, 4 bits:
// 22 / 35, 29 / 35, 42 / 36.
constexpr long long kChunkCols = 64;

size_t up16(size_t x) { return (x + 15) / 16 * 16; }

// The launch: kernel, columns (query rows) per block, CTAs, workspace layout.
struct Launch {
  bool chunk;
  int NC, ctas;
  long long max_blocks;
  bool big;  // the plan does not fit in shared memory
  size_t o_meta, o_gpre, o_tpre, o_ng, bytes;
};

Launch plan_launch(const AttnArgs& a) {
  Launch c{};
  const View& v = a.v;
  int dev = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&c.ctas, cudaDevAttrMultiProcessorCount, dev);
  // columns per block: 16 where a sequence has more than 8 (K and V are read
  // once for all; D 256 has no registers for them), 4 where it has no more
  const long long cols = (long long)v.rows * a.rep;
  c.chunk = v.cu && cols > kChunkCols * v.B;
  c.NC = c.chunk ? (v.D == 256 ? 128 : 256) : cols > 8ll * v.B ? (v.D < 256 ? 16 : 8) : (cols > 4ll * v.B ? 8 : 4);
  const int NC = c.NC, NT = NC > 8 ? 2 : 1;
  c.max_blocks = v.cu ? cols / NC + v.B : (long long)v.B * ((a.rep + NC - 1) / NC);
  c.big = v.B > kPlanMax || c.max_blocks > kPlanMax;
  const size_t piece = c.chunk ? (size_t)NC * (v.D + 2) * 4
                               : (size_t)(16 * NT + v.D / 16 * NT * 128) * 4;
  c.o_meta = 2 * (size_t)c.ctas * piece;
  c.o_gpre = c.o_meta + (size_t)c.ctas * 16;
  c.bytes = c.o_gpre;
  if (c.big) {
    c.o_tpre = up16(c.o_gpre + (size_t)(v.B + 1) * 4);
    c.o_ng = c.o_tpre + (size_t)(c.max_blocks + 1) * 8;
    c.bytes = up16(c.o_ng + 4);
  }
  return c;
}

bool vec_ok(const AttnArgs& a) {
  return reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.q_row % 8 == 0 && a.q_head % 8 == 0;
}

}  // namespace

size_t paged_attn_workspace(const AttnArgs& a) { return plan_launch(a).bytes; }

int32_t launch_paged_attn(const AttnArgs& a, void* ws, size_t, cudaStream_t st) {
  const Launch c = plan_launch(a);
  if (c.max_blocks * a.v.Hkv > 0x7fffffff) return fail(KVQ_ERR_ARG, "paged: too many rows * heads in one call");
  uint8_t* p = static_cast<uint8_t*>(ws);
  Work w{};
  w.slots = reinterpret_cast<float*>(p);
  w.meta = reinterpret_cast<int4*>(p + c.o_meta);
  if (c.big) {
    w.gpre = reinterpret_cast<int*>(p + c.o_gpre);
    w.tpre = reinterpret_cast<long long*>(p + c.o_tpre);
    w.ng = reinterpret_cast<int*>(p + c.o_ng);
  }
  w.max_blocks = (int)c.max_blocks;
  w.vec = vec_ok(a);
  int dev = 0;
  KVQ_CUDA_TRY(cudaGetDevice(&dev));
  if (c.chunk) {
    if (a.v.bits == 4)
      return a.bf16 ? launch_chunk<4, true>(a, w, c.ctas, dev, st)
                    : launch_chunk<4, false>(a, w, c.ctas, dev, st);
    return a.bf16 ? launch_chunk<8, true>(a, w, c.ctas, dev, st)
                  : launch_chunk<8, false>(a, w, c.ctas, dev, st);
  }
  if (a.v.bits == 4)
    return a.bf16 ? launch_cols<4, true>(a, w, c.NC, c.ctas, dev, st)
                  : launch_cols<4, false>(a, w, c.NC, c.ctas, dev, st);
  return a.bf16 ? launch_cols<8, true>(a, w, c.NC, c.ctas, dev, st)
                : launch_cols<8, false>(a, w, c.NC, c.ctas, dev, st);
}

}  // namespace paged
}  // namespace kvq
