// kvq_paged_api.cu — C entry points of the paged quantized cache: argument
// checks, workspaces, launches.
#include <cmath>
#include <mutex>
#include <new>
#include <string>

#include "kvq_paged.cuh"

using namespace kvq;

namespace {

// Every device array starts at a multiple of its elements' size (a null one
// does): the kernels load whole elements.
bool aligned(const void* p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

// Whether the contiguous rows that a call writes at `out` share memory with the
// rows [rows][heads][D] it reads at `in` (element strides rs, hs).
bool shares(const void* out, const void* in, int64_t rows, int64_t heads, int64_t D, int64_t out_heads,
            int64_t rs, int64_t hs) {
  if (rs < 0) {
    in = static_cast<const uint16_t*>(in) + (rows - 1) * rs;
    rs = -rs;
  }
  const int64_t a = reinterpret_cast<intptr_t>(out), b = a + rows * out_heads * D * 2, len = 2 * D, step = 2 * rs;
  for (int64_t h = 0; h < heads; h++) {
    const int64_t x = reinterpret_cast<intptr_t>(in) + 2 * h * hs;  // rows at x + r * step, len bytes each
    if (x >= b) continue;
    // the first row that ends behind a
    const int64_t r = x + len > a ? 0 : step ? (a - (x + len)) / step + 1 : rows;
    if (r < rows && x + r * step < b) return true;
  }
  return false;
}

int32_t make_view(const kvq_paged* c, const kvq_paged_batch* b, paged::View& v) {
  if (!c || !b) return fail(KVQ_ERR_ARG, "paged: NULL cache / batch");
  if (!c->pool || !c->status) return fail(KVQ_ERR_ARG, "paged: NULL pool / status");
  if (reinterpret_cast<uintptr_t>(c->pool) % 16) return fail(KVQ_ERR_ARG, "paged: pool must be 16-byte aligned");
  if (c->num_pages <= 0 || c->kv_heads <= 0) return fail(KVQ_ERR_ARG, "paged: num_pages and kv_heads must be positive");
  int shift = 4;
  while (shift < 8 && (1 << shift) != c->page_size) shift++;
  if ((1 << shift) != c->page_size) return fail(KVQ_ERR_ARG, "paged: page_size must be 16, 32, 64, 128 or 256");
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(KVQ_ERR_ARG, "paged: head_dim must be 64, 128 or 256");
  if (c->bits != 4 && c->bits != 8) return fail(KVQ_ERR_ARG, "paged: bits must be 4 or 8");
  if ((c->group_size != 32 && c->group_size != 64 && c->group_size != 128) || c->group_size > c->head_dim)
    return fail(KVQ_ERR_ARG, "paged: group_size must be 32, 64 or 128 and at most head_dim");
  if (c->dtype != KVQ_DTYPE_FLOAT16 && c->dtype != KVQ_DTYPE_BFLOAT16)
    return fail(KVQ_ERR_ARG, "paged: dtype must be KVQ_DTYPE_FLOAT16 or KVQ_DTYPE_BFLOAT16");
  if (b->batch < 0 || b->rows < 0 || b->max_pages < 0) return fail(KVQ_ERR_ARG, "paged: batch, rows and max_pages must be >= 0");
  if (b->batch > 0 && (!b->seq_lens || (b->max_pages > 0 && !b->page_table)))
    return fail(KVQ_ERR_ARG, "paged: NULL page_table / seq_lens");
  if (!aligned(c->status, 4) || !aligned(b->page_table, 4) || !aligned(b->seq_lens, 4) || !aligned(b->cu_rows, 4))
    return fail(KVQ_ERR_ARG, "paged: status, page_table, seq_lens and cu_rows must be 4-byte aligned");
  if (b->table_stride < b->max_pages && b->batch > 1) return fail(KVQ_ERR_ARG, "paged: table_stride smaller than max_pages");
  if (((int64_t)b->max_pages << shift) > 0x7fffffff) return fail(KVQ_ERR_ARG, "paged: max_pages * page_size passes 2^31");
  v = paged::View{};
  v.pool = static_cast<uint8_t*>(c->pool);
  v.status = c->status;
  v.num_pages = c->num_pages;
  v.page_shift = shift;
  v.page_mask = c->page_size - 1;
  v.tiles_shift = shift - 4;
  v.Hkv = c->kv_heads;
  v.D = c->head_dim;
  v.bits = c->bits;
  v.gs = c->group_size;
  v.tile_bytes = 2 * paged::half_tile_bytes(v.D, v.bits, v.gs);
  v.table = b->page_table;
  v.table_stride = b->table_stride;
  v.seq_lens = b->seq_lens;
  v.cu = b->cu_rows;
  v.B = b->batch;
  v.max_pages = b->max_pages;
  v.rows = b->rows;
  return KVQ_OK;
}

int32_t make_attn(const kvq_paged* c, const kvq_paged_batch* b, int32_t q_heads, bool decode,
                  paged::AttnArgs& a) {
  a = paged::AttnArgs{};
  int32_t rc = make_view(c, b, a.v);
  if (rc) return rc;
  if (q_heads <= 0 || q_heads % c->kv_heads) return fail(KVQ_ERR_ARG, "paged: q_heads must be a positive multiple of kv_heads");
  if (decode) a.v.cu = nullptr;
  if (!a.v.cu && a.v.rows != a.v.B) return fail(KVQ_ERR_ARG, "paged: rows must equal batch without cu_rows");
  a.Hq = q_heads;
  a.rep = q_heads / c->kv_heads;
  a.bf16 = c->dtype == KVQ_DTYPE_BFLOAT16;
  return KVQ_OK;
}

// The library's own stream-ordered pool on `dev` (the current device) for
// workspaces of calls that bring none.  Memory stays in it: the default pool
// gives it back to the driver at every synchronization, and taking it again
// costs hundreds of microseconds.
std::mutex g_pool_mu;
cudaMemPool_t g_pool[64] = {};

int32_t scratch_pool(int dev, cudaMemPool_t* out) {
  if (dev < 0 || dev >= 64) return fail(KVQ_ERR_ARG, "device ordinal out of range");
  std::lock_guard<std::mutex> lk(g_pool_mu);
  if (!g_pool[dev]) {
    cudaMemPoolProps props = {};
    props.allocType = cudaMemAllocationTypePinned;
    props.location.type = cudaMemLocationTypeDevice;
    props.location.id = dev;
    cudaMemPool_t pool = nullptr;
    // the first call may be one that is being captured, where a pool cannot be
    // made otherwise
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    KVQ_CUDA_TRY(cudaThreadExchangeStreamCaptureMode(&mode));
    uint64_t keep = UINT64_MAX;
    cudaError_t e = cudaMemPoolCreate(&pool, &props);
    if (e == cudaSuccess) e = cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep);
    const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) return cuda_fail(e, "cudaMemPoolCreate");
    if (back != cudaSuccess) return cuda_fail(back, "cudaThreadExchangeStreamCaptureMode");
    g_pool[dev] = pool;
  }
  *out = g_pool[dev];
  return KVQ_OK;
}

int32_t sdpa(const kvq_paged* c, const kvq_paged_batch* b, bool decode, const void* q,
             int32_t q_heads, const int64_t* q_strides, float scale, int32_t window, int32_t sinks,
             void* out, void* workspace, size_t workspace_bytes, void* stream) {
  paged::AttnArgs a;
  int32_t rc = make_attn(c, b, q_heads, decode, a);
  if (rc) return rc;
  if (window < 0 || sinks < 0) return fail(KVQ_ERR_ARG, "paged: window and sinks must be >= 0");
  if (!std::isfinite(scale)) return fail(KVQ_ERR_ARG, "paged: scale must be finite");
  // a window as long as the table holds hides nothing
  if ((int64_t)window >= ((int64_t)a.v.max_pages << a.v.page_shift)) window = 0;
  if (a.v.rows == 0 || a.v.B == 0) return KVQ_OK;
  if (!q || !q_strides || !out) return fail(KVQ_ERR_ARG, "paged: NULL q / q_strides / out");
  if (!aligned(q, 2) || !aligned(out, 2)) return fail(KVQ_ERR_ARG, "paged: q and out must be 2-byte aligned");
  const bool packed = (q_heads == 1 || q_strides[1] == a.v.D) && (a.v.rows == 1 || q_strides[0] == (int64_t)q_heads * a.v.D);
  if (!(out == q && packed) && shares(out, q, a.v.rows, q_heads, a.v.D, q_heads, q_strides[0], q_strides[1]))
    return fail(KVQ_ERR_ARG, "paged: out overlaps q (it may be q itself when q is contiguous)");
  a.q = static_cast<const uint16_t*>(q);
  a.q_row = q_strides[0];
  a.q_head = q_strides[1];
  a.out = static_cast<uint16_t*>(out);
  const uintptr_t at = reinterpret_cast<uintptr_t>(out);
  a.out_align = at % 16 == 0 ? 2 : at % 4 == 0 ? 1 : 0;  // head_dim elements are a multiple of 16 bytes
  a.scale = scale;
  a.window = window;
  a.sinks = window > 0 ? sinks : 0;
  DeviceGuard guard(c->device);
  if (!guard.ok) return fail(KVQ_ERR_CUDA, "cannot select the cache's device");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t need = paged::paged_attn_workspace(a);
  if (workspace) {
    if (workspace_bytes < need)
      return fail(KVQ_ERR_WORKSPACE, "workspace too small: " + std::to_string(need) + " bytes needed");
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(KVQ_ERR_ARG, "paged: workspace must be 16-byte aligned");
    return paged::launch_paged_attn(a, workspace, need, st);
  }
  if (!need) return paged::launch_paged_attn(a, nullptr, 0, st);
  void* ws = nullptr;
  cudaMemPool_t pool = nullptr;
  if ((rc = scratch_pool(c->device, &pool))) return rc;
  KVQ_CUDA_TRY(cudaMallocFromPoolAsync(&ws, need, pool, st));
  rc = paged::launch_paged_attn(a, ws, need, st);
  const cudaError_t e = cudaFreeAsync(ws, st);
  if (!rc && e != cudaSuccess) return cuda_fail(e, "cudaFreeAsync(paged workspace)");
  return rc;
}

// Reads and clears the error flag in one step: a kernel of another stream may
// raise it at any time, and what it raises after this is the next check's.
__global__ void take_status(int* status, int* taken) { *taken = atomicExch(status, 0); }

// No exception leaves a C entry (bookkeeping maps and messages allocate).
template <class F>
int32_t guarded(F&& f) noexcept {
  try {
    return f();
  } catch (...) {
    try {
      return fail(KVQ_ERR_OOM, "out of host memory");
    } catch (...) {
      return KVQ_ERR_OOM;
    }
  }
}

}  // namespace

extern "C" {

int32_t kvq_paged_tile_bytes(const kvq_paged* c, size_t* bytes) {
  return guarded([&]() -> int32_t {
    if (!bytes) return fail(KVQ_ERR_ARG, "bytes is NULL");
    static int32_t dummy;
    if (!c) return fail(KVQ_ERR_ARG, "paged: NULL cache / batch");
    kvq_paged shape = *c;  // the pool itself need not exist yet
    shape.pool = reinterpret_cast<void*>(static_cast<uintptr_t>(16));
    shape.status = &dummy;
    kvq_paged_batch none{};
    paged::View v;
    int32_t rc = make_view(&shape, &none, v);
    if (rc) return rc;
    *bytes = (size_t)v.tile_bytes;
    return KVQ_OK;
  });
}

int32_t kvq_paged_append(const kvq_paged* c, const kvq_paged_batch* b, const void* k, const void* v,
                         const int64_t* k_strides, const int64_t* v_strides, const kvq_rope* rope,
                         const void* q, int32_t q_heads, const int64_t* q_strides, void* q_out,
                         void* stream) {
  return guarded([&]() -> int32_t {
    paged::AppendArgs a{};
    int32_t rc = make_view(c, b, a.v);
    if (rc) return rc;
    if (!a.v.cu && a.v.rows != a.v.B) return fail(KVQ_ERR_ARG, "paged: rows must equal batch without cu_rows");
    if (q && (q_heads <= 0 || !q_strides || !q_out)) return fail(KVQ_ERR_ARG, "paged: q needs q_heads, q_strides and q_out");
    if (q && q_out == q &&
        ((q_heads > 1 && q_strides[1] != a.v.D) || (a.v.rows > 1 && q_strides[0] != (int64_t)q_heads * a.v.D)))
      return fail(KVQ_ERR_ARG, "paged: q can be rotated in place only when it is contiguous");
    a.rope.base = 1.0;
    a.rope.scale = a.rope.pre = 1.0;
    if (rope) {
      if (rope->dims < 0 || rope->dims > a.v.D || rope->dims % 2)
        return fail(KVQ_ERR_ARG, "paged: rope dims must be even and within head_dim");
      if (rope->dims > 0 && !rope->freqs && !(rope->base > 0.0f))
        return fail(KVQ_ERR_ARG, "paged: rope base must be positive (or freqs given)");
      if (!aligned(rope->freqs, 4)) return fail(KVQ_ERR_ARG, "paged: rope freqs must be 4-byte aligned");
      a.rope.dims = rope->dims;
      a.rope.half = rope->dims / 2;
      a.rope.traditional = rope->traditional != 0;
      a.rope.base = rope->base;
      a.rope.scale = rope->scale != 0.0f ? rope->scale : 1.0f;
      a.rope.pre = rope->pre_scale != 0.0f ? rope->pre_scale : 1.0f;
      a.rope.freqs = rope->freqs;
    }
    if (a.v.rows == 0 || a.v.B == 0) return KVQ_OK;
    if (!k || !v || !k_strides || !v_strides) return fail(KVQ_ERR_ARG, "paged: NULL k / v / strides");
    if (!aligned(k, 2) || !aligned(v, 2) || (q && (!aligned(q, 2) || !aligned(q_out, 2))))
      return fail(KVQ_ERR_ARG, "paged: k, v, q and q_out must be 2-byte aligned");
    if (q && (shares(q_out, k, a.v.rows, a.v.Hkv, a.v.D, q_heads, k_strides[0], k_strides[1]) ||
              shares(q_out, v, a.v.rows, a.v.Hkv, a.v.D, q_heads, v_strides[0], v_strides[1]) ||
              (q_out != q && shares(q_out, q, a.v.rows, q_heads, a.v.D, q_heads, q_strides[0], q_strides[1]))))
      return fail(KVQ_ERR_ARG, "paged: q_out overlaps k, v or (other than as q itself) q");
    a.k = static_cast<const uint16_t*>(k);
    a.val = static_cast<const uint16_t*>(v);
    a.k_row = k_strides[0];
    a.k_head = k_strides[1];
    a.v_row = v_strides[0];
    a.v_head = v_strides[1];
    if (q) {
      a.q = static_cast<const uint16_t*>(q);
      a.q_row = q_strides[0];
      a.q_head = q_strides[1];
      a.q_out = static_cast<uint16_t*>(q_out);
      a.Hq = q_heads;
    }
    a.bf16 = c->dtype == KVQ_DTYPE_BFLOAT16;
    DeviceGuard guard(c->device);
    if (!guard.ok) return fail(KVQ_ERR_CUDA, "cannot select the cache's device");
    return paged::launch_paged_append(a, static_cast<cudaStream_t>(stream));
  });
}

int32_t kvq_paged_sdpa_workspace(const kvq_paged* c, const kvq_paged_batch* b, int32_t q_heads,
                                 int32_t decode, size_t* bytes) {
  return guarded([&]() -> int32_t {
    if (!bytes) return fail(KVQ_ERR_ARG, "bytes is NULL");
    paged::AttnArgs a;
    int32_t rc = make_attn(c, b, q_heads, decode != 0, a);
    if (rc) return rc;
    DeviceGuard guard(c->device);
    if (!guard.ok) return fail(KVQ_ERR_CUDA, "cannot select the cache's device");
    *bytes = paged::paged_attn_workspace(a);
    return KVQ_OK;
  });
}

int32_t kvq_paged_sdpa_decode(const kvq_paged* c, const kvq_paged_batch* b, const void* q,
                              int32_t q_heads, const int64_t* q_strides, float scale,
                              int32_t window, int32_t sinks, void* out, void* workspace,
                              size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int32_t {
    return sdpa(c, b, true, q, q_heads, q_strides, scale, window, sinks, out, workspace,
                workspace_bytes, stream);
  });
}

int32_t kvq_paged_sdpa_prefill(const kvq_paged* c, const kvq_paged_batch* b, const void* q,
                               int32_t q_heads, const int64_t* q_strides, float scale,
                               int32_t window, int32_t sinks, void* out, void* workspace,
                               size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int32_t {
    return sdpa(c, b, false, q, q_heads, q_strides, scale, window, sinks, out, workspace,
                workspace_bytes, stream);
  });
}

int32_t kvq_paged_check(const kvq_paged* c, void* stream) {
  return guarded([&]() -> int32_t {
    if (!c || !c->status) return fail(KVQ_ERR_ARG, "paged: NULL cache / status");
    DeviceGuard guard(c->device);
    if (!guard.ok) return fail(KVQ_ERR_CUDA, "cannot select the cache's device");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    KVQ_CUDA_TRY(cudaStreamSynchronize(st));
    int flag = 0;
    cudaMemPool_t pool = nullptr;
    int32_t rc = scratch_pool(c->device, &pool);
    if (rc) return rc;
    int* taken = nullptr;
    KVQ_CUDA_TRY(cudaMallocFromPoolAsync(reinterpret_cast<void**>(&taken), sizeof(int), pool, st));
    take_status<<<1, 1, 0, st>>>(c->status, taken);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaMemcpyAsync(&flag, taken, sizeof(int), cudaMemcpyDeviceToHost, st);
    const cudaError_t f = cudaFreeAsync(taken, st), w = cudaStreamSynchronize(st);
    for (cudaError_t x : {e, f, w})
      if (x != cudaSuccess) return cuda_fail(x, "kvq_paged_check");
    if (!flag) return KVQ_OK;
    if (flag & 2) return fail(KVQ_ERR_CUDA, "a paged kernel gave up waiting (its results are not valid)");
    return fail(KVQ_ERR_STATE,
                "a paged call met a row without a place, a page number outside the pool or a length "
                "beyond the page table (rows skipped, keys masked)");
  });
}

}  // extern "C"
