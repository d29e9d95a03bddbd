// pb_kvattn.cuh -- what the two attention kernels over the paged K/V cache
// share (pb_kvattn.cu: one token per sequence; pb_kvprefill.cu: prompt
// chunks): arguments and their checks, the search of the line of work, copies.
#pragma once
#include "pb_kv.cuh"
#include <atomic>
#include <climits>

namespace {

struct AttnKvArgs {
  KvPool p;
  const int* len;
  const int* start;     // prefill: row offsets [n_seq + 1]
  const char* q;
  char* out;
  long long ldq, ldo;   // bytes
  int n_rows, nh, grp, max_len, window, sinks;
  float scale2;         // scale * log2(e): the softmax runs in powers of two
  float* lse;           // [row][nh]: log2 of the softmax sum (only for the weights)
};

PB_DEV float kv_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The probabilities of an fp16 cache carry a factor 2^UP, in the product with V
// and in the sum: they are 2^(s - kv_ref(m)) under the maximum m. None where a
// score's own step in fp32 (2^-4 and more) could bring them past fp16's range.
// Factors between maxima go by kv_ref as well, so that they agree with it.
template <int UP>
PB_DEV float kv_ref(float m) {
  return UP == 0 || !(fabsf(m) < 1048576.0f) ? m : m - (float)UP;
}

// Sequences laid end to end on a line, count(i) units each: the line's length
// and, for the unit pick(length), its sequence and that sequence's first unit
// (b = -1 when it lies past the line: the caller has no work then). A thread
// of the CTA's T sums a run of sequences; the runs are scanned.
template <int T, typename C, typename F>
PB_DEV void kv_locate(int n_seq, C count, F pick, int& total, int& b, int& first) {
  __shared__ int wsum[T / 32], found[2];
  if (n_seq == 1) {      // no search: one sequence's latency counts
    total = count(0);
    const int x = pick(total);
    b = x >= 0 && x < total ? 0 : -1;
    first = 0;
    return;
  }
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  if (n_seq <= 32) {     // a lane per sequence, each warp for itself: no barrier
    const int own = lane < n_seq ? count(lane) : 0;
    int inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    total = __shfl_sync(0xffffffffu, inc, 31);
    const int x = pick(total);
    const unsigned at = __ballot_sync(0xffffffffu, x >= inc - own && x < inc);
    b = __ffs((int)at) - 1;      // -1: none
    first = __shfl_sync(0xffffffffu, inc - own, b & 31);
    return;
  }
  const int per = (n_seq + T - 1) / T, b0 = min(n_seq, t * per), b1 = min(n_seq, b0 + per);
  int own = 0;
  for (int i = b0; i < b1; i++) own += count(i);
  int inc = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) wsum[warp] = inc;
  if (t == 0) found[0] = -1;
  __syncthreads();
  int pre = inc - own;
  total = 0;
#pragma unroll
  for (int w = 0; w < T / 32; w++) {
    if (w < warp) pre += wsum[w];
    total += wsum[w];
  }
  const int x = pick(total);
  if (x >= pre && x < pre + own) {
    for (int i = b0; i < b1; i++) {
      const int n = count(i);
      if (x < pre + n) {
        found[0] = i;
        found[1] = pre;
        break;
      }
      pre += n;
    }
  }
  __syncthreads();
  b = found[0];
  first = found[1];
}

PB_DEV uint32_t kv_s32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
PB_DEV void kv_cp16(uint32_t dst, const char* src, bool in) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
PB_DEV void kv_cp16(uint32_t dst, const char* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
PB_DEV void kv_cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
PB_DEV void kv_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// the checks of an attention call of `rows` query rows; fills a but for its
// prefill part
inline int attn_check(const char* who, const pb_kv_pages* c, const pb_kv_attention_args* g, int rows, AttnKvArgs* a) {
  if (!g) return pb_set_error(PB_EINVAL, "%s: null argument", who);
  if (int rc = kv_pool(who, c, g->n_seq, g->table, g->table_ld, &a->p)) return rc;
  if (rows < 0) return pb_set_error(PB_EINVAL, "%s: %d rows", who, rows);
  if (rows == 0 || g->n_seq == 0) return PB_OK;      // nothing to do: the caller returns
  if (!g->len || !g->q || !g->out) return pb_set_error(PB_EINVAL, "%s: null argument", who);
  if (g->out_dtype != PB_DT_F16 && g->out_dtype != PB_DT_BF16)
    return pb_set_error(PB_ENOTSUP, "%s: out_dtype %d (fp16 or bf16)", who, g->out_dtype);
  if (g->n_heads <= 0 || g->n_heads % c->n_kv || g->n_heads / c->n_kv > 16)
    return pb_set_error(PB_ENOTSUP, "%s: %d query heads over %d K/V heads (a whole number, at most 16)", who, g->n_heads, c->n_kv);
  if (g->window < 0 || g->sinks < 0 || !(g->scale > 0.0f) || g->scale > 1e30f)
    return pb_set_error(PB_EINVAL, "%s: window %d, %d sinks, scale %g", who, g->window, g->sinks, (double)g->scale);
  const long long wide = (long long)g->n_heads * c->head_dim;
  if (g->ldq < wide || g->ldo < wide || ((reinterpret_cast<size_t>(g->q) | reinterpret_cast<size_t>(g->out)) & 15) ||
      ((g->ldq | g->ldo) & 7))
    return pb_set_error(PB_EINVAL, "%s: q and out rows must be 16-byte aligned (row strides %lld, %lld)", who, g->ldq, g->ldo);
  if (kv_overlap(g->q, ((size_t)(rows - 1) * g->ldq + wide) * 2, g->out, ((size_t)(rows - 1) * g->ldo + wide) * 2))
    return pb_set_error(PB_EINVAL, "%s: out overlaps q", who);
  const int most = g->table_ld * c->page_size;
  a->len = g->len;
  a->q = static_cast<const char*>(g->q);
  a->out = static_cast<char*>(g->out);
  a->ldq = g->ldq * 2;
  a->ldo = g->ldo * 2;
  a->n_rows = rows;
  a->nh = g->n_heads;
  a->grp = g->n_heads / c->n_kv;
  a->max_len = g->max_len <= 0 || g->max_len > most ? most : g->max_len;
  a->window = g->window;
  a->sinks = g->window > 0 ? g->sinks : 0;
  a->scale2 = g->scale * 1.4426950408889634f;
  return PB_OK;
}
inline int attn_scratch(const char* who, const pb_kv_attention_args* g, long long need) {
  if (need > 0 && (!g->scratch || g->scratch_bytes < need || (reinterpret_cast<size_t>(g->scratch) & 15)))
    return pb_set_error(PB_EINVAL, "%s: scratch of %lld bytes, %lld needed (16-byte aligned)", who, g->scratch_bytes, need);
  return PB_OK;
}

// dynamic shared memory above 48 KB is allowed once per device and kernel
template <typename K>
inline int kv_smem(K k, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  PB_TRY_CUDA(cudaGetDevice(&dev));
  if (dev < 64 && (done.load(std::memory_order_acquire) >> dev) & 1) return PB_OK;
  PB_TRY_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
  return PB_OK;
}

template <typename... KArgs, typename... Args>
inline int kv_launch(void (*k)(KArgs...), unsigned grid, int block, int smem, cudaStream_t st, bool pdl, const char* name, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k, args...);
  if (e != cudaSuccess) return pb_set_error(PB_ECUDA, "%s: %s", name, cudaGetErrorString(e));
  pb_count_launch();
  return PB_OK;
}

}  // namespace
