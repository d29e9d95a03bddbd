// pb_kvattn.cu -- attention over the paged K/V cache: one new token per
// sequence (pb_kv_decode) and the last rows of each sequence (pb_kv_prefill).
#include "pb_kv.cuh"
#include <climits>

namespace {

struct AttnKvArgs {
  KvPool p;
  const int* len;
  const int* start;     // prefill: row offsets [n_seq + 1]; null: row b is sequence b's one token
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

// sequence and own cache row of a query row; false when it has none
PB_DEV bool kv_row_of(const AttnKvArgs& a, int r, int& b, int& t) {
  if (!a.start) {
    b = r;
    t = kv_len(a.len[b], a.max_len) - 1;
    return true;
  }
  int lo = 0, hi = a.p.n_seq;   // the last sequence whose start is <= r
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.start[mid] <= r) lo = mid;
    else hi = mid;
  }
  b = lo;
  if (r < a.start[lo] || r >= a.start[lo + 1]) return false;
  t = kv_len(a.len[b], a.max_len) - (a.start[lo + 1] - r);
  return true;
}

// one CTA of 4 warps per query row and head, a key per warp and turn
template <int D, int CT, int OT>
__global__ void __launch_bounds__(128) k_kv_attn(AttnKvArgs a) {
  constexpr int E = D / 64;   // pairs per lane
  __shared__ float sm[4], sl[4], so[4][D];
  const int r = blockIdx.x / a.nh, h = blockIdx.x % a.nh, kh = h / a.grp;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int b, t;
  if (!kv_row_of(a, r, b, t)) return;
  const int* trow = a.p.table + (size_t)b * a.p.table_ld;
  float2 q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    q[e] = kv_up<CT>(*reinterpret_cast<const unsigned*>(a.q + (long long)r * a.ldq + (size_t)h * D * 2 + (e * 32 + lane) * 4));
    o[e] = make_float2(0.0f, 0.0f);
  }
  float m = -INFINITY, l = 0.0f;
  const int lo = a.window > 0 ? max(0, t + 1 - a.window) : 0, ns = min(a.sinks, lo), n = ns + (t + 1 - lo);
  for (int i = warp; i < n; i += 4) {
    const int j = i < ns ? i : lo + i - ns;
    const int page = kv_page(a.p, trow, j);
    if (page < 0) continue;
    const long long at = (long long)page * a.p.ps + (long long)kh * a.p.hs + (long long)(j & ((1 << a.p.shift) - 1)) * a.p.rs;
    float s = 0.0f;
    float2 v[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
      const float2 k = kv_up<CT>(*reinterpret_cast<const unsigned*>(a.p.k + at + (e * 32 + lane) * 4));
      v[e] = kv_up<CT>(*reinterpret_cast<const unsigned*>(a.p.v + at + (e * 32 + lane) * 4));
      s += q[e].x * k.x + q[e].y * k.y;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= a.scale2;
    const float mn = fmaxf(m, s), c = kv_ex2(m - mn), p = kv_ex2(s - mn);
    l = l * c + p;
    m = mn;
#pragma unroll
    for (int e = 0; e < E; e++) { o[e].x = o[e].x * c + p * v[e].x; o[e].y = o[e].y * c + p * v[e].y; }
  }
  if (lane == 0) { sm[warp] = m; sl[warp] = l; }
#pragma unroll
  for (int e = 0; e < E; e++) *reinterpret_cast<float2*>(&so[warp][(e * 32 + lane) * 2]) = o[e];
  __syncthreads();
  if (threadIdx.x < D / 2) {
    float mm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), ll = 0.0f;
    float2 x = make_float2(0.0f, 0.0f);
    if (mm != -INFINITY) {
      for (int w = 0; w < 4; w++) {
        const float c = kv_ex2(sm[w] - mm);
        ll += c * sl[w];
        x.x += c * so[w][2 * threadIdx.x];
        x.y += c * so[w][2 * threadIdx.x + 1];
      }
      x.x /= ll;
      x.y /= ll;
    }
    *reinterpret_cast<unsigned*>(a.out + (long long)r * a.ldo + (size_t)h * D * 2 + threadIdx.x * 4) = kv_down<OT>(x.x, x.y);
    if (a.lse && threadIdx.x == 0) a.lse[(size_t)r * a.nh + h] = ll > 0.0f ? mm + log2f(ll) : -INFINITY;
  }
}

// the weights: a warp per cache row and K/V head adds the row's probability
// under every query head of the group
template <int D, int CT>
__global__ void __launch_bounds__(128) k_kv_weight(AttnKvArgs a) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.y / a.p.n_kv, kh = blockIdx.y % a.p.n_kv;
  const int j = blockIdx.x * 4 + (threadIdx.x >> 5), t = kv_len(a.len[b], a.max_len) - 1;
  if (j > t || (a.window > 0 && j <= t - a.window && j >= a.sinks)) return;
  const int page = kv_page(a.p, a.p.table + (size_t)b * a.p.table_ld, j);
  if (page < 0) return;
  const int row = j & ((1 << a.p.shift) - 1);
  const char* kp = a.p.k + (long long)page * a.p.ps + (long long)kh * a.p.hs + (long long)row * a.p.rs;
  float sum = 0.0f;
  for (int g = 0; g < a.grp; g++) {
    const int h = kh * a.grp + g;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const float2 k = kv_up<CT>(*reinterpret_cast<const unsigned*>(kp + (e * 32 + lane) * 4));
      const float2 q = kv_up<CT>(*reinterpret_cast<const unsigned*>(a.q + (long long)b * a.ldq + (size_t)h * D * 2 + (e * 32 + lane) * 4));
      s += q.x * k.x + q.y * k.y;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    sum += kv_ex2(s * a.scale2 - a.lse[(size_t)b * a.nh + h]);
  }
  if (lane == 0) a.p.w[((size_t)page * a.p.n_kv + kh) * (1 << a.p.shift) + row] += sum;
}

int attn_check(const char* who, const pb_kv_pages* c, const KvPool& p, const int* d_len, int* max_len, int table_ld, int rows,
               int n_heads, const void* d_q, long long ldq, float scale, int window, int sinks, const void* d_out, int out_dtype,
               long long ldo, AttnKvArgs* a) {
  if (!d_len || !d_q || !d_out) return pb_set_error(PB_EINVAL, "%s: null argument", who);
  if (out_dtype != PB_DT_F16 && out_dtype != PB_DT_BF16)
    return pb_set_error(PB_ENOTSUP, "%s: out_dtype %d (fp16 or bf16)", who, out_dtype);
  if (n_heads <= 0 || n_heads % c->n_kv || n_heads / c->n_kv > 16)
    return pb_set_error(PB_ENOTSUP, "%s: %d query heads over %d K/V heads (a whole number, at most 16)", who, n_heads, c->n_kv);
  if (rows < 0 || window < 0 || sinks < 0 || !(scale > 0.0f) || scale > 1e30f)
    return pb_set_error(PB_EINVAL, "%s: %d rows, window %d, %d sinks, scale %g", who, rows, window, sinks, (double)scale);
  const long long wide = (long long)n_heads * c->head_dim;
  if (ldq < wide || ldo < wide || ((reinterpret_cast<size_t>(d_q) | reinterpret_cast<size_t>(d_out)) & 15) || ((ldq | ldo) & 7))
    return pb_set_error(PB_EINVAL, "%s: q and out rows must be 16-byte aligned (row strides %lld, %lld)", who, ldq, ldo);
  if (rows > 0 && kv_overlap(d_q, ((size_t)(rows - 1) * ldq + wide) * 2, d_out, ((size_t)(rows - 1) * ldo + wide) * 2))
    return pb_set_error(PB_EINVAL, "%s: out overlaps q", who);
  if (*max_len <= 0 || *max_len > table_ld * c->page_size) *max_len = table_ld * c->page_size;
  a->p = p;
  a->len = d_len;
  a->q = static_cast<const char*>(d_q);
  a->out = static_cast<char*>(const_cast<void*>(d_out));
  a->ldq = ldq * 2;
  a->ldo = ldo * 2;
  a->n_rows = rows;
  a->nh = n_heads;
  a->grp = n_heads / c->n_kv;
  a->max_len = *max_len;
  a->window = window;
  a->sinks = window > 0 ? sinks : 0;
  a->scale2 = scale * 1.4426950408889634f;
  return PB_OK;
}

template <int D>
void attn_launch(const AttnKvArgs& a, int ct, int ot, cudaStream_t st) {
  const unsigned g = (unsigned)((long long)a.n_rows * a.nh);
  if (ct == PB_DT_F16) {
    if (ot == PB_DT_F16) k_kv_attn<D, PB_DT_F16, PB_DT_F16><<<g, 128, 0, st>>>(a);
    else k_kv_attn<D, PB_DT_F16, PB_DT_BF16><<<g, 128, 0, st>>>(a);
  } else {
    if (ot == PB_DT_F16) k_kv_attn<D, PB_DT_BF16, PB_DT_F16><<<g, 128, 0, st>>>(a);
    else k_kv_attn<D, PB_DT_BF16, PB_DT_BF16><<<g, 128, 0, st>>>(a);
  }
}

}  // namespace

extern "C" long long pb_kv_decode_scratch(const pb_kv_pages* c, int n_seq, int max_len, int n_heads, int accumulate) {
  if (!c || n_seq < 0 || max_len < 0 || n_heads <= 0) return -1;
  return accumulate ? (long long)n_seq * n_heads * 4 : 0;
}

extern "C" int pb_kv_decode(const pb_kv_pages* c, int n_seq, const int* d_table, int table_ld, const int* d_len, int max_len,
                            int n_heads, const void* d_q, long long ldq, float scale, int window, int sinks, int accumulate,
                            void* d_out, int out_dtype, long long ldo, void* d_scratch, long long scratch_bytes, void* stream) {
  KvPool p{};
  AttnKvArgs a{};
  if (int rc = kv_pool("pb_kv_decode", c, n_seq, d_table, table_ld, &p)) return rc;
  if (int rc = attn_check("pb_kv_decode", c, p, d_len, &max_len, table_ld, n_seq, n_heads, d_q, ldq, scale, window, sinks, d_out,
                          out_dtype, ldo, &a))
    return rc;
  if (accumulate && !c->weight) return pb_set_error(PB_EINVAL, "pb_kv_decode: the cache keeps no weights");
  const long long need = pb_kv_decode_scratch(c, n_seq, max_len, n_heads, accumulate);
  if (need > 0 && (!d_scratch || scratch_bytes < need))
    return pb_set_error(PB_EINVAL, "pb_kv_decode: scratch of %lld bytes, %lld needed", scratch_bytes, need);
  if (n_seq == 0) return PB_OK;
  cudaStream_t st = (cudaStream_t)stream;
  a.lse = accumulate ? static_cast<float*>(d_scratch) : nullptr;
  if (c->head_dim == 64) attn_launch<64>(a, c->dtype, out_dtype, st);
  else attn_launch<128>(a, c->dtype, out_dtype, st);
  PB_LAUNCHED("k_kv_attn");
  if (accumulate) {
    const dim3 g((unsigned)((max_len + 3) / 4), (unsigned)(n_seq * c->n_kv));
    if (c->head_dim == 64) {
      if (c->dtype == PB_DT_F16) k_kv_weight<64, PB_DT_F16><<<g, 128, 0, st>>>(a);
      else k_kv_weight<64, PB_DT_BF16><<<g, 128, 0, st>>>(a);
    } else {
      if (c->dtype == PB_DT_F16) k_kv_weight<128, PB_DT_F16><<<g, 128, 0, st>>>(a);
      else k_kv_weight<128, PB_DT_BF16><<<g, 128, 0, st>>>(a);
    }
    PB_LAUNCHED("k_kv_weight");
  }
  return PB_OK;
}

extern "C" long long pb_kv_prefill_scratch(const pb_kv_pages* c, int n_seq, int max_len, int n_tok, int n_heads) {
  if (!c || n_seq < 0 || max_len < 0 || n_tok < 0 || n_heads <= 0) return -1;
  return 0;
}

extern "C" int pb_kv_prefill(const pb_kv_pages* c, int n_seq, const int* d_table, int table_ld, const int* d_start,
                             const int* d_len, int max_len, int n_tok, int n_heads, const void* d_q, long long ldq, float scale,
                             int window, int sinks, void* d_out, int out_dtype, long long ldo, void* d_scratch,
                             long long scratch_bytes, void* stream) {
  KvPool p{};
  AttnKvArgs a{};
  if (int rc = kv_pool("pb_kv_prefill", c, n_seq, d_table, table_ld, &p)) return rc;
  if (!d_start) return pb_set_error(PB_EINVAL, "pb_kv_prefill: null argument");
  if (int rc = attn_check("pb_kv_prefill", c, p, d_len, &max_len, table_ld, n_tok, n_heads, d_q, ldq, scale, window, sinks, d_out,
                          out_dtype, ldo, &a))
    return rc;
  if (n_seq == 0 || n_tok == 0) return PB_OK;
  if ((long long)n_tok * n_heads > INT_MAX) return pb_set_error(PB_EINVAL, "pb_kv_prefill: %d tokens of %d heads", n_tok, n_heads);
  a.start = d_start;
  cudaStream_t st = (cudaStream_t)stream;
  if (c->head_dim == 64) attn_launch<64>(a, c->dtype, out_dtype, st);
  else attn_launch<128>(a, c->dtype, out_dtype, st);
  PB_LAUNCHED("k_kv_attn");
  return PB_OK;
}
