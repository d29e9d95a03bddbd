// pb_kv.cu -- the paged K/V cache: append (head norms, rotation and store in
// one pass) and evict (the rows of largest accumulated weight to fresh pages).
#include "pb_kvattn.cuh"

namespace {

// ------------------------------------------------------------------ append
// Per token and head of D values: y = x w / sqrt(mean(x^2) + eps), then for
// i < half the pair (y_i, y_{i+D/2}) turned by the token's angle. All of it in
// fp32 with one rounding at the store. V heads are only rounded.
//
// Bytes bound it (each row in, each row out) as long as the instructions stay
// few: D / 16 lanes hold a head, each 8 values and their 8 partners of the
// rotation (16-byte loads and stores, nothing to exchange but the mean's
// sum), a warp 4 (D 128) or 8 (D 64) heads at a time, two such groups' loads
// in flight. A warp takes one token and every parts-th of its groups; its
// angles stay in registers, the norm weights in shared memory. (One lane per 8
// consecutive values, with shuffles for the partners, needed twice the
// instructions: 74 us for 8191 tokens of 32/8 heads x 128 in bf16, now 43,
// 4.8 TB/s; without any arithmetic 36.)
struct AppendArgs {
  KvPool p;
  const char* x;
  long long ldx, ldq;      // bytes
  char* q;
  const int* seq;
  const int* slot;
  const int* pos;          // null: the slot
  const float *qn, *kn, *cs, *sn;
  int xa;                  // bytes that every row of x is aligned to: 16, 8, 4 or 2
  int n_tok, nh, half, n_rope, rows, parts, n_qk, n_groups;   // groups of query and key heads, and with those of value heads
  float eps;
};

template <int XT>
struct KvRaw {             // 8 values
  uint4 a, b;
};
PB_DEV unsigned ap_ld16(const char* p) {
  unsigned short r;
  asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(r) : "l"(p));
  return r;
}
PB_DEV uint4 ap_ld(const char* p, int xa) {     // 16 bytes at less than 16-byte alignment
  uint4 r;
  if (xa == 8) {
    const uint2 x = pb_ldg_stream64(p), y = pb_ldg_stream64(p + 8);
    r = make_uint4(x.x, x.y, y.x, y.y);
  } else if (xa == 4) {
    r = make_uint4(pb_ldg_stream32(p), pb_ldg_stream32(p + 4), pb_ldg_stream32(p + 8), pb_ldg_stream32(p + 12));
  } else {
    r = make_uint4(ap_ld16(p) | ap_ld16(p + 2) << 16, ap_ld16(p + 4) | ap_ld16(p + 6) << 16,
                   ap_ld16(p + 8) | ap_ld16(p + 10) << 16, ap_ld16(p + 12) | ap_ld16(p + 14) << 16);
  }
  return r;
}
// VEC: rows on 16 bytes. A projection with a value per head behind v (gates)
// has other rows.
template <int XT, bool VEC>
PB_DEV void ap_load(KvRaw<XT>& r, const char* p, int xa) {
  r.a = VEC ? pb_ldg_stream(p) : ap_ld(p, xa);
  if (XT == PB_DT_F32) r.b = VEC ? pb_ldg_stream(p + 16) : ap_ld(p + 16, xa);
}
template <int XT>
PB_DEV void ap_up(const KvRaw<XT>& r, float (&x)[8]) {
  if (XT == PB_DT_F32) {
    const unsigned u[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __uint_as_float(u[i]);
  } else {
    const unsigned u[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = kv_up<XT>(u[i]);
      x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
  }
}
template <int CT>
PB_DEV uint4 ap_down(const float (&y)[8]) {
  return make_uint4(kv_down<CT>(y[0], y[1]), kv_down<CT>(y[2], y[3]), kv_down<CT>(y[4], y[5]), kv_down<CT>(y[6], y[7]));
}
PB_DEV void ap_floats(const float* p, int n, float past, float (&o)[8]) {   // p[0 .. 7], `past` from n on
  if (n >= 8 && (reinterpret_cast<size_t>(p) & 15) == 0) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(p)), y = __ldg(reinterpret_cast<const float4*>(p) + 1);
    o[0] = x.x; o[1] = x.y; o[2] = x.z; o[3] = x.w; o[4] = y.x; o[5] = y.y; o[6] = y.z; o[7] = y.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = i < n ? __ldg(p + i) : past;
  }
}


// packed pairs of fp32 (each operation rounds on its own)
typedef unsigned long long ap_f2;
PB_DEV ap_f2 ap_pk(float a, float b) {
  ap_f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
PB_DEV void ap_upk(ap_f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
PB_DEV ap_f2 ap_fma2(ap_f2 a, ap_f2 b, ap_f2 c) {
  ap_f2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
PB_DEV ap_f2 ap_mul2(ap_f2 a, ap_f2 b) {
  ap_f2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

constexpr int AP_W = 8;    // warps per CTA
constexpr int AP_U = 2;    // groups whose loads are in flight together

template <int D, int XT, int CT, bool VEC>
__global__ void __launch_bounds__(32 * AP_W, XT == PB_DT_F32 ? 3 : 4) k_kv_append(AppendArgs a) {
  constexpr int L = D / 16, HPW = 32 / L, XB = XT == PB_DT_F32 ? 4 : 2;
  __shared__ __align__(16) float nw[2][D];   // the norms' weights, of queries and of keys
  for (int i = threadIdx.x; i < 2 * D; i += 32 * AP_W) {
    const float* w = i < D ? a.qn : a.kn;
    nw[i / D][i % D] = w ? __ldg(w + i % D) : 1.0f;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, l = lane % L, sub = lane / L;
  const long long unit = (long long)blockIdx.x * AP_W + (threadIdx.x >> 5);
  const int t = (int)(unit / a.parts), part = (int)(unit % a.parts);
  if (t >= a.n_tok) return;
  const int nk = a.p.n_kv;
  const char* x0 = a.x + (long long)t * a.ldx + l * 8 * XB;
  // head of this lane in group g: query and key heads, then (from n_qk on) value heads
  auto head = [&](int g) { return g < a.n_qk ? g * HPW + sub : a.nh + nk + (g - a.n_qk) * HPW + sub; };
  auto live = [&](int g, int h) { return g < a.n_groups && h < (g < a.n_qk ? a.nh + nk : a.nh + 2 * nk); };
  KvRaw<XT> lo[AP_U], hi[AP_U];
  auto fetch = [&](int g, int u) {
    const int h = head(g);
    if (live(g, h)) {
      ap_load<XT, VEC>(lo[u], x0 + (size_t)h * (D * XB), a.xa);
      ap_load<XT, VEC>(hi[u], x0 + (size_t)h * (D * XB) + D / 2 * XB, a.xa);
    } else {
      lo[u].a = lo[u].b = hi[u].a = hi[u].b = make_uint4(0, 0, 0, 0);
    }
  };
#pragma unroll
  for (int u = 0; u < AP_U; u++) fetch(part + u * a.parts, u);   // before the look-ups of the destination

  const int seq = __ldg(a.seq + t), slot = __ldg(a.slot + t), pos = a.pos ? __ldg(a.pos + t) : slot;
  if ((unsigned)seq >= (unsigned)a.p.n_seq || (unsigned)slot >= (unsigned)a.rows) return;
  if (a.half > 0 && (unsigned)pos >= (unsigned)a.n_rope) return;
  const int page = kv_page(a.p, a.p.table + (size_t)seq * a.p.table_ld, slot);
  if (page < 0) return;
  const int row = slot & ((1 << a.p.shift) - 1);
  const long long at = (long long)page * a.p.ps + (long long)row * a.p.rs + l * 16;
  char* q0 = a.q + (long long)t * a.ldq + l * 16;
  float c[8], s[8];        // of pairs 8l .. 8l + 7
  ap_floats(a.cs + (size_t)pos * a.half + 8 * l, a.half - 8 * l, 1.0f, c);
  ap_floats(a.sn + (size_t)pos * a.half + 8 * l, a.half - 8 * l, 0.0f, s);
  const bool whole = a.half == D / 2;

  for (int g0 = part; g0 < a.n_groups; g0 += AP_U * a.parts) {
#pragma unroll
    for (int u = 0; u < AP_U; u++) {
      const int g = g0 + u * a.parts;
      if (g >= a.n_groups) break;      // warp-uniform
      const int h = head(g);
      const bool on = live(g, h);
      float x[8], y[8];
      ap_up<XT>(lo[u], x);
      ap_up<XT>(hi[u], y);
      fetch(g + AP_U * a.parts, u);    // the slot's next group
      if (g >= a.n_qk) {
        if (!on) continue;
        const int kh = h - a.nh - nk;
        char* v = a.p.v + at + (long long)kh * a.p.hs;
        *reinterpret_cast<uint4*>(v) = ap_down<CT>(x);
        *reinterpret_cast<uint4*>(v + D) = ap_down<CT>(y);
        if (a.p.w && l == 0) a.p.w[((size_t)page * nk + kh) * (1 << a.p.shift) + row] = 0.0f;
        continue;
      }
      const bool isq = h < a.nh;
      ap_f2 X[4], Y[4], sq = 0ull;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        X[i] = ap_pk(x[2 * i], x[2 * i + 1]);
        Y[i] = ap_pk(y[2 * i], y[2 * i + 1]);
        sq = ap_fma2(X[i], X[i], ap_fma2(Y[i], Y[i], sq));
      }
      float ss, s1;
      ap_upk(sq, ss, s1);
      ss += s1;
#pragma unroll
      for (int o = 1; o < L; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = (isq ? a.qn : a.kn) ? rsqrtf(ss * (1.0f / D) + a.eps) : 1.0f;
      const ap_f2 R = ap_pk(r, r);
      const ulonglong2* wl = reinterpret_cast<const ulonglong2*>(nw[isq ? 0 : 1] + 8 * l);
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const ulonglong2 w = wl[i], z = wl[i + D / 8];
        X[2 * i] = ap_mul2(X[2 * i], ap_mul2(R, w.x)); X[2 * i + 1] = ap_mul2(X[2 * i + 1], ap_mul2(R, w.y));
        Y[2 * i] = ap_mul2(Y[2 * i], ap_mul2(R, z.x)); Y[2 * i + 1] = ap_mul2(Y[2 * i + 1], ap_mul2(R, z.y));
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const ap_f2 C = ap_pk(c[2 * i], c[2 * i + 1]), S = ap_pk(s[2 * i], s[2 * i + 1]), T = ap_pk(-s[2 * i], -s[2 * i + 1]);
        const ap_f2 n0 = ap_fma2(Y[i], T, ap_mul2(X[i], C)), n1 = ap_fma2(X[i], S, ap_mul2(Y[i], C));
        float p, q, v, w;
        ap_upk(X[i], x[2 * i], x[2 * i + 1]);
        ap_upk(Y[i], y[2 * i], y[2 * i + 1]);
        ap_upk(n0, p, q);
        ap_upk(n1, v, w);
        if (whole || 8 * l + 2 * i < a.half) { x[2 * i] = p; y[2 * i] = v; }
        if (whole || 8 * l + 2 * i + 1 < a.half) { x[2 * i + 1] = q; y[2 * i + 1] = w; }
      }
      if (!on) continue;
      char* o = isq ? q0 + (size_t)h * (D * 2) : a.p.k + at + (long long)(h - a.nh) * a.p.hs;
      *reinterpret_cast<uint4*>(o) = ap_down<CT>(x);
      *reinterpret_cast<uint4*>(o + D) = ap_down<CT>(y);
    }
  }
}

template <int D, int XT, int CT>
void ap_launch_t(const AppendArgs& a, dim3 grid, cudaStream_t st) {
  if (a.xa == 16) k_kv_append<D, XT, CT, true><<<grid, 32 * AP_W, 0, st>>>(a);
  else k_kv_append<D, XT, CT, false><<<grid, 32 * AP_W, 0, st>>>(a);
}
template <int D, int XT>
void ap_launch(const AppendArgs& a, int ct, dim3 grid, cudaStream_t st) {
  if (ct == PB_DT_F16) ap_launch_t<D, XT, PB_DT_F16>(a, grid, st);
  else ap_launch_t<D, XT, PB_DT_BF16>(a, grid, st);
}

// ------------------------------------------------------------------- evict
// One CTA per sequence and K/V head finds the rows that stay: the first
// `sinks`, the last `recent`, and of the others the `need` of largest weight
// (equal weights: the lowest row first), by a radix select on the weights'
// bits (non-negative floats order as integers; anything not above zero counts
// as zero), then lists them in order with ballots. A row on no page is left
// out, whichever it is: moved nowhere, it must not count as a row of the new
// cache, where it would be seen. One sequence of 1087 rows
// to 1024: 10.7 us with the gather; the passes' barriers bound it, not its few
// bytes.
struct EvictArgs {
  KvPool p;
  const int* len;
  int* new_len;
  const int* dst;       // table of the fresh pages
  int dst_ld, max_len, budget, sinks, recent;
  int lcap;             // rows of a list: min(budget, max_len)
  int* list;            // [sequence][kv head][lcap], -1 behind the last kept row; null: no sequence passes the budget
  int staged;           // rows whose keys fit in shared memory
  bool in_place;        // new_len is len
};

constexpr int EV_T = 1024;
static_assert(EV_T == 32 * 32, "one lane of warp 0 scans each warp's sum");

constexpr unsigned EV_GONE = 0xffffffffu;   // the key of a row on no page; no weight has it

PB_DEV unsigned ev_key(const EvictArgs& a, const int* trow, int h, int j) {
  const int page = kv_page(a.p, trow, j);
  if (page < 0) return EV_GONE;
  const float w = a.p.w[((size_t)page * a.p.n_kv + h) * (1 << a.p.shift) + (j & ((1 << a.p.shift) - 1))];
  return w > 0.0f ? __float_as_uint(w) : 0u;
}

__global__ void __launch_bounds__(EV_T) k_kv_select(EvictArgs a) {
  extern __shared__ unsigned keys[];
  __shared__ int hist[2048];
  __shared__ int wsum[EV_T / 32], wsum2[EV_T / 32];
  __shared__ int s_bin, s_need, s_gone[2];   // (rows on no page: among those that compete, and the others)
  const int b = blockIdx.x / a.p.n_kv, h = blockIdx.x % a.p.n_kv;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  pb_grid_launch_dependents();
  const int len = kv_len(a.len[b], a.max_len);
  if (len <= a.budget) return;   // every row stays: no list
  const int* trow = a.p.table + (size_t)b * a.p.table_ld;
  const int lo = min(a.sinks, len), hi = max(lo, len - a.recent);   // [lo, hi) competes
  if (t < 2) s_gone[t] = 0;
  __syncthreads();
  for (int j = t << a.p.shift; j < len; j += EV_T << a.p.shift)
    if (kv_page(a.p, trow, j) < 0) {
      const int end = min(len, j + (1 << a.p.shift)), in = max(0, min(end, hi) - max(j, lo));
      atomicAdd(&s_gone[0], in);
      atomicAdd(&s_gone[1], end - j - in);
    }
  const int m = min(hi, a.staged);
  for (int j = lo + t; j < m; j += EV_T) keys[j] = ev_key(a, trow, h, j);
  __syncthreads();
  const bool gaps = s_gone[0] + s_gone[1] > 0;
  const int kept = min(a.budget, len - s_gone[0] - s_gone[1]);
  int need = kept - (len - (hi - lo) - s_gone[1]);   // how many of [lo, hi) stay (>= 0: sinks + recent <= budget)
  const bool all = need == hi - lo - s_gone[0];
  auto key = [&](int j) { return j < a.staged ? keys[j] : ev_key(a, trow, h, j); };

  unsigned prefix = 0, mask = 0;
  if (need > 0 && !all) {
    for (int pass = 0; pass < 3; pass++) {
      const int sh = pass == 0 ? 20 : (pass == 1 ? 10 : 0), nb = pass == 0 ? 2048 : 1024;
      for (int i = t; i < nb; i += EV_T) hist[i] = 0;
      __syncthreads();
      for (int j = lo + t; j < hi; j += EV_T) {
        const unsigned k = key(j);
        if (k != EV_GONE && (k & mask) == prefix) atomicAdd(&hist[(k >> sh) & (nb - 1)], 1);
      }
      __syncthreads();
      // the bin, counted from the top, in which the need-th largest key lies
      const int per = nb / EV_T;   // 2 or 1 bins per thread, from the top
      int own = 0;
      for (int i = 0; i < per; i++) own += hist[nb - 1 - (t * per + i)];
      int inc = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (lane == 31) wsum[warp] = inc;
      __syncthreads();
      if (warp == 0) {
        int v = wsum[lane], x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        wsum[lane] = x - v;
      }
      __syncthreads();
      int before = wsum[warp] + inc - own;   // keys in the bins above this thread's
      for (int i = 0; i < per; i++) {
        const int bin = nb - 1 - (t * per + i), n = hist[bin];
        if (before < need && before + n >= need) { s_bin = bin; s_need = need - before; }
        before += n;
      }
      __syncthreads();
      prefix |= (unsigned)s_bin << sh;
      mask |= (unsigned)(nb - 1) << sh;
      need = s_need;
      __syncthreads();
    }
  }
  // kept, if on a page: outside [lo, hi), a key above prefix, or one of the
  // first `need` keys equal to it; with `all`, every one. (need == 0 here only
  // when nothing of [lo, hi) stays.)
  const bool none = need == 0;
  auto keep = [&](int j, bool& gt, bool& eq) {
    if (j < lo || j >= hi) {
      gt = !gaps || kv_page(a.p, trow, j) >= 0;
    } else if (!none) {
      const unsigned k = key(j);
      gt = k != EV_GONE && (all || k > prefix);
      eq = !all && k == prefix;
    }
  };
  int* out = a.list + (size_t)blockIdx.x * a.lcap;
  const int seg = (len + EV_T - 1) / EV_T * 32, j0 = warp * seg, j1 = min(len, j0 + seg);
  int ngt = 0, neq = 0;
  for (int j = j0 + lane; j - lane < j1; j += 32) {
    bool gt = false, eq = false;
    if (j < j1) keep(j, gt, eq);
    ngt += __popc(__ballot_sync(0xffffffffu, gt));
    neq += __popc(__ballot_sync(0xffffffffu, eq));
  }
  if (lane == 0) { wsum[warp] = ngt; wsum2[warp] = neq; }
  __syncthreads();
  int pgt = 0, peq = 0;
  for (int w = 0; w < warp; w++) { pgt += wsum[w]; peq += wsum2[w]; }
  const unsigned lt = (1u << lane) - 1u;
  for (int j = j0 + lane; j - lane < j1; j += 32) {
    bool gt = false, eq = false;
    if (j < j1) keep(j, gt, eq);
    const unsigned bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    const int e = peq + __popc(be & lt);
    const int d = pgt + __popc(bg & lt) + min(e, need);
    if ((gt || (eq && e < need)) && d < a.lcap) out[d] = j;
    pgt += __popc(bg);
    peq += __popc(be);
  }
  for (int d = kept + t; d < a.lcap; d += EV_T) out[d] = -1;
}

// rows of sequence row trow, of its first len, that lie on a page; for a whole CTA
template <int T>
PB_DEV int ev_named(const KvPool& p, const int* trow, int len) {
  __shared__ int part[T / 32];
  int n = 0;
  for (int j = threadIdx.x << p.shift; j < len; j += T << p.shift)
    if (kv_page(p, trow, j) >= 0) n += min(1 << p.shift, len - j);
#pragma unroll
  for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0;
#pragma unroll
  for (int w = 0; w < T / 32; w++) n += part[w];
  return n;
}

// The kept rows to the fresh pages: D / 8 lanes per row, K and V and the
// weight, EV_R rows per lane group with all their loads in flight. A sequence
// within the budget has no list (for 16 sequences of 2500 to 4352 rows, most
// of them within 4096, lists of all rows cost 96 against 86 us): row i is row
// i, unless a page before it is missing. That is looked up beside the rows'
// loads, and only then the rows are found by counting. 16
// sequences of 2500 to 4352 rows to 4096, 32/8 heads x 128: 87 us with the
// select (17 of them, hardly beside the gather), 5.3 TB/s over the whole call.
constexpr int EV_R = 4, EV_GT = 256;

// rows c0 .. c0 + C - 1 of a sequence within the budget some of whose pages
// are missing: the pages in order, EV_GT at a time, with the rows before each
template <int D>
__device__ __noinline__ void ev_gather_named(const EvictArgs& a, int b, int h, int c0, int len) {
  constexpr int LPH = D / 8, G = EV_GT / LPH, C = G * EV_R;
  __shared__ int from_row[C], wsum[EV_GT / 32];
  const int t = threadIdx.x, ps = 1 << a.p.shift;
  const int* trow = a.p.table + (size_t)b * a.p.table_ld;
  for (int i = t; i < C; i += EV_GT) from_row[i] = -1;
  int base = 0;
  for (int j0 = 0; j0 < len && base < c0 + C; j0 += EV_GT << a.p.shift) {
    const int j = j0 + (t << a.p.shift), own = j < len && kv_page(a.p, trow, j) >= 0 ? min(ps, len - j) : 0;
    int inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if ((t & 31) >= o) inc += v;
    }
    __syncthreads();
    if ((t & 31) == 31) wsum[t >> 5] = inc;
    __syncthreads();
    int first = base + inc - own;
    for (int x = 0; x < EV_GT / 32; x++) {
      if (x < t >> 5) first += wsum[x];
      base += wsum[x];
    }
    for (int i = max(first, c0); i < min(first + own, c0 + C); i++) from_row[i - c0] = j + i - first;
  }
  __syncthreads();
  const int l = t % LPH;
  for (int r = t / LPH; r < C; r += G) {
    const int j = from_row[r], i = c0 + r;
    if (j < 0) break;
    const int sp = kv_page(a.p, trow, j), dp = kv_page(a.p, a.dst + (size_t)b * a.dst_ld, i);
    if (dp < 0) continue;
    const long long from = (long long)sp * a.p.ps + (long long)h * a.p.hs + (long long)(j & (ps - 1)) * a.p.rs + l * 16;
    const long long to = (long long)dp * a.p.ps + (long long)h * a.p.hs + (long long)(i & (ps - 1)) * a.p.rs + l * 16;
    *reinterpret_cast<uint4*>(a.p.k + to) = *reinterpret_cast<const uint4*>(a.p.k + from);
    *reinterpret_cast<uint4*>(a.p.v + to) = *reinterpret_cast<const uint4*>(a.p.v + from);
    if (l == 0)
      a.p.w[((size_t)dp * a.p.n_kv + h) * ps + (i & (ps - 1))] = a.p.w[((size_t)sp * a.p.n_kv + h) * ps + (j & (ps - 1))];
  }
}

template <int D>
__global__ void __launch_bounds__(EV_GT) k_kv_gather(const __grid_constant__ EvictArgs a, int chunks) {
  constexpr int LPH = D / 8, G = EV_GT / LPH, C = G * EV_R;   // lane groups, rows per CTA
  const int bh = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int b = bh / a.p.n_kv, h = bh % a.p.n_kv;
  const int t = threadIdx.x, l = t % LPH, g = t / LPH, c0 = chunk * C;
  const int len = kv_len(a.len[b], a.max_len), n = min(len, a.budget);   // (n: no more rows than that)
  const int ps = 1 << a.p.shift;
  const int* trow = a.p.table + (size_t)b * a.p.table_ld;
  const int* drow = a.dst + (size_t)b * a.dst_ld;
  const bool listed = len > a.budget;
  const int* list = a.list + ((size_t)b * a.p.n_kv + h) * a.lcap;
  pb_grid_launch_dependents();
  bool gone = false;
  if (!listed)
    for (int j = t << a.p.shift; j < min(n, c0 + C); j += EV_GT << a.p.shift) gone |= kv_page(a.p, trow, j) < 0;
  pb_grid_wait();      // the lists
  uint4 kk[EV_R], vv[EV_R];
  float w[EV_R];
  int to[EV_R];        // the fresh page, or -1
#pragma unroll
  for (int r = 0; r < EV_R; r++) {
    const int i = c0 + g + r * G;
    to[r] = -1;
    if (i >= n) continue;
    const int j = listed ? list[i] : i;
    if (j < 0) continue;
    const int sp = kv_page(a.p, trow, j), dp = kv_page(a.p, drow, i);
    if (sp < 0 || dp < 0) continue;
    const long long from = (long long)sp * a.p.ps + (long long)h * a.p.hs + (long long)(j & (ps - 1)) * a.p.rs + l * 16;
    to[r] = dp;
    kk[r] = *reinterpret_cast<const uint4*>(a.p.k + from);
    vv[r] = *reinterpret_cast<const uint4*>(a.p.v + from);
    w[r] = a.p.w[((size_t)sp * a.p.n_kv + h) * ps + (j & (ps - 1))];
  }
  if (!listed && __syncthreads_or(gone)) {
    ev_gather_named<D>(a, b, h, c0, len);
  } else {
#pragma unroll
    for (int r = 0; r < EV_R; r++) {
      if (to[r] < 0) continue;
      const int row = (c0 + g + r * G) & (ps - 1);
      const long long at = (long long)to[r] * a.p.ps + (long long)h * a.p.hs + (long long)row * a.p.rs + l * 16;
      *reinterpret_cast<uint4*>(a.p.k + at) = kk[r];
      *reinterpret_cast<uint4*>(a.p.v + at) = vv[r];
      if (l == 0) a.p.w[((size_t)to[r] * a.p.n_kv + h) * ps + row] = w[r];
    }
  }
  if (chunk == 0 && h == 0 && !a.in_place) {
    const int m = min(ev_named<EV_GT>(a.p, trow, len), a.budget);
    if (t == 0) a.new_len[b] = m;
  }
}

// The lengths where they replace the old ones, which every CTA of the gather
// reads: a kernel of its own behind it. (Apart from them, the gather's first
// CTA of each sequence writes them.)
constexpr int EV_LT = 128;
__global__ void __launch_bounds__(EV_LT) k_kv_lengths(EvictArgs a) {
  const int b = blockIdx.x;
  const int n = min(ev_named<EV_LT>(a.p, a.p.table + (size_t)b * a.p.table_ld, kv_len(a.len[b], a.max_len)), a.budget);
  pb_grid_wait();
  if (threadIdx.x == 0) a.new_len[b] = n;
}

}  // namespace

int kv_pool(const char* who, const pb_kv_pages* c, int n_seq, const int* d_table, int table_ld, KvPool* p) {
  if (!c || !c->k || !c->v || (n_seq > 0 && !d_table)) return pb_set_error(PB_EINVAL, "%s: null argument", who);
  if (c->dtype != PB_DT_F16 && c->dtype != PB_DT_BF16)
    return pb_set_error(PB_ENOTSUP, "%s: cache dtype %d (fp16 or bf16)", who, c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128)
    return pb_set_error(PB_ENOTSUP, "%s: head_dim %d (64 or 128)", who, c->head_dim);
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return pb_set_error(PB_ENOTSUP, "%s: page_size %d (16, 32, 64, 128 or 256)", who, c->page_size);
  if (c->n_pages <= 0 || c->n_kv <= 0 || c->n_kv > 1024 || n_seq < 0 || n_seq > (1 << 20) ||
      (n_seq > 0 && table_ld <= 0) || table_ld > (1 << 30) / c->page_size)
    return pb_set_error(PB_EINVAL, "%s: %d pages, %d K/V heads, %d sequences, table of %d pages", who, c->n_pages, c->n_kv,
                        n_seq, table_ld);
  if (((reinterpret_cast<size_t>(c->k) | reinterpret_cast<size_t>(c->v)) & 15) ||
      ((c->page_stride | c->head_stride | c->row_stride) & 7))
    return pb_set_error(PB_EINVAL, "%s: rows are 16-byte aligned (strides are multiples of 8 elements)", who);
  // the strides, smallest first, must each step over everything below it:
  // no two rows of the pool share memory
  struct { long long st; int n; } d[3] = {{c->page_stride, c->n_pages}, {c->head_stride, c->n_kv}, {c->row_stride, c->page_size}};
  for (int i = 0; i < 2; i++)
    for (int j = 0; j < 2 - i; j++)
      if (d[j].st > d[j + 1].st) { const auto x = d[j]; d[j] = d[j + 1]; d[j + 1] = x; }
  long long span = c->head_dim, below = 8;
  for (int i = 0; i < 3; i++) {
    if (d[i].n == 1) continue;
    // (2^38 elements, and whole multiples of the next smaller stride: what a tensor map takes)
    if (d[i].st < span || d[i].st > (1ll << 38) / d[i].n || d[i].st % below)
      return pb_set_error(PB_EINVAL, "%s: strides %lld (page), %lld (head), %lld (row): rows overlap, or one is not a multiple of the next smaller",
                          who, c->page_stride, c->head_stride, c->row_stride);
    span += d[i].st * (d[i].n - 1);
    below = d[i].st;
  }
  p->k = static_cast<char*>(c->k);
  p->v = static_cast<char*>(c->v);
  p->w = c->weight;
  p->table = d_table;
  p->ps = c->page_stride * 2;
  p->hs = c->head_stride * 2;
  p->rs = c->row_stride * 2;
  p->table_ld = table_ld;
  p->n_pages = c->n_pages;
  p->n_kv = c->n_kv;
  p->n_seq = n_seq;
  p->shift = 31 - __builtin_clz((unsigned)c->page_size);
  return PB_OK;
}

extern "C" int pb_kv_append(const pb_kv_pages* c, const pb_kv_append_args* g, void* stream) {
  if (!g) return pb_set_error(PB_EINVAL, "pb_kv_append: null argument");
  const int n_tok = g->n_tok, n_heads = g->n_heads, half = g->half, x_dtype = g->x_dtype;
  const long long ldx = g->ldx, ldq = g->ldq;
  AppendArgs a{};
  if (int rc = kv_pool("pb_kv_append", c, g->n_seq, g->table, g->table_ld, &a.p)) return rc;
  const int D = c->head_dim;
  if (n_tok == 0) return PB_OK;
  if (!g->qkv || !g->seq || !g->slot || !g->q) return pb_set_error(PB_EINVAL, "pb_kv_append: null argument");
  if (x_dtype != PB_DT_BF16 && x_dtype != PB_DT_F32 && x_dtype != PB_DT_F16)
    return pb_set_error(PB_EINVAL, "pb_kv_append: x_dtype %d", x_dtype);
  if (n_tok < 0 || n_heads <= 0 || n_heads > 65536) return pb_set_error(PB_EINVAL, "pb_kv_append: %d tokens, %d heads", n_tok, n_heads);
  if (half < 0 || half > D / 2 || (half > 0 && (!g->cos || !g->sin || g->n_rope <= 0)))
    return pb_set_error(PB_EINVAL, "pb_kv_append: half %d of head_dim %d, %d positions", half, D, g->n_rope);
  const long long wide = (long long)(n_heads + 2 * c->n_kv) * D;
  const int xb = x_dtype == PB_DT_F32 ? 4 : 2;
  if (ldx < wide || ldq < (long long)n_heads * D) return pb_set_error(PB_EINVAL, "pb_kv_append: row strides %lld, %lld", ldx, ldq);
  const size_t xa = reinterpret_cast<size_t>(g->qkv) | (n_tok > 1 ? (size_t)(ldx * xb) : 0) | 16;
  a.xa = (int)(xa & ~(xa - 1));
  if (a.xa < xb || ((reinterpret_cast<size_t>(g->q) | (size_t)(ldq * 2)) & 15))
    return pb_set_error(PB_EINVAL, "pb_kv_append: q rows must be 16-byte aligned, those of qkv aligned to its elements");
  if (kv_overlap(g->qkv, ((size_t)(n_tok - 1) * ldx + wide) * xb, g->q, ((size_t)(n_tok - 1) * ldq + (size_t)n_heads * D) * 2))
    return pb_set_error(PB_EINVAL, "pb_kv_append: q overlaps qkv");
  a.x = static_cast<const char*>(g->qkv);
  a.ldx = ldx * xb;
  a.q = static_cast<char*>(g->q);
  a.ldq = ldq * 2;
  a.seq = g->seq; a.slot = g->slot; a.pos = g->pos;
  a.qn = g->qnorm; a.kn = g->knorm; a.cs = g->cos; a.sn = g->sin;
  a.n_tok = n_tok; a.nh = n_heads; a.half = half; a.n_rope = g->n_rope;
  a.rows = g->table_ld * c->page_size;
  a.eps = g->eps;
  // few tokens: a warp per group of heads; many: up to 6 groups a warp (12,
  // a whole token of 48 heads, left a longer tail: 47 against 43 us; 1 paid
  // the look-ups each time: 81)
  const int hpw = 512 / D, nk = c->n_kv;
  a.n_qk = (n_heads + nk + hpw - 1) / hpw;
  a.n_groups = a.n_qk + (nk + hpw - 1) / hpw;
  const long long per = (long long)n_tok * a.n_groups / ((long long)pb_num_sms() * 24);
  const int iters = per < 1 ? 1 : (per > 6 ? 6 : (int)per);
  a.parts = (a.n_groups + iters - 1) / iters;
  const long long blocks = ((long long)n_tok * a.parts + AP_W - 1) / AP_W;
  if (blocks > INT_MAX) return pb_set_error(PB_EINVAL, "pb_kv_append: %d tokens", n_tok);
  const dim3 grid((unsigned)blocks);
  cudaStream_t st = (cudaStream_t)stream;
  if (D == 64) {
    if (x_dtype == PB_DT_BF16) ap_launch<64, PB_DT_BF16>(a, c->dtype, grid, st);
    else if (x_dtype == PB_DT_F16) ap_launch<64, PB_DT_F16>(a, c->dtype, grid, st);
    else ap_launch<64, PB_DT_F32>(a, c->dtype, grid, st);
  } else {
    if (x_dtype == PB_DT_BF16) ap_launch<128, PB_DT_BF16>(a, c->dtype, grid, st);
    else if (x_dtype == PB_DT_F16) ap_launch<128, PB_DT_F16>(a, c->dtype, grid, st);
    else ap_launch<128, PB_DT_F32>(a, c->dtype, grid, st);
  }
  PB_LAUNCHED("k_kv_append");
  return PB_OK;
}

extern "C" long long pb_kv_evict_scratch(const pb_kv_pages* c, int n_seq, int max_len, int budget) {
  if (!c || n_seq < 0 || c->n_kv <= 0 || budget <= 0) return -1;
  if (max_len <= 0) return n_seq == 0 && max_len == 0 ? 0 : -1;
  const long long cap = max_len > budget ? budget : 0;   // no list when nothing can pass the budget
  return (long long)n_seq * c->n_kv * cap * 4;
}

extern "C" int pb_kv_evict(const pb_kv_pages* c, const pb_kv_evict_args* g, void* stream) {
  if (!g) return pb_set_error(PB_EINVAL, "pb_kv_evict: null argument");
  const int n_seq = g->n_seq, table_ld = g->table_ld, budget = g->budget, sinks = g->sinks, recent = g->recent, dst_ld = g->dst_ld;
  int max_len = g->max_len;
  EvictArgs a{};
  if (int rc = kv_pool("pb_kv_evict", c, n_seq, g->table, table_ld, &a.p)) return rc;
  if (n_seq == 0) return PB_OK;
  if (!c->weight || !g->len || !g->dst_table || !g->new_len) return pb_set_error(PB_EINVAL, "pb_kv_evict: null argument");
  if (g->dst_table == g->table) return pb_set_error(PB_EINVAL, "pb_kv_evict: the fresh pages must not be the old ones");
  if (max_len <= 0 || max_len > table_ld * c->page_size) max_len = table_ld * c->page_size;
  if (budget <= 0 || sinks < 0 || recent < 0 || sinks > budget || recent > budget - sinks)
    return pb_set_error(PB_EINVAL, "pb_kv_evict: budget %d, %d first and %d last rows", budget, sinks, recent);
  const int cap = budget < max_len ? budget : max_len;
  if (dst_ld <= 0 || dst_ld < (cap + c->page_size - 1) / c->page_size)
    return pb_set_error(PB_EINVAL, "pb_kv_evict: %d rows need more than %d pages", cap, dst_ld);
  const long long need = pb_kv_evict_scratch(c, n_seq, max_len, budget);
  if (need > 0 && (!g->scratch || g->scratch_bytes < need || (reinterpret_cast<size_t>(g->scratch) & 15)))
    return pb_set_error(PB_EINVAL, "pb_kv_evict: scratch of %lld bytes, %lld needed (16-byte aligned)", g->scratch_bytes, need);
  a.in_place = g->new_len == g->len;
  if (!a.in_place && kv_overlap(g->len, (size_t)n_seq * 4, g->new_len, (size_t)n_seq * 4))
    return pb_set_error(PB_EINVAL, "pb_kv_evict: new_len is len, or apart from it");
  a.len = g->len; a.new_len = g->new_len; a.dst = g->dst_table; a.dst_ld = dst_ld;
  a.max_len = max_len; a.budget = budget; a.sinks = sinks; a.recent = recent;
  a.lcap = cap;
  a.list = max_len > budget ? static_cast<int*>(g->scratch) : nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  if (max_len > budget) {
    // keys in shared memory up to 40 KB (no opt-in needed), the rest re-read
    a.staged = max_len < 8192 ? max_len : 8192;
    k_kv_select<<<n_seq * c->n_kv, EV_T, (size_t)a.staged * 4, st>>>(a);
    PB_LAUNCHED("k_kv_select");
  }
  const int per = EV_GT / (c->head_dim / 8) * EV_R, chunks = (cap + per - 1) / per;
  const long long blocks = (long long)n_seq * c->n_kv * chunks;
  if (blocks > INT_MAX) return pb_set_error(PB_EINVAL, "pb_kv_evict: %d sequences of %d rows", n_seq, cap);
  const bool pdl = max_len > budget;   // (behind the select)
  int rc = c->head_dim == 64 ? kv_launch(k_kv_gather<64>, (unsigned)blocks, EV_GT, 0, st, pdl, "k_kv_gather", a, chunks)
                             : kv_launch(k_kv_gather<128>, (unsigned)blocks, EV_GT, 0, st, pdl, "k_kv_gather", a, chunks);
  if (!rc && a.in_place) rc = kv_launch(k_kv_lengths, (unsigned)n_seq, EV_LT, 0, st, true, "k_kv_lengths", a);
  return rc;
}
