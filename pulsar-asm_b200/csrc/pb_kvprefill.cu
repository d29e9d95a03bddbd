// pb_kvprefill.cu -- attention of the last rows of each sequence over the
// paged K/V cache (prompt chunks; causal, window and sinks) on the tensor
// cores: tcgen05.mma kind::f16 with the scores, the probabilities and the
// output in TMEM.
//
// 4 D n_heads flops per visible pair of rows bound it, together with one
// exponential per pair and head (16 per clock and SM: as long as the matrix
// products at D = 128, twice as long at D = 64). So both have to run at once:
//  - a CTA takes up to 256 rows of one K/V head, in two groups of 128: a row
//    is one of the heads of the group and a token, so that short chunks fill
//    the tiles and a K/V tile serves all heads at once. Key tiles are 64 rows.
//  - per group, the scores S = Q K^T of a tile go to one of two TMEM buffers;
//    128 threads (a row each) turn them into probabilities, in place, while
//    the tensor cores work on the other group and on the next tile's scores;
//    O += P V takes P from TMEM and accumulates in TMEM.
//  - the running maximum only moves when a row's scores pass it by more than
//    2^8; the output is rescaled in TMEM then, which is rare. The sum of a row
//    stays with its thread. Any maximum that is near enough gives the same
//    quotient; so does a factor in the probabilities and their sum, which an
//    fp16 cache has (2^7).
// Warp 1 brings the queries, warp 0 K and V tiles, by TMA (a box per page, or part of one, and 64
// columns, in the 128-byte swizzle the tensor cores read; a table entry that
// names no page becomes a box outside the pool, which reads as zeros), warps 2
// and 3 issue the two groups' matrix products, warps 4-7 and 8-11 are the two
// groups' softmax (a warp reads its quarter of the TMEM lanes). In a tile at
// the end of what the queries see, V rows behind it are set to zero: they may
// hold anything, and 0 times that must be 0.
// 8192 tokens of 32/8 heads x 128 take 470 to 485 us, by the clock that the
// power cap leaves (1160 TFLOP/s at 474): tensor pipe and
// exponentials each busy half the time (56 %), the steps of the two groups
// meeting imperfectly. A ragged batch of 5 prompts to 4000 tokens with a
// window of 256, 16/4 x 128: 74 us; of a CTA's 12 some 4 pass until its first
// scores (search, first copies) and 2 at its end (the rows go out), beside 5
// to 7 tiles of 1 us. A chunk of 32 tokens against 4131 rows: 17 us, two
// launches and the join of the splits. (The queries by a warp of their own
// took the ragged batch from 77.5 to 73.9 us; asking for the next CTA's
// queries into L2 ahead of it gained nothing.)
// All waits are bounded; a wait that gives up
// records an error (pb_kv_status); copies and products in flight are waited
// for and the TMEM is freed before the CTA ends.
#include "pb_kvattn.cuh"
#include <cuda.h>
#include <mutex>

namespace {

constexpr int PF_KT = 64;                 // key rows per tile
constexpr int PF_MMA = 2;                 // the warp that issues the first group's products, the next one the second's
constexpr unsigned long long PF_WAIT_NS = 1000000000ull;

// (One group per CTA and two CTAs an SM took as long or longer on every shape
// tried, at the time: 515 against 500 us for 8192 tokens of 32/8 heads x 128, 419 against
// 393 at head_dim 64, 86 against 82 for the ragged batch with a window.)
constexpr int NG = 2;                     // groups of 128 rows per CTA
template <int D>
struct PfGeo {
  static constexpr int T = 128 + 128 * NG;        // threads
  static constexpr int Q = 128 * D * 2;           // bytes of a group's queries
  static constexpr int KV = PF_KT * D * 2;        // bytes of a K (or V) tile
  static constexpr int NST = D == 128 ? 5 : 8;    // stages of the K ring, and of the V ring
  static constexpr int SMEM = NG * Q + NST * 2 * KV + 1024;
  static constexpr int COLS = 512;                // TMEM columns allocated
  static constexpr uint32_t O_COL = NG * 128;     // S: group * 128 + buffer * 64; O: O_COL + group * D
};

struct PfArgs {
  AttnKvArgs a;
  int d_row, d_head, box;   // which of the tensor map's dimensions 1-3 are the row and the head (the third is the page); rows per box
  int tq, ns, out_bf16;     // tokens per group of 128 rows; splits of the key line
  float* part;              // [split][row][head][D] unnormalised sums (ns > 1)
  float2* ml;               // [split][row][head] maximum and sum
};

// waits that gave up on this device, by their role (1 to 15). The counts only
// grow: the host compares them with those that it reported last, so no record
// is lost between a read and a reset.
constexpr int PF_ROLES = 16;
__device__ unsigned kv_pf_gave_up[PF_ROLES];

PB_DEV void pf_init(uint64_t* b, unsigned c) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(kv_s32(b)), "r"(c) : "memory");
}
PB_DEV void pf_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(kv_s32(b)) : "memory");
}
PB_DEV bool pf_try(uint64_t* b, unsigned par) {
  uint32_t ok;
  asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(ok) : "r"(kv_s32(b)), "r"(par) : "memory");
  return ok != 0;
}
PB_DEV unsigned long long pf_now() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// A wait ends after about a second: it then records the role that gave up and
// raises the CTA's stop flag, at which every further wait returns at once. The
// roles run on through their loops (all accesses stay in bounds), so copies
// and products end and the TMEM is freed; the result is void.
PB_DEV void pf_wait_slow(uint64_t* b, unsigned par, volatile int* stop, int role, unsigned long long limit = PF_WAIT_NS) {
  const unsigned long long t0 = pf_now();
  for (unsigned i = 1; !pf_try(b, par); i++) {
    if ((i & 63) == 0) {
      if (*stop) return;
      if (pf_now() - t0 > limit) {
        *stop = 1;
        atomicAdd(&kv_pf_gave_up[role], 1u);
        return;
      }
    }
  }
}
PB_DEV void pf_wait(uint64_t* b, unsigned par, volatile int* stop, int role) {
  if (!pf_try(b, par)) pf_wait_slow(b, par, stop, role);
}
// the same whatever the other roles did: products in flight before the exit
PB_DEV void pf_drain(uint64_t* b, unsigned par) {
  const unsigned long long t0 = pf_now();
  for (unsigned i = 0; !pf_try(b, par); i++)
    if ((i & 63) == 63 && pf_now() - t0 > PF_WAIT_NS) return;
}
PB_DEV void pf_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
PB_DEV void pf_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
PB_DEV void pf_commit(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(kv_s32(b)) : "memory");
}
PB_DEV bool pf_elect() {
  uint32_t one;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(one));
  return one != 0;
}
// shared-memory descriptors, 128-byte swizzle (layout 2), version 1. K-major
// (Q, K): 8-row groups 1024 bytes apart. Row-major V as the N-major operand:
// 64-column panels `lbo` bytes apart, 8-key groups 1024 bytes apart.
PB_DEV uint64_t pf_desc(uint32_t at, uint32_t lbo) {
  return (uint64_t)((at >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}
PB_DEV void pf_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
PB_DEV void pf_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
#define PF_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define PF_W8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
// 32 consecutive columns of this thread's TMEM lane
PB_DEV void pf_ld32(uint32_t at, unsigned* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : PF_R8(v, 0), PF_R8(v, 8), PF_R8(v, 16), PF_R8(v, 24) : "r"(at));
}
PB_DEV void pf_ld16(uint32_t at, unsigned* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : PF_R8(v, 0), PF_R8(v, 8) : "r"(at));
}
PB_DEV void pf_st16(uint32_t at, const unsigned* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
               ::PF_W8(v, 0), PF_W8(v, 8), "r"(at) : "memory");
}
PB_DEV void pf_st8(uint32_t at, const unsigned* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::PF_W8(v, 0), "r"(at) : "memory");
}
PB_DEV void pf_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
PB_DEV void pf_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// packed pairs of fp32, each operation rounded on its own
typedef unsigned long long pf_f2;
PB_DEV pf_f2 pf_pk(float a, float b) {
  pf_f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
PB_DEV void pf_upk(pf_f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
PB_DEV pf_f2 pf_fma2(pf_f2 a, pf_f2 b, pf_f2 c) {
  pf_f2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
PB_DEV pf_f2 pf_add2(pf_f2 a, pf_f2 b) {
  pf_f2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
PB_DEV float pf_max3(float a, float b, float c) {   // NaN if any is
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
PB_DEV void pf_expect(uint64_t* b, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(kv_s32(b)), "r"(bytes) : "memory");
}
PB_DEV void pf_tma2(uint32_t dst, const CUtensorMap* m, int c0, int c1, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(m), "r"(c0), "r"(c1), "r"(kv_s32(bar)) : "memory");
}
PB_DEV void pf_tma(uint32_t dst, const CUtensorMap* m, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
               ::"r"(dst), "l"(m), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(kv_s32(bar)) : "memory");
}

// rows of q of sequence b: the first, and how many
PB_DEV int pf_count(const AttnKvArgs& a, int b, int& s0) {
  s0 = min(max(__ldg(a.start + b), 0), a.n_rows);
  return max(0, min(__ldg(a.start + b + 1), a.n_rows) - s0);
}

// the key tiles of one CTA: those of the sinks, then from the first query's
// window on (all of them where the two meet), to the last query's row
struct PfLine {
  int lo, sinks, end, nst, lot, nt;
};
PB_DEV PfLine pf_line(const AttnKvArgs& a, int t_first, int t_last) {
  PfLine s;
  s.end = max(0, t_last + 1);
  s.lo = a.window > 0 ? min(max(0, t_first + 1 - a.window), s.end) : 0;
  s.sinks = min(a.sinks, s.lo);
  s.nst = (s.sinks + PF_KT - 1) / PF_KT;
  s.lot = s.lo / PF_KT;
  if (s.nst >= s.lot) s.nst = s.lot = 0;
  s.nt = s.nst + (s.end + PF_KT - 1) / PF_KT - s.lot;
  return s;
}
// bits 0 .. x - 1
PB_DEV unsigned long long pf_below(int x) { return x <= 0 ? 0ull : (x >= 64 ? ~0ull : (1ull << x) - 1ull); }
// a tile with rows that no query of the CTA sees
PB_DEV bool pf_edge(const PfLine& s, int k0) { return k0 + PF_KT > s.end || (k0 < s.lo && k0 + PF_KT > s.sinks); }
PB_DEV int pf_key(const PfLine& s, int i) { return (i < s.nst ? i : i - s.nst + s.lot) * PF_KT; }

// P2: the probabilities as two numbers of the cache's type, for an output with
// more bits than that has; the second ones take the other half of the scores'
// columns, and a second product with V (8192 tokens of 32/8 heads x 128: 615
// against 505 us on one GPU; the ragged batch with a window 81 against 74).
// Elsewhere one number has to do, and in an output of the same type its
// rounding shows beside the output's own (bf16, ragged batch: error against 64
// bits 0.0022 of the output, 0.0016 with two).
template <int D, int CT, bool P2>
__global__ void __launch_bounds__(PfGeo<D>::T, 1) k_kv_prefill(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mq,
             PfArgs p) {
  typedef PfGeo<D> G;
  constexpr int NST = G::NST, KP = PF_KT * 128, QP = 128 * 128;   // bytes of a 64-column panel of K or V, of Q
  // log2: how far a score may pass the row's maximum before that moves, and the factor of the probabilities. In fp16,
  // what lies below 2^-25 would be 0 in the product with V but not in the sum, and many such rows together may be all
  // that an output has (a first row far above a long rest); so the two take all of the range above 1 and what is lost
  // lies below 2^-32. (Moving at 2^4 with a factor of 2^11: 513 against 478 us for 8192 tokens of 32/8 heads x 128.)
  constexpr int LAG = 8, UP = CT == PB_DT_F16 ? 15 - LAG : 0;
  extern __shared__ __align__(128) char psm_raw[];
  __shared__ uint64_t kfull[NST], kempty[NST], vfull[NST], vempty[NST], sfull[NG][2], pready[NG][2], pvdone[NG], ofin[NG], lock[4], qfull, vfix[3], done[NG];
  __shared__ uint32_t tbase;
  __shared__ int stop_f;
  const AttnKvArgs& a = p.a;
  char* smq = psm_raw + ((1024u - (kv_s32(psm_raw) & 1023u)) & 1023u);
  char* smk = smq + NG * G::Q;     // stage: K, V
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pb_grid_launch_dependents();
  if (warp == PF_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(kv_s32(&tbase)), "n"(G::COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 32) {             // (warp 1: the barriers, then the queries)
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mq) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
    for (int i = 0; i < NST; i++) {
      pf_init(&kfull[i], 1);
      pf_init(&vfull[i], 1);
    }
    for (int g = 0; g < NG; g++) {
      for (int i = 0; i < 2; i++) { pf_init(&sfull[g][i], 1); pf_init(&pready[g][i], 128); }
      pf_init(&pvdone[g], 1);
      pf_init(&ofin[g], 1);
      pf_init(&done[g], 1);
    }
    for (int i = 0; i < 4; i++) pf_init(&lock[i], 1);
    for (int i = 0; i < 3; i++) pf_init(&vfix[i], 1);
    pf_init(&qfull, 1);
    stop_f = 0;
  }
  __syncwarp();

  // ---- which rows: the last tiles of the line (the longest keys) first
  const int split = blockIdx.x % p.ns, kh = blockIdx.x / p.ns % a.p.n_kv, idx = blockIdx.x / p.ns / a.p.n_kv;
  int total, b, first;
  kv_locate<G::T>(a.p.n_seq, [&](int i) {
                    int s0;
                    asm volatile("prefetch.global.L1 [%0];" ::"l"(a.len + i));
                    return (pf_count(a, i, s0) + NG * p.tq - 1) / (NG * p.tq);
                  },
                  [&](int n) { return idx < n ? n - 1 - idx : n; }, total, b, first);
  if (idx >= total || b < 0) {         // CTA-uniform: no work
    pf_fence_before();
    __syncthreads();
    pf_fence_after();
    if (warp == PF_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "n"(G::COLS));
    return;
  }
  int row0;
  const int cnt = pf_count(a, b, row0), tok0 = (total - 1 - idx - first) * NG * p.tq, ntok = min(NG * p.tq, cnt - tok0);
  row0 += tok0;
  const int len = kv_len(__ldg(a.len + b), a.max_len), t0 = len - cnt + tok0;   // cache row of the first token (negative: before the cache)
  const PfLine line = pf_line(a, t0, t0 + ntok - 1);
  int i0 = 0, n = line.nt;
  if (p.ns > 1) {    // (nt is below 2^24, ns at most 160)
    i0 = (int)((unsigned)line.nt * split / (unsigned)p.ns);
    n = (int)((unsigned)line.nt * (split + 1) / (unsigned)p.ns) - i0;
  }
  const int ng = ntok > p.tq ? 2 : 1;   // groups with rows
  const int* trow = a.p.table + (size_t)b * a.p.table_ld;

  if (warp == 1) {
    if (lane < NST) {
      pf_init(&kempty[lane], ng);
      pf_init(&vempty[lane], ng);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // the pages of 8 tiles, 4 blocks of 16 rows each, a lane for each
  constexpr int BT = PF_KT / 16, AHEAD = 32 / BT;
  auto pages = [&](int i) {
    const int j = pf_key(line, i0 + i + lane / BT) + lane % BT * 16;
    const int e = i + lane / BT < n && j < line.end ? __ldg(trow + (j >> a.p.shift)) : -1;
    return (unsigned)e < (unsigned)a.p.n_pages ? e : a.p.n_pages;   // the box behind the last page: zeros
  };
  int now = warp == 0 ? pages(0) : 0;
  pf_fence_before();
  __syncthreads();
  pf_fence_after();
  const uint32_t tmem = tbase;
  volatile int* stop = &stop_f;

  if (warp == 0) {
    // ------------------------------------------------------------ copies
    int pg = 0, st = 0, sf = 0;
    unsigned epar = 1, fpar = 0;
    int fixes = 0;    // at most 3: where the sinks end, where the window begins, the last tile
    // a tile's V is looked at LATER tiles on: by then others are on their way
    // (fewer than NST, so that issuing them has not waited for this one's product)
    constexpr int LATER = 2;
    for (int i = 0; i < n + LATER; i++) {
      if (i < n) {
        const int k0 = pf_key(line, i0 + i), it = i % AHEAD;
        if (it == 0) {
          if (i > 0) now = pg;
          if (i + AHEAD < n) pg = pages(i + AHEAD);   // (for 8 tiles on)
        }
        const uint32_t ks = kv_s32(smk) + st * (2 * G::KV);
#pragma unroll
        for (int z = 0; z < 2; z++) {        // K, then V
          if (i >= NST) pf_wait(z ? &vempty[st] : &kempty[st], epar, stop, 1);
          __syncwarp();
          uint64_t* bar = z ? &vfull[st] : &kfull[st];
          if (lane == 0) pf_expect(bar, G::KV);
          for (int r = 0; r < PF_KT; r += p.box) {
            const int page = __shfl_sync(0xffffffffu, now, it * BT + (r >> 4)), row = (k0 + r) & ((1 << a.p.shift) - 1);
            if (lane == 0) {
              const int c1 = p.d_row == 1 ? row : (p.d_head == 1 ? kh : page), c2 = p.d_row == 2 ? row : (p.d_head == 2 ? kh : page),
                        c3 = p.d_row == 3 ? row : (p.d_head == 3 ? kh : page);
#pragma unroll
              for (int c = 0; c < D / 64; c++) pf_tma(ks + z * G::KV + c * KP + r * 128, z ? &mv : &mk, c * 64, c1, c2, c3, bar);
            }
          }
        }
        if (++st == NST) { st = 0; epar ^= 1; }
      }
      if (i >= LATER) {   // V rows behind what is seen
        const int k0 = pf_key(line, i0 + i - LATER);
        if (pf_edge(line, k0)) {
          pf_wait(&vfull[sf], fpar, stop, 9);
          char* vs = smk + sf * (2 * G::KV) + G::KV;
          for (int u = lane; u < PF_KT * (D / 8); u += 32) {
            const int r = u & (PF_KT - 1), j = k0 + r;
            if (j >= line.end || (j < line.lo && j >= line.sinks))
              *reinterpret_cast<uint4*>(vs + (u / PF_KT >> 3) * KP + r * 128 + (u / PF_KT & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && fixes < 3) pf_arrive(&vfix[fixes]);
          fixes++;
        }
        if (++sf == NST) { sf = 0; fpar ^= 1; }
      }
    }
    // no copy may land after the CTA ends: every tile was waited for by the products; where those
    // gave up, by time
    if (*stop) {
      const unsigned long long t1 = pf_now();
      while (pf_now() - t1 < 1000000ull) {}
    }
  } else if (warp == 1) {
    // the queries, beside the first keys: a box of tq tokens and 64 columns for each head (rows past the
    // sequence's last token are another's or zeros, and go nowhere)
    if (n > 0) {
      const int per = a.grp * (D / 64);
      if (lane == 0) pf_expect(&qfull, ng * per * (p.tq * 128));
      __syncwarp();
      for (int u = lane; u < ng * per; u += 32) {
        const int g = u / per, h = u % per / (D / 64), c = u % (D / 64);
        pf_tma2(kv_s32(smq) + g * G::Q + c * QP + h * p.tq * 128, &mq, (kh * a.grp + h) * D + c * 64, row0 + g * p.tq, &qfull);
      }
    }
  } else if (warp == PF_MMA || warp == PF_MMA + 1) {
    // ---------------------------------------------------- matrix products
    // kind::f16: D fp32 (bits 4-5 = 1), A and B fp16 (0) or bf16 (1) at bits 7 and 10, B N-major at bit 16,
    // N / 8 at bits 17-22, M / 16 at bits 24-28
    constexpr uint32_t ty = CT == PB_DT_BF16 ? 1u : 0u;
    constexpr uint32_t base = (1u << 4) | (ty << 7) | (ty << 10) | (8u << 24);
    constexpr uint32_t id_s = base | ((uint32_t)(PF_KT >> 3) << 17), id_o = base | (1u << 16) | ((uint32_t)(D >> 3) << 17);
    const uint64_t dq = pf_desc(kv_s32(smq), 16), dk = pf_desc(kv_s32(smk), 16), dv = pf_desc(kv_s32(smk) + G::KV, KP);
    // A warp per group, in which one elected thread waits and issues: with a
    // warp-wide wait, its vote and election, a step's waits took half its
    // time; operands that ptxas does not see as uniform cost 100 cycles per
    // product instead of 25 (a product takes 48 to 64); and one thread for
    // both groups spent 1900 cycles a step on its own waits and commits.
    const int g = warp - PF_MMA;
    if (g < ng && pf_elect()) {
      // scores of tile j
      auto scores = [&](int j, int st, unsigned par) {
        pf_wait(&kfull[st], par, stop, 2);
        // the buffer held P of tile j - 2: its product is done
        if (j >= 2) pf_wait(&pvdone[g], (unsigned)j & 1u, stop, 3);
        pf_fence_after();
        const uint64_t kb = dk + (uint64_t)(st * ((2 * G::KV) >> 4)), qb = dq + (uint64_t)((g * G::Q) >> 4);
        const uint32_t d = tmem + g * 128 + (uint32_t)(j & 1) * 64;
#pragma unroll
        for (int k = 0; k < D / 16; k++)
          pf_mma_ss(d, qb + (uint64_t)(((k >> 2) * QP + (k & 3) * 32) >> 4), kb + (uint64_t)(((k >> 2) * KP + (k & 3) * 32) >> 4),
                    id_s, k > 0);
        pf_commit(&sfull[g][j & 1]);
        pf_commit(&kempty[st]);
      };
      // The groups are held half a step apart, so that one's exponentials
      // fall beside the other's other work: the second group's next scores
      // wait for the first's probabilities, and the first's next but one for
      // the second's. (At their own pace they fell into step: 540 us instead
      // of 502, at the time, for 8192 tokens of 32/8 heads x 128; a share of
      // the exponentials by polynomial on the FMA pipe, 509 in step, did not
      // help further here.)
      int fixes = 0;                    // edge tiles so far
      int st = 0, s1 = 1, s2 = 2;                  // stages of tiles i, i + 1, i + 2
      unsigned p0 = 0, p1 = 0, p2 = 0;       // and the parities of their use
      if (n > 0) {
        pf_wait(&qfull, 0, stop, 10);
        scores(0, 0, 0);
        if (g == 0 && n > 1) scores(1, 1, 0);
      }
      for (int i = 0; i < n; i++) {
        const bool edge = pf_edge(line, pf_key(line, i0 + i));
        if (g == 1 && i + 1 < n) {
          pf_wait(&pready[0][i & 1], (unsigned)(i >> 1) & 1u, stop, 7);
          scores(i + 1, s1, p1);
        }
        pf_wait(&vfull[st], p0, stop, 13);
        if (edge && fixes < 3) pf_wait(&vfix[fixes++], 0, stop, 11);
        pf_wait(&pready[g][i & 1], (unsigned)(i >> 1) & 1u, stop, 4);
        if (g == 1) pf_arrive(&lock[i & 3]);
        pf_fence_after();
        const uint64_t vb = dv + (uint64_t)(st * ((2 * G::KV) >> 4));
        const uint32_t pb = tmem + g * 128 + (uint32_t)(i & 1) * 64, o = tmem + G::O_COL + g * D;
#pragma unroll
        for (int k = 0; k < (P2 ? 2 : 1) * (PF_KT / 16); k++)
          pf_mma_ts(o, pb + k * 8, vb + (uint64_t)((k % (PF_KT / 16) * 2048) >> 4), id_o, i > 0 || k > 0);
        pf_commit(i + 1 < n ? &pvdone[g] : &ofin[g]);
        pf_commit(&vempty[st]);
        if (g == 0 && i + 2 < n) {
          // (of four, as the other thread may be up to three tiles ahead)
          if (ng == 2) pf_wait(&lock[i & 3], (unsigned)(i >> 2) & 1u, stop, 12);
          scores(i + 2, s2, p2);
        }
        st = s1;
        p0 = p1;
        s1 = s2;
        p1 = p2;
        if (++s2 == NST) { s2 = 0; p2 ^= 1; }
      }
      // every product has completed before the TMEM is freed (bounded)
      pf_commit(&done[g]);
      pf_drain(&done[g], 0);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax
    const int g = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t to = tl + G::O_COL + (uint32_t)(g * D);
    const int tk = g * p.tq + r % p.tq, hq = r / p.tq;         // token within the CTA, head within the group
    const bool live = hq < a.grp && tk < ntok;
    const int t = t0 + min(tk, ntok - 1);                      // the row's own cache row
    const int wlo = a.window > 0 ? t + 1 - a.window : 0;       // it sees [wlo, t] and [0, sinks)
    // of the group: what all rows see, for tiles that need no masks
    const int ta = t0 + min(g * p.tq, ntok - 1), tb = t0 + min((g + 1) * p.tq - 1, ntok - 1);
    const int whi = a.window > 0 ? tb + 1 - a.window : 0;
    float m = -INFINITY, ms = 0.0f, l = 0.0f;                  // maximum of the raw scores, what is taken off the scaled ones, sum
    // does every 16-row block of the line have its page? (while the first tile is on its way)
    bool gap = false;
    if (g < ng)
      for (int u = lane; u < n * (PF_KT / 16); u += 32) {
        const int j = pf_key(line, i0 + u / (PF_KT / 16)) + u % (PF_KT / 16) * 16;
        if (j < line.end && kv_page(a.p, trow, j) < 0) gap = true;
      }
    const bool gaps = __any_sync(0xffffffffu, gap);
    const pf_f2 sc2 = pf_pk(a.scale2, a.scale2);
    const float over = (float)LAG / a.scale2;
    float thr = -INFINITY;                                     // m + over
    const int steps = g < ng ? n : 0;
    for (int i = 0; i < steps; i++) {
      const int k0 = pf_key(line, i0 + i);
      const uint32_t ts = tl + (uint32_t)(g * 128 + (i & 1) * 64);
      unsigned bad = 0;
      if (gaps) {
        const int j = k0 + (lane & (PF_KT / 16 - 1)) * 16;
        bad = ~__ballot_sync(0xffffffffu, j >= line.end || kv_page(a.p, trow, j) >= 0) & ((1u << (PF_KT / 16)) - 1u);
      }
      pf_wait(&sfull[g][i & 1], (unsigned)(i >> 1) & 1u, stop, 5);
      __syncwarp();
      pf_fence_after();
      unsigned s[PF_KT];
      pf_ld32(ts, s);
      pf_ld32(ts + 32, s + 32);
      pf_wait_ld();
      const bool masked = bad || k0 + PF_KT - 1 > ta || (k0 < whi && k0 + PF_KT > a.sinks);   // warp-uniform
      if (__builtin_expect(masked, 0)) {
        unsigned long long v = pf_below(t - k0 + 1) & (~pf_below(wlo - k0) | pf_below(a.sinks - k0));
#pragma unroll
        for (int u = 0; u < PF_KT / 16; u++)
          if ((bad >> u) & 1u) v &= ~(0xffffull << (16 * u));
#pragma unroll
        for (int k = 0; k < PF_KT; k++) s[k] = (v >> k) & 1ull ? s[k] : 0xff800000u;
      }
      float x[4];
#pragma unroll
      for (int u = 0; u < 4; u++) x[u] = __uint_as_float(s[u]);
#pragma unroll
      for (int k = 4; k + 8 <= PF_KT; k += 8)
#pragma unroll
        for (int u = 0; u < 4; u++) x[u] = pf_max3(x[u], __uint_as_float(s[k + 2 * u]), __uint_as_float(s[k + 2 * u + 1]));
      const float mx = pf_max3(pf_max3(x[0], x[1], pf_max3(__uint_as_float(s[60]), __uint_as_float(s[61]), __uint_as_float(s[62]))),
                               __uint_as_float(s[63]), pf_max3(x[2], x[3], x[2]));
      // the reference maximum: the first one, and a new one when a score
      // passes it by 2^8. A NaN or +inf makes the row's sum, and so its output, NaN.
      // (A row that is not one, where the group's heads do not fill 128 rows, multiplies whatever
      // shared memory held and must not ask for anything: with NaN there 3000 tokens of 12/2 heads x 64
      // took 59 us instead of 49.)
      const bool over_it = live && !(mx <= thr);
      if (__any_sync(0xffffffffu, over_it)) {
        const bool move = mx > thr;
        const float now_ms = kv_ref<UP>(mx * a.scale2);
        const float f = !move ? 1.0f : (m == -INFINITY ? 0.0f : kv_ex2(ms - now_ms));
        if (move) { m = mx; ms = now_ms; thr = mx + over; }
        if (over_it && !(mx < INFINITY)) l = __int_as_float(0x7fffffff);
        l *= f;
        if (i > 0) {   // the output so far, which the product of tile i - 1 has completed
          pf_wait(&pvdone[g], (unsigned)(i - 1) & 1u, stop, 6);
          __syncwarp();
          pf_fence_after();
#pragma unroll 2
          for (int e = 0; e < D; e += 16) {
            unsigned o[16];
            pf_ld16(to + e, o);
            pf_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            pf_st16(to + e, o);
          }
        }
      }
      // p = 2^(scale2 s - ms), rounded to the cache's type, which the product
      // with V needs; the sum takes the unrounded ones
      const pf_f2 nms = pf_pk(-ms, -ms);
      pf_f2 y[2] = {0ull, 0ull};
#pragma unroll
      for (int q = 0; q < 4; q++) {
        unsigned w[8], z[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
          float u, v;
          pf_upk(pf_fma2(pf_pk(__uint_as_float(s[16 * q + 2 * k]), __uint_as_float(s[16 * q + 2 * k + 1])), sc2, nms), u, v);
          u = kv_ex2(u);
          v = kv_ex2(v);
          y[k & 1] = pf_add2(y[k & 1], pf_pk(u, v));
          w[k] = kv_down<CT>(u, v);
          if (P2) {              // what that rounding left
            const float2 x = kv_up<CT>(w[k]);
            z[k] = kv_down<CT>(u - x.x, v - x.y);
          }
        }
        pf_st8(ts + q * 8, w);
        if (P2) pf_st8(ts + PF_KT / 2 + q * 8, z);
      }
      float ya, yb, yc, yd;
      pf_upk(y[0], ya, yb);
      pf_upk(y[1], yc, yd);
      l += (ya + yb) + (yc + yd);
      pf_wait_st();
      pf_fence_before();
      pf_arrive(&pready[g][i & 1]);
    }
    if (g < ng) {
      if (n > 0) {
        pf_wait(&ofin[g], 0, stop, 8);   // (a barrier of its own: pvdone may be one or two phases on)
        __syncwarp();
      }
      pf_fence_after();
      const int row = row0 + tk, h = kh * a.grp + hq;   // (of a live row)
      const float f = l != 0.0f ? 1.0f / l : 0.0f;       // nothing seen: zeros
      const size_t at = ((size_t)split * a.n_rows + row) * a.nh + h;
      if (p.ns == 1) {
        // by way of the (now idle) queries' rows, so that a warp writes whole rows together
        char* sr = smq + g * G::Q + r * 128;
#pragma unroll
        for (int e = 0; e < D; e += 64) {
          unsigned o[64];
          if (n > 0) {
            pf_ld32(to + e, o);
            pf_ld32(to + e + 32, o + 32);
            pf_wait_ld();
          } else {
#pragma unroll
            for (int k = 0; k < 64; k++) o[k] = 0u;
          }
#pragma unroll
          for (int k = 0; k < 64; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
#pragma unroll
          for (int k = 0; k < 8; k++) {
            uint4 w;
            unsigned* x = &w.x;
#pragma unroll
            for (int z = 0; z < 4; z++) {
              const float y0 = __uint_as_float(o[8 * k + 2 * z]), y1 = __uint_as_float(o[8 * k + 2 * z + 1]);
              x[z] = p.out_bf16 ? kv_down<PB_DT_BF16>(y0, y1) : kv_down<PB_DT_F16>(y0, y1);
            }
            const int c = e / 8 + k;
            *reinterpret_cast<uint4*>(sr + (c >> 3) * QP + (((c & 7) ^ (r & 7)) << 4)) = w;
          }
        }
        __syncwarp();
        // D / 8 lanes write a row; where it goes is known to the lane whose row it is
        constexpr int CPR = D / 8, RP = 32 / CPR;
        const int c = lane % CPR;
        const long long off = live ? (long long)row * a.ldo + h * (D * 2) : -1;
        const char* from = smq + g * G::Q + (c >> 3) * QP + (warp & 3) * (32 * 128);
#pragma unroll
        for (int i0 = 0; i0 < 32; i0 += RP) {
          const int i = i0 + lane / CPR;
          const long long to_row = __shfl_sync(0xffffffffu, off, i);
          if (to_row >= 0)
            *reinterpret_cast<uint4*>(a.out + to_row + c * 16) =
                *reinterpret_cast<const uint4*>(from + i * 128 + (((c & 7) ^ (i & 7)) << 4));
        }
      } else if (n > 0) {
#pragma unroll
        for (int e = 0; e < D; e += 16) {
          unsigned o[16];
          pf_ld16(to + e, o);
          pf_wait_ld();
          if (live)
#pragma unroll
            for (int k = 0; k < 16; k += 4)
              *reinterpret_cast<uint4*>(p.part + at * D + e + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
        }
      }
      if (live && p.ns > 1) p.ml[at] = make_float2(n > 0 ? ms : -INFINITY, n > 0 ? l : 0.0f);
    }
    pf_fence_before();
  }
  __syncthreads();
  if (warp == PF_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(G::COLS));
}

// The splits of each row and head joined, by D / 4 lanes: a lane reads the
// maximum and sum of every (D / 4)-th split, the factors go around by shuffle,
// and the sums of 8 splits are in flight together. A row belongs to a sequence
// or it is left alone.
template <int D>
__global__ void __launch_bounds__(128) k_kv_prefill_join(PfArgs p) {
  const AttnKvArgs& a = p.a;
  constexpr int L = D / 4, MOST = 160 / L;      // lanes per head; splits per lane (at most one split per SM)
  const int unit = (blockIdx.x * 128 + threadIdx.x) / L, l = threadIdx.x % L, e = l * 4;
  const int row = unit / a.nh, h = unit % a.nh;
  bool mine = row < a.n_rows;
  if (mine) {
    // the sequences are in ascending order: the last that starts at or before the row, if it reaches it
    int lo = 0, hi = a.p.n_seq;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(a.start + mid) <= row) lo = mid;
      else hi = mid;
    }
    int s0;
    const int c = pf_count(a, lo, s0);
    mine = row >= s0 && row < s0 + c;
  }
  pb_grid_wait();
  // (every lane of a head has the same `mine`; the others follow for the shuffles)
  const size_t step = (size_t)a.n_rows * a.nh, at = mine ? (size_t)row * a.nh + h : 0;
  float2 q[MOST];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < MOST; i++) {
    const int s = i * L + l;
    q[i] = mine && s < p.ns ? __ldcg(p.ml + s * step + at) : make_float2(-INFINITY, 0.0f);
    if (q[i].y != 0.0f) m = fmaxf(m, q[i].x);      // an empty split wrote no sums
  }
#pragma unroll
  for (int o = L / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float ll = 0.0f;
#pragma unroll
  for (int i = 0; i < MOST; i++) {
    q[i].x = q[i].y != 0.0f ? kv_ex2(q[i].x - m) : 0.0f;
    ll += q[i].x * q[i].y;
  }
#pragma unroll
  for (int o = L / 2; o; o >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, o);
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < MOST; i++) {
    if (i * L >= p.ns) break;
    const int n = min(L, p.ns - i * L);
#pragma unroll 8
    for (int k = 0; k < n; k++) {
      const float f = __shfl_sync(0xffffffffu, q[i].x, (threadIdx.x & 31) / L * L + k);
      if (!mine || f == 0.0f) continue;
      const float4 z = __ldcg(reinterpret_cast<const float4*>(p.part + ((i * L + k) * step + at) * D + e));
      y.x += f * z.x; y.y += f * z.y; y.z += f * z.z; y.w += f * z.w;
    }
  }
  if (!mine) return;
  const float f = ll != 0.0f ? 1.0f / ll : 0.0f;
  char* o = a.out + (long long)row * a.ldo + (size_t)h * (D * 2) + e * 2;
  uint2 w;
  if (p.out_bf16) w = make_uint2(kv_down<PB_DT_BF16>(y.x * f, y.y * f), kv_down<PB_DT_BF16>(y.z * f, y.w * f));
  else w = make_uint2(kv_down<PB_DT_F16>(y.x * f, y.y * f), kv_down<PB_DT_F16>(y.z * f, y.w * f));
  *reinterpret_cast<uint2*>(o) = w;
}

// launch shape: CTAs of NG * tq tokens, and splits of the key line where those
// leave SMs idle (at least 4 tiles each)
struct PfPlan {
  int tq, ns;
  long long items, part, ml;   // CTAs per split; floats
};
PfPlan pf_plan(const pb_kv_pages* c, int n_seq, int max_len, int n_tok, int n_heads, int window, int sinks) {
  PfPlan p{};
  const int grp = n_heads / c->n_kv;
  p.tq = 128 / (grp > 0 ? grp : 1) / 8 * 8;       // whole 8-row groups of the swizzle
  const int tok = NG * p.tq;
  p.items = ((long long)n_tok / tok + (n_seq < n_tok ? n_seq : n_tok)) * c->n_kv;
  long long tiles = (max_len + PF_KT - 1) / PF_KT;
  if (window > 0) {
    const long long seen = ((long long)window + tok + 2 * PF_KT - 1) / PF_KT + ((long long)sinks + PF_KT - 1) / PF_KT;
    if (seen < tiles) tiles = seen;
  }
  long long ns = p.items > 0 ? pb_num_sms() / p.items : 1;
  if (ns > tiles / 4) ns = tiles / 4;
  p.ns = ns < 1 ? 1 : (ns > 160 ? 160 : (int)ns);     // (what the join's lanes hold)
  const long long rows = (long long)p.ns * n_tok * n_heads;
  p.part = p.ns > 1 ? rows * c->head_dim : 0;
  p.ml = p.ns > 1 ? rows * 2 : 0;
  return p;
}

// The pools as tensors of rank 4, dimension 0 the columns, the others by
// ascending stride; a box is up to 64 rows of one page and 64 columns.
typedef CUresult (*PfEncode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
int pf_maps(const pb_kv_pages* c, PfArgs* p, CUtensorMap* mk, CUtensorMap* mv, CUtensorMap* mq) {
  static std::atomic<void*> fn{nullptr};
  void* f = fn.load(std::memory_order_acquire);
  if (!f) {
    cudaDriverEntryPointQueryResult found;
    PB_TRY_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || !f) return pb_set_error(PB_ECUDA, "pb_kv_prefill: no cuTensorMapEncodeTiled");
    fn.store(f, std::memory_order_release);
  }
  struct Dim { long long st; int n, box, what; } d[3] = {{c->row_stride, c->page_size, c->page_size < PF_KT ? c->page_size : PF_KT, 0},
                                                         {c->head_stride, c->n_kv, 1, 1},
                                                         {c->page_stride, c->n_pages, 1, 2}};
  p->box = d[0].box;
  // a dimension of size 1 takes part with the stride behind the larger ones
  long long far = c->head_dim;
  for (const Dim& x : d)
    if (x.n > 1 && x.st * x.n > far) far = x.st * x.n;
  for (Dim& x : d)
    if (x.n == 1) x.st = far;
  for (int i = 0; i < 2; i++)
    for (int j = 0; j < 2 - i; j++)
      if (d[j].st > d[j + 1].st) { const Dim x = d[j]; d[j] = d[j + 1]; d[j + 1] = x; }
  cuuint64_t dims[4] = {(cuuint64_t)c->head_dim}, strides[3];
  cuuint32_t box[4] = {64}, one[4] = {1, 1, 1, 1};
  for (int i = 0; i < 3; i++) {
    dims[i + 1] = (cuuint64_t)d[i].n;
    strides[i] = (cuuint64_t)d[i].st * 2;
    box[i + 1] = (cuuint32_t)d[i].box;
    if (d[i].what == 0) p->d_row = i + 1;
    if (d[i].what == 1) p->d_head = i + 1;
  }
  const CUtensorMapDataType ty = c->dtype == PB_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  for (int i = 0; i < 2; i++) {
    const CUresult r = reinterpret_cast<PfEncode>(f)(i ? mv : mk, ty, 4, i ? c->v : c->k, dims, strides, box, one,
                                                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return pb_set_error(PB_EINVAL, "pb_kv_prefill: strides the tensor map does not take (%d)", (int)r);
  }
  // the queries as a matrix [token][head and column]
  const cuuint64_t qdims[2] = {(cuuint64_t)p->a.nh * c->head_dim, (cuuint64_t)p->a.n_rows};
  const cuuint64_t qstride[1] = {(cuuint64_t)p->a.ldq};
  const cuuint32_t qbox[2] = {64, (cuuint32_t)p->tq};
  const CUresult r = reinterpret_cast<PfEncode>(f)(mq, ty, 2, const_cast<char*>(p->a.q), qdims, qstride, qbox, one,
                                                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return pb_set_error(PB_EINVAL, "pb_kv_prefill: a row stride of q that the tensor map does not take (%d)", (int)r);
  return PB_OK;
}

template <int D, int CT, bool P2>
int pf_run(const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq, const PfArgs& p, const PfPlan& pl, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  if (int rc = kv_smem(k_kv_prefill<D, CT, P2>, PfGeo<D>::SMEM, done)) return rc;
  if (int rc = kv_launch(k_kv_prefill<D, CT, P2>, (unsigned)(pl.items * p.ns), PfGeo<D>::T, PfGeo<D>::SMEM, st, false, "k_kv_prefill",
                         mk, mv, mq, p))
    return rc;
  if (p.ns == 1) return PB_OK;
  const long long blocks = ((long long)p.a.n_rows * p.a.nh * (D / 4) + 127) / 128;
  return kv_launch(k_kv_prefill_join<D>, (unsigned)blocks, 128, 0, st, true, "k_kv_prefill_join", p);
}
template <int D>
int pf_types(const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq, const PfArgs& p, const PfPlan& pl, int ct, cudaStream_t st) {
  if (ct == PB_DT_F16) return pf_run<D, PB_DT_F16, false>(mk, mv, mq, p, pl, st);
  return p.out_bf16 ? pf_run<D, PB_DT_BF16, false>(mk, mv, mq, p, pl, st) : pf_run<D, PB_DT_BF16, true>(mk, mv, mq, p, pl, st);
}

}  // namespace

extern "C" long long pb_kv_prefill_scratch(const pb_kv_pages* c, int n_seq, int max_len, int n_tok, int n_heads) {
  if (!c || n_seq < 0 || n_tok < 0 || n_heads <= 0 || c->n_kv <= 0 || n_heads / c->n_kv > 16) return -1;
  if (max_len <= 0) return n_seq == 0 && max_len == 0 ? 0 : -1;
  // (a window may need fewer splits: the whole cache's need covers both)
  const PfPlan p = pf_plan(c, n_seq, max_len, n_tok, n_heads, 0, 0);
  return 4 * (p.part + p.ml);
}

extern "C" int pb_kv_prefill(const pb_kv_pages* c, const pb_kv_attention_args* g, void* stream) {
  PfArgs p{};
  if (int rc = attn_check("pb_kv_prefill", c, g, g ? g->n_tok : 0, &p.a)) return rc;
  const int n_tok = g->n_tok, n_heads = g->n_heads;
  if (g->n_seq == 0 || n_tok == 0) return PB_OK;
  if (!g->start) return pb_set_error(PB_EINVAL, "pb_kv_prefill: null argument");
  const PfPlan pl = pf_plan(c, g->n_seq, p.a.max_len, n_tok, n_heads, g->window, g->sinks);
  if (pl.items * pl.ns > INT_MAX || (long long)n_tok * n_heads > INT_MAX)
    return pb_set_error(PB_EINVAL, "pb_kv_prefill: %d tokens of %d heads", n_tok, n_heads);
  if (int rc = attn_scratch("pb_kv_prefill", g, 4 * (pl.part + pl.ml))) return rc;
  p.a.start = g->start;
  p.tq = pl.tq;
  p.ns = pl.ns;
  p.out_bf16 = g->out_dtype == PB_DT_BF16;
  p.part = static_cast<float*>(g->scratch);
  p.ml = reinterpret_cast<float2*>(p.part + pl.part);
  cudaStream_t st = (cudaStream_t)stream;
  CUtensorMap mk, mv, mq;
  if (int rc = pf_maps(c, &p, &mk, &mv, &mq)) return rc;
  return c->head_dim == 64 ? pf_types<64>(mk, mv, mq, p, pl, c->dtype, st) : pf_types<128>(mk, mv, mq, p, pl, c->dtype, st);
}

extern "C" int pb_kv_status(void* stream) {
  static std::mutex mu;
  static unsigned reported[64][PF_ROLES];
  int dev = 0;
  PB_TRY_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return pb_set_error(PB_ENOTSUP, "pb_kv_status: device %d", dev);
  PB_TRY_CUDA(cudaStreamSynchronize((cudaStream_t)stream));
  std::lock_guard<std::mutex> lk(mu);
  unsigned now[PF_ROLES];
  PB_TRY_CUDA(cudaMemcpyFromSymbolAsync(now, kv_pf_gave_up, sizeof now, 0, cudaMemcpyDeviceToHost, (cudaStream_t)stream));
  PB_TRY_CUDA(cudaStreamSynchronize((cudaStream_t)stream));
  int role = 0;
  for (int i = 0; i < PF_ROLES; i++) {
    if (now[i] != reported[dev][i]) role = i;
    reported[dev][i] = now[i];
  }
  return role ? pb_set_error(PB_ECUDA, "k_kv_prefill: a bounded wait gave up (role %d)", role) : PB_OK;
}

namespace {
// the prompt kernel's wait on a barrier that nothing arrives at: it gives up
// after `limit` and records that; the next one then returns at once
__global__ void k_test_kv_wait(unsigned long long limit) {
  __shared__ uint64_t bar;
  __shared__ int stop;
  if (threadIdx.x == 0) {
    pf_init(&bar, 1);
    stop = 0;
    pf_wait_slow(&bar, 0, &stop, 14, limit);
    pf_wait_slow(&bar, 0, &stop, 15, limit);
  }
}
}  // namespace
// test hook (not part of the public ABI)
extern "C" int pb_test_kv_wait(unsigned long long limit_ns, void* stream) {
  k_test_kv_wait<<<1, 32, 0, (cudaStream_t)stream>>>(limit_ns);
  PB_LAUNCHED("k_test_kv_wait");
  return PB_OK;
}
