// pb_kvattn.cu -- attention of one new token per sequence over the paged K/V
// cache (pb_kv_decode), and the weights eviction goes by.
#include "pb_kvattn.cuh"

namespace {

// ------------------------------------------------------------------ decode
// One token per sequence. The work is the K/V bytes: 2 D elements per seen
// row and K/V head, 4 D (n_heads / n_kv) flops on them, so HBM bounds it and
// the rest has to keep out of the way:
//  - the heads of a group share each row: S^T = K Q^T and O^T = V^T P^T as
//    m16n8k16 matrix products with the group's heads as the 8 columns (two
//    column tiles for groups of 9 to 16), K and V as they lie in memory;
//  - every warp streams its own rows through a private ring of shared memory
//    (16-byte asynchronous copies, rows that are not seen filled with zeros
//    and never read), with running maximum and sum per head: no barrier
//    until a piece of work ends;
//  - the tiles of all sequences and K/V heads form one line, cut into equal
//    pieces, one per CTA, whatever the lengths are; a sequence and head that a
//    cut goes through is joined by a second, small kernel from the pieces'
//    unnormalised sums, in the order of the line (the same bits every time).
// Two sequences of 65537 and 131071 rows, 32/8 heads x 128 bf16: 139 to 142 us,
// 6.4 to 6.5 TB/s, the rate of a plain copy. 64 ragged ones of 16 to 2048 rows, 32/8 x
// 64: 30 us, 4.5 TB/s; there each warp's chain of a tile's steps is what is
// left (58 % of the DRAM's cycles, 32 % of the issue slots, tensor pipe 9 %).
// One of 1029 rows: 6.7 us, the latency of two launches and one tile.
constexpr int DC_W = 4;      // warps per CTA

template <int D>
struct DcGeo {
  static constexpr int KT = 2048 / D;            // rows per warp and tile: 4 KB of K, 4 KB of V
  static constexpr int TILE = DC_W * KT;         // rows per tile
  static constexpr int NB = KT / 16;             // 16-row blocks: one page each
  static constexpr int NS = 2;                   // ring stages per warp: with 3 CTAs an SM faster than 3 stages and 2 CTAs
                                                 // (64 ragged: 29.7 against 32.1 us, long: 138 against 146, at the time): a warp's step is
                                                 // a chain of some 3000 cycles, which other warps have to fill
  static constexpr int RING = DC_W * NS * 8192;
  static constexpr int OP = 64 + 4;              // padded row of the merge buffer: 64 columns at a time, so
                                                 // that the join's CTAs fit beside two of these
  static constexpr int SMEM = RING + DC_W * 8 * OP * 4 + DC_W * 8 * 8;
};

struct DcArgs {
  AttnKvArgs a;
  float* part;       // [2 grid][grp][D] unnormalised sums of pieces that are not a whole item
  float* ml;         // [2 grid][grp][2] their maximum and sum
  float* score;      // [item][max_len][grp2] log2-scaled scores (only for the weights)
  int grid, grp2, out_bf16;
};

// tiles of sequence b: those of the sinks, then those from the window's first
// row on (all of them where the two meet). At least one, so that a sequence
// that sees nothing is written too.
struct DcSeq {
  int len, lo, sinks, nst, lot, nt;
};
template <int TILE>
PB_DEV DcSeq dc_seq(const AttnKvArgs& a, int b) {
  DcSeq s;
  s.len = kv_len(__ldg(a.len + b), a.max_len);
  s.lo = a.window > 0 ? max(0, s.len - a.window) : 0;
  s.sinks = min(a.sinks, s.lo);
  s.nst = (s.sinks + TILE - 1) / TILE;
  s.lot = s.lo / TILE;
  if (s.nst >= s.lot) s.nst = s.lot = 0;
  s.nt = max(1, s.nst + (s.len + TILE - 1) / TILE - s.lot);
  return s;
}

// the pieces: one per CTA, none of them empty
PB_DEV int dc_pieces(const DcArgs& d, int total) { return min(d.grid, total); }
// piece w of `grid` over `total` tiles begins at tile total w / grid
PB_DEV int dc_cut(int w, int total, int grid) { return (int)((long long)total * w / grid); }
// the piece that holds tile x
PB_DEV int dc_piece(int x, int total, int grid) { return (int)((((long long)x + 1) * grid - 1) / total); }

PB_DEV void kv_ldm(uint32_t at, unsigned (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
PB_DEV void kv_ldmt(uint32_t at, unsigned (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <int CT>
PB_DEV void kv_mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  if (CT == PB_DT_F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
PB_DEV unsigned kv_trans(unsigned x) {
  unsigned y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// a place on the line of tiles
struct DcAt {
  DcSeq s;
  int b, kh, t;
};
template <int TILE>
PB_DEV void dc_next(const AttnKvArgs& a, DcAt& w) {
  if (++w.t < w.s.nt) return;
  w.t = 0;
  if (++w.kh < a.p.n_kv) return;
  w.kh = 0;
  if (++w.b < a.p.n_seq) w.s = dc_seq<TILE>(a, w.b);
}

// output of one group: normalised rows, or the piece's sums
template <int D>
PB_DEV void dc_store(const DcArgs& d, int b, int h, int e, const float4& x) {
  char* o = d.a.out + (long long)b * d.a.ldo + (size_t)h * (D * 2) + e * 2;
  uint2 w;
  if (d.out_bf16) w = make_uint2(kv_down<PB_DT_BF16>(x.x, x.y), kv_down<PB_DT_BF16>(x.z, x.w));
  else w = make_uint2(kv_down<PB_DT_F16>(x.x, x.y), kv_down<PB_DT_F16>(x.z, x.w));
  *reinterpret_cast<uint2*>(o) = w;
}

// P2: the probabilities as two numbers of the cache's type, the second what the
// rounding of the first left, so that the output's own rounding is the largest
// error: for every output but bf16 of an fp16 cache, which has that with one
// (error against 64 bits of fp16 from bf16, 2 and 3 rows: 0.0002 instead of
// 0.0007 of the output; of bf16 from bf16, long: 0.0016 instead of 0.0020).
// Long caches take the same time (139.6 against 139.2 us), a window with sinks
// 63.9 against 63.8; with 64 ragged sequences, whose fp16 cache and bf16
// output do without, it would be 30.0 against 29.6.
template <int D, int CT, int NT, bool P2>
__global__ void __launch_bounds__(32 * DC_W, NT == 1 ? 3 : 2) k_kv_decode(DcArgs d) {
  typedef DcGeo<D> G;
  constexpr int KT = G::KT, TILE = G::TILE, NB = G::NB, NS = G::NS, CPR = D / 8, RS = 32 / CPR;
  constexpr int UP = CT == PB_DT_F16 ? 15 : 0;      // log2 of the probabilities' factor
  extern __shared__ __align__(128) char dsm[];
  const AttnKvArgs& a = d.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pb_grid_launch_dependents();
  int total, b, first;
  kv_locate<32 * DC_W>(a.p.n_seq, [&](int i) { return dc_seq<TILE>(a, i).nt * a.p.n_kv; }, [&](int n) { return dc_cut(blockIdx.x, n, dc_pieces(d, n)); }, total, b, first);
  const int pieces = dc_pieces(d, total);
  if ((int)blockIdx.x >= pieces || b < 0) return;   // CTA-uniform
  const int x0 = dc_cut(blockIdx.x, total, pieces), x1 = dc_cut(blockIdx.x + 1, total, pieces);
  DcAt at;
  at.b = b;
  at.s = dc_seq<TILE>(a, b);
  at.kh = (x0 - first) / at.s.nt;
  at.t = (x0 - first) % at.s.nt;

  // ---- the issuing side, NS - 1 tiles ahead
  char* ring = dsm + warp * (NS * 8192);
  const int cc = lane % CPR, rr = lane / CPR;
  const uint32_t ring0 = kv_s32(ring);
  uint32_t soff[16 / RS];   // this lane's chunk of its rows in a 16-row block, swizzled by the row
#pragma unroll
  for (int i = 0; i < 16 / RS; i++) {
    const int r = rr + i * RS;
    soff[i] = r * (D * 2) + ((cc ^ (r & 7)) << 4);
  }
  const long long step = (long long)RS * a.p.rs, lane_off = (long long)rr * a.p.rs + cc * 16;
  DcAt ia = at;
  int ix = x0, islot = 0;
  unsigned vbits = 0;       // validity of the 16-row blocks in flight, newest lowest
  int pg[NB];
  auto key0 = [&](const DcAt& w) {
    return (w.t < w.s.nst ? w.t : w.t - w.s.nst + w.s.lot) * TILE + warp * KT;
  };
  auto pages = [&]() {      // the pages of the tile to be issued next
    const int* trow = a.p.table + (size_t)ia.b * a.p.table_ld;
    const int j = key0(ia);
#pragma unroll
    for (int n = 0; n < NB; n++) pg[n] = j + n * 16 < ia.s.len ? __ldg(trow + ((j + n * 16) >> a.p.shift)) : -1;
  };
  pages();
  auto issue = [&]() {
    if (ix < x1) {
      const int j = key0(ia);
      const uint32_t st = ring0 + islot * 8192;
#pragma unroll
      for (int n = 0; n < NB; n++) {
        const bool ok = (unsigned)pg[n] < (unsigned)a.p.n_pages;
        vbits = (vbits << 1) | (ok ? 1u : 0u);
        const int j0 = j + n * 16;
        const uint32_t dst = st + n * (16 * D * 2);
        const bool some = ok && j0 < ia.s.len;
        const long long off = (some ? (long long)pg[n] * a.p.ps + (long long)(j0 & ((1 << a.p.shift) - 1)) * a.p.rs : 0) +
                              (long long)ia.kh * a.p.hs + lane_off;
        const char *kp = a.p.k + off, *vp = a.p.v + off;
        if (some && j0 + 16 <= ia.s.len && (j0 >= ia.s.lo || j0 + 16 <= ia.s.sinks)) {   // all 16 rows: no tests, no sizes
#pragma unroll
          for (int i = 0; i < 16 / RS; i++) {
            kv_cp16(dst + soff[i], kp);
            kv_cp16(dst + 4096 + soff[i], vp);
            kp += step;
            vp += step;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16 / RS; i++) {
            const int r = j0 + rr + i * RS;
            const bool in = ok && r < ia.s.len && (r >= ia.s.lo || r < ia.s.sinks);
            kv_cp16(dst + soff[i], in ? kp : a.p.k, in);
            kv_cp16(dst + 4096 + soff[i], in ? vp : a.p.v, in);
            kp += step;
            vp += step;
          }
        }
      }
      if (++ix < x1) {
        const int was = ia.b, kw = ia.kh;
        dc_next<TILE>(a, ia);
        pages();
        if (ia.b != was || ia.kh != kw) {   // the next group's queries on their way to L1
          const char* q = a.q + (long long)ia.b * a.ldq + (size_t)ia.kh * a.grp * (D * 2);
          if (lane * 128 < a.grp * D * 2) asm volatile("prefetch.global.L1 [%0];" ::"l"(q + lane * 128));
        }
      }
      if (++islot == NS) islot = 0;
    } else {
      vbits <<= NB;
    }
    kv_cp_commit();
  };
#pragma unroll
  for (int i = 0; i < NS - 1; i++) issue();

  // ---- the consuming side
  const int g = lane >> 2, c = lane & 3;
  unsigned qf[NT][D / 16][2];
  float o[NT][D / 16][4], m[NT][2], l[NT][2];
  int slot = 0;
  // ldmatrix: lane i gives the address of row i % 8 of matrix i / 8. K (rows
  // = keys): matrices (keys 0-7, dims 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15)
  const int lr = lane & 7, lq = lane >> 3;
  const int krow = lr + (lq & 1) * 8, kch = lq >> 1;
  // V transposed (rows = dims): (dims 0-7, keys 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15)
  const int vrow = lr + (lq >> 1) * 8, vch = lq & 1;
  float* mo = reinterpret_cast<float*>(dsm + G::RING);
  float* mml = mo + DC_W * 8 * G::OP;
  bool fresh = true;
  int t0 = at.t;            // first tile of this piece in its item
  for (int x = x0; x < x1; x++) {
    if (fresh) {
      fresh = false;
      t0 = at.t;
      const char* q = a.q + (long long)at.b * a.ldq + (size_t)at.kh * a.grp * (D * 2);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        const int h = n * 8 + g;
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
#pragma unroll
          for (int u = 0; u < 2; u++)
            qf[n][k][u] = h < a.grp ? __ldg(reinterpret_cast<const unsigned*>(q + (size_t)h * (D * 2) + (k * 16 + u * 8 + 2 * c) * 2)) : 0u;
        }
#pragma unroll
        for (int k = 0; k < D / 16; k++)
#pragma unroll
          for (int u = 0; u < 4; u++) o[n][k][u] = 0.0f;
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
      }
    }
    kv_cp_wait<NS - 2>();
    __syncwarp();           // the tile has landed for every lane, and its predecessor's slot is free
    const unsigned vb = vbits >> ((NS - 2) * NB);
    issue();
    const int j = key0(at);
    const uint32_t ks = ring0 + slot * 8192, vs = ks + 4096;
    if (++slot == NS) slot = 0;
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const int j0 = j + nb * 16;
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
      for (int k = 0; k < D / 16; k++) {
        unsigned f[4];
        kv_ldm(ks + (nb * 16 + krow) * (D * 2) + (((2 * k + kch) ^ (krow & 7)) << 4), f);
#pragma unroll
        for (int n = 0; n < NT; n++) kv_mma<CT>(s[n], f, qf[n][k][0], qf[n][k][1]);
      }
      const bool okb = (vb >> (NB - 1 - nb)) & 1u;
      const bool whole = okb && j0 + 16 <= at.s.len && (j0 >= at.s.lo || j0 + 16 <= at.s.sinks);   // warp-uniform
      const int ja = j0 + g, jb = ja + 8;
      const bool ina = whole || (okb && ja < at.s.len && (ja >= at.s.lo || ja < at.s.sinks));
      const bool inb = whole || (okb && jb < at.s.len && (jb >= at.s.lo || jb < at.s.sinks));
#pragma unroll
      for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
          s[n][u] = ina ? s[n][u] * a.scale2 : -INFINITY;
          s[n][2 + u] = inb ? s[n][2 + u] * a.scale2 : -INFINITY;
        }
        if (d.score) {
          const int h = n * 8 + 2 * c;
          if (h < d.grp2) {
            float* sp = d.score + (((size_t)at.b * a.p.n_kv + at.kh) * a.max_len + ja) * d.grp2 + h;
            if (ina) *reinterpret_cast<float2*>(sp) = make_float2(s[n][0], s[n][1]);
            if (inb) *reinterpret_cast<float2*>(sp + 8 * d.grp2) = make_float2(s[n][2], s[n][3]);
          }
        }
        float mx[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          mx[u] = fmaxf(s[n][u], s[n][2 + u]);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], w));
          mx[u] = fmaxf(mx[u], m[n][u]);
        }
        if (__any_sync(0xffffffffu, mx[0] > m[n][0] || mx[1] > m[n][1])) {
#pragma unroll
          for (int u = 0; u < 2; u++) {
            const float f = mx[u] > m[n][u] ? kv_ex2(kv_ref<UP>(m[n][u]) - kv_ref<UP>(mx[u])) : 1.0f;
            m[n][u] = mx[u];
            l[n][u] *= f;
#pragma unroll
            for (int k = 0; k < D / 16; k++) { o[n][k][u] *= f; o[n][k][2 + u] *= f; }
          }
        }
        // p in the cache's type for the matrix product; their sum in fp32 from before that rounding. In
        // fp16, times 2^15, in the sum as well: what lies below 2^-25 of the largest would be 0 there,
        // and many such rows together may be all that an output has (a first row far above the rest).
        float p[4];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const float r = m[n][u] == -INFINITY ? 0.0f : kv_ref<UP>(m[n][u]);
          p[u] = kv_ex2(s[n][u] - r);
          p[2 + u] = kv_ex2(s[n][2 + u] - r);
          l[n][u] += p[u] + p[2 + u];
        }
        const unsigned w0 = kv_down<CT>(p[0], p[1]), w1 = kv_down<CT>(p[2], p[3]);
        const unsigned b0 = kv_trans(w0), b1 = kv_trans(w1);
        unsigned c0 = 0, c1 = 0;
        if (P2) {                // what that rounding left
          const float2 x = kv_up<CT>(w0), y = kv_up<CT>(w1);
          c0 = kv_trans(kv_down<CT>(p[0] - x.x, p[1] - x.y));
          c1 = kv_trans(kv_down<CT>(p[2] - y.x, p[3] - y.y));
        }
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
          unsigned f[4];
          kv_ldmt(vs + (nb * 16 + vrow) * (D * 2) + (((2 * k + vch) ^ (vrow & 7)) << 4), f);
          kv_mma<CT>(o[n][k], f, b0, b1);
          if (P2) kv_mma<CT>(o[n][k], f, c0, c1);
        }
      }
    }
    const bool ends = at.t == at.s.nt - 1;
    if (ends || x == x1 - 1) {
      // the piece of this group is done: merge the warps
      const bool whole = t0 == 0 && ends;
      const int slot_p = 2 * blockIdx.x + (t0 == 0 ? 1 : 0);
#pragma unroll
      for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) l[n][u] += __shfl_xor_sync(0xffffffffu, l[n][u], w);
        }
#pragma unroll
        for (int half = 0; half < D / 64; half++) {
#pragma unroll
          for (int u = 0; u < 2; u++) {
            float* row = mo + (warp * 8 + 2 * c + u) * G::OP;
#pragma unroll
            for (int k = 0; k < 4; k++) {
              row[k * 16 + g] = o[n][half * 4 + k][u];
              row[k * 16 + g + 8] = o[n][half * 4 + k][2 + u];
            }
            if (g == 0) { mml[(warp * 8 + 2 * c + u) * 2] = kv_ref<UP>(m[n][u]); mml[(warp * 8 + 2 * c + u) * 2 + 1] = l[n][u]; }
          }
          __syncthreads();
          {
            const int h = threadIdx.x / 16, e = (threadIdx.x % 16) * 4, hg = n * 8 + h;      // 8 heads x 16 float4
            if (hg < a.grp) {
              float mm = -INFINITY, ll = 0.0f;
#pragma unroll
              for (int w = 0; w < DC_W; w++) mm = fmaxf(mm, mml[(w * 8 + h) * 2]);
              const float r = mm == -INFINITY ? 0.0f : mm;
              float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
              for (int w = 0; w < DC_W; w++) {
                const float f = kv_ex2(mml[(w * 8 + h) * 2] - r);
                const float4 z = *reinterpret_cast<const float4*>(mo + (w * 8 + h) * G::OP + e);
                ll += f * mml[(w * 8 + h) * 2 + 1];
                y.x += f * z.x; y.y += f * z.y; y.z += f * z.z; y.w += f * z.w;
              }
              const bool first_of = half == 0 && e == 0;
              if (whole) {
                const float f = ll != 0.0f ? 1.0f / ll : 0.0f;   // nothing seen: zeros
                dc_store<D>(d, at.b, at.kh * a.grp + hg, half * 64 + e, make_float4(y.x * f, y.y * f, y.z * f, y.w * f));
                if (a.lse && first_of) a.lse[(size_t)at.b * a.nh + at.kh * a.grp + hg] = mm + log2f(ll);
              } else {
                *reinterpret_cast<float4*>(d.part + ((size_t)slot_p * a.grp + hg) * D + half * 64 + e) = y;
                if (first_of) *reinterpret_cast<float2*>(d.ml + ((size_t)slot_p * a.grp + hg) * 2) = make_float2(mm, ll);
              }
            }
          }
          __syncthreads();
        }
      }
      fresh = true;
    }
    dc_next<TILE>(a, at);
  }
  kv_cp_wait<0>();
}

// One CTA per sequence and K/V head joins the pieces of a group that was cut,
// always in the same order: the pieces' factors first (a warp per head), then
// the sums, a float4 per thread; where a group has fewer of those than the CTA
// threads, slices of the pieces go to the others, so that the loads of all
// pieces are in flight at once (a thread per float4 alone took 11 us to join
// 32 pieces). JN_T is 512 for few groups, 128 where the CTAs fill the GPU
// several times and most groups are whole (64 x 8 groups: 33 against 35 us
// for the whole call).

template <int D, int JN_T>
__global__ void __launch_bounds__(JN_T) k_kv_join(DcArgs d) {
  const AttnKvArgs& a = d.a;
  constexpr int TILE = DcGeo<D>::TILE;
  extern __shared__ float fac[];      // [head][piece]
  __shared__ float4 sum[JN_T];
  __shared__ float inv[16];
  __shared__ int wsum[JN_T / 32][2];
  const int b = blockIdx.x / a.p.n_kv, kh = blockIdx.x % a.p.n_kv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pb_grid_launch_dependents();
  // tiles of the sequences before b, and of all
  int pre = 0, total = 0;
  for (int i = threadIdx.x; i < a.p.n_seq; i += JN_T) {
    const int n = dc_seq<TILE>(a, i).nt;
    total += n;
    if (i < b) pre += n;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    pre += __shfl_xor_sync(0xffffffffu, pre, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (lane == 0) { wsum[warp][0] = pre; wsum[warp][1] = total; }
  __syncthreads();
  pre = total = 0;
#pragma unroll
  for (int w = 0; w < JN_T / 32; w++) { pre += wsum[w][0]; total += wsum[w][1]; }
  pre *= a.p.n_kv;
  total *= a.p.n_kv;
  const int nt = dc_seq<TILE>(a, b).nt, s = pre + kh * nt;
  const int pieces = dc_pieces(d, total);
  const int w0 = dc_piece(s, total, pieces), np = dc_piece(s + nt - 1, total, pieces) - w0 + 1;
  pb_grid_wait();
  if (np == 1) return;     // whole: written by its CTA
  // piece k of this group lies in slot 2 (w0 + k), the first one in 2 w0 + 1
  for (int h = warp; h < a.grp; h += JN_T / 32) {
    float mm = -INFINITY, ll = 0.0f;
    for (int k = lane; k < np; k += 32) mm = fmaxf(mm, __ldcg(d.ml + ((size_t)(2 * (w0 + k) + (k == 0)) * a.grp + h) * 2));
#pragma unroll
    for (int o = 16; o; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    const float r = mm == -INFINITY ? 0.0f : mm;
    for (int k = lane; k < np; k += 32) {
      const float2 q = __ldcg(reinterpret_cast<const float2*>(d.ml + ((size_t)(2 * (w0 + k) + (k == 0)) * a.grp + h) * 2));
      const float f = kv_ex2(q.x - r);
      fac[h * np + k] = f;
      ll += f * q.y;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, o);
    if (lane == 0) {
      inv[h] = ll != 0.0f ? 1.0f / ll : 0.0f;
      if (a.lse) a.lse[(size_t)b * a.nh + kh * a.grp + h] = mm + log2f(ll);
    }
  }
  __syncthreads();
  const int items = a.grp * (D / 4), pass = min(items, JN_T), slices = JN_T / pass;
  const int slice = threadIdx.x / pass;
  for (int i = threadIdx.x % pass; i < items; i += pass) {      // one round, unless items > JN_T
    const int h = i / (D / 4), e = (i % (D / 4)) * 4;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (slice < slices) {
      const int k0 = np * slice / slices, k1 = np * (slice + 1) / slices;
#pragma unroll 8
      for (int k = k0; k < k1; k++) {
        const float4 z = __ldcg(reinterpret_cast<const float4*>(d.part + ((size_t)(2 * (w0 + k) + (k == 0)) * a.grp + h) * D + e));
        const float f = fac[h * np + k];
        y.x += f * z.x; y.y += f * z.y; y.z += f * z.z; y.w += f * z.w;
      }
    }
    if (slices > 1) {            // (one round then: every thread is here)
      sum[threadIdx.x] = y;
      __syncthreads();
      if (slice == 0)
        for (int s2 = 1; s2 < slices; s2++) {
          const float4 z = sum[s2 * pass + i];
          y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
        }
    }
    const float f = inv[h];
    if (slice == 0) dc_store<D>(d, b, kh * a.grp + h, e, make_float4(y.x * f, y.y * f, y.z * f, y.w * f));
  }
}

// The weights: a thread per seen row and K/V head adds the row's
// probabilities under the heads of the group, from the kept scores. The same
// line of tiles, in finer pieces: its few loads depend on one another, so it
// takes many small CTAs (with one piece per CTA of the attention this kernel
// took 46 us of a decode step of 16 sequences of 2048 to 4352 rows, 32/8
// heads x 128; in 32 per SM it takes 12, cold, of the step's 51).
template <int D>
__global__ void __launch_bounds__(DcGeo<D>::TILE) k_kv_weight(DcArgs d) {
  constexpr int TILE = DcGeo<D>::TILE;
  const AttnKvArgs& a = d.a;
  int total, b, first;
  kv_locate<TILE>(a.p.n_seq, [&](int i) { return dc_seq<TILE>(a, i).nt * a.p.n_kv; },
                  [&](int n) { return dc_cut(blockIdx.x, n, min(n, (int)gridDim.x)); }, total, b, first);
  const int pieces = min(total, (int)gridDim.x);
  if ((int)blockIdx.x >= pieces || b < 0) return;
  const int x0 = dc_cut(blockIdx.x, total, pieces), x1 = dc_cut(blockIdx.x + 1, total, pieces);
  DcAt at;
  at.b = b;
  at.s = dc_seq<TILE>(a, b);
  at.kh = (x0 - first) / at.s.nt;
  at.t = (x0 - first) % at.s.nt;
  pb_grid_wait();
  for (int x = x0; x < x1; x++, dc_next<TILE>(a, at)) {
    const int j = (at.t < at.s.nst ? at.t : at.t - at.s.nst + at.s.lot) * TILE + threadIdx.x;
    if (j >= at.s.len || (j < at.s.lo && j >= at.s.sinks)) continue;
    const int page = kv_page(a.p, a.p.table + (size_t)at.b * a.p.table_ld, j);
    if (page < 0) continue;
    float* w = a.p.w + ((size_t)page * a.p.n_kv + at.kh) * (1 << a.p.shift) + (j & ((1 << a.p.shift) - 1));
    const float* sp = d.score + (((size_t)at.b * a.p.n_kv + at.kh) * a.max_len + j) * d.grp2;
    const float* lp = a.lse + (size_t)at.b * a.nh + at.kh * a.grp;
    const float was = *w;
    float sum = 0.0f;
    for (int h = 0; h < a.grp; h += 2) {
      const float2 s = __ldcg(reinterpret_cast<const float2*>(sp + h));
      sum += kv_ex2(s.x - __ldcg(lp + h));
      if (h + 1 < a.grp) sum += kv_ex2(s.y - __ldcg(lp + h + 1));
    }
    *w = was + sum;
  }
}

// launch shape and scratch of a decode call
struct DcPlan {
  int grid, grp2;
  bool join;
  long long part, ml, lse, score;   // floats
};
template <int D>
DcPlan dc_plan_t(int n_seq, int n_kv, int max_len, int grp, int accumulate) {
  DcPlan p{};
  const long long most = (max_len + DcGeo<D>::TILE - 1) / DcGeo<D>::TILE, items = (long long)n_seq * n_kv;
  const long long all = items * (most > 0 ? most : 1), cap = (grp > 8 ? 2LL : 3LL) * pb_num_sms();
  p.grid = (int)(all < cap ? all : cap);
  p.grp2 = (grp + 1) / 2 * 2;
  // a sequence of one tile cannot be cut
  p.join = most > 1;
  p.part = p.join ? 2LL * p.grid * grp * D : 0;
  p.ml = p.join ? 2LL * p.grid * grp * 2 : 0;
  p.lse = accumulate ? (items * grp + 3) / 4 * 4 : 0;
  p.score = accumulate ? items * max_len * p.grp2 : 0;
  return p;
}
DcPlan dc_plan(const pb_kv_pages* c, int n_seq, int max_len, int n_heads, int accumulate) {
  return c->head_dim == 64 ? dc_plan_t<64>(n_seq, c->n_kv, max_len, n_heads / c->n_kv, accumulate)
                           : dc_plan_t<128>(n_seq, c->n_kv, max_len, n_heads / c->n_kv, accumulate);
}

template <int D, int CT, int NT, bool P2>
int dc_launch(const DcArgs& d, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  if (int rc = kv_smem(k_kv_decode<D, CT, NT, P2>, DcGeo<D>::SMEM, done)) return rc;
  return kv_launch(k_kv_decode<D, CT, NT, P2>, (unsigned)d.grid, 32 * DC_W, DcGeo<D>::SMEM, st, false, "k_kv_decode", d);
}

template <int D>
int dc_run(const DcArgs& d, int ct, bool join, cudaStream_t st) {
  const bool two = d.a.grp > 8;
  int rc;
  if (ct == PB_DT_F16 && d.out_bf16) rc = two ? dc_launch<D, PB_DT_F16, 2, false>(d, st) : dc_launch<D, PB_DT_F16, 1, false>(d, st);
  else if (ct == PB_DT_F16) rc = two ? dc_launch<D, PB_DT_F16, 2, true>(d, st) : dc_launch<D, PB_DT_F16, 1, true>(d, st);
  else rc = two ? dc_launch<D, PB_DT_BF16, 2, true>(d, st) : dc_launch<D, PB_DT_BF16, 1, true>(d, st);
  if (rc) return rc;
  // (a group's pieces: at most one per tile and per CTA)
  const int tiles = (d.a.max_len + DcGeo<D>::TILE - 1) / DcGeo<D>::TILE, np = d.grid < tiles ? d.grid : tiles;
  if (join) {
    const unsigned groups = (unsigned)(d.a.p.n_seq * d.a.p.n_kv);
    rc = (int)groups <= 2 * pb_num_sms() ? kv_launch(k_kv_join<D, 512>, groups, 512, d.a.grp * np * 4, st, true, "k_kv_join", d)
                                         : kv_launch(k_kv_join<D, 128>, groups, 128, d.a.grp * np * 4, st, true, "k_kv_join", d);
    if (rc) return rc;
  }
  if (d.score) {
    const long long all = (long long)d.a.p.n_seq * d.a.p.n_kv * (tiles > 0 ? tiles : 1), cap = 32LL * pb_num_sms();
    rc = kv_launch(k_kv_weight<D>, (unsigned)(all < cap ? all : cap), DcGeo<D>::TILE, 0, st, true, "k_kv_weight", d);
  }
  return rc;
}

}  // namespace

extern "C" long long pb_kv_decode_scratch(const pb_kv_pages* c, int n_seq, int max_len, int n_heads, int accumulate) {
  if (!c || n_seq < 0 || n_heads <= 0 || c->n_kv <= 0 || (c->head_dim != 64 && c->head_dim != 128)) return -1;
  if (max_len <= 0) return n_seq == 0 && max_len == 0 ? 0 : -1;
  const DcPlan p = dc_plan(c, n_seq, max_len, n_heads, accumulate);
  return 4 * (p.part + p.ml + p.lse + p.score);
}

extern "C" int pb_kv_decode(const pb_kv_pages* c, const pb_kv_attention_args* g, void* stream) {
  DcArgs d{};
  if (int rc = attn_check("pb_kv_decode", c, g, g ? g->n_seq : 0, &d.a)) return rc;
  const int n_seq = g->n_seq, max_len = d.a.max_len, accumulate = g->accumulate;
  if (n_seq == 0) return PB_OK;
  if (accumulate && !c->weight) return pb_set_error(PB_EINVAL, "pb_kv_decode: the cache keeps no weights");
  if ((long long)n_seq * c->n_kv * ((max_len + 63) / 64) > INT_MAX)
    return pb_set_error(PB_EINVAL, "pb_kv_decode: %d sequences of %d rows", n_seq, max_len);
  const DcPlan pl = dc_plan(c, n_seq, max_len, g->n_heads, accumulate);
  if (int rc = attn_scratch("pb_kv_decode", g, 4 * (pl.part + pl.ml + pl.lse + pl.score))) return rc;
  float* f = static_cast<float*>(g->scratch);
  d.part = f;
  d.ml = f + pl.part;
  d.a.lse = accumulate ? d.ml + pl.ml : nullptr;
  d.score = accumulate ? d.a.lse + pl.lse : nullptr;
  d.grid = pl.grid;
  d.grp2 = pl.grp2;
  d.out_bf16 = g->out_dtype == PB_DT_BF16;
  cudaStream_t st = (cudaStream_t)stream;
  return c->head_dim == 64 ? dc_run<64>(d, c->dtype, pl.join, st) : dc_run<128>(d, c->dtype, pl.join, st);
}
