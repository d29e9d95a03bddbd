// pb_kv.cuh -- the paged K/V cache shared by its operators (pb_kv.cu: append
// and evict; pb_kvattn.cu: attention): the pool as the kernels see it, the
// argument checks, and the element types (fp16 or bf16 rows, 16-byte vectors).
#pragma once
#include "pb_common.cuh"
#include "pb_internal.h"
#include <cuda_bf16.h>

// Row j of sequence b is row j & (page_size - 1) of page table[b][j >> shift];
// strides in bytes (64-bit: a long cache passes 2^31 elements). A table entry
// outside [0, n_pages) names no page: its rows are not seen, stored or moved.
struct KvPool {
  char* k;
  char* v;
  float* w;            // accumulated weights [page][kv head][row], or null
  const int* table;
  long long ps, hs, rs;
  int table_ld, n_pages, shift, n_kv, n_seq;
};

// the checks every entry point makes of a cache and its table; fills p
int kv_pool(const char* who, const pb_kv_pages* c, int n_seq, const int* d_table, int table_ld, KvPool* p);
// [a, a + an) and [b, b + bn) (bytes) share memory
inline bool kv_overlap(const void* a, size_t an, const void* b, size_t bn) {
  const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
  return x < y + bn && y < x + an;
}

// page of row j, or -1
PB_DEV int kv_page(const KvPool& p, const int* trow, int j) {
  const int e = __ldg(trow + (j >> p.shift));
  return (unsigned)e < (unsigned)p.n_pages ? e : -1;
}
// the length the operators use: never past the table or the caller's bound
PB_DEV int kv_len(int len, int max_len) { return len < 0 ? 0 : (len < max_len ? len : max_len); }

// a pair of elements <-> fp32; DT is PB_DT_F16 or PB_DT_BF16. Stores round to
// nearest even, once, from fp32 (an fp16 overflow becomes an infinity).
template <int DT>
PB_DEV float2 kv_up(unsigned w) {
  if (DT == PB_DT_BF16) return make_float2(pb_lo2f(w), pb_hi2f(w));
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
template <int DT>
PB_DEV unsigned kv_down(float a, float b) {
  unsigned r;
  if (DT == PB_DT_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
