// flashb: what the paged kernels share (fb_long_decode.cu, fb_paged_append.cu, fb_paged_attend.cu): the pool of pages, a
// step's rows and where their tokens lie.
#pragma once
#include "fb_long.cuh"

namespace fb {

// The pool: `pages` pages of `page` = 1 << shift slots; byte strides per page, head and slot.
struct PagedPool {
  unsigned char *k, *v;
  long long k_sb, k_sh, k_sl, v_sb, v_sh, v_sl;
  int pages, NKV, page, shift;
};
// Slot j of row b lies in page table[b table_sb + (j >> shift)]; entries outside [0, pages) are pages that are not there.
struct PagedTable {
  const int* table;
  long long table_sb;
  int pages, page, shift;
};
// A step's tokens 0 .. T - 1: row b's run is [offsets[b], offsets[b + 1]) (null: token b), its last one at slot
// lengths[b] - 1.
struct PagedRows {
  const long long *lengths, *offsets;
  int rows, T, S;                       // S: slots that a row's table entries span
};

// The rows whose runs hold tokens t .. t + N - 1, -1: none; lane i < N gets that of t + i.  A warp together: rows whose run
// begins at the token or before, counted 32 at a time with no load waiting for another (a search by halves is a chain of
// them).
template <int N>
__device__ __forceinline__ int paged_rows(const PagedRows& r, int t) {
  const int lane = threadIdx.x & 31;
  if (!r.offsets) return t + lane < r.rows ? t + lane : -1;
  int n[N], mine = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) n[i] = 0;
#pragma unroll 4
  for (int b = lane; b <= r.rows; b += 32) {
    if (b < r.rows) asm volatile("prefetch.global.L1 [%0];" ::"l"(r.lengths + b));    // the row's is read next
    const long long f = r.offsets[b];
#pragma unroll
    for (int i = 0; i < N; ++i) n[i] += f <= t + i;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    n[i] = __reduce_add_sync(FULL, n[i]);
    mine = lane == i ? n[i] : mine;
  }
  return mine <= r.rows ? mine - 1 : -1;
}
// That of one token, for every lane.
__device__ __forceinline__ int paged_row(const PagedRows& r, int t) { return __shfl_sync(FULL, paged_rows<1>(r, t), 0); }
// How many tokens of row b's run come after token t, itself counted.
__device__ __forceinline__ long long paged_left(const PagedRows& r, int b, int t) {
  return r.offsets ? r.offsets[b + 1] - t : 1;
}

}  // namespace fb

namespace fbh {
// Checks a public pool descriptor and fills the kernels' form.
int paged_pool(const fb_paged_cache* c, fb::PagedPool* out);
// Checks the number of rows and of table entries per row.
int paged_width(const fb_paged_cache* c, int rows, int width);
// Refuses an out [T, NH, 128] that shares memory with q or the cache.
int paged_apart(const fb::PagedPool& c, int T, int NH, const void* q, int64_t q_st, int64_t q_sh, const void* out, int64_t o_st,
                int64_t o_sh);
}  // namespace fbh
