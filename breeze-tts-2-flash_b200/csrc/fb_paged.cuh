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

// The row whose run holds token t, -1: none.  A warp together: rows whose run begins at t or before, counted 32 at a time
// with no load waiting for another (a search by halves is a chain of them).
__device__ __forceinline__ int paged_row(const PagedRows& r, int t) {
  if (!r.offsets) return t < r.rows ? t : -1;
  const int lane = threadIdx.x & 31;
  int n = 0;
#pragma unroll 4
  for (int b = lane; b <= r.rows; b += 32) n += r.offsets[b] <= t;
  n = __reduce_add_sync(FULL, n);
  return n <= r.rows ? n - 1 : -1;
}
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
// Single-token attention (fb_long_decode.cu; arguments checked by the caller) of the rows whose run is one token (offsets
// null: token b is row b's), and the floats of workspace that it takes.
int paged_decode_floats(const fb_paged_cache* cache, int rows, int width, int NH, int window, int sinks, int64_t* floats);
int paged_decode(const fb_paged_cache* cache, const fb::PagedPool& pool, const int32_t* table, int64_t table_sb, int rows,
                 int width, const int64_t* lengths, const int64_t* offsets, int T, const void* q, int64_t q_st,
                 int64_t q_sh, int NH, int window, int sinks, float scaling, float* ws, void* out, int64_t o_st,
                 int64_t o_sh, void* stream);
}  // namespace fbh
