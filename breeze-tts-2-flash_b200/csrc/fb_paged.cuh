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

// One token and head over the visible keys `row` of batch row b, one at a time: four dims a lane; the output row in bf16, 0
// without a key in a page of the pool.  The weight is fp32 and one factor, so that an infinity in a visible slot comes out as
// itself: for tokens that saw nothing, or whose output is not finite.  h: KV head; q: the token's head.  (0.6 us a key, which
// only a row with an infinity or a NaN in V takes; eight keys' loads together took 0.3, but 64 registers that spill into the
// kernels that call it, 1% of them.)
__device__ __forceinline__ uint2 paged_one(const PagedPool& pool, const PagedTable& t, const LongRow& row, float scale, int b, int h,
                                           const bf16* q) {
  constexpr float SHIFT = -24.f;                  // sums of 2^16 keys stay in fp32's range for every finite V
  const int lane = threadIdx.x & 31;
  const unsigned char *kb = pool.k + h * pool.k_sh + 8 * lane, *vb = pool.v + h * pool.v_sh + 8 * lane;
  const int* table = t.table + b * t.table_sb;
  const uint2 qw = *reinterpret_cast<const uint2*>(q + 4 * lane);
  float m = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  bool some = false;
#pragma unroll 4
  for (int i = 0; i < row.n; ++i) {
    const int j = (int)row.slot(i), page = table[j >> t.shift], in = j & (t.page - 1);
    if ((unsigned)page >= (unsigned)t.pages) continue;
    some = true;
    const uint2 kw = *reinterpret_cast<const uint2*>(kb + page * pool.k_sb + in * pool.k_sl);
    const uint2 vw = *reinterpret_cast<const uint2*>(vb + page * pool.v_sb + in * pool.v_sl);
    const float s = scale * warp_sum(lo_f(qw.x) * lo_f(kw.x) + hi_f(qw.x) * hi_f(kw.x) + lo_f(qw.y) * lo_f(kw.y) +
                                     hi_f(qw.y) * hi_f(kw.y));
    const float mn = fmaxf(m, s), f = m > -INFINITY ? ex2(m - mn) : 0.f;
    const float w = mn > -INFINITY ? ex2(s - mn + SHIFT) : (s == -INFINITY ? 0.f : s);
    m = mn;
    sum = sum * f + w;
    o[0] = o[0] * f + w * lo_f(vw.x);
    o[1] = o[1] * f + w * hi_f(vw.x);
    o[2] = o[2] * f + w * lo_f(vw.y);
    o[3] = o[3] * f + w * hi_f(vw.y);
  }
  const float inv = some ? 1.f / sum : 0.f;       // scores of -inf alone: 0 / 0, as softmax has it
  return make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
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
