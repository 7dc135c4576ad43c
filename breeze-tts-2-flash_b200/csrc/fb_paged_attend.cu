// flashb: attention of a step's new tokens (a run of any length per row) over a paged cache, on the 5th-generation tensor
// cores.
//
//   out_t = softmax(scaling q_t k^T over the slots that t sees) v, fp32, rounded once; without a visible slot 0.
//
// The pipeline is fb_long_prefill.cu's: 128 rows a CTA, 64-key tiles of two 32-key segments, S = Q K^T and O += P V issued by
// a thread each, P kept in TMEM, four softmax warps with a thread per row, two CTAs an SM.  What differs:
//
// Rows of a tile are the run's tokens in order with the G heads of a KV head inner, so a run of few tokens fills the first
// warps alone; the others do not take part.  Keys come from pages: a tile in one page is one box, else 32-key segments are
// boxes of 32 slots or two of 16.  An entry that is no page is loaded from past the pool's end, which reads as zeros, and
// its slots get no weight.
//
// The weights are 2^(s - m - 24) with a reference m of the row's own that is hardly ever moved: they are taken with the old
// m first, and only when a tile's sum shows that some score passed it by 2^8 is the tile's maximum worked out, O and the
// sum rescaled and the weights taken again.  (The maximum first, for every tile: 600 instead of 530 us at the largest
// case below.  The sums are exact either way; sum and reference are fp32.)
//
// P goes to bf16, one part, as in the prefill: the tensor cores take it in V's type, half a step of 2^-8 off at most.  Against
// 64 bits the output is 2.0e-3 to 2.4e-3 off, where single tokens, whose kernel takes P in two parts, have 1.7e-3, their own
// rounding.  A second part here would need half as much again of the tensor cores (1536 cycles for the two tiles of an SM,
// which take 1500 in all now) and 32 columns of TMEM more for either buffer of P, where S, P and O of two CTAs fill all 512.
//
// Pieces.  A step can be one run of a few tokens over a long row, or many rows of which some are long.  So the key tiles of
// a query tile are cut into s pieces of about C; a CTA takes one piece of the list that lengths and offsets, on the device,
// come to (nothing is read on the host).  C is chosen among those with which the list fills one round or about two, and whole
// query tiles, by what they take.  Up to 32 rows, and query tiles for one round at most, every CTA works this out itself,
// a row a lane (1 us; a prompt of 17 tokens over 2000 slots 13.8 us, 16.0 with a kernel before it).  For more rows
// paged_plan_kernel (one CTA) writes the list, 4 us: many CTAs that each work it out took up to 9% longer.  Where rows are too
// short to cut, CTAs just find their query tiles.  Pieces of a query tile leave (reference, sum, unnormalised out) in the
// workspace and paged_merge_kernel joins them in order: no atomics, the same inputs give the same bits.
//
// Rows of one token are runs as others are.  (The single-token kernel for them, in a launch of its own, measured before pieces
// were priced as they are now: 128 instead of 133 us for 512 tokens beside 63 single ones over long rows, but 19 instead of 14
// over short ones, and 5 us where there are none.)
//
// Slots that no row of the CTA sees may hold anything: in V they are zeroed in shared memory (0 times a NaN is NaN), in K
// their scores are replaced.  A row whose output is not finite all the same (a NaN that another row of the tile sees), though
// its weights' sum is a number, is computed again, one visible key at a time.
//
// Measured on a B200 (in a CUDA graph, 16 heads over 4): 2048 tokens over 32768 slots of one row 520 to 577 us by the box, 983
// to 1090 TFLOP/s, in pages of 16 to 128 alike; 801 tokens of 32 rows over a window of 2048 (131 MB) 46 us; 512 tokens of one
// row beside one each of 63, over up to 8000 slots (530 MB), 97 to 129 us by their lengths, 116 on average over ten sets of
// them; two prompts of 197 tokens 9.1 us, in a table of 16384 slots, by whose width the form is chosen, 11.5.  A tile takes
// 1500 cycles with two CTAs an SM: 700 to 870 are exponentials (the unit's bound for both CTAs is 1024), 100 the read of S,
// 240 masks, the rest waits and stores; issuing S takes its thread 480 cycles and P V 290, both beside the exponentials.
// Under the largest case's load clocks fall to 1.5 GHz.  With few keys a piece it is beginning and ending (9000 cycles) that
// counts.  Tried and slower: one copying warp for K and V (8 boxes one after the other take 900 cycles), a flag for missing
// pages read in the loop (6%), arrivals by one lane a warp (4%), P V's waits by one lane (10%), the second CTA of an SM begun
// half a tile later (the same), copies to L2 a buffer ahead (4 to 30%: more boxes), half of Q in the place of P's second
// buffer in TMEM (3 to 10%).
#include <climits>

#include "fb_long_tc.cuh"
#include "fb_paged.cuh"

namespace fb {

constexpr int PT_WHOLE = 8;                       // query tiles of so few key tiles stay whole, without a plan
constexpr int PT_MIN = 6;                         // key tiles of a piece, at least
constexpr int PT_WAVES = 2;                       // rounds of CTAs that the list of pieces may be cut for (and an eighth)
constexpr float PT_LIMIT = 0x1p-16f;              // 2^(8 + LP_SHIFT): a tile's weights below it leave the reference as it is
// What a list costs, in the time of a key tile: the longest piece + PT_COST where it fits one round of the SMs, else what all
// pieces are to an SM's place and a share PT_LAST of the longest; and where anything is cut PT_JOIN a round (parts written and
// read again) and PT_JOINS.  Fitted to 430 lists of 45 drawn steps (pieces of 5 to 128 tiles, and whole): its choices take
// 1.5% more time than the best of each step, 7% at most; those by rounds x (longest + 5) 7%, 36% at most.
constexpr float PT_COST = 8.f, PT_LAST = 0.5f, PT_JOIN = 2.f, PT_JOINS = 4.f;

struct PagedPiece;

struct alignas(64) PagedAttendArgs {
  CUtensorMap tq, tk, tv, tks, tvs;     // Q tile; K, V: boxes of 64 slots, and of 32 or 16 (of K half of the dims)
  PagedPool pool;
  PagedTable t;
  PagedRows r;
  const bf16* q;
  long long q_st, q_sh;
  int NH, NKV, G, nq, window, sinks;    // nq = 128 / G tokens a CTA; window 0: none
  int lq, lg;                           // log2 of nq and of G
  int per, pieces, list, cuts;          // rows per thread of the plan; CTAs that the SMs hold a KV head, 0: query tiles stay
  float rounds;                         // whole; entries of the list, of them cut at most; 1 / pieces
  int per32;                            // rows per lane where a CTA finds its query tile itself
  float scale;                          // scaling x log2(e)
  bf16* out;
  long long o_st, o_sh;
  float* po;                            // pieces: unnormalised out [slot][128][128],
  float2* ml;                           //   maximum and sum [slot][128]
  PagedPiece* plan;                     // [list]
  int4* cut;                            // [cuts / 2] query tiles of two pieces and more (first token, tokens, pieces, slot),
                                        //   then their number
  unsigned* err;
};

// Row b's run: n tokens from t0 on, the first at slot p0.
struct PagedSpan {
  int t0, n, p0;
};
__device__ __forceinline__ PagedSpan paged_span(const PagedRows& r, long long f, long long e, long long len) {
  const int t0 = (int)min(max(f, 0ll), (long long)r.T), t1 = (int)min(max(e, (long long)t0), (long long)r.T);
  const long long p0 = min(max(len, 0ll), (long long)r.S) - (e - t0);
  return PagedSpan{t0, t1 - t0, (int)max(p0, -0x40000000ll)};
}
__device__ __forceinline__ PagedSpan paged_span(const PagedRows& r, int b) {
  return paged_span(r, r.offsets[b], r.offsets[b + 1], r.lengths[b]);
}
// The key segments of tokens at slots p_lo .. p_hi: ns of sinks from slot 0 on, then those from base to p_hi; lo: the first
// slot that the window of any of them holds.
struct PagedSegs {
  int lo, base, ns, n;
  __device__ __forceinline__ int at(int s) const { return s < ns ? LP_SEG * s : base + LP_SEG * (s - ns); }
};
__device__ __forceinline__ PagedSegs paged_segs(const PagedAttendArgs& a, int p_lo, int p_hi) {
  PagedSegs g;
  g.lo = a.window > 0 ? max(p_lo - a.window + 1, 0) : 0;
  g.base = g.lo & ~(LP_SEG - 1);
  g.ns = min((a.sinks + LP_SEG - 1) / LP_SEG, g.base / LP_SEG);
  g.n = p_hi < 0 ? 0 : g.ns + (p_hi - g.base) / LP_SEG + 1;
  return g;
}
// A row's query tiles and the key tiles of its last one (the most that one has).  Not inlined, nor the plan's other parts
// repeated: the plan is one pass over cold instructions, which cost it more than its arithmetic.
__device__ __noinline__ int2 paged_tiles(const PagedAttendArgs& a, int b) {
  const PagedSpan x = paged_span(a.r, b);
  if (x.n <= 0) return make_int2(0, 0);
  const int p_hi = x.p0 + x.n - 1;
  return make_int2((x.n + a.nq - 1) >> a.lq, (paged_segs(a, p_hi - min(x.n, a.nq) + 1, p_hi).n + 1) >> 1);
}

// Pieces of a query tile of k key tiles, about C = 1 / r in each.
__device__ __forceinline__ int paged_cut(int k, float r) { return max(1, (int)ceilf((float)k * r)); }

// Piece i of s of the tokens tok .. tok + nt - 1 of row b, the first at slot p_lo; slot: its place in the workspace.
struct alignas(16) PagedPiece {
  int b, tok, nt, p_lo, i, s, slot, pad;   // b = -1: none
};

// What a list of n pieces, of so many key tiles in all and in the longest, costs.
__device__ __forceinline__ float paged_price(const PagedAttendArgs& a, int n, float work, float longest, bool cut) {
  const float rounds = (float)n * a.rounds;
  const float p = n <= a.pieces ? longest + PT_COST : (work + PT_COST * (float)n) * a.rounds + PT_LAST * longest;
  return cut ? p + rounds * PT_JOIN + PT_JOINS : p;
}
// 1 / (key tiles of a piece) for which the list has room in a round of the SMs, or (j = 1) comes to about two: a query tile
// has up to one piece more than its key tiles come to.  0: no room.
__device__ __forceinline__ float paged_room(const PagedAttendArgs& a, int j, int units, float work) {
  const float room = (float)((j + 1) * a.pieces) - (j ? 0.6f : 1.f) * (float)units;
  return room > 0.f ? fminf(__fdividef(room, work), 1.f / PT_MIN) : 0.f;
}

constexpr int PP_THREADS = 256, PP_WARPS = PP_THREADS / 32;
constexpr int PP_ROWS = 1024;              // rows whose tiles are kept in shared memory

// The list: rows in order, a row's latest query tiles first (they have the most keys), a query tile's pieces in order.
__global__ void __launch_bounds__(PP_THREADS) paged_plan_kernel(const __grid_constant__ PagedAttendArgs a) {
  __shared__ int2 s_k[PP_ROWS];
  __shared__ int s_units[PP_WARPS], s_longest[PP_WARPS], s_n[PT_WAVES][PP_WARPS], s_most[PT_WAVES][PP_WARPS];
  __shared__ int s_before[PP_THREADS], s_slots[PP_THREADS], s_cut[PP_THREADS], s_w[PP_WARPS][3];
  __shared__ float s_work[PP_WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  const int b0 = tid * a.per, b1 = min(b0 + a.per, a.r.rows);
  auto tiles = [&](int b) { return b < PP_ROWS ? s_k[b] : paged_tiles(a, b); };
  // what there is: key tiles, query tiles, the longest row
  float w = 0.f;
  int units = 0, longest = 0;
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    const int2 k = paged_tiles(a, b);
    if (b < PP_ROWS) s_k[b] = k;
    w += (float)k.x * (float)k.y;
    units += k.x;
    longest = max(longest, k.y);
  }
  float r = 0.f;                        // 1 / (key tiles of a piece), 0: query tiles stay whole
  if (a.pieces > 0) {
    w = warp_sum(w);
    units = __reduce_add_sync(FULL, units);
    longest = __reduce_max_sync(FULL, longest);
    if (lane == 0) s_work[warp] = w, s_units[warp] = units, s_longest[warp] = longest;
    __syncthreads();
    w = warp_sum(lane < PP_WARPS ? s_work[lane] : 0.f);
    units = __reduce_add_sync(FULL, lane < PP_WARPS ? s_units[lane] : 0);
    longest = __reduce_max_sync(FULL, lane < PP_WARPS ? s_longest[lane] : 0);
    // candidates: what a piece may hold for the list to fit that many rounds of the SMs
    float c[PT_WAVES];
    int n[PT_WAVES], most[PT_WAVES];
#pragma unroll
    for (int j = 0; j < PT_WAVES; ++j) {
      c[j] = paged_room(a, j, units, w);
      n[j] = most[j] = 0;
    }
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      const int2 x = tiles(b);
#pragma unroll
      for (int j = 0; j < PT_WAVES; ++j) {
        const int s = paged_cut(x.y, c[j]);
        n[j] += x.x * s;
        most[j] = max(most[j], (int)__fdividef((float)(x.y + s - 1), (float)s));
      }
    }
#pragma unroll
    for (int j = 0; j < PT_WAVES; ++j) {
      n[j] = __reduce_add_sync(FULL, n[j]);
      most[j] = __reduce_max_sync(FULL, most[j]);
      if (lane == 0) s_n[j][warp] = n[j], s_most[j][warp] = most[j];
    }
    __syncthreads();
    // the cheapest of those and of whole query tiles; the places in the workspace are enough for `cuts` pieces
    float price = paged_price(a, units, w, (float)longest, false);
#pragma unroll
    for (int j = 0; j < PT_WAVES; ++j) {
      const int count = __reduce_add_sync(FULL, lane < PP_WARPS ? s_n[j][lane] : 0);
      const float len = (float)__reduce_max_sync(FULL, lane < PP_WARPS ? s_most[j][lane] : 0);
      const float p = paged_price(a, count, w, len, true);
      if (p < price && count <= a.cuts) price = p, r = c[j];
    }
  }
  int np = 0, ns = 0, nc = 0;
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    const int2 k = tiles(b);
    const int s = paged_cut(k.y, r);
    np += k.x * s;
    ns += s > 1 ? k.x * s : 0;
    nc += s > 1 ? k.x : 0;
  }
  int before = np, slots = ns, cuts = nc;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(FULL, before, o), z = __shfl_up_sync(FULL, slots, o), v = __shfl_up_sync(FULL, cuts, o);
    if (lane >= o) {
      before += y;
      slots += z;
      cuts += v;
    }
  }
  if (lane == 31) s_w[warp][0] = before, s_w[warp][1] = slots, s_w[warp][2] = cuts;
  __syncthreads();
  int total = 0, used = 0, joins = 0;
#pragma unroll
  for (int i = 0; i < PP_WARPS; ++i) {
    if (i == warp) before += total, slots += used, cuts += joins;
    total += s_w[i][0];
    used += s_w[i][1];
    joins += s_w[i][2];
  }
  s_before[tid] = before - np;
  s_slots[tid] = slots - ns;
  s_cut[tid] = cuts - nc;
  __syncthreads();
#pragma unroll 1
  for (int x = tid; x < a.list; x += PP_THREADS) {
    PagedPiece p{-1, 0, 0, 0, 0, 1, used, 0};
    if (x < total) {
      int o = 0;                        // the last thread whose pieces begin at x or before
#pragma unroll 1
      for (int h = PP_THREADS / 2; h > 0; h >>= 1)
        if (s_before[o + h] <= x) o += h;
      int at = s_before[o], slot = s_slots[o], join = s_cut[o], b = o * a.per, s, n;
#pragma unroll 1
      for (;; ++b) {
        const int2 k = tiles(b);
        s = paged_cut(k.y, r);
        n = k.x * s;
        if (x < at + n) break;
        at += n;
        slot += s > 1 ? n : 0;
        join += s > 1 ? k.x : 0;
      }
      const PagedSpan span = paged_span(a.r, b);
      const int rem = x - at, u = rem / s, q0 = (n / s - 1 - u) << a.lq;
      p = PagedPiece{b, span.t0 + q0, min(a.nq, span.n - q0), span.p0 + q0, rem - u * s, s, slot + rem, 0};
      if (s > 1 && p.i == 0) a.cut[join + u] = make_int4(p.tok, p.nt, s, p.slot);
    }
    *reinterpret_cast<int4*>(&a.plan[x]) = *reinterpret_cast<const int4*>(&p);
    reinterpret_cast<int4*>(&a.plan[x])[1] = reinterpret_cast<const int4*>(&p)[1];
  }
  if (tid == 0 && a.cuts > 1) a.cut[a.cuts / 2] = make_int4(joins, 0, 0, 0);
}

// Piece x of the list, for a CTA without a plan: a warp, lane i has rows [i per32, ..), the first four of them in registers
// (108 rows of two tokens: 24 us; a row after the other, each load behind the last, 30).  CUT (a row a lane): cut as the plan
// would; the first head's CTAs also write what the merge needs.  Else query tiles stay whole.
template <bool CUT>
__device__ __forceinline__ void paged_find(const PagedAttendArgs& a, int x, int h, int lane, PagedPiece* piece) {
  constexpr int R = CUT ? 1 : 4;
  const int b0 = min(lane * a.per32, a.r.rows), b1 = min(b0 + a.per32, a.r.rows);
  long long f[R + 1], len[R];
  int q[R], k[R], n = 0, slots = 0, joins = 0;               // query tiles of the rows, key tiles of their last
  f[0] = a.r.offsets[b0];
#pragma unroll
  for (int i = 0; i < R; ++i) f[i + 1] = a.r.offsets[min(b0 + i + 1, b1)], len[i] = a.r.lengths[min(b0 + i, a.r.rows - 1)];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const PagedSpan y = paged_span(a.r, f[i], f[i + 1], len[i]);
    const int p_hi = y.p0 + y.n - 1;
    q[i] = b0 + i < b1 ? (y.n + a.nq - 1) >> a.lq : 0;
    k[i] = CUT && q[i] > 0 ? (paged_segs(a, p_hi - min(y.n, a.nq) + 1, p_hi).n + 1) >> 1 : 0;
    n += q[i];
  }
  float r = 0.f;
  if (CUT) {
    float w = 0.f;
    int longest = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) w += (float)q[i] * (float)k[i], longest = max(longest, k[i]);
    w = warp_sum(w);
    const int units = __reduce_add_sync(FULL, n);
    longest = __reduce_max_sync(FULL, longest);
    float price = paged_price(a, units, w, (float)longest, false);
#pragma unroll
    for (int j = 0; j < PT_WAVES; ++j) {
      const float c = paged_room(a, j, units, w);
      int count = 0, most = 0;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int s = paged_cut(k[i], c);
        count += q[i] * s;
        most = max(most, (int)__fdividef((float)(k[i] + s - 1), (float)s));
      }
      count = __reduce_add_sync(FULL, count);
      const float p = paged_price(a, count, w, (float)__reduce_max_sync(FULL, most), true);
      if (p < price && count <= a.cuts) price = p, r = c;
    }
    n = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int s = paged_cut(k[i], r);
      n += q[i] * s;
      slots += s > 1 ? q[i] * s : 0;
      joins += s > 1 ? q[i] : 0;
    }
  } else {
#pragma unroll 1
    for (int b = b0 + R; b < b1; ++b) n += (paged_span(a.r, b).n + a.nq - 1) >> a.lq;
  }
  int before = n, slot = slots, join = joins;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(FULL, before, o);
    const int z = CUT ? __shfl_up_sync(FULL, slot, o) : 0, v = CUT ? __shfl_up_sync(FULL, join, o) : 0;
    if (lane >= o) before += y, slot += z, join += v;
  }
  if (CUT && lane == 31 && x == 0 && h == 0 && a.cuts > 1) a.cut[a.cuts / 2] = make_int4(join, 0, 0, 0);
  if (x >= before || x < before - n) {
    if (lane == 31 && x >= before) *piece = PagedPiece{-1, 0, 0, 0, 0, 1, 0, 0};
    return;
  }
  int at = x - (before - n), b = b0, tiles = q[0];           // the lane's piece `at`, of row b
  const int s = CUT ? paged_cut(k[0], r) : 1;
  slot -= slots;
  join -= joins;
  PagedSpan span = paged_span(a.r, f[0], f[1], len[0]);
#pragma unroll
  for (int i = 1; i < R; ++i)
    if (b == b0 + i - 1 && at >= tiles) at -= tiles, ++b, tiles = q[i], span = paged_span(a.r, f[i], f[i + 1], len[i]);
  if (!CUT)
#pragma unroll 1
    while (at >= tiles) {
      at -= tiles, ++b;
      span = paged_span(a.r, b);
      tiles = (span.n + a.nq - 1) >> a.lq;
    }
  const int u = CUT ? at / s : at, q0 = (tiles - 1 - u) << a.lq;
  const PagedPiece p{b, span.t0 + q0, min(a.nq, span.n - q0), span.p0 + q0, at - u * s, s, slot + at, 0};
  *piece = p;
  if (CUT && s > 1 && p.i == 0 && h == 0) a.cut[join + u] = make_int4(p.tok, p.nt, s, p.slot);
}

constexpr int PT_THREADS = 256;                  // 4 softmax warps; one each for S, P V, the copies of K and of V
constexpr int PT_K = 3;                          // buffers of K: with two, S waited for K a quarter of the time
struct alignas(16) PagedShared {
  uint64_t bar_k[PT_K], bar_s[PT_K], bar_v[2], bar_p[2], bar_o[2], bar_f;
  uint32_t tslot;
  int bad;
  PagedPiece piece;
};
constexpr int PT_SMEM = LP_Q + (PT_K + 2) * LP_KV + (int)sizeof(PagedShared);
static_assert(2 * (PT_SMEM + 1024) <= 228 * 1024, "two CTAs an SM");

// The token at slot p of row b, its head hq, again: where it saw nothing, or its output is not finite.
__device__ __noinline__ uint2 paged_again(const PagedAttendArgs& a, int b, int p, int hq, const bf16* q) {
  return paged_one(a.pool, a.t, long_row((long long)p + 1, 0, a.r.S, a.window, a.sinks), a.scale, b, hq / a.G, q);
}

// Pieces come from the plan (PT_PLAN), or CTAs find theirs: of query tiles that stay whole, or cut.
enum { PT_FIND, PT_CUT, PT_PLAN };
template <int HOW>
__global__ void __launch_bounds__(PT_THREADS, 2) paged_attend_kernel(const __grid_constant__ PagedAttendArgs a) {
  // nothing but this: with 1 KB of the system's, two CTAs fill an SM, and the base is at a 1024-byte boundary (checked)
  extern __shared__ __align__(1024) unsigned char sq[];                   // Q; the output tile at the end
  unsigned char* sk = sq + LP_Q;                                          // [PT_K]
  unsigned char* sv = sk + PT_K * LP_KV;                                  // [2]
  PagedShared& sh = *reinterpret_cast<PagedShared*>(sv + 2 * LP_KV);
  uint64_t *bar_k = sh.bar_k, *bar_v = sh.bar_v, *bar_s = sh.bar_s, *bar_p = sh.bar_p, *bar_o = sh.bar_o, &bar_f = sh.bar_f;
  uint32_t& tslot = sh.tslot;
  int& s_bad = sh.bad;
  PagedPiece& s_piece = sh.piece;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int x = blockIdx.x / a.NKV, h = blockIdx.x - x * a.NKV;
  if (tid == 0) {
    s_bad = 0;
    if (smem_u32(sq) & 1023u) set_error(a.err, FB_ERR_DEVICE);
    for (const CUtensorMap* m : {&a.tq, &a.tk, &a.tv, &a.tks, &a.tvs})
      asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
  }
  pdl_wait();
  pdl_trigger();
  PagedPiece piece;
  if constexpr (HOW == PT_PLAN) {
    piece = a.plan[x];
  } else {
    if (warp == 0) paged_find<HOW == PT_CUT>(a, x, h, lane, &s_piece);
    __syncthreads();
    piece = s_piece;
  }
  if (piece.b < 0) return;
  const int p_lo = piece.p_lo, p_hi = p_lo + piece.nt - 1;
  const int live = piece.nt * a.G, warps = (live + 31) >> 5;
  const PagedSegs seg = paged_segs(a, p_lo, p_hi);
  const int all = (seg.n + 1) >> 1;
  const int first = (int)((long long)all * piece.i / piece.s), tiles = (int)((long long)all * (piece.i + 1) / piece.s) - first;
  const int segs = seg.n - 2 * first;               // segments from the piece's first tile on
  const int* table = a.t.table + piece.b * a.t.table_sb;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_v[i], 1);
      mbar_init(&bar_p[i], 32 * warps);
      mbar_init(&bar_o[i], 1);
    }
    for (int i = 0; i < PT_K; ++i) {
      mbar_init(&bar_k[i], 1);
      mbar_init(&bar_s[i], 1);
    }
    mbar_init(&bar_f, 32 * warps);
    fence_mbar_init();
  }
  if (warp == 4) tc_alloc(&tslot, LP_COLS);
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tslot, t_o = tmem + 128;
  // whether any row of the tile sees a slot of [j, j + n)
  auto seen = [&](int j, int n) { return j <= p_hi && (j + n > seg.lo || j < a.sinks); };

  // A tile is one box where it lies in one page, else boxes of `small` slots: of K one half of the dims each (its 64 keys
  // are rows of one operand), of V both (a step of its product takes 16 keys, whose halves may lie anywhere).
  const int small = min(a.t.page, LP_SEG);
  auto whole = [&](int t) {
    const int sg = 2 * (first + t);
    return segs - 2 * t >= 2 && a.t.page >= LP_TILE && (seg.at(sg) & (LP_TILE - 1)) == 0 && sg != seg.ns - 1;
  };

  if (warp == 4 || warp == 7) {                    // copies of K, of V; the warp holds the entries of 16 tiles
    const bool is_v = warp == 7;
    const int mask = a.t.page - 1, qc = (lane >> 1) & 3;             // lane 2 c + i: quarter c (16 slots), half i
    // lane 4 i + c: the page of quarter c of tile 8 g + i of the piece
    auto entries = [&](int g) {
      const int tl = 8 * g + (lane >> 2);
      int e = -1;
      if (tl < tiles) {
        const int sg = 2 * (first + tl) + ((lane >> 1) & 1), j = seg.at(sg) + 16 * (lane & 1);
        // of a page that any row sees a slot of: a box may begin before the first of them
        if (sg < seg.n && j < a.r.S && seen(j & -a.t.page, a.t.page)) e = table[j >> a.t.shift];
      }
      return (unsigned)e < (unsigned)a.t.pages ? e : a.t.pages;      // past the pool: zeros
    };
    int e0 = entries(0), e1 = entries(1), buf = 0;
    unsigned parity = 1;                           // of the buffer's last use
    uint64_t *full = is_v ? bar_v : bar_k, *freed = is_v ? bar_o : bar_s;
    const int bufs = is_v ? 2 : PT_K;
    const CUtensorMap *big = is_v ? &a.tv : &a.tk, *little = is_v ? &a.tvs : &a.tks;
    bool ok = true;
    int t = 0;
    for (; t < tiles; ++t) {
      // everything but the copy itself before the wait
      const int sg = 2 * (first + t), n = min(2, segs - 2 * t);
      const int pg = __shfl_sync(FULL, (t >> 3) & 1 ? e1 : e0, ((t & 7) << 2) + qc);
      const bool one = whole(t);
      const int j = (one ? seg.at(sg) : seg.at(sg + (qc >> 1)) + 16 * (qc & 1)) & mask;
      const bool mine = one ? lane == 0
                            : (qc >> 1) < n && lane < 8 && (small == LP_SEG / 2 || (qc & 1) == 0) && (!is_v || (lane & 1) == 0);
      unsigned char* dst = (is_v ? sv : sk) + buf * LP_KV;
      if (!one) dst += is_v ? qc * (LP_KV / 4) : (lane & 1) * (LP_KV / 2) + qc * (LP_KV / 8);
      const unsigned bytes = (unsigned)(n * (LP_KV / 2) + (!is_v && t == 0 ? LP_Q : 0));
      // free: S of t - 3 has read its K, P V of t - 2 its V
      if (t >= bufs && !lp_wait_warp(&freed[buf], parity, a.err)) {
        ok = false;
        break;
      }
      if (lane == 0) mbar_arrive_expect_tx(&full[buf], bytes);
      // a lane a box: one thread after the other takes 40 ns each
      if (mine) lp_load(dst, one ? big : little, j, one || is_v ? 0 : lane & 1, h, pg, &full[buf]);
      if (!is_v && t == 0 && lane == 0)
        asm volatile(
            "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
            "[%6];" ::"r"(smem_u32(sq)),
            "l"(&a.tq), "r"(0), "r"(h * a.G), "r"(piece.tok), "r"(0), "r"(smem_u32(&full[buf]))
            : "memory");
      __syncwarp();
      if (++buf == bufs) buf = 0, parity ^= 1;
      if ((t & 7) == 7) {                          // the next group of eight tiles but one
        if ((t >> 3) & 1) e1 = entries((t >> 3) + 2);
        else e0 = entries((t >> 3) + 2);
      }
    }
    // no copy may be in flight when the CTA ends (after a wait that gave up: nobody else waits for them)
    if (!ok)
      for (int i = max(0, t - bufs); i < t; ++i) lp_wait_warp(&full[i % bufs], (i / bufs) & 1, a.err);
  } else if (warp == 5) {                          // S: one thread
    const uint64_t dq = tc_desc_sw128(smem_u32(sq)), dk = tc_desc_sw128(smem_u32(sk));
    auto step = [&](auto buf, int t, unsigned parity) -> bool {
      constexpr int B = decltype(buf)::value;
      if (t >= tiles || !lp_wait(&bar_k[B], parity, a.err)) return false;
      if (t >= 1 && !lp_wait(&bar_f, (t - 1) & 1, a.err)) return false;   // the last tile's scores are in registers
      tc_after();
      const uint32_t idesc = segs - 2 * t >= 2 ? tc_idesc(2 * LP_SEG) : tc_idesc(LP_SEG);
#pragma unroll
      for (int s = 0; s < LG_D / 16; ++s)
        tc_mma(tmem, dq + (((s >> 2) * (LP_Q / 2) + (s & 3) * 32) >> 4),
               dk + ((B * LP_KV + (s >> 2) * (LP_KV / 2) + (s & 3) * 32) >> 4), s > 0, idesc);
      tc_commit(&bar_s[B]);
      return true;
    };
    if (lane == 0) {
      unsigned parity = 0;
      for (int t = 0; step(std::integral_constant<int, 0>(), t, parity) &&
                      step(std::integral_constant<int, 1>(), t + 1, parity) &&
                      step(std::integral_constant<int, 2>(), t + 2, parity);
           t += PT_K)
        parity ^= 1;
    }
    __syncwarp();
  } else if (warp == 6) {                          // P V
    // dims contiguous: two halves of 64, 8-key groups; in a box of n slots the halves are n x 128 bytes apart, and the next
    // box is n x 256 on
    const uint64_t dv = tc_desc(smem_u32(sv), LP_KV / 2, 1024, 2), ds = tc_desc(smem_u32(sv), small * 128, 1024, 2);
    const int odd = small == LP_SEG ? 2048 : 4096;   // 16 keys on
    auto step = [&](auto buf, int t) -> bool {
      constexpr int B = decltype(buf)::value;
      const bool one = whole(t);                   // worked out before the waits: between P and its product every cycle counts
      if (!lp_wait_warp(&bar_v[B], (t >> 1) & 1, a.err)) return false;
      bool zeroed = false;
      for (int s = 0; s < 2 && 2 * t + s < segs; ++s) {              // slots that no row of the tile sees
        const int j0 = seg.at(2 * (first + t) + s);
        const uint32_t see = lp_bits(seg.lo - j0, p_hi + 1 - j0) | lp_bits(0, min(a.sinks, p_hi + 1) - j0);
        if (see == FULL) continue;
        zeroed = true;
        const int rows = one ? LP_TILE : small;
        for (int i = lane; i < LP_SEG * 16; i += 32)
          if (!((see >> (i >> 4)) & 1u)) {
            const int key = LP_SEG * s + (i >> 4), in = key & (rows - 1);
            *reinterpret_cast<uint4*>(sv + B * LP_KV + (key - in) * 256 + ((i >> 3) & 1) * rows * 128 + in * 128 + (i & 7) * 16) =
                make_uint4(0, 0, 0, 0);
          }
      }
      if (zeroed) {
        fence_proxy_async();
        __syncwarp();
      }
      if (!lp_wait_warp(&bar_p[B], (t >> 1) & 1, a.err)) return false;
      tc_after();
      if (lane == 0) {
        constexpr uint32_t idesc = tc_idesc(LG_D) | (1u << 16);   // V: dims contiguous
        const bool half = segs - 2 * t < 2;
        if (one) {
#pragma unroll
          for (int s = 0; s < 4; ++s)
            lp_mma_ts(t_o, tmem + 64 + 32 * B + 8 * s, dv + ((B * LP_KV + 2048 * s) >> 4), idesc, s > 0 || t > 0);
        } else {
#pragma unroll
          for (int s = 0; s < 4; ++s)
            if (s < 2 || !half)
              lp_mma_ts(t_o, tmem + 64 + 32 * B + 8 * s, ds + ((B * LP_KV + (s >> 1) * 8192 + (s & 1) * odd) >> 4), idesc,
                        s > 0 || t > 0);
        }
        tc_commit(&bar_o[B]);
      }
      __syncwarp();
      return true;
    };
    for (int t = 0; t < tiles; t += 2)
      if (!step(std::integral_constant<int, 0>(), t) || (t + 1 < tiles && !step(std::integral_constant<int, 1>(), t + 1)))
        break;
  } else if (warp < warps) {
    const int r = tid, l = r >> a.lg;
    const bool mine = r < live;
    const int p = mine ? p_lo + l : -1;                     // a row without a token: its weights may be anything
    const uint32_t my = (uint32_t)(warp * 32) << 16;
    const int wnd = a.window > 0 ? a.window : 0x40000000;   // none: more than any row has
    const uint64_t scale2 = f2(a.scale, a.scale);
    // entries that are no page, among those of the piece's slots that are seen (known before the loop: with a flag of the
    // copying warp's read in every tile the loop was 6% slower)
    bool hole = false;
#pragma unroll 4
    for (int i = tid; i < 4 * tiles; i += 32 * warps) {
      const int sg = 2 * first + (i >> 1), j = seg.at(sg) + 16 * (i & 1);
      if (sg < seg.n && j < a.r.S && seen(j, 16)) hole |= (unsigned)table[j >> a.t.shift] >= (unsigned)a.t.pages;
    }
    if (hole) s_bad = 1;
    named_sync(1, 32 * warps);
    const bool holes = s_bad != 0;
    // the reference m of the weights, 2^(score - m + LP_SHIFT); fresh: none yet (a row that sees nothing needs none)
    float m = p < 0 ? 0.f : -INFINITY, off = 0.f, sum = 0.f;
    bool fresh = p >= 0, ok = true;
    int sb = 0;                                    // S's barrier of the next tile, its parity
    unsigned sp = 0;
    for (int t = 0; t < tiles; ++t) {
      ok = lp_wait_warp(&bar_s[sb], sp, a.err);
      if (++sb == PT_K) sb = 0, sp ^= 1;
      if (!ok) break;
      tc_after();
      float s[LP_TILE];
      lp_ld64(tmem + my, s);                       // half a tile: the rest is old scores, past every p and masked below
      tc_before();
      mbar_arrive(&bar_f);
#pragma unroll
      for (int sg = 0; sg < 2; ++sg) {
        const int j0 = seg.at(2 * (first + t) + sg);
        if (j0 + LP_SEG - 1 > p_lo || (p_hi - j0 >= wnd && j0 + LP_SEG > a.sinks) || holes) {
          // the row's keys of the segment as bits: slots p - window + 1 .. p and the sinks
          uint32_t see = lp_bits(p - wnd + 1 - j0, p + 1 - j0) | lp_bits(0, min(p + 1, a.sinks) - j0);
          if (holes) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int j = j0 + 16 * c;
              if (j < a.r.S && seen(j, 16) && (unsigned)table[j >> a.t.shift] >= (unsigned)a.t.pages) see &= ~(0xffffu << (16 * c));
            }
          }
#pragma unroll
          for (int c = 0; c < LP_SEG; ++c) s[LP_SEG * sg + c] = (see >> c) & 1u ? s[LP_SEG * sg + c] : -INFINITY;
        }
      }
      // P's buffer: free once P V of t - 2 is done (asked here, needed after the exponentials)
      const bool free = t < 2 || mbar_test(&bar_o[t & 1], ((t - 2) >> 1) & 1);
      uint32_t w[32];
      uint64_t part[2];
      auto weights = [&] {
        const uint64_t off2 = f2(off, off);
        part[0] = part[1] = 0;
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float2 e = f2_get(f2_fma(f2(s[2 * c], s[2 * c + 1]), scale2, off2));
          const float p0 = ex2(e.x), p1 = ex2(e.y);
          part[c & 1] = f2_add(part[c & 1], f2(p0, p1));
          w[c] = pack_bf16(p0, p1);
        }
      };
      bool move = __any_sync(FULL, fresh);
      float2 u;
      if (!move) {
        // the tile's sum tells whether a score passes the reference by 2^8
        weights();
        u = f2_get(f2_add(part[0], part[1]));
        move = __any_sync(FULL, mine && !(u.x + u.y <= PT_LIMIT));
      }
      if (move) {
        float x[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < 64; c += 4) {
          x[(c >> 2) & 3] = max3(x[(c >> 2) & 3], s[c], s[c + 1]);
          x[((c >> 2) + 2) & 3] = max3(x[((c >> 2) + 2) & 3], s[c + 2], s[c + 3]);
        }
        // scale > 0 (checked): the maximum of the scaled scores
        const float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * a.scale;
        const bool up = mx > -INFINITY && (fresh || mx > m);
        const float f = up ? (fresh ? 0.f : ex2(m - mx)) : 1.f;
        if (up) {
          m = mx;
          fresh = false;
          off = LP_SHIFT - mx;
        }
        sum *= f;
        if (t > 0) {
          ok = lp_wait_warp(&bar_o[(t - 1) & 1], ((t - 1) >> 1) & 1, a.err);
          if (!ok) break;
          tc_after();
#pragma unroll 1
          for (int c = 0; c < LG_D; c += 32) {
            float o[32];
            lp_ld32(t_o + my + c, o);
            uint32_t v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(o[i] * f);
            lp_st32(t_o + my + c, v);
          }
        }
        weights();
        u = f2_get(f2_add(part[0], part[1]));
      }
      sum += u.x + u.y;
      if (!__all_sync(FULL, free)) {
        ok = lp_wait_warp(&bar_o[t & 1], ((t - 2) >> 1) & 1, a.err);
        if (!ok) break;
      }
      tc_after();
      lp_st32(tmem + my + 64 + 32 * (t & 1), w);
      tc_before();
      mbar_arrive(&bar_p[t & 1]);
    }
    if (ok && tiles > 1) ok = lp_wait_warp(&bar_o[tiles & 1], ((tiles - 2) >> 1) & 1, a.err);
    if (ok && tiles > 0) ok = lp_wait_warp(&bar_o[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1, a.err);
    tc_after();
    if (piece.s > 1) {
      // ---- a piece: the row's part, unnormalised
      const long long at = (long long)piece.slot * a.NKV + h;
      if (mine) a.ml[at * LP_ROWS + r] = make_float2(m, sum);
      // through shared memory (K and V are read), so that a store is a whole row
      unsigned char* st = sk + warp * (32 * LG_D * 4);
#pragma unroll 1
      for (int c = 0; c < LG_D; c += 32) {
        float o[32];
        if (tiles > 0 && ok) {
          lp_ld32(t_o + my + c, o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<float4*>(st + lane * (LG_D * 4) + ((((c + i) >> 2) ^ lane) << 4)) =
              make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
      }
      __syncwarp();
      float* po = a.po + (at * LP_ROWS + warp * 32) * LG_D + 4 * lane;
      const int rows = min(32, live - warp * 32);
#pragma unroll 4
      for (int i = 0; i < rows; ++i)
        *reinterpret_cast<float4*>(po + i * LG_D) = *reinterpret_cast<const float4*>(st + i * (LG_D * 4) + ((lane ^ i) << 4));
    } else {
      // ---- the whole row, through shared memory (over Q, with its swizzle) to 16-byte stores of whole rows
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const uint64_t inv2 = f2(inv, inv);
      uint64_t odd = 0;                              // becomes NaN with the first value that is not finite
#pragma unroll 1
      for (int c = 0; c < LG_D; c += 32) {
        float o[32];
        if (tiles > 0 && ok) {
          lp_ld32(t_o + my + c, o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint64_t x = f2(o[2 * i], o[2 * i + 1]);
          odd = f2_fma(x, 0, odd);
          const float2 y = f2_get(f2_fma(x, inv2, 0));
          w[i] = pack_bf16(y.x, y.y);
        }
        unsigned char* d = sq + (c >> 6) * (LP_Q / 2) + r * 128;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint4*>(d + (((((c & 63) >> 3) + i) ^ (r & 7)) << 4)) =
              make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      }
      const float2 od = f2_get(odd);
      const bool bad = sum == 0.f || (sum > 0.f && !(od.x + od.y == 0.f));   // (a NaN of the weights stays one)
      __syncwarp();
      const int half = lane >> 4, c = lane & 15;
#pragma unroll 4
      for (int i = 0; i < 32; i += 2) {
        const int rr = warp * 32 + i + half, ll = rr >> a.lg, gg = rr & (a.G - 1);
        const uint4 y = *reinterpret_cast<const uint4*>(sq + (c >> 3) * (LP_Q / 2) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4));
        if (rr < live && ok)
          *reinterpret_cast<uint4*>(a.out + (long long)(piece.tok + ll) * a.o_st + (h * a.G + gg) * a.o_sh + 8 * c) = y;
      }
      // rows that are not finite, or saw nothing: the warp, a row at a time
      for (unsigned todo = __ballot_sync(FULL, bad && ok && mine); todo; todo &= todo - 1) {
        const int rr = warp * 32 + __ffs(todo) - 1, ll = rr >> a.lg, hq = h * a.G + (rr & (a.G - 1));
        const long long t = piece.tok + ll;
        const uint2 y = paged_again(a, piece.b, p_lo + ll, hq, a.q + t * a.q_st + hq * a.q_sh);
        *reinterpret_cast<uint2*>(a.out + t * a.o_st + hq * a.o_sh + 4 * lane) = y;
      }
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 4) {
    tc_after();
    tc_dealloc(tmem, LP_COLS);
  }
}

// Joins the pieces of the query tiles that were cut, in their order: a warp a row, the CTAs that the SMs hold go round (how
// many rows there are only the device knows).  For 801 tokens of 32 rows in 3 pieces (24 MB) 7.5 us, 1.5 of them the launch; with a
// CTA for every 16 rows that there might be 8.7, two rows a warp at a time 8 to 10.
constexpr int PM_THREADS = 256, PM_CTAS = 4;
__global__ void __launch_bounds__(PM_THREADS, PM_CTAS) paged_merge_kernel(const __grid_constant__ PagedAttendArgs a) {
  constexpr int W = PM_THREADS / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  const long long n = (long long)a.cut[a.cuts / 2].x * a.NKV * LP_ROWS, step = (long long)a.NKV * LP_ROWS;
#pragma unroll 1
  for (long long k = (long long)blockIdx.x * W + warp; k < n; k += (long long)gridDim.x * W) {
    const int xh = (int)(k / LP_ROWS), x = xh / a.NKV, h = xh - x * a.NKV;
    const int4 cut = a.cut[x];
    // (turned from tile to tile: a warp's rows would be the same in each, and tiles of few tokens all with the same warps)
    const int pieces = cut.z, live = cut.y * a.G, r = (int)(k + 5 * xh) & (LP_ROWS - 1);
    if (r >= live) continue;
    const long long at = ((long long)cut.w * a.NKV + h) * LP_ROWS + r;
    const float2* ml = a.ml + at;
    const float* po = a.po + at * LG_D + 4 * lane;
    // four pieces at a time, their loads together
    float M = -INFINITY, L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int s0 = 0; s0 < pieces; s0 += 4) {
      float2 y[4];
      float4 o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = min(s0 + i, pieces - 1);
        y[i] = ml[s * step];
        o[i] = *reinterpret_cast<const float4*>(po + s * step * LG_D);
      }
      const float m = fmaxf(fmaxf(fmaxf(y[0].x, y[1].x), fmaxf(y[2].x, y[3].x)), M);
      const float g = M > -INFINITY ? ex2(M - m) : 0.f;
      M = m;
      L *= g;
      O.x *= g, O.y *= g, O.z *= g, O.w *= g;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (s0 + i < pieces) {
          const float f = y[i].x > -INFINITY ? ex2(y[i].x - m) : 0.f;
          L += y[i].x > -INFINITY ? f * y[i].y : y[i].y;     // nothing, or a NaN
          O.x += f * o[i].x;
          O.y += f * o[i].y;
          O.z += f * o[i].z;
          O.w += f * o[i].w;
        }
    }
    const float f = 1.f / L;
    uint2 y = make_uint2(pack_bf16(O.x * f, O.y * f), pack_bf16(O.z * f, O.w * f));
    const int l = r >> a.lg, hq = h * a.G + (r & (a.G - 1));
    const long long t = cut.x + l;
    if (__any_sync(FULL, L == 0.f || (L > 0.f && !isfinite(O.x + O.y + O.z + O.w)))) {
      const int b = paged_row(a.r, (int)t);
      const PagedSpan span = paged_span(a.r, b);
      y = paged_again(a, b, span.p0 + (int)t - span.t0, hq, a.q + t * a.q_st + hq * a.q_sh);
    }
    *reinterpret_cast<uint2*>(a.out + t * a.o_st + hq * a.o_sh + 4 * lane) = y;
  }
}

}  // namespace fb

namespace {
using namespace fb;

int paged_group(const fb_paged_cache* c, int NH) {
  FB_CHECK_ARG(NH >= c->NKV && NH % c->NKV == 0, "paged_attend: %d query heads over %d key/value heads", NH, c->NKV);
  const int G = NH / c->NKV;
  if (G != 1 && G != 2 && G != 4 && G != 8) {
    fbh::set_msg("paged_attend: GQA group %d not built (1, 2, 4, 8)", G);
    return FB_ERR_UNSUPPORTED;
  }
  return FB_OK;
}

struct PagedPlan {
  int pieces;                           // a KV head, 0: query tiles stay whole
  bool direct;                          // nothing to cut: no plan, CTAs find their query tiles
  int64_t units, list, cuts, slots, off_ml, off_plan, off_cut, ws_floats;
};
int paged_plan_host(const fb_paged_cache* c, int rows, int width, int T, int NH, int window, int sinks, PagedPlan* p) {
  const int nq = LP_ROWS / (NH / c->NKV);
  const int64_t S = (int64_t)width * c->page, runs = rows < T ? rows : T;
  const int64_t units = (T + runs * (nq - 1)) / nq;                // query tiles, at most
  p->units = units;
  // key tiles of a query tile, at most
  int64_t keys = S;
  if (window > 0 && (int64_t)window + sinks + nq + 3 * LP_SEG < S) keys = (int64_t)window + sinks + nq + 3 * LP_SEG;
  const int64_t most = (keys + LP_TILE - 1) / LP_TILE;
  // CTAs that the SMs hold.  By the device's SMs, not the calling thread's budget: the workspace's size goes by it.
  p->pieces = most > PT_WHOLE ? (2 * fbh::num_sms() + c->NKV - 1) / c->NKV : 0;
  p->direct = p->pieces == 0;
  // a list is cut for PT_WAVES rounds at most (one where query tiles fill less than half of it: two gain nothing by the price
  // below rows of 12800 slots) and into pieces of PT_MIN at least, or is its query tiles
  p->cuts = 2 * units <= p->pieces ? p->pieces : (int64_t)PT_WAVES * p->pieces + p->pieces / 8;
  if (p->cuts > units * ((most + PT_MIN - 1) / PT_MIN)) p->cuts = units * ((most + PT_MIN - 1) / PT_MIN);
  p->list = units > p->cuts ? units : p->cuts;
  FB_CHECK_ARG(p->list * c->NKV <= 0x7fffffff, "paged_attend: too many tokens, rows and heads");
  p->slots = p->cuts * c->NKV;
  p->off_ml = p->slots * LP_ROWS * LG_D;
  p->off_plan = p->off_ml + p->slots * LP_ROWS * 2;
  p->off_cut = p->off_plan + (p->direct ? 0 : p->list * (int64_t)(sizeof(PagedPiece) / 4));
  p->ws_floats = p->off_cut + (p->cuts > 1 ? p->cuts / 2 + 1 : 0) * 4;
  return FB_OK;
}

// The pool as (64 dims, slots, half, heads, pages); boxes of `rows` slots x `halves`.
int paged_map(CUtensorMap* m, const PagedPool& c, bool v, int rows, int halves) {
  const unsigned long long dims[5] = {64, (unsigned long long)c.page, 2, (unsigned long long)c.NKV, (unsigned long long)c.pages};
  const unsigned long long st[4] = {(unsigned long long)(v ? c.v_sl : c.k_sl), 128,
                                    (unsigned long long)(c.NKV > 1 ? (v ? c.v_sh : c.k_sh) : 2 * LG_D),
                                    (unsigned long long)(c.pages > 1 ? (v ? c.v_sb : c.k_sb) : 2 * LG_D)};
  const unsigned bx[5] = {64, (unsigned)rows, (unsigned)halves, 1, 1};
  return fbh::tmap_bf16(m, v ? c.v : c.k, 5, dims, st, bx);
}

}  // namespace

extern "C" int64_t flashb_paged_attend_ws_floats(const fb_paged_cache* cache, int rows, int width, int T, int NH,
                                                 int window, int sinks) {
  PagedPool pool;
  PagedPlan p{};
  if (fbh::paged_pool(cache, &pool) || fbh::paged_width(cache, rows, width) || paged_group(cache, NH)) return -1;
  if (T < 1 || sinks < 0) {
    fbh::set_msg("paged_attend: bad shape T=%d sinks=%d", T, sinks);
    return -1;
  }
  if (paged_plan_host(cache, rows, width, T, NH, window, sinks, &p)) return -1;
  return p.ws_floats;
}

extern "C" int flashb_paged_attend(const fb_paged_cache* cache, const int32_t* table, int64_t table_sb, int rows, int width,
                                   const int64_t* lengths, const int64_t* offsets, int T, const void* q, int64_t q_st,
                                   int64_t q_sh, int NH, int window, int sinks, float scaling, float* ws, int64_t ws_floats,
                                   void* out, int64_t o_st, int64_t o_sh, void* stream) {
  PagedAttendArgs a{};
  int rc = fbh::paged_pool(cache, &a.pool);
  if (!rc) rc = fbh::paged_width(cache, rows, width);
  if (!rc) rc = paged_group(cache, NH);
  if (rc) return rc;
  FB_CHECK_ARG(table && lengths && offsets && q && out, "paged_attend: null pointer argument");
  FB_CHECK_ARG(table_sb >= 0, "paged_attend: table stride %lld", (long long)table_sb);
  FB_CHECK_ARG(T >= 1 && (int64_t)T * NH <= 0x7fffffff, "paged_attend: %d tokens of %d heads", T, NH);
  FB_CHECK_ARG(sinks >= 0, "paged_attend: sinks %d", sinks);
  FB_CHECK_ARG(scaling > 0.f && scaling * LG_LOG2E < INFINITY, "paged_attend: scaling must be positive, and finite times log2(e)");
  FB_CHECK_ARG((((uintptr_t)q | (uintptr_t)out) & 15) == 0 && (q_st | q_sh | o_st | o_sh) % 8 == 0,
               "paged_attend: tensors must be 16-byte aligned with strides multiple of 8 elements");
  FB_CHECK_ARG((T == 1 || (q_st > 0 && o_st > 0)) && (NH == 1 || (q_sh > 0 && o_sh > 0)),
               "paged_attend: strides must be positive");
  FB_CHECK_ARG((cache->pages == 1 || (cache->k_sb > 0 && cache->v_sb > 0)) && (cache->NKV == 1 || (cache->k_sh > 0 && cache->v_sh > 0)),
               "paged_attend: strides of the cache must be positive");
  FB_CHECK_ARG(!fbh::long_box_folds(fbh::long_box(out, 1, T, NH, 0, 2 * o_st, 2 * o_sh, 2 * LG_D)),
               "paged_attend: rows of out share memory");
  rc = fbh::paged_apart(a.pool, T, NH, q, q_st, q_sh, out, o_st, o_sh);
  if (rc) return rc;
  a.t = PagedTable{table, table_sb, a.pool.pages, a.pool.page, a.pool.shift};
  a.r = PagedRows{(const long long*)lengths, (const long long*)offsets, rows, T, width * a.pool.page};
  a.q = (const bf16*)q, a.q_st = q_st, a.q_sh = q_sh, a.NH = NH, a.G = NH / cache->NKV;
  a.window = window > 0 && window < a.r.S ? window : 0, a.sinks = sinks < a.r.S ? sinks : a.r.S;
  a.scale = scaling * LG_LOG2E, a.out = (bf16*)out, a.o_st = o_st, a.o_sh = o_sh;
  PagedPlan p{};
  rc = paged_plan_host(cache, rows, width, T, NH, window, sinks, &p);
  if (rc) return rc;
  FB_CHECK_ARG(p.ws_floats == 0 || (ws && ((uintptr_t)ws & 15) == 0 && ws_floats >= p.ws_floats),
               "paged_attend: workspace of %lld floats, %lld needed", (long long)ws_floats, (long long)p.ws_floats);
  a.NKV = cache->NKV, a.nq = LP_ROWS / a.G, a.lg = a.G == 1 ? 0 : a.G == 2 ? 1 : a.G == 4 ? 2 : 3, a.lq = 7 - a.lg;
  a.per = (rows + PP_THREADS - 1) / PP_THREADS, a.per32 = (rows + 31) / 32;
  a.pieces = p.pieces, a.list = (int)p.list, a.cuts = (int)p.cuts;
  a.rounds = p.pieces ? 1.f / p.pieces : 0.f;
  a.po = ws, a.ml = (float2*)(ws + p.off_ml), a.plan = p.direct ? nullptr : (PagedPiece*)(ws + p.off_plan);
  a.cut = (int4*)(ws + p.off_cut);
  a.err = fbh::device_err_ptr();
  const unsigned long long qd[4] = {64, (unsigned long long)NH, (unsigned long long)T, 2};
  const unsigned long long qs[3] = {(unsigned long long)(NH > 1 ? q_sh : LG_D) * 2, (unsigned long long)(T > 1 ? q_st : LG_D) * 2, 128};
  const unsigned qb[4] = {64, (unsigned)a.G, (unsigned)a.nq, 2};
  rc = fbh::tmap_bf16(&a.tq, q, 4, qd, qs, qb);
  const int small = cache->page < LP_SEG ? cache->page : LP_SEG;
  if (!rc) rc = paged_map(&a.tks, a.pool, false, small, 1);
  if (!rc) rc = paged_map(&a.tvs, a.pool, true, small, 2);
  if (cache->page >= LP_TILE) {
    if (!rc) rc = paged_map(&a.tk, a.pool, false, LP_TILE, 2);
    if (!rc) rc = paged_map(&a.tv, a.pool, true, LP_TILE, 2);
  } else {
    a.tk = a.tks, a.tv = a.tvs;          // not used
  }
  if (rc) return rc;
  const int how = p.direct ? PT_FIND : rows <= 32 && p.units <= p.pieces ? PT_CUT : PT_PLAN;
  const void* attend = how == PT_FIND  ? (const void*)paged_attend_kernel<PT_FIND>
                       : how == PT_CUT ? (const void*)paged_attend_kernel<PT_CUT>
                                       : (const void*)paged_attend_kernel<PT_PLAN>;
  static int attr_done[64][3] = {{0}};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_done[dev][how]) {
    const cudaError_t e = cudaFuncSetAttribute(attend, cudaFuncAttributeMaxDynamicSharedMemorySize, PT_SMEM);
    if (e != cudaSuccess) {
      fbh::set_msg("paged_attend: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
      return FB_ERR_CUDA;
    }
    if (dev < 64) attr_done[dev][how] = 1;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  void* args[] = {(void*)&a};
  if (how == PT_PLAN) rc = fbh::launch_pdl((const void*)paged_plan_kernel, dim3(1), dim3(PP_THREADS), 0, st, args, true);
  if (!rc) rc = fbh::launch_pdl(attend, dim3((unsigned)(p.list * a.NKV)), dim3(PT_THREADS), PT_SMEM, st, args, true);
  if (rc || p.cuts < 2) return rc;
  const int64_t joins = (p.cuts / 2 * a.NKV * LP_ROWS + PM_THREADS / 32 - 1) / (PM_THREADS / 32);
  const int64_t at_once = (int64_t)PM_CTAS * fbh::grid_sms();
  return fbh::launch_pdl((const void*)paged_merge_kernel, dim3((unsigned)(joins < at_once ? joins : at_once)),
                         dim3(PM_THREADS), 0, st, args, true);
}
