// flashb: the new tokens of many rows into a paged cache, with the head norms and the rotary embedding on the way.
//
// qkv [T, (NH + 2 NKV) 128] holds each token's raw q | k | v heads.  Per q and k head, in fp32 and rounded to bf16 once:
//   y = w x / sqrt(mean(x^2) + eps)                      (with a norm weight)
//   z_i = A (y_i cos t - y_i' sin t),  z_i' = A (y_i' cos t + y_i sin t),   t = 2 pi position turns_i    (the first `rot` dims)
// for the pairs (i, i') = (i, i + rot / 2), or (2 i, 2 i + 1) interleaved.  q goes to q_out, k and v to their slots.
//
// The angle: position x turns in 64 bits, less its whole turns, then sincospi in fp32.  In fp32 the product alone would be
// off by 2^-24 of the angle, 0.01 radians at position 200000 of the fastest pair.
//
// Bound: 512 (NH + 2 NKV) bytes a token, read and written once; for a few tokens a chain of loads (offsets, lengths, page).
// A warp takes units of up to twelve heads through a ring of its own in shared memory (bulk copies of 3 KB, three under
// way), eight lanes a head; the first copies are issued before the tokens' places are known.  Places (up to seven tokens a
// warp, no load waiting for another token's) and one sine and cosine for each pair and token are worked out once a CTA.
//
// Measured on a B200 (in a CUDA graph): 16391 tokens of 24 heads (201 MB) 39 us, 0.79 of the measured copy bandwidth, with
// head norms 40 us; one token of 128 rows 3.0 us, of 2 rows 2.9 us.  Sixteen lanes a head (and one round of CTAs) 41 us, 53
// with norms (twice the instructions a head) and 3.4 for one token.  Rings of five units of eight heads 42 us, 30 instead of
// 23 for tokens of twelve heads (a unit of eight and one of four); three CTAs an SM 45; loads straight to registers, six a
// thread, 48 to 58 whatever the occupancy (too few bytes under way).
#include <climits>

#include "fb_long_tc.cuh"
#include "fb_paged.cuh"

namespace fb {

constexpr int PA_THREADS = 256, PA_WARPS = PA_THREADS / 32;
constexpr int PA_CTAS = 2;               // an SM: 100 KB
constexpr int PA_EACH = 7;               // tokens of a CTA whose places a warp finds, at most
constexpr int PA_TOKENS = PA_EACH * PA_WARPS;
constexpr int PA_HEADS = 12;             // heads of a unit, at most
constexpr int PA_RING = 3;               // units of a warp under way
constexpr int PA_SLOT = PA_HEADS * LG_D * 2;
constexpr int PA_SMEM = PA_WARPS * PA_RING * PA_SLOT + PA_TOKENS * (LG_D / 2) * (int)sizeof(float2);

struct PagedAppendArgs {
  PagedPool pool;
  PagedTable t;
  PagedRows r;
  const bf16* qkv;
  long long ldq;
  int NH, NKV, rot, interleaved, tokens, each;   // tokens of a CTA, heads of a unit
  const bf16 *q_norm, *k_norm;
  float eps, amplitude;
  const double* turns;
  const long long* positions;
  bf16* q_out;
  long long o_st, o_sh;
  unsigned* err;
};

__device__ __forceinline__ uint4 paged_pack(const float* v) {
  return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}

__global__ void __launch_bounds__(PA_THREADS, PA_CTAS) paged_append_kernel(const __grid_constant__ PagedAppendArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char* ring = smem + (threadIdx.x >> 5) * (PA_RING * PA_SLOT);
  float2(*s_cs)[LG_D / 2] = reinterpret_cast<float2(*)[LG_D / 2]>(smem + PA_WARPS * PA_RING * PA_SLOT);
  __shared__ __align__(8) uint64_t bars[PA_WARPS][PA_RING];
  __shared__ long long s_pos[PA_TOKENS];
  __shared__ unsigned char *s_k[PA_TOKENS], *s_v[PA_TOKENS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, l = tid & 7;
  const int t0 = blockIdx.x * a.tokens, tokens = min(a.tokens, a.r.T - t0), pairs = a.rot >> 1, heads = a.NH + 2 * a.NKV;
  // a lane's two runs of eight dims.  Half layout: the second run holds the first one's partners, or is not turned either;
  // interleaved: every run holds whole pairs.
  const int l2 = l - (pairs >> 3);
  const int d1 = a.interleaved || l2 < 0 ? 8 * l : a.rot + 16 * l2;
  const int d2 = a.interleaved ? LG_D / 2 + 8 * l : l2 < 0 ? pairs + 8 * l : d1 + 8;
  const bool turn1 = d1 < a.rot, turn2 = d2 < a.rot;
  uint64_t* bar = bars[warp];
  if (lane == 0) {
    for (int i = 0; i < PA_RING; ++i) mbar_init(&bar[i], 1);
    fence_mbar_init();
  }
  pdl_wait();
  pdl_trigger();
  // ---- a unit: `each` heads of a token; warp w takes units w, w + PA_WARPS, .. through its ring
  const int per = (heads + a.each - 1) / a.each, units = tokens * per;
  auto copy = [&](int u, int slot) {                         // lane 0
    const int j = u / per, h = (u - j * per) * a.each;
    const unsigned bytes = min(a.each, heads - h) * (LG_D * 2);
    mbar_arrive_expect_tx(&bar[slot], bytes);
    bulk_g2s(ring + slot * PA_SLOT, a.qkv + (t0 + j) * a.ldq + h * LG_D, bytes, &bar[slot]);
  };
  if (lane == 0)
    for (int i = 0; i < PA_RING; ++i)
      if (warp + i * PA_WARPS < units) copy(warp + i * PA_WARPS, i);
  __syncwarp();
  uint4 qn[2]{}, kn[2]{};
  if (a.q_norm) {
    qn[0] = *reinterpret_cast<const uint4*>(a.q_norm + d1), qn[1] = *reinterpret_cast<const uint4*>(a.q_norm + d2);
    kn[0] = *reinterpret_cast<const uint4*>(a.k_norm + d1), kn[1] = *reinterpret_cast<const uint4*>(a.k_norm + d2);
  }
  // ---- the tokens' places (a few a warp), the turns of their pairs
  const int each = (a.tokens + PA_WARPS - 1) / PA_WARPS;
  if (warp * each < tokens) {
    const int j = warp * each + lane, t = t0 + j;
    const int b = paged_rows<PA_EACH>(a.r, t0 + warp * each);
    if (lane < each && j < tokens) {
      unsigned char *k = nullptr, *v = nullptr;
      long long pos = LLONG_MIN;                             // no row's token
      if (b >= 0) {
        const long long slot = a.r.lengths[b] - paged_left(a.r, b, t);
        pos = a.positions ? a.positions[t] : slot;
        if (slot >= 0 && slot < a.r.S) {
          const int page = a.t.table[b * a.t.table_sb + (slot >> a.t.shift)];
          if ((unsigned)page < (unsigned)a.t.pages) {
            const long long in = slot & (a.t.page - 1);
            k = a.pool.k + page * a.pool.k_sb + in * a.pool.k_sl;
            v = a.pool.v + page * a.pool.v_sb + in * a.pool.v_sl;
          }
        }
      }
      s_pos[j] = pos;
      s_k[j] = k;
      s_v[j] = v;
    }
  }
  const int p = tid & 63;                                    // a pair a thread, every fourth token
  const double turns = p < pairs ? a.turns[p] : 0.;
  __syncthreads();
  if (p < pairs)
#pragma unroll 1
    for (int t = tid >> 6; t < tokens; t += PA_THREADS / 64) {
      const double x = (double)s_pos[t] * turns;
      float s, c;
      sincospif(2.f * (float)(x - rint(x)), &s, &c);
      s_cs[t][p] = make_float2(a.amplitude * c, a.amplitude * s);
    }
  __syncthreads();
  // ---- the heads, four at a time
  const unsigned mask = 0xffu << (lane & 24);
  int slot = 0;
  unsigned phase = 0;
#pragma unroll 1
  for (int u = warp; u < units; u += PA_WARPS) {
    const int j = u / per, h0 = (u - j * per) * a.each, n = min(a.each, heads - h0);
    float2 cs[8];
    if (turn1) {
      const int p1 = a.interleaved ? 4 * l : 8 * l, p2 = a.interleaved ? LG_D / 4 + 4 * l : 8 * l + 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        cs[e] = s_cs[j][p1 + e];
        cs[4 + e] = s_cs[j][p2 + e];
      }
    }
    const bool live = s_pos[j] != LLONG_MIN;
    unsigned char *kp = s_k[j], *vp = s_v[j];
    bf16* qp = a.q_out + (t0 + j) * a.o_st;
    if (!lp_wait_warp(&bar[slot], phase, a.err)) {           // no copy may be in flight when the CTA ends
      for (int i = 1; i < PA_RING; ++i)
        if (u + i * PA_WARPS < units) lp_wait_warp(&bar[(slot + i) % PA_RING], slot + i < PA_RING ? phase : phase ^ 1, a.err);
      break;
    }
    const bf16* x = reinterpret_cast<const bf16*>(ring + slot * PA_SLOT);
#pragma unroll 1
    for (int i = lane >> 3; i < n; i += 4) {
      const int h = h0 + i;
      const uint4 x1 = *reinterpret_cast<const uint4*>(x + i * LG_D + d1), x2 = *reinterpret_cast<const uint4*>(x + i * LG_D + d2);
      if (h >= a.NH + a.NKV) {
        if (live && vp) {
          bf16* y = reinterpret_cast<bf16*>(vp + (h - a.NH - a.NKV) * a.pool.v_sh);
          *reinterpret_cast<uint4*>(y + d1) = x1;
          *reinterpret_cast<uint4*>(y + d2) = x2;
        }
        continue;
      }
      float v[16];
      cvt8(x1, v);
      cvt8(x2, v + 8);
      if (a.q_norm) {
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s0 += v[e] * v[e], s1 += v[8 + e] * v[8 + e];
        s0 += s1;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) s0 += __shfl_xor_sync(mask, s0, o);
        const float f = rsqrtf(s0 * (1.f / LG_D) + a.eps);
        float g[16];
        cvt8(h < a.NH ? qn[0] : kn[0], g);
        cvt8(h < a.NH ? qn[1] : kn[1], g + 8);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] *= f * g[e];
      }
      if (a.interleaved) {                                   // (dims that do not turn stay: 0 x an infinity is not 0)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < 4 ? turn1 : turn2) {
            const float q = v[2 * e], m = v[2 * e + 1];
            v[2 * e] = q * cs[e].x - m * cs[e].y;
            v[2 * e + 1] = m * cs[e].x + q * cs[e].y;
          }
      } else if (turn1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float q = v[e], m = v[8 + e];
          v[e] = q * cs[e].x - m * cs[e].y;
          v[8 + e] = m * cs[e].x + q * cs[e].y;
        }
      }
      bf16* y = h < a.NH ? qp + h * a.o_sh : reinterpret_cast<bf16*>(kp + (h - a.NH) * a.pool.k_sh);
      if (live && (h < a.NH || kp)) {
        *reinterpret_cast<uint4*>(y + d1) = paged_pack(v);
        *reinterpret_cast<uint4*>(y + d2) = paged_pack(v + 8);
      }
    }
    __syncwarp();
    if (lane == 0 && u + PA_RING * PA_WARPS < units) copy(u + PA_RING * PA_WARPS, slot);
    if (++slot == PA_RING) slot = 0, phase ^= 1;
  }
}

}  // namespace fb

namespace fbh {

int paged_pool(const fb_paged_cache* c, fb::PagedPool* out) {
  FB_CHECK_ARG(c, "paged cache: null descriptor");
  FB_CHECK_ARG(c->pages >= 1 && c->NKV >= 1, "paged cache: bad shape pages=%d NKV=%d", c->pages, c->NKV);
  FB_CHECK_ARG(c->page >= 16 && c->page <= (1 << 20) && (c->page & (c->page - 1)) == 0,
               "paged cache: pages of %d slots (a power of two, 16 to 2^20)", c->page);
  FB_CHECK_ARG(c->k && c->v && ((uintptr_t)c->k & 15) == 0 && ((uintptr_t)c->v & 15) == 0,
               "paged cache: keys and values: not null, 16-byte aligned");
  const int64_t st[6] = {c->k_sb, c->k_sh, c->k_sl, c->v_sb, c->v_sh, c->v_sl};
  for (int64_t x : st)
    FB_CHECK_ARG(x >= 0 && x % 8 == 0 && x < (1ll << 38), "paged cache: strides must be multiples of 8 elements");
  FB_CHECK_ARG(c->k_sl >= fb::LG_D && c->v_sl >= fb::LG_D, "paged cache: slot strides below the row (%d)", fb::LG_D);
  out->k = (unsigned char*)c->k, out->v = (unsigned char*)c->v;
  out->k_sb = 2 * c->k_sb, out->k_sh = 2 * c->k_sh, out->k_sl = 2 * c->k_sl;
  out->v_sb = 2 * c->v_sb, out->v_sh = 2 * c->v_sh, out->v_sl = 2 * c->v_sl;
  out->pages = c->pages, out->NKV = c->NKV, out->page = c->page;
  out->shift = 0;
  while ((1 << out->shift) < c->page) ++out->shift;
  return FB_OK;
}

int paged_width(const fb_paged_cache* c, int rows, int width) {
  FB_CHECK_ARG(rows >= 1 && width >= 1, "paged rows: bad shape rows=%d width=%d", rows, width);
  FB_CHECK_ARG((int64_t)width * c->page <= 0x3fffff00, "paged rows: %d pages of %d slots a row", width, c->page);
  return FB_OK;
}

int paged_apart(const fb::PagedPool& c, int T, int NH, const void* q, int64_t q_st, int64_t q_sh, const void* out, int64_t o_st,
                int64_t o_sh) {
  const LongBox o = long_box(out, 1, T, NH, 0, 2 * o_st, 2 * o_sh, 2 * fb::LG_D);
  FB_CHECK_ARG(!long_boxes_meet(o, long_box(q, 1, T, NH, 0, 2 * q_st, 2 * q_sh, 2 * fb::LG_D)),
               "paged attention: out and q share memory");
  FB_CHECK_ARG(!long_boxes_meet(o, long_box(c.k, c.pages, c.NKV, c.page, c.k_sb, c.k_sh, c.k_sl, 2 * fb::LG_D)) &&
                   !long_boxes_meet(o, long_box(c.v, c.pages, c.NKV, c.page, c.v_sb, c.v_sh, c.v_sl, 2 * fb::LG_D)),
               "paged attention: out and the cache share memory");
  return FB_OK;
}

}  // namespace fbh

extern "C" int flashb_paged_append(const fb_paged_cache* cache, const int32_t* table, int64_t table_sb, int rows, int width,
                                   const int64_t* lengths, const int64_t* offsets, int T, const void* qkv, int64_t ldq,
                                   int NH, const void* q_norm, const void* k_norm, float eps, const double* turns, int rot,
                                   int interleaved, float amplitude, const int64_t* positions, void* q_out, int64_t o_st,
                                   int64_t o_sh, void* stream) {
  using namespace fb;
  PagedAppendArgs a{};
  int rc = fbh::paged_pool(cache, &a.pool);
  if (!rc) rc = fbh::paged_width(cache, rows, width);
  if (rc) return rc;
  FB_CHECK_ARG(table && lengths && qkv && q_out, "paged_append: null pointer argument");
  FB_CHECK_ARG(table_sb >= 0, "paged_append: table stride %lld", (long long)table_sb);
  FB_CHECK_ARG(T >= 1 && NH >= 1, "paged_append: bad shape T=%d NH=%d", T, NH);
  FB_CHECK_ARG(offsets || T == rows, "paged_append: %d tokens of %d rows without offsets", T, rows);
  FB_CHECK_ARG((q_norm == nullptr) == (k_norm == nullptr), "paged_append: q_norm and k_norm come together");
  FB_CHECK_ARG(rot >= 0 && rot <= LG_D && rot % 16 == 0, "paged_append: %d rotated dims (a multiple of 16 up to %d)", rot, LG_D);
  FB_CHECK_ARG(rot == 0 || (turns && ((uintptr_t)turns & 7) == 0), "paged_append: rotation without its turns");
  const int heads = NH + 2 * cache->NKV;
  FB_CHECK_ARG((int64_t)heads * LG_D <= 0x7fffffff / 8, "paged_append: too many heads");
  FB_CHECK_ARG(ldq >= (int64_t)heads * LG_D && ldq % 8 == 0, "paged_append: row stride of qkv %lld", (long long)ldq);
  FB_CHECK_ARG(o_st > 0 && o_sh > 0 && (o_st | o_sh) % 8 == 0, "paged_append: strides of q_out: positive multiples of 8");
  FB_CHECK_ARG((((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)q_norm | (uintptr_t)k_norm) & 15) == 0,
               "paged_append: tensors must be 16-byte aligned");
  const fbh::LongBox out = fbh::long_box(q_out, 1, T, NH, 0, 2 * o_st, 2 * o_sh, 2 * LG_D);
  const fbh::LongBox in = fbh::long_box(qkv, 1, T, heads, 0, 2 * ldq, 2 * LG_D, 2 * LG_D);
  const fbh::LongBox k = fbh::long_box(a.pool.k, a.pool.pages, a.pool.NKV, a.pool.page, a.pool.k_sb, a.pool.k_sh, a.pool.k_sl, 2 * LG_D);
  const fbh::LongBox v = fbh::long_box(a.pool.v, a.pool.pages, a.pool.NKV, a.pool.page, a.pool.v_sb, a.pool.v_sh, a.pool.v_sl, 2 * LG_D);
  FB_CHECK_ARG(!fbh::long_box_folds(out), "paged_append: rows of q_out share memory");
  FB_CHECK_ARG((q_out == qkv && (o_st == ldq || T == 1) && (o_sh == LG_D || NH == 1)) || !fbh::long_boxes_meet(out, in),
               "paged_append: q_out and qkv share memory and are not the same");
  FB_CHECK_ARG(!fbh::long_box_folds(k) && !fbh::long_box_folds(v) && !fbh::long_boxes_meet(k, v),
               "paged_append: slots of the cache share memory");
  FB_CHECK_ARG(!fbh::long_boxes_meet(k, in) && !fbh::long_boxes_meet(v, in) && !fbh::long_boxes_meet(k, out) &&
                   !fbh::long_boxes_meet(v, out),
               "paged_append: the cache shares memory with qkv or q_out");
  a.t = PagedTable{table, table_sb, a.pool.pages, a.pool.page, a.pool.shift};
  a.r = PagedRows{(const long long*)lengths, (const long long*)offsets, rows, T, width * a.pool.page};
  a.qkv = (const bf16*)qkv, a.ldq = ldq, a.NH = NH, a.NKV = cache->NKV, a.rot = rot, a.interleaved = interleaved != 0;
  a.q_norm = (const bf16*)q_norm, a.k_norm = (const bf16*)k_norm, a.eps = eps, a.amplitude = amplitude;
  a.turns = turns, a.positions = (const long long*)positions;
  a.q_out = (bf16*)q_out, a.o_st = o_st, a.o_sh = o_sh;
  const int at_once = PA_CTAS * fbh::grid_sms();
  // Rounds of CTAs, all of them full (20000 tokens in CTAs of 56 56 us, in two rounds 46).  Where there are no norms to work
  // out, shorter CTAs begin and end beside others' streams: 16391 tokens in CTAs of 56 41 us, of 28 38 us; with norms 40 and 43.
  const int most = q_norm ? PA_TOKENS : 32, rounds = (T - 1) / (at_once * most) + 1;
  a.tokens = (T - 1) / (at_once * rounds) + 1;
  const int parts = (heads + PA_HEADS - 1) / PA_HEADS;       // of a token, equal but for whole fours of heads
  a.each = a.tokens * parts >= PA_WARPS ? ((heads + parts - 1) / parts + 3) / 4 * 4 : 4;   // few tokens: a unit for every warp
  a.err = fbh::device_err_ptr();
  static int attr_done[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(paged_append_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PA_SMEM);
    if (e != cudaSuccess) {
      fbh::set_msg("paged_append: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
      return FB_ERR_CUDA;
    }
    if (dev < 64) attr_done[dev] = 1;
  }
  void* args[] = {(void*)&a};
  return fbh::launch_pdl((const void*)paged_append_kernel, dim3((T - 1) / a.tokens + 1), dim3(PA_THREADS), PA_SMEM,
                         (cudaStream_t)stream, args, true);
}
