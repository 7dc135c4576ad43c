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
// Bound: 512 (NH + 2 NKV) bytes a token, read and written once.  A CTA takes up to four tokens: each thread first issues
// all its 16-byte loads (a half-warp per head), then works out one sine and cosine for a pair and token, shared through
// shared memory by the token's heads.
#include <climits>

#include "fb_paged.cuh"

namespace fb {

constexpr int PA_THREADS = 256;
constexpr int PA_TOKENS = 4;             // tokens of a CTA
constexpr int PA_HALVES = PA_THREADS / 16;

struct PagedAppendArgs {
  PagedPool pool;
  PagedTable t;
  PagedRows r;
  const bf16* qkv;
  long long ldq;
  int NH, NKV, rot, interleaved, tokens;
  const bf16 *q_norm, *k_norm;
  float eps, amplitude;
  const double* turns;
  const long long* positions;
  bf16* q_out;
  long long o_st, o_sh;
};

__global__ void __launch_bounds__(PA_THREADS) paged_append_kernel(const __grid_constant__ PagedAppendArgs a) {
  __shared__ float2 s_cs[PA_TOKENS][LG_D / 2];
  __shared__ long long s_slot[PA_TOKENS];
  __shared__ unsigned char *s_k[PA_TOKENS], *s_v[PA_TOKENS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, half = tid >> 4, l = tid & 15;
  const int t0 = blockIdx.x * a.tokens, heads = a.NH + 2 * a.NKV;
  pdl_wait();
  pdl_trigger();
  if (warp < a.tokens) {
    const int t = t0 + warp;
    const int b = t < a.r.T ? paged_row(a.r, t) : -1;
    if (lane == 0) {
      unsigned char *k = nullptr, *v = nullptr;
      long long pos = -1;
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
      s_slot[warp] = b >= 0 ? pos : LLONG_MIN;
      s_k[warp] = k;
      s_v[warp] = v;
    }
  }
  __syncthreads();
  const int pairs = a.rot >> 1;
  for (int i = tid; i < a.tokens * pairs; i += PA_THREADS) {
    const int t = i / pairs, p = i - t * pairs;
    const long long pos = s_slot[t];
    if (pos == LLONG_MIN) continue;
    const double x = (double)pos * a.turns[p];
    float s, c;
    sincospif(2.f * (float)(x - rint(x)), &s, &c);
    s_cs[t][p] = make_float2(a.amplitude * c, a.amplitude * s);
  }
  __syncthreads();
  for (int i = half; i < a.tokens * heads; i += PA_HALVES) {
    const int ti = i / heads, hd = i - ti * heads, t = t0 + ti;
    const bool live = t < a.r.T && s_slot[ti] != LLONG_MIN;
    const bool is_q = hd < a.NH, is_v = hd >= a.NH + a.NKV;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (live) w = *reinterpret_cast<const uint4*>(a.qkv + t * a.ldq + hd * LG_D + 8 * l);
    if (!is_v) {
      float x[8];
      cvt8(w, x);
      const bf16* nw = is_q ? a.q_norm : a.k_norm;
      const unsigned mask = 0xffffu << (16 * (half & 1));   // the two halves of a warp may be at different kinds of heads
      if (nw) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float f = rsqrtf(ss * (1.f / LG_D) + a.eps);
        float g[8];
        cvt8(*reinterpret_cast<const uint4*>(nw + 8 * l), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= f * g[e];
      }
      if (a.rot > 0) {
        if (a.interleaved) {
          if (8 * l < a.rot) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 cs = s_cs[ti][4 * l + e];
              const float p = x[2 * e], m = x[2 * e + 1];
              x[2 * e] = p * cs.x - m * cs.y;
              x[2 * e + 1] = m * cs.x + p * cs.y;
            }
          }
        } else {
          const int step = a.rot >> 4, my = l < step ? 0 : 1;   // lanes from a dim to its pair
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            y[e] = __shfl_sync(mask, x[e], (lane & 16) + (8 * l < a.rot ? (my ? l - step : l + step) : l));
          if (8 * l < a.rot) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 cs = s_cs[ti][8 * (my ? l - step : l) + e];
              x[e] = x[e] * cs.x + (my ? y[e] : -y[e]) * cs.y;
            }
          }
        }
      }
      w = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
    }
    if (!live) continue;
    if (is_q) {
      *reinterpret_cast<uint4*>(a.q_out + t * a.o_st + hd * a.o_sh + 8 * l) = w;
    } else {
      unsigned char* p = is_v ? s_v[ti] : s_k[ti];
      const int h = hd - a.NH - (is_v ? a.NKV : 0);
      if (p) *reinterpret_cast<uint4*>(p + h * (is_v ? a.pool.v_sh : a.pool.k_sh) + 16 * l) = w;
    }
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
  a.tokens = PA_TOKENS;
  void* args[] = {(void*)&a};
  return fbh::launch_pdl((const void*)paged_append_kernel, dim3((T - 1) / a.tokens + 1), dim3(PA_THREADS), 0,
                         (cudaStream_t)stream, args, true);
}
