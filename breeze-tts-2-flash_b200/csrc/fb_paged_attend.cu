// flashb: attention of a step's new tokens (a run of any length per row) over a paged cache.
//
//   out_t = softmax(scaling q_t k^T over the slots that t sees) v, fp32, rounded once; without a visible slot 0.
//
// A warp per token and query head, one key at a time, four dims a lane.
#include "fb_paged.cuh"

namespace fb {

struct PagedAttendArgs {
  PagedPool pool;
  PagedTable t;
  PagedRows r;
  const bf16* q;
  long long q_st, q_sh;
  int NH, G, window, sinks;
  float scale;                          // scaling x log2(e)
  bf16* out;
  long long o_st, o_sh;
};

// P x 2^-24: the unnormalised sums of 2^16 keys stay in fp32's range for every finite V
constexpr float PT_SHIFT = -24.f;

// One token and head over its visible keys, one at a time: four dims a lane; the row in bf16.
__device__ uint2 paged_one(const PagedAttendArgs& a, int b, int p, int hq, const bf16* q) {
  const int lane = threadIdx.x & 31, h = hq / a.G;
  const LongRow row = long_row((long long)p + 1, 0, a.r.S, a.window, a.sinks);
  const unsigned char *kb = a.pool.k + h * a.pool.k_sh + 8 * lane, *vb = a.pool.v + h * a.pool.v_sh + 8 * lane;
  const int* table = a.t.table + b * a.t.table_sb;
  const uint2 qw = *reinterpret_cast<const uint2*>(q + 4 * lane);
  float m = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  bool some = false;
#pragma unroll 4
  for (int i = 0; i < row.n; ++i) {
    const int j = (int)row.slot(i), page = table[j >> a.t.shift], in = j & (a.t.page - 1);
    if ((unsigned)page >= (unsigned)a.t.pages) continue;
    some = true;
    const uint2 kw = *reinterpret_cast<const uint2*>(kb + page * a.pool.k_sb + in * a.pool.k_sl);
    const uint2 vw = *reinterpret_cast<const uint2*>(vb + page * a.pool.v_sb + in * a.pool.v_sl);
    const float s = a.scale * warp_sum(lo_f(qw.x) * lo_f(kw.x) + hi_f(qw.x) * hi_f(kw.x) + lo_f(qw.y) * lo_f(kw.y) +
                                       hi_f(qw.y) * hi_f(kw.y));
    const float mn = fmaxf(m, s), f = m > -INFINITY ? ex2(m - mn) : 0.f;
    const float w = mn > -INFINITY ? ex2(s - mn + PT_SHIFT) : (s == -INFINITY ? 0.f : s);
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

__global__ void __launch_bounds__(128) paged_attend_kernel(const __grid_constant__ PagedAttendArgs a) {
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  const int t = i / a.NH, hq = i - t * a.NH;
  if (t >= a.r.T) return;
  const int b = paged_row(a.r, t);
  if (b < 0) return;
  const long long len = min(max(a.r.lengths[b], 0ll), (long long)a.r.S);
  const int p = (int)(len - paged_left(a.r, b, t));
  const uint2 w = paged_one(a, b, p, hq, a.q + t * a.q_st + hq * a.q_sh);
  *reinterpret_cast<uint2*>(a.out + t * a.o_st + hq * a.o_sh + 4 * lane) = w;
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

}  // namespace

extern "C" int64_t flashb_paged_attend_ws_floats(const fb_paged_cache* cache, int rows, int width, int T, int NH,
                                                 int window, int sinks) {
  PagedPool pool;
  if (fbh::paged_pool(cache, &pool) || fbh::paged_width(cache, rows, width) || paged_group(cache, NH)) return -1;
  return 0;
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
  FB_CHECK_ARG(scaling > 0.f, "paged_attend: scaling must be positive");
  FB_CHECK_ARG((((uintptr_t)q | (uintptr_t)out) & 15) == 0 && (q_st | q_sh | o_st | o_sh) % 8 == 0,
               "paged_attend: tensors must be 16-byte aligned with strides multiple of 8 elements");
  FB_CHECK_ARG((T == 1 || (q_st > 0 && o_st > 0)) && (NH == 1 || (q_sh > 0 && o_sh > 0)),
               "paged_attend: strides must be positive");
  FB_CHECK_ARG(!fbh::long_box_folds(fbh::long_box(out, 1, T, NH, 0, 2 * o_st, 2 * o_sh, 2 * LG_D)),
               "paged_attend: rows of out share memory");
  a.t = PagedTable{table, table_sb, a.pool.pages, a.pool.page, a.pool.shift};
  a.r = PagedRows{(const long long*)lengths, (const long long*)offsets, rows, T, width * a.pool.page};
  a.q = (const bf16*)q, a.q_st = q_st, a.q_sh = q_sh, a.NH = NH, a.G = NH / cache->NKV;
  a.window = window > 0 && window < a.r.S ? window : 0, a.sinks = sinks < a.r.S ? sinks : a.r.S;
  a.scale = scaling * LG_LOG2E, a.out = (bf16*)out, a.o_st = o_st, a.o_sh = o_sh;
  (void)ws, (void)ws_floats;
  void* args[] = {(void*)&a};
  return fbh::launch_pdl((const void*)paged_attend_kernel, dim3((unsigned)(((int64_t)T * NH + 3) / 4)), dim3(128), 0,
                         (cudaStream_t)stream, args, true);
}
