// flashb: attention of a run of tokens over a long cache with a sliding window and first tokens that stay visible.
//
// q [B, NH, L, 128] holds the tokens at slots q_start .. q_start + L - 1 of k / v [B, NKV, S, 128].  The token at slot
// p of row b sees slot j when start_b <= j <= p and (j > p - window or j < start_b + sinks);
//   out = softmax(scaling q k^T over those) v in fp32, rounded once; a token without a visible key (p < start_b) gives 0.
//
// long_row_kernel: a CTA per (token, head, row), a warp per quarter of the visible keys, four dims a lane.
#include "fb_long.cuh"

namespace fb {

struct LongPrefillArgs {
  const bf16 *q, *k, *v;
  long long q_sb, q_sh, q_sl, k_sb, k_sh, k_sl, v_sb, v_sh, v_sl;
  const long long* starts;
  int B, NH, NKV, L, q_start, window, sinks;
  float scale;                          // scaling x log2(e)
  bf16* out;
  long long o_sb, o_sl, o_sh;
};

__global__ void __launch_bounds__(128) long_row_kernel(const __grid_constant__ LongPrefillArgs a) {
  __shared__ float s_o[4][LG_D], s_m[4], s_l[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int l = blockIdx.x, hq = blockIdx.y, b = blockIdx.z, h = hq / (a.NH / a.NKV);
  pdl_wait();
  pdl_trigger();
  const int p = a.q_start + l;
  // the tokens up to p; a row that begins after p has none
  const LongRow row = long_row(p + 1, a.starts ? a.starts[b] : 0, p + 1, a.window, a.sinks);
  float qf[4];
  const bf16* qp = a.q + b * a.q_sb + hq * a.q_sh + l * a.q_sl;
#pragma unroll
  for (int e = 0; e < 4; ++e) qf[e] = b2f(qp[4 * lane + e]) * a.scale;
  const bf16* kb = a.k + b * a.k_sb + h * a.k_sh + 4 * lane;
  const bf16* vb = a.v + b * a.v_sb + h * a.v_sh + 4 * lane;
  float m = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = warp; i < row.n; i += 4) {
    const long long j = row.slot(i);
    const uint2 kw = *reinterpret_cast<const uint2*>(kb + j * a.k_sl), vw = *reinterpret_cast<const uint2*>(vb + j * a.v_sl);
    const float s = warp_sum(qf[0] * lo_f(kw.x) + qf[1] * hi_f(kw.x) + qf[2] * lo_f(kw.y) + qf[3] * hi_f(kw.y));
    const float mn = fmaxf(m, s), f = m > -INFINITY ? ex2(m - mn) : 0.f, w = mn > -INFINITY ? ex2(s - mn) : 0.f;
    m = mn;
    sum = sum * f + w;
    o[0] = o[0] * f + w * lo_f(vw.x);
    o[1] = o[1] * f + w * hi_f(vw.x);
    o[2] = o[2] * f + w * lo_f(vw.y);
    o[3] = o[3] * f + w * hi_f(vw.y);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) s_o[warp][4 * lane + e] = o[e];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = sum;
  }
  __syncthreads();
  const float M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float L = 0.f, O = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = s_m[w] > -INFINITY ? ex2(s_m[w] - M) : 0.f;
    if (f != 0.f) {
      L += f * s_l[w];
      O += f * s_o[w][threadIdx.x];
    }
  }
  a.out[b * a.o_sb + l * a.o_sl + hq * a.o_sh + threadIdx.x] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L);
}

}  // namespace fb

extern "C" int flashb_long_prefill(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_sl, const void* k, int64_t k_sb,
                                   int64_t k_sh, int64_t k_sl, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_sl,
                                   int B, int NH, int NKV, int L, int S, int q_start, const int64_t* starts, int window,
                                   int sinks, float scaling, void* out, int64_t o_sb, int64_t o_sl, int64_t o_sh,
                                   void* stream) {
  using namespace fb;
  FB_CHECK_ARG(q && k && v && out, "long_prefill: null pointer argument");
  FB_CHECK_ARG(B >= 1 && L >= 1 && NKV >= 1 && NH >= NKV && NH % NKV == 0, "long_prefill: bad shape B=%d NH=%d NKV=%d L=%d",
               B, NH, NKV, L);
  const int G = NH / NKV;
  if (G != 1 && G != 2 && G != 4 && G != 8) {
    fbh::set_msg("long_prefill: GQA group %d not built (1, 2, 4, 8)", G);
    return FB_ERR_UNSUPPORTED;
  }
  FB_CHECK_ARG(q_start >= 0 && (int64_t)q_start + L <= S, "long_prefill: tokens at slots %d .. of a cache of %d", q_start, S);
  FB_CHECK_ARG(sinks >= 0, "long_prefill: sinks %d", sinks);
  FB_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) == 0 &&
                   (q_sb | q_sh | q_sl | k_sb | k_sh | k_sl | v_sb | v_sh | v_sl | o_sb | o_sl | o_sh) % 8 == 0,
               "long_prefill: tensors must be 16-byte aligned with strides multiple of 8 elements");
  FB_CHECK_ARG(q_sl >= LG_D && k_sl >= LG_D && v_sl >= LG_D && NH <= 65535 && B <= 65535, "long_prefill: bad strides or grid");
  LongPrefillArgs a{(const bf16*)q, (const bf16*)k, (const bf16*)v, q_sb, q_sh, q_sl, k_sb, k_sh, k_sl, v_sb, v_sh, v_sl,
                    (const long long*)starts, B, NH, NKV, L, q_start, window > 0 ? window : 0, sinks,
                    scaling * LG_LOG2E, (bf16*)out, o_sb, o_sl, o_sh};
  void* args[] = {(void*)&a};
  return fbh::launch_pdl((const void*)long_row_kernel, dim3(L, NH, B), dim3(128), 0, (cudaStream_t)stream, args, true);
}
