// flashb: eviction from a KV cache by accumulated attention weight.
//
// Row b holds keys in slots [st, len).  With at most `keep` of them everything stays; else the first `sinks`, the
// last `recent` and, of the others, the keep - sinks - recent slots of largest accumulated weight (equal weights: the
// lower slot; NaN above everything) stay.  Each KV head chooses for itself.  What stays moves, in slot order, to
// slots 0, 1, .. of another cache, its weight with it; kept[i] is the slot it came from.
//
// One launch.  A CTA finds the weight of the last slot that stays by radix selection (8 bits a pass over order-preserving
// integer keys, held in shared memory), counts the slots that stay below each thread's run of slots, and then copies its
// share of them.  With few rows several CTAs share one: each selects for itself (a few microseconds, and no exchange),
// and copies its part.  Bound: HBM, the kept rows read and written once (1 KB a slot in bf16).
// Measured on a B200: 64 rows of up to 8192 slots to 2048 (478 MB) 99 us, 0.74 of the measured copy bandwidth; the same rows
// in 4 bits 70 us, 0.31; one stream's 1920 slots to 1023 9 us.  What is lost at many rows: the selection, 17 us (64 slots
// kept of the same rows), during which memory is idle, and uneven ends (256 CTAs of one ragged row each on 148 SMs: 40 have
// one CTA, the others two).  The places of the kept slots matter little: adjacent instead of scattered, 98 us for 99 (in 4 bits
// 62 for 72).  In 4 bits a row is 64 bytes, so 8 of a warp's 32 lanes copy codes, and the scales take a second loop.
// Half the warps copying while the others select took 102 us for 101 then.
#include "fb_long.cuh"

namespace fb {

constexpr int EV_THREADS = 512;
constexpr int EV_KEYS = 11776;       // keys held in shared memory (46 KB); rows with more read the weights again
constexpr int EV_ROWS = 4;           // rows in flight per warp of the copy

struct EvictArgs {
  LongCache c, d;
  const float* acc;
  long long acc_sb, acc_sh;
  const long long *lengths, *starts;
  int NKV, S, keep, sinks, recent, row_bytes;
  int* kept;                       // [B, NKV, keep]
  long long* lengths_out;          // [B]
  float* acc_out;
  long long acco_sb, acco_sh;
  int acc_n;                       // slots of acc_out
  int staged;                      // keys that fit the launch's shared memory
};

// Larger weight -> larger integer; -0 as 0, NaN above all.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if (w != w) return 0xffffffffu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(EV_THREADS, 2) evict_kernel(const __grid_constant__ EvictArgs a) {
  extern __shared__ uint32_t s_key[];
  __shared__ int s_hist[256];
  __shared__ unsigned long long s_w[EV_THREADS / 32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x, ns = gridDim.x;
  const int r = blockIdx.y, b = r / a.NKV, h = r - b * a.NKV;
  pdl_wait();
  pdl_trigger();
  const LongRow row = long_row(a.lengths[b], a.starts ? a.starts[b] : 0, a.S, 0, 0);
  const float* acc = a.acc + b * a.acc_sb + h * a.acc_sh;
  int* kept = a.kept + (long long)r * a.keep;
  const int n = min(row.n, a.keep);
  const int k0 = (int)((long long)n * split / ns), k1 = (int)((long long)n * (split + 1) / ns);   // this CTA's share
  if (split == 0) {
    if (h == 0 && tid == 0) a.lengths_out[b] = n;
    for (int i = n + tid; i < a.keep; i += EV_THREADS) kept[i] = -1;
  }
  if (row.n <= a.keep) {
    for (int i = k0 + tid; i < k1; i += EV_THREADS) kept[i] = row.st + i;
  } else {
    // the first `sinks` and the last `recent` stay; m of the others
    for (int i = k0 + tid; i < k1; i += EV_THREADS) {
      if (i < a.sinks) kept[i] = row.st + i;
      else if (i >= a.keep - a.recent) kept[i] = row.st + row.n - (a.keep - i);
    }
    const int base = row.st + a.sinks, len = row.n - a.sinks - a.recent, m = a.keep - a.sinks - a.recent;
    if (m > 0) {
      const bool staged = len <= a.staged;
      if (staged)
        for (int i = tid; i < len; i += EV_THREADS) s_key[i] = weight_key(acc[base + i]);
      auto key = [&](int i) { return staged ? s_key[i] : weight_key(acc[base + i]); };
      // the m-th largest key, digit by digit from the top
      uint32_t prefix = 0, mask = 0;
      int need = m;
      for (int sh = 24; sh >= 0; sh -= 8) {
        if (tid < 256) s_hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < len; i += EV_THREADS) {
          const uint32_t k = key(i);
          if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> sh) & 255u], 1);
        }
        __syncthreads();
        if (warp == 0) {                     // the digit at which the count from the top reaches `need`
          const int d0 = 255 - 8 * lane;
          int sum = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) sum += s_hist[d0 - j];
          int upto = sum;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(FULL, upto, o);
            if (lane >= o) upto += y;
          }
          int left = need - (upto - sum);
          if (left > 0 && left <= sum) {     // one lane: the total is at least `need`
            int d = d0;
            while (s_hist[d] < left) left -= s_hist[d--];
            s_need = left;
            s_prefix = prefix | ((uint32_t)d << sh);
          }
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;                       // so many of the slots whose key is `prefix` stay: the lowest ones
        mask |= 255u << sh;
      }
      // a run of slots per thread (of odd length: no bank conflicts), its slots above and at the threshold
      const int run = ((len + EV_THREADS - 1) / EV_THREADS) | 1;
      const int i0 = min(len, tid * run), i1 = min(len, i0 + run);
      unsigned long long mine = 0;           // above | at << 32
      for (int i = i0; i < i1; ++i) {
        const uint32_t k = key(i);
        mine += k > prefix ? 1ull : (k == prefix ? 1ull << 32 : 0ull);
      }
      unsigned long long x = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(FULL, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) s_w[warp] = x;
      __syncthreads();
      x -= mine;
      for (int w = 0; w < warp; ++w) x += s_w[w];
      int above = (int)(x & 0xffffffffu), tie = (int)(x >> 32);
      for (int i = i0; i < i1; ++i) {
        const uint32_t k = key(i);
        const bool stays = k > prefix || (k == prefix && tie < need);
        const int at = a.sinks + above + min(tie, need);
        if (stays && at >= k0 && at < k1) kept[at] = base + i;
        above += k > prefix;
        tie += k == prefix;
      }
    }
  }
  __syncthreads();
  // ---- the copy: a warp per EV_ROWS slots; lanes 0-15 keys, 16-31 values, 16 bytes each (4 bits: four lanes, and the
  // scales)
  const bool is_v = lane >= 16;
  const int c = lane & 15;
  const bool on = 16 * c < a.row_bytes;
  const unsigned char* src = (is_v ? a.c.v + b * a.c.v_sb + h * a.c.v_sh : a.c.k + b * a.c.k_sb + h * a.c.k_sh) + 16 * c;
  unsigned char* dst = const_cast<unsigned char*>(is_v ? a.d.v + b * a.d.v_sb + h * a.d.v_sh : a.d.k + b * a.d.k_sb + h * a.d.k_sh) + 16 * c;
  const long long sp = is_v ? a.c.v_sp : a.c.k_sp, dp = is_v ? a.d.v_sp : a.d.k_sp;
  for (int i = k0 + warp * EV_ROWS; i < k1; i += EV_ROWS * (EV_THREADS / 32)) {
    uint4 w[EV_ROWS];
    const int mine = lane < EV_ROWS && i + lane < k1 ? kept[i + lane] : 0;
#pragma unroll
    for (int j = 0; j < EV_ROWS; ++j) {
      const int from = __shfl_sync(FULL, mine, j);
      if (on && i + j < k1) w[j] = ld_nc_v4(src + from * sp);
    }
#pragma unroll
    for (int j = 0; j < EV_ROWS; ++j)
      if (on && i + j < k1) *reinterpret_cast<uint4*>(dst + (i + j) * dp) = w[j];
  }
  if (a.c.ks) {
    for (int i = k0 + (tid >> 1); i < k1; i += EV_THREADS / 2) {
      const int from = kept[i];
      const unsigned char* s = (tid & 1) ? a.c.vs + b * a.c.vs_sb + h * a.c.vs_sh + from * a.c.vs_sp
                                         : a.c.ks + b * a.c.ks_sb + h * a.c.ks_sh + from * a.c.ks_sp;
      unsigned char* d =
          const_cast<unsigned char*>((tid & 1) ? a.d.vs + b * a.d.vs_sb + h * a.d.vs_sh + (long long)i * a.d.vs_sp
                                               : a.d.ks + b * a.d.ks_sb + h * a.d.ks_sh + (long long)i * a.d.ks_sp);
      *reinterpret_cast<uint2*>(d) = *reinterpret_cast<const uint2*>(s);
    }
  }
  if (a.acc_out) {
    float* ao = a.acc_out + b * a.acco_sb + h * a.acco_sh;
    for (int i = k0 + tid; i < k1; i += EV_THREADS) ao[i] = acc[kept[i]];
    if (split == ns - 1)
      for (int i = n + tid; i < a.acc_n; i += EV_THREADS) ao[i] = 0.f;
  }
}

}  // namespace fb

extern "C" int flashb_kv_evict(const fb_kv_cache* cache, const float* acc, int64_t acc_sb, int64_t acc_sh,
                               const int64_t* lengths, const int64_t* starts, int keep, int sinks, int recent,
                               const fb_kv_cache* into, float* acc_out, int64_t acco_sb, int64_t acco_sh, int acc_n,
                               int32_t* kept, int64_t* lengths_out, void* stream) {
  fb::EvictArgs a{};
  int rc = fbh::long_cache(cache, &a.c);
  if (rc) return rc;
  rc = fbh::long_cache(into, &a.d);
  if (rc) return rc;
  FB_CHECK_ARG(acc && lengths && kept && lengths_out, "kv_evict: null pointer argument");
  FB_CHECK_ARG(into->bits == cache->bits && into->B == cache->B && into->NKV == cache->NKV,
               "kv_evict: the two caches differ in bits, rows or heads");
  FB_CHECK_ARG(cache->bits == 16 || (into->k_scale == cache->k_scale && into->v_scale == cache->v_scale),
               "kv_evict: the two caches differ in their tensor scales");
  FB_CHECK_ARG(lengths_out != lengths && lengths_out != starts, "kv_evict: the outputs may not be the inputs");
  FB_CHECK_ARG(keep >= 1 && keep <= into->S && sinks >= 0 && recent >= 0 && (int64_t)sinks + recent <= keep,
               "kv_evict: keep %d of %d slots with %d first and %d last", keep, into->S, sinks, recent);
  FB_CHECK_ARG(!acc_out || acc_n >= keep, "kv_evict: acc_out holds %d slots, %d stay", acc_n, keep);
  FB_CHECK_ARG((int64_t)cache->B * cache->NKV <= 65535, "kv_evict: more than 65535 rows and heads");
  rc = fbh::long_cache_written(into, a.d, "kv_evict");
  if (rc) return rc;
  fbh::LongBox from[4], to[4];
  const int nf = fbh::long_cache_boxes(cache, a.c, from), nt = fbh::long_cache_boxes(into, a.d, to);
  for (int i = 0; i < nf; ++i)
    for (int j = 0; j < nt; ++j)
      FB_CHECK_ARG(!fbh::long_boxes_meet(from[i], to[j]), "kv_evict: the two caches share memory");
  const auto weights = [&](const float* w, int64_t sb, int64_t sh, int n) {
    return fbh::long_box(w, cache->B, cache->NKV, 1, 4 * sb, 4 * sh, 0, 4ll * n);
  };
  FB_CHECK_ARG(!acc_out || !fbh::long_boxes_meet(weights(acc, acc_sb, acc_sh, cache->S), weights(acc_out, acco_sb, acco_sh, acc_n)),
               "kv_evict: acc and acc_out share memory");
  FB_CHECK_ARG(!acc_out || !fbh::long_box_folds(weights(acc_out, acco_sb, acco_sh, acc_n)), "kv_evict: rows of acc_out share memory");
  a.acc = acc, a.acc_sb = acc_sb, a.acc_sh = acc_sh;
  a.lengths = (const long long*)lengths, a.starts = (const long long*)starts;
  a.NKV = cache->NKV, a.S = cache->S, a.keep = keep, a.sinks = sinks, a.recent = recent;
  a.row_bytes = cache->bits == 16 ? 2 * fb::LG_D : fb::LG_D / 2;
  a.kept = kept, a.lengths_out = (long long*)lengths_out;
  a.acc_out = acc_out, a.acco_sb = acco_sb, a.acco_sh = acco_sh, a.acc_n = acc_out ? acc_n : 0;
  a.staged = cache->S < fb::EV_KEYS ? cache->S : fb::EV_KEYS;
  void* args[] = {(void*)&a};
  // two CTAs fit an SM; with fewer rows than that a row is shared, down to some tens of slots a CTA
  const int rows = cache->B * cache->NKV, slots = 2 * fbh::grid_sms();
  int split = slots / rows;
  if (split > (keep + 63) / 64) split = (keep + 63) / 64;
  if (split < 1) split = 1;
  return fbh::launch_pdl((const void*)fb::evict_kernel, dim3(split, rows), dim3(fb::EV_THREADS),
                         sizeof(uint32_t) * a.staged, (cudaStream_t)stream, args, true);
}
