// flashb: eviction from a KV cache by accumulated attention weight.
//
// Row b holds keys in slots [st, len).  With at most `keep` of them everything stays; else the first `sinks`, the
// last `recent` and, of the others, the keep - sinks - recent slots of largest accumulated weight (equal weights: the
// lower slot; NaN above everything) stay.  Each KV head chooses for itself.  What stays moves, in slot order, to
// slots 0, 1, .. of another cache, its weight with it; kept[i] is the slot it came from.
//
// Two launches.  evict_select_kernel (a CTA per row and KV head) finds the weight of the last slot that stays by
// radix selection (8 bits a pass over order-preserving integer keys) and writes the kept slots by a running count in
// slot order.  evict_move_kernel copies them.  Bound: HBM, the kept rows read and written once (1 KB a slot in bf16).
#include "fb_long.cuh"

namespace fb {

constexpr int EV_THREADS = 1024;

struct EvictArgs {
  LongCache c, d;
  const float* acc;
  long long acc_sb, acc_sh;
  const long long *lengths, *starts;
  int NKV, S, dS, keep, sinks, recent, row_bytes;
  int* kept;                       // [B, NKV, keep]
  long long* lengths_out;          // [B]
  float* acc_out;
  long long acco_sb, acco_sh;
  int acc_n;                       // slots of acc_out
};

// Larger weight -> larger integer; -0 as 0, NaN above all.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if (w != w) return 0xffffffffu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(EV_THREADS) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  __shared__ int s_hist[256];
  __shared__ int s_w[EV_THREADS / 32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = blockIdx.x, b = r / a.NKV, h = r - b * a.NKV;
  pdl_wait();
  pdl_trigger();
  const LongRow row = long_row(a.lengths[b], a.starts ? a.starts[b] : 0, a.S, 0, 0);
  const float* acc = a.acc + b * a.acc_sb + h * a.acc_sh + row.st;
  int* kept = a.kept + (long long)r * a.keep;
  const int n = min(row.n, a.keep);
  if (h == 0 && tid == 0) a.lengths_out[b] = n;
  for (int i = n + tid; i < a.keep; i += EV_THREADS) kept[i] = -1;
  if (row.n <= a.keep) {
    for (int i = tid; i < n; i += EV_THREADS) kept[i] = row.st + i;
    return;
  }
  const int lo = a.sinks, hi = row.n - a.recent, m = a.keep - a.sinks - a.recent;   // choose m of [lo, hi)
  // the m-th largest key of [lo, hi): digit by digit from the top
  uint32_t prefix = 0, mask = 0;
  int need = m;
  if (m > 0) {
    for (int sh = 24; sh >= 0; sh -= 8) {
      if (tid < 256) s_hist[tid] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += EV_THREADS) {
        const uint32_t k = weight_key(acc[i]);
        if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> sh) & 255u], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int left = need, d = 255;
        while (d > 0 && s_hist[d] < left) left -= s_hist[d--];
        s_need = left;
        s_prefix = prefix | ((uint32_t)d << sh);
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;                 // so many of the slots whose key is `prefix` stay: the lowest ones
      mask |= 255u << sh;
      __syncthreads();
    }
  }
  // in slot order: every slot above the threshold and the first `need` at it
  int done = 0, ties = 0;
  for (int i0 = 0; i0 < row.n; i0 += EV_THREADS) {
    const int i = i0 + tid;
    int above = 0, tie = 0;
    if (i < row.n) {
      if (i < lo || i >= hi) above = 1;
      else if (m > 0) {
        const uint32_t k = weight_key(acc[i]);
        above = k > prefix;
        tie = k == prefix;
      }
    }
    // running counts of both, packed
    int x = above | (tie << 16);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(FULL, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_w[warp] = x;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < EV_THREADS / 32; ++w) {
      if (w < warp) before += s_w[w];
      all += s_w[w];
    }
    __syncthreads();
    const int tr = ties + ((before + x) >> 16) - tie;                       // ties below this slot
    const int ar = done + ((before + x) & 0xffff) - above;                  // forced or above, below this slot
    const bool stays = above || (tie && tr < need);
    if (stays) kept[ar + min(tr, need)] = row.st + i;
    done += all & 0xffff;
    ties += all >> 16;
  }
}

// A warp per kept slot: lanes 0-15 keys, 16-31 values (bf16: 16 bytes a lane); 4 bits: 16 bytes a lane of four, and
// the scales
__global__ void __launch_bounds__(256) evict_move_kernel(const __grid_constant__ EvictArgs a) {
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.y, b = r / a.NKV, h = r - b * a.NKV;
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
  pdl_wait();
  pdl_trigger();
  if (i >= max(a.keep, a.acc_n)) return;
  const int from = i < a.keep ? a.kept[(long long)r * a.keep + i] : -1;
  if (lane == 0 && a.acc_out && i < a.acc_n)
    a.acc_out[b * a.acco_sb + h * a.acco_sh + i] = from >= 0 ? a.acc[b * a.acc_sb + h * a.acc_sh + from] : 0.f;
  if (from < 0) return;
  const bool is_v = lane >= 16;
  const int c = lane & 15;
  const unsigned char* s = is_v ? a.c.v + b * a.c.v_sb + h * a.c.v_sh + from * a.c.v_sp
                                : a.c.k + b * a.c.k_sb + h * a.c.k_sh + from * a.c.k_sp;
  unsigned char* d = const_cast<unsigned char*>(is_v ? a.d.v + b * a.d.v_sb + h * a.d.v_sh + (long long)i * a.d.v_sp
                                                     : a.d.k + b * a.d.k_sb + h * a.d.k_sh + (long long)i * a.d.k_sp);
  if (16 * c < a.row_bytes) *reinterpret_cast<uint4*>(d + 16 * c) = ld_nc_v4(s + 16 * c);
  if (a.c.ks && c == 0) {
    const unsigned char* ss = is_v ? a.c.vs + b * a.c.vs_sb + h * a.c.vs_sh + from * a.c.vs_sp
                                   : a.c.ks + b * a.c.ks_sb + h * a.c.ks_sh + from * a.c.ks_sp;
    unsigned char* ds =
        const_cast<unsigned char*>(is_v ? a.d.vs + b * a.d.vs_sb + h * a.d.vs_sh + (long long)i * a.d.vs_sp
                                        : a.d.ks + b * a.d.ks_sb + h * a.d.ks_sh + (long long)i * a.d.ks_sp);
    *reinterpret_cast<uint2*>(ds) = *reinterpret_cast<const uint2*>(ss);
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
  FB_CHECK_ARG(into->k != cache->k && into->v != cache->v, "kv_evict: the cache cannot be evicted into itself");
  FB_CHECK_ARG(keep >= 1 && keep <= into->S && sinks >= 0 && recent >= 0 && (int64_t)sinks + recent <= keep,
               "kv_evict: keep %d of %d slots with %d first and %d last", keep, into->S, sinks, recent);
  FB_CHECK_ARG(!acc_out || acc_n >= keep, "kv_evict: acc_out holds %d slots, %d stay", acc_n, keep);
  FB_CHECK_ARG((int64_t)cache->B * cache->NKV <= 65535, "kv_evict: more than 65535 rows and heads");
  a.acc = acc, a.acc_sb = acc_sb, a.acc_sh = acc_sh;
  a.lengths = (const long long*)lengths, a.starts = (const long long*)starts;
  a.NKV = cache->NKV, a.S = cache->S, a.dS = into->S, a.keep = keep, a.sinks = sinks, a.recent = recent;
  a.row_bytes = cache->bits == 16 ? 2 * fb::LG_D : fb::LG_D / 2;
  a.kept = kept, a.lengths_out = (long long*)lengths_out;
  a.acc_out = acc_out, a.acco_sb = acco_sb, a.acco_sh = acco_sh, a.acc_n = acc_out ? acc_n : 0;
  void* args[] = {(void*)&a};
  const int rows = cache->B * cache->NKV;
  rc = fbh::launch_pdl((const void*)fb::evict_select_kernel, dim3(rows), dim3(fb::EV_THREADS), 0, (cudaStream_t)stream,
                       args, true);
  if (rc) return rc;
  const int n = keep > a.acc_n ? keep : a.acc_n;
  return fbh::launch_pdl((const void*)fb::evict_move_kernel, dim3((n + 7) / 8, rows), dim3(256), 0,
                         (cudaStream_t)stream, args, true);
}
