// flashb: what a model's logits say about given tokens: log probability, entropy, rank, and the likeliest alternatives.
//
// Per row x of logits, z = x / temperature, m = max z, Z = sum exp(z - m):
// (without the largest's own 1: log Z = log1p(the others' sum))
//   logprob = z_token - m - log Z,  entropy = log Z - sum exp(z - m) (z - m) / Z,
//   rank = how many ids come before the token, top = the first k ids and their log probabilities,
// where ids are ordered by logit, equal ones by id, a NaN first (the greedy sampler's order).
//
// A CTA per row: the maximum, the sums, then one pass per alternative.
#include <climits>

#include "fb_paged.cuh"
#include "fb_sample.cuh"

namespace fb {

constexpr int SC_THREADS = 256, SC_WARPS = SC_THREADS / 32;

struct ScoresArgs {
  const void* x;
  long long ld;
  int rows, V, top;
  const long long* tokens;
  float inv;                            // 1 / temperature
  float *logprob, *entropy, *top_logprob;
  long long *rank, *top_id;
};

// The order of ids as one number: a larger one comes first.
__device__ __forceinline__ unsigned long long score_key(float x, int id) {
  const unsigned hi = x != x ? 0xffffffffu : f2ord(x + 0.f);       // -0 equals 0
  return ((unsigned long long)hi << 32) | (0xffffffffu - (unsigned)id);
}
template <typename T>
__device__ __forceinline__ float score_at(const T* x, int i) {
  if constexpr (sizeof(T) == 4) return x[i];
  else return __uint_as_float((uint32_t)x[i] << 16);
}
template <typename T, class F>
__device__ __forceinline__ T block_reduce(T v, T* s, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(FULL, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int w = 1; w < SC_WARPS; ++w) v = f(v, s[w]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(SC_THREADS) scores_kernel(const __grid_constant__ ScoresArgs a) {
  __shared__ float s_f[SC_WARPS];
  __shared__ int s_i[SC_WARPS];
  __shared__ unsigned long long s_k[SC_WARPS];
  const int r = blockIdx.x, tid = threadIdx.x;
  pdl_wait();
  pdl_trigger();
  const T* x = reinterpret_cast<const T*>(a.x) + (long long)r * a.ld;
  const auto add = [](auto p, auto q) { return p + q; };
  const auto larger = [](unsigned long long p, unsigned long long q) { return p > q ? p : q; };
  const long long token = a.tokens[r];
  const bool known = token >= 0 && token < a.V;
  const float xt = known ? score_at(x, (int)token) : 0.f;
  const unsigned long long kt = known ? score_key(xt, (int)token) : 0ull;
  unsigned long long first = 0;
  int before = 0;
  for (int i = tid; i < a.V; i += SC_THREADS) {
    const unsigned long long key = score_key(score_at(x, i), i);
    first = larger(first, key);
    before += key > kt;
  }
  first = block_reduce(first, s_k, larger);
  before = block_reduce(before, s_i, add);
  const int i0 = (int)(0xffffffffu - (unsigned)first);
  const float m = score_at(x, i0);
  const bool none = !(fabsf(m) < INFINITY);              // no distribution: a NaN or +inf first, or -inf alone
  // the first id's own 1 stays out of the sum, so that what the others add to an almost certain one is not rounded away
  float rest = 0.f, dot = 0.f;
  for (int i = tid; i < a.V; i += SC_THREADS) {
    const float d = (score_at(x, i) - m) * a.inv, e = i == i0 ? 0.f : __expf(d);
    rest += e;
    if (e > 0.f) dot -= e * d;
  }
  rest = block_reduce(rest, s_f, add);
  dot = block_reduce(dot, s_f, add);
  const float logz = log1pf(rest);
  if (tid == 0) {
    a.logprob[r] = none ? NAN : known ? (xt - m) * a.inv - logz : -INFINITY;
    a.entropy[r] = none ? NAN : logz + dot / (1.f + rest);
    a.rank[r] = before;
  }
  unsigned long long last = ULLONG_MAX;
  for (int k = 0; k < a.top; ++k) {
    unsigned long long best = 0;
    for (int i = tid; i < a.V; i += SC_THREADS) {
      const unsigned long long key = score_key(score_at(x, i), i);
      if (key < last && key > best) best = key;
    }
    last = block_reduce(best, s_k, larger);
    if (tid == 0) {
      const int id = (int)(0xffffffffu - (unsigned)last);
      a.top_id[(long long)r * a.top + k] = id;
      a.top_logprob[(long long)r * a.top + k] = none ? NAN : (score_at(x, id) - m) * a.inv - logz;
    }
  }
}

}  // namespace fb

extern "C" int flashb_token_scores(const void* logits, int is_bf16, int64_t ld, int rows, int V, const int64_t* tokens,
                                   float temperature, int top, float* logprob, float* entropy, int64_t* rank,
                                   int64_t* top_id, float* top_logprob, void* stream) {
  using namespace fb;
  FB_CHECK_ARG(logits && tokens && logprob && entropy && rank && (top == 0 || (top_id && top_logprob)),
               "token_scores: null pointer argument");
  FB_CHECK_ARG(rows >= 1 && V >= 1 && V <= (1 << 24), "token_scores: bad shape rows=%d V=%d", rows, V);
  FB_CHECK_ARG(top >= 0 && top <= 32 && top <= V, "token_scores: %d alternatives of %d ids (0 to 32)", top, V);
  FB_CHECK_ARG(temperature > 0.f && temperature < INFINITY && 1.f / temperature < INFINITY, "token_scores: temperature must be positive and finite");
  FB_CHECK_ARG(ld >= V || rows == 1, "token_scores: row stride %lld below %d", (long long)ld, V);
  FB_CHECK_ARG(((uintptr_t)logits & (is_bf16 ? 1 : 3)) == 0, "token_scores: logits not aligned to their type");
  ScoresArgs a{};
  a.x = logits, a.ld = ld, a.rows = rows, a.V = V, a.top = top, a.tokens = (const long long*)tokens;
  a.inv = 1.f / temperature;
  a.logprob = logprob, a.entropy = entropy, a.top_logprob = top_logprob;
  a.rank = (long long*)rank, a.top_id = (long long*)top_id;
  void* args[] = {(void*)&a};
  return fbh::launch_pdl(is_bf16 ? (const void*)scores_kernel<uint16_t> : (const void*)scores_kernel<float>, dim3(rows),
                         dim3(SC_THREADS), 0, (cudaStream_t)stream, args, true);
}
