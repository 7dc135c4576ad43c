// flashb: what a model's logits say about given tokens: log probability, entropy, rank, and the likeliest alternatives.
//
// Per row x of logits, z = x / temperature, m = max z, Z = sum exp(z - m):
//   logprob = z_token - m - log Z,  entropy = log Z - sum exp(z - m) (z - m) / Z,
//   rank = how many ids come before the token, top = the first k ids and their log probabilities,
// where ids are ordered by logit, equal ones by id, a NaN first (the greedy sampler's order).
//
// Bound: the row is read once from memory.  A CTA per row, 16-byte loads; a thread keeps, over its vectors,
//   the sums of e = 2^(x c - R) and of e (x c - R) with c = log2(e) / temperature and a reference R of its own, which moves
//   only when a vector's maximum passes it by 2^16 (the sums are exact either way);
//   the two largest vector maxima, and which vector holds the largest, whose sums are kept apart.
// The block's threshold for the alternatives is the least of the warps' k / W-th largest thread maxima: at least k logits
// reach it.  Only vectors that reach it are read again (from L1 or L2; mostly one each of some tens of threads), what they
// hold of it is collected, and each of those finds its place by counting the others above it.
// The largest logit's own 1 stays out of the sum (its vector's sum is worked out again without it): what the others add to
// an almost certain token's 1 is not rounded away.
//
// Rows that the fast path cannot take go through scores_slow, a pass per alternative: a NaN or +inf, -inf alone, logits
// past 2^60, more than SC_CAP logits at the threshold (rows of equal logits), fewer finite logits than alternatives.
#include <climits>

#include "fb_long.cuh"
#include "fb_sample.cuh"

namespace fb {

constexpr int SC_MAX = 512;             // threads of a CTA, at most
constexpr int SC_CAP = 1024;            // logits collected for the alternatives
constexpr float SC_LOW = -1e6f;         // 2 to it is 0; what -inf is taken for in e (x c - R)
constexpr float SC_LN2 = 0.6931471805599453f;

struct ScoresArgs {
  const void* x;
  long long ld;
  int rows, V, top;
  const long long* tokens;
  float inv, c;                         // 1 / temperature; that x log2(e)
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
  for (int w = 1; w < (int)blockDim.x / 32; ++w) v = f(v, s[w]);
  return v;
}
struct ScoreKeyMax {
  __device__ unsigned long long operator()(unsigned long long p, unsigned long long q) const { return p > q ? p : q; }
};
struct ScoreAdd {
  template <typename T>
  __device__ T operator()(T p, T q) const { return p + q; }
};

// Any row, by a pass for the maximum, one for the sums and one per alternative.
template <typename T>
__device__ __noinline__ void scores_slow(const ScoresArgs& a, int r) {
  __shared__ float s_f[SC_MAX / 32];
  __shared__ int s_i[SC_MAX / 32];
  __shared__ unsigned long long s_k[SC_MAX / 32];
  const int tid = threadIdx.x, step = blockDim.x;
  const T* x = reinterpret_cast<const T*>(a.x) + (long long)r * a.ld;
  const long long token = a.tokens[r];
  const bool known = token >= 0 && token < a.V;
  const float xt = known ? score_at(x, (int)token) : 0.f;
  const unsigned long long kt = known ? score_key(xt, (int)token) : 0ull;
  unsigned long long first = 0;
  int before = 0;
  for (int i = tid; i < a.V; i += step) {
    const unsigned long long key = score_key(score_at(x, i), i);
    first = key > first ? key : first;
    before += key > kt;
  }
  first = block_reduce(first, s_k, ScoreKeyMax());
  before = block_reduce(before, s_i, ScoreAdd());
  const int i0 = (int)(0xffffffffu - (unsigned)first);
  const float m = score_at(x, i0);
  const bool none = !(fabsf(m) < INFINITY);              // no distribution: a NaN or +inf first, or -inf alone
  float rest = 0.f, dot = 0.f;
  for (int i = tid; i < a.V; i += step) {
    const float d = (score_at(x, i) - m) * a.inv, e = i == i0 ? 0.f : __expf(d);
    rest += e;
    if (e > 0.f) dot -= e * d;
  }
  rest = block_reduce(rest, s_f, ScoreAdd());
  dot = block_reduce(dot, s_f, ScoreAdd());
  const float logz = log1pf(rest);
  if (tid == 0) {
    a.logprob[r] = none ? NAN : known ? (xt - m) * a.inv - logz : -INFINITY;
    a.entropy[r] = none ? NAN : logz + dot / (1.f + rest);
    a.rank[r] = before;
  }
  unsigned long long last = ULLONG_MAX;
  for (int k = 0; k < a.top; ++k) {
    unsigned long long best = 0;
    for (int i = tid; i < a.V; i += step) {
      const unsigned long long key = score_key(score_at(x, i), i);
      if (key < last && key > best) best = key;
    }
    last = block_reduce(best, s_k, ScoreKeyMax());
    if (tid == 0) {
      const int id = (int)(0xffffffffu - (unsigned)last);
      a.top_id[(long long)r * a.top + k] = id;
      a.top_logprob[(long long)r * a.top + k] = none ? NAN : (score_at(x, id) - m) * a.inv - logz;
    }
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {       // a NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
__global__ void __launch_bounds__(SC_MAX, 2) scores_kernel(const __grid_constant__ ScoresArgs a) {
  constexpr int N = 16 / sizeof(T);                      // logits of a vector
  constexpr int UNROLL = 4;
  __shared__ unsigned s_max[SC_MAX / 32], s_thr[SC_MAX / 32];
  __shared__ float s_sum[SC_MAX / 32], s_dot[SC_MAX / 32];
  __shared__ int s_cnt[SC_MAX / 32], s_n;
  __shared__ unsigned long long s_key[SC_CAP];
  const int r = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, step = blockDim.x, W = step >> 5;
  if (tid == 0) s_n = 0;
  pdl_wait();
  pdl_trigger();
  const T* x = reinterpret_cast<const T*>(a.x) + (long long)r * a.ld;
  const long long token = a.tokens[r];
  const bool known = token >= 0 && token < a.V;
  const float xt = known ? score_at(x, (int)token) : INFINITY;
  // logits before the first 16-byte boundary and behind the last whole vector: one each for the first threads ("vector -1")
  const int head = min(a.V, (int)(((16u - ((unsigned)(uintptr_t)x & 15u)) & 15u) / sizeof(T)));
  const int nv = (a.V - head) / N, odd = a.V - nv * N;
  const int mine = tid < odd ? (tid < head ? tid : nv * N + tid) : -1;   // the thread's odd logit
  const T* body = x + head;

  const float c = a.c;
  float R = -0x1p100f, sum = 0.f, dot = 0.f, bs = 0.f, bd = 0.f, tm = -INFINITY, tm2 = -INFINITY;
  int iv = -2, cnt = 0;                                  // iv: the vector that holds tm (-2: none)
  auto unpack = [&](const uint4& w, float (&f)[N]) {
    if constexpr (N == 8) {
      cvt8(w, f);
    } else {
      f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
    }
  };
  // e and e y of one logit
  auto term = [&](float v, float& s, float& d) {
    const float y = max_nan(fmaf(v, c, -R), SC_LOW), e = ex2(y);
    s += e;
    d = fmaf(e, y, d);
  };
  auto feed = [&](const float (&f)[N], int v, int base) {
    float vm = fmaxf(f[0], f[1]);
#pragma unroll
    for (int i = 2; i < N; ++i) vm = fmaxf(vm, f[i]);
    if (vm * c > R + 16.f) {
      const float n = vm * c, g = ex2(R - n), by = R - n;
      dot = g * fmaf(by, sum, dot);
      bd = g * fmaf(by, bs, bd);
      sum *= g;
      bs *= g;
      R = n;
    }
    const uint64_t c2 = f2(c, c), r2 = f2(-R, -R);
    uint64_t s2 = 0, d2 = 0;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 y = f2_get(f2_fma(f2(f[i], f[i + 1]), c2, r2));
      const float y0 = max_nan(y.x, SC_LOW), y1 = max_nan(y.y, SC_LOW);
      const uint64_t e = f2(ex2(y0), ex2(y1));
      s2 = f2_add(s2, e);
      d2 = f2_fma(e, f2(y0, y1), d2);
    }
    const float2 s = f2_get(s2), d = f2_get(d2);
    const float vs = s.x + s.y, vd = d.x + d.y;
    const bool nb = vm > tm;
    sum += nb ? bs : vs;
    dot += nb ? bd : vd;
    bs = nb ? vs : bs;
    bd = nb ? vd : bd;
    tm2 = nb ? tm : fmaxf(tm2, vm);
    tm = fmaxf(tm, vm);
    iv = nb ? v : iv;
    if (vm >= xt) {
#pragma unroll
      for (int i = 0; i < N; ++i) cnt += f[i] > xt || (f[i] == xt && base + i < token);
    }
  };
  const uint4* vec = reinterpret_cast<const uint4*>(body);
  for (int v0 = tid; v0 < nv; v0 += UNROLL * step) {
    uint4 w[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (v0 + u * step < nv) w[u] = vec[v0 + u * step];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (v0 + u * step < nv) {
        float f[N];
        unpack(w[u], f);
        feed(f, v0 + u * step, head + (v0 + u * step) * N);
      }
  }
  if (mine >= 0) {
    float f[N];
    f[0] = score_at(x, mine);
#pragma unroll
    for (int i = 1; i < N; ++i) f[i] = -INFINITY;
    feed(f, -1, mine);
  }

  // ---- the maximum and the threshold
  const unsigned key = iv == -2 ? 0u : f2ord(tm + 0.f);
  {
    const unsigned top = __reduce_max_sync(FULL, key);
    unsigned k = key, at = top;
    const int kw = (a.top + W - 1) / W;
    for (int i = 1; i < kw && at > 0; ++i) {             // the next largest lane, one lane at a time
      if (lane == __ffs(__ballot_sync(FULL, k == at)) - 1) k = 0;
      at = __reduce_max_sync(FULL, k);
    }
    if (lane == 0) {
      s_max[warp] = top;
      s_thr[warp] = at;
    }
  }
  __syncthreads();
  unsigned M = 0, thr = 0xffffffffu;
  int holder = 0;
  for (int w = 0; w < W; ++w) {
    if (s_max[w] > M) M = s_max[w], holder = w;
    thr = min(thr, s_thr[w]);
  }
  const float xm = ord2f(M), hi = xm * c, lo = fmaf(xm, c, -hi);
  bool fast = M != 0 && fabsf(hi) < 0x1p60f;
  const bool owner = warp == holder && lane == __ffs(__ballot_sync(FULL, key == M)) - 1;
  if (fast) {
    // ---- the vectors that reach the threshold, and the largest's without its own 1
    if ((a.top > 0 && key >= thr && iv != -2) || owner) {
      bool skip = owner;
      auto collect = [&](float v, int id) {
        const unsigned k = f2ord(v + 0.f);
        if (a.top > 0 && k >= thr && v > -INFINITY) {     // a vector of -inf alone is not looked at again, so none is collected
          const int n = atomicAdd(&s_n, 1);
          if (n < SC_CAP) s_key[n] = ((unsigned long long)k << 32) | (0xffffffffu - (unsigned)id);
        }
      };
      if (owner) bs = bd = 0.f;
      auto again = [&](int v) {                          // the largest's vector
        if (v == -1) {
          const float f = score_at(x, mine);
          collect(f, mine);
        } else {
          float f[N];
          unpack(vec[v], f);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            collect(f[i], head + v * N + i);
            if (owner) {
              if (skip && f[i] == xm) skip = false;
              else term(f[i], bs, bd);
            }
          }
        }
      };
      again(iv);
      if (a.top > 0 && iv != -2 && tm2 > -INFINITY && f2ord(tm2 + 0.f) >= thr) {
        for (int v = tid; v < nv; v += step)
          if (v != iv) {
            float f[N];
            unpack(vec[v], f);
#pragma unroll
            for (int i = 0; i < N; ++i) collect(f[i], head + v * N + i);
          }
        if (mine >= 0 && iv != -1) collect(score_at(x, mine), mine);
      }
    }
    const float by = (hi - R) + lo, g = ex2(-by), all = sum + bs;
    float rest = g * all, ent = g * fmaf(by, all, -(dot + bd));
    rest = warp_sum(rest);
    ent = warp_sum(ent);
    cnt = __reduce_add_sync(FULL, cnt);
    if (lane == 0) {
      s_sum[warp] = rest;
      s_dot[warp] = ent;
      s_cnt[warp] = cnt;
    }
  }
  __syncthreads();
  float rest = 0.f, ent = 0.f;
  int before = 0;
  if (fast) {
    for (int w = 0; w < W; ++w) {
      rest += s_sum[w];
      ent += s_dot[w];
      before += s_cnt[w];
    }
    fast = rest == rest && s_n <= SC_CAP && s_n >= a.top;   // fewer: -inf among the alternatives
  }
  if (!fast) {
    scores_slow<T>(a, r);
    return;
  }
  const float logz = log1pf(rest);
  if (tid == 0) {
    a.logprob[r] = known ? (xt - xm) * a.inv - logz : -INFINITY;
    a.entropy[r] = logz + SC_LN2 * ent / (1.f + rest);
    a.rank[r] = known ? before : a.V;
  }
  const int n = s_n;
  for (int i = tid; i < n; i += step) {
    const unsigned long long k = s_key[i];
    int at = 0;
    for (int j = 0; j < n; ++j) at += s_key[j] > k;
    if (at < a.top) {
      a.top_id[(long long)r * a.top + at] = (int)(0xffffffffu - (unsigned)k);
      a.top_logprob[(long long)r * a.top + at] = (ord2f((unsigned)(k >> 32)) - xm) * a.inv - logz;
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
  a.inv = 1.f / temperature, a.c = a.inv * LG_LOG2E;
  a.logprob = logprob, a.entropy = entropy, a.top_logprob = top_logprob;
  a.rank = (long long*)rank, a.top_id = (long long*)top_id;
  // two vectors a thread or more, up to the CTA's limit
  const int vectors = V / (is_bf16 ? 8 : 4);
  int threads = 32;
  while (threads < SC_MAX && threads * 4 <= vectors) threads *= 2;
  void* args[] = {(void*)&a};
  return fbh::launch_pdl(is_bf16 ? (const void*)scores_kernel<uint16_t> : (const void*)scores_kernel<float>, dim3(rows),
                         dim3(threads), 0, (cudaStream_t)stream, args, true);
}
