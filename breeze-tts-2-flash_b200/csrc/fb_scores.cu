// flashb: what a model's logits say about given tokens: log probability, entropy, rank, and the likeliest alternatives.
//
// Per row x of logits, z = x / temperature, m = max z, Z = sum exp(z - m):
//   logprob = z_token - m - log Z,  entropy = log Z - sum exp(z - m) (z - m) / Z,
//   rank = how many ids come before the token, top = the first k ids and their log probabilities,
// where ids are ordered by logit, equal ones by id, a NaN first (the greedy sampler's order).
//
// Bound: the row is read once from memory, and an exponential a logit takes three quarters of that time.  A CTA per row,
// units of 32 bytes; a thread keeps, over its units,
//   the sums of e = 2^(x c - R) and of e (x c - R) with c = log2(e) / temperature and a reference R of its own, which moves
//   only when a unit's maximum passes it by 2^16 (the sums are exact either way);
//   the three largest unit maxima, which units hold the first two, and the first one's sums apart from the rest.
// The block's threshold for the alternatives is the least of the warps' k / W-th largest unit maxima (of each thread's first,
// where k / W is small, else of its first two): at least k logits reach it.  Only units that reach it are read again (from
// L1 or L2; mostly one each of some tens of threads), what they hold of it is collected, and each of those finds its place by
// counting the others above it.
// The largest logit's own 1 stays out of the sum (its unit's sum is worked out again without it): what the others add to
// an almost certain token's 1 is not rounded away.
//
// Measured on a B200 (in a CUDA graph): 4095 rows of 32003 in bf16 with 20 alternatives (262 MB) 73 us, 0.55 of the measured
// copy bandwidth; 1088 rows of 2049 in fp32 with 8 (9 MB) 6.6 us; 17 rows 3.9 us.  The first is bound by issue (0.7 of the
// slots; 12.5 instructions a logit in all, 1 of them an exponential).
//
// Rows that the fast path cannot take go through scores_slow, a pass per alternative: a NaN or +inf, -inf alone, a largest
// logit of more than 2^27 temperatures, temperatures past 10^29, more than SC_CAP logits at the threshold (rows of equal
// logits), fewer finite logits than alternatives.
#include <cfloat>
#include <climits>
#include <cmath>

#include "fb_long.cuh"
#include "fb_sample.cuh"

namespace fb {

constexpr int SC_MAX = 512;             // threads of a CTA, at most
constexpr int SC_CAP = 1024;            // logits collected for the alternatives
constexpr int SC_EACH = 16;             // so many of them a lane, at most, where they are thinned out first
// Exponents x c on the fast path.  The largest one of a row is below SC_FAR in size: an exponent less its own rounding (the
// first reference of a unit) is then 2^3 at most, and 2^5 for those that are masked by a finite value.  Threads begin at
// SC_START; what lies below is taken for `low`, whose exponent is SC_START to twice that at every temperature: finite, never
// above a reference, and 0 beside the row's largest.  (A fixed -2^100 for it: products past fp32's range at temperatures
// below 5e-9, exponentials of more than a reference above 1.44, and masked ids of some probability from 10^28 on.)
constexpr float SC_FAR = 0x1p28f, SC_START = -0x1p30f;
constexpr float SC_LN2 = 0.6931471805599453f;

struct ScoresArgs {
  const void* x;
  long long ld;
  int rows, V, top;
  const long long* tokens;
  float inv, c, low;                    // 1 / temperature; that x log2(e); the least logit of the fast path (-inf: none)
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
// (x - m) / temperature, m the row's maximum.  A difference past fp32's range may be within it once divided: from halves.
__device__ __forceinline__ float score_below(float x, float m, float inv) {
  const float d = x - m;
  return d == -INFINITY ? (0.5f * x - 0.5f * m) * inv * 2.f : d * inv;
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
    const float d = score_below(score_at(x, i), m, a.inv), e = i == i0 ? 0.f : __expf(d);
    rest += e;
    if (e > 0.f) dot -= e * d;
  }
  rest = block_reduce(rest, s_f, ScoreAdd());
  dot = block_reduce(dot, s_f, ScoreAdd());
  const float logz = log1pf(rest);
  if (tid == 0) {
    a.logprob[r] = none ? NAN : known ? score_below(xt, m, a.inv) - logz : -INFINITY;
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
      a.top_logprob[(long long)r * a.top + k] = none ? NAN : score_below(score_at(x, id), m, a.inv) - logz;
    }
  }
}

// Logits below `low` (a power of two: exact in bf16), -inf among them, as `low`; a NaN stays.
template <typename T>
__device__ __forceinline__ uint32_t score_clamp(uint32_t w, float low) {
  uint32_t r;
  if constexpr (sizeof(T) == 4) asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(__float_as_uint(low)));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"((__float_as_uint(low) >> 16) * 0x10001u));
  return r;
}

// A unit: 32 bytes of logits.
struct ScoreUnit {
  uint4 w[2];
};
__device__ __forceinline__ uint32_t score_max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ float score_max(const ScoreUnit& u) {
  const uint32_t w[8] = {u.w[0].x, u.w[0].y, u.w[0].z, u.w[0].w, u.w[1].x, u.w[1].y, u.w[1].z, u.w[1].w};
  if constexpr (sizeof(T) == 4) {
    float m = __uint_as_float(w[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, __uint_as_float(w[i]));
    return m;
  } else {
    const uint32_t m = score_max2(score_max2(score_max2(w[0], w[1]), score_max2(w[2], w[3])),
                                  score_max2(score_max2(w[4], w[5]), score_max2(w[6], w[7])));
    return fmaxf(lo_f(m), hi_f(m));
  }
}
// How many of the unit's logits are `th` (a number of the logits' type) or more.
template <typename T>
__device__ __forceinline__ int score_count(const ScoreUnit& u, float th) {
  const uint32_t w[8] = {u.w[0].x, u.w[0].y, u.w[0].z, u.w[0].w, u.w[1].x, u.w[1].y, u.w[1].z, u.w[1].w};
  if constexpr (sizeof(T) == 4) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) n += __uint_as_float(w[i]) >= th;
    return n;
  } else {                                               // ones in bf16, added in pairs (at most 8 each: exact)
    const uint32_t t = (__float_as_uint(th) >> 16) * 0x10001u;
    uint32_t n[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) asm("set.ge.bf16x2.bf16x2 %0, %1, %2;" : "=r"(n[i]) : "r"(w[i]), "r"(t));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < o; ++i) asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(n[i]) : "r"(n[i + o]));
    return (int)(lo_f(n[0]) + hi_f(n[0]));
  }
}

template <typename T>
__global__ void __launch_bounds__(SC_MAX, 2) scores_kernel(const __grid_constant__ ScoresArgs a) {
  constexpr int N = 32 / sizeof(T);                      // logits of a unit
  __shared__ unsigned s_max[SC_MAX / 32], s_thr[SC_MAX / 32];
  __shared__ float s_sum[SC_MAX / 32], s_dot[SC_MAX / 32];
  __shared__ int s_cnt[SC_MAX / 32], s_n, s_kept;
  __shared__ unsigned long long s_key[SC_CAP];
  const int r = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, step = blockDim.x, W = step >> 5;
  if (tid == 0) s_n = 0;
  pdl_wait();
  pdl_trigger();
  const T* x = reinterpret_cast<const T*>(a.x) + (long long)r * a.ld;
  // logits before the first 32-byte boundary and behind the last whole unit: one each for the first threads ("unit -1")
  const int head = min(a.V, (int)(((32u - ((unsigned)(uintptr_t)x & 31u)) & 31u) / sizeof(T)));
  const int nu = (a.V - head) / N, odd = a.V - nu * N;
  const int mine = tid < odd ? (tid < head ? tid : nu * N + tid) : -1;   // the thread's odd logit
  const uint4* body = reinterpret_cast<const uint4*>(x + head);

  const float c = a.c;
  const uint64_t c2 = f2(c, c);
  float R = SC_START, sum = 0.f, dot = 0.f, bs = 0.f, bd = 0.f, tm = -INFINITY, tm2 = -INFINITY, tm3 = -INFINITY;
  int iu = -2, iu2 = -2, cnt = 0;                        // the units that hold tm and tm2 (-2: none)
  // f(pair of logits, the first one's place in the unit)
  auto pairs = [&](const ScoreUnit& u, auto f) {
    const uint32_t w[8] = {u.w[0].x, u.w[0].y, u.w[0].z, u.w[0].w, u.w[1].x, u.w[1].y, u.w[1].z, u.w[1].w};
    if constexpr (N == 16) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f(lo_f(w[i]), hi_f(w[i]), 2 * i);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) f(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]), 2 * i);
    }
  };
  auto clamped = [&](const ScoreUnit& u) {
    ScoreUnit o;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      o.w[i] = make_uint4(score_clamp<T>(u.w[i].x, a.low), score_clamp<T>(u.w[i].y, a.low), score_clamp<T>(u.w[i].z, a.low),
                          score_clamp<T>(u.w[i].w, a.low));
    return o;
  };
  auto whole = [&](int v) { return ScoreUnit{body[2 * v], body[2 * v + 1]}; };
  auto unit = [&](int v) {
    ScoreUnit u;
    if (v >= 0) {
      u = whole(v);
    } else {                                             // the odd logit, and -inf
      const uint32_t none = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u, f = __float_as_uint(score_at(x, mine));
      u.w[0] = u.w[1] = make_uint4(none, none, none, none);
      u.w[0].x = sizeof(T) == 4 ? f : 0xff800000u | f >> 16;
    }
    return u;
  };
  // the next unit is under way while one is worked on; the first before the token, whose logit is a load behind a load
  int v = mine >= 0 ? -1 : tid;
  ScoreUnit next;
  if (v < nu) next = unit(v);
  const long long token = a.tokens[r];
  const bool known = token >= 0 && token < a.V;
  const int tok = known ? (int)token : 0;
  const float xt = known ? score_at(x, tok) + 0.f : INFINITY;
  const float above = known ? ord2f(f2ord(xt) + (sizeof(T) == 4 ? 1u : 0x10000u)) : NAN;   // the type's next number
  auto feed = [&](const ScoreUnit& raw, int v, int base) {
    const float vm = score_max<T>(raw);
    if (vm * c > R + 16.f) {
      const float n = vm * c, g = ex2(R - n), by = R - n;
      dot = g * fmaf(by, sum, dot);
      bd = g * fmaf(by, bs, bd);
      sum *= g;
      bs *= g;
      R = n;
    }
    const uint64_t r2 = f2(-R, -R);
    uint64_t s2 = 0, d2 = 0;
    pairs(clamped(raw), [&](float p, float q, int) {
      const uint64_t y2 = f2_fma(f2(p, q), c2, r2);
      const float2 y = f2_get(y2);
      const uint64_t e = f2(ex2(y.x), ex2(y.y));
      s2 = f2_add(s2, e);
      d2 = f2_fma(e, y2, d2);
    });
    const float2 s = f2_get(s2), d = f2_get(d2);
    const float vs = s.x + s.y, vd = d.x + d.y;
    const bool nb = vm > tm, nb2 = vm > tm2;
    sum += nb ? bs : vs;
    dot += nb ? bd : vd;
    bs = nb ? vs : bs;
    bd = nb ? vd : bd;
    tm3 = fmaxf(tm3, fminf(tm2, vm));
    tm2 = fmaxf(tm2, fminf(tm, vm));
    tm = fmaxf(tm, vm);
    iu2 = nb ? iu : nb2 ? v : iu2;
    iu = nb ? v : iu;
    if (vm >= xt) {
      cnt += score_count<T>(raw, base + N <= tok ? xt : above);
      if (base <= tok && tok < base + N)                 // equal logits of lower ids
        pairs(raw, [&](float p, float q, int i) { cnt += (p == xt && base + i < tok) + (q == xt && base + i + 1 < tok); });
    }
  };
#pragma unroll 1
  while (v < nu) {
    const ScoreUnit u = next;
    const int w = v < 0 ? tid : v + step;
    if (w < nu) next = whole(w);
    feed(u, v, v < 0 ? mine : head + v * N);
    v = w;
  }
  if (mine >= 0 && xt == -INFINITY) cnt -= min(N - 1, max(0, tok - mine - 1));   // what stood beside the odd logit

  // ---- the maximum and the threshold
  const unsigned key = iu == -2 ? 0u : f2ord(tm + 0.f);
  {
    const unsigned top = __reduce_max_sync(FULL, key);
    unsigned k = key, at = top;
    const int kw = (a.top + W - 1) / W;
    if (kw <= 5) {
      for (int i = 1; i < kw && at > 0; ++i) {           // the next largest lane, one lane at a time
        if (lane == __ffs(__ballot_sync(FULL, k == at)) - 1) k = 0;
        at = __reduce_max_sync(FULL, k);
      }
    } else {                                             // the lanes' first and second units sorted, the largest first
      unsigned k2 = f2ord(tm2 + 0.f);
#pragma unroll
      for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int o = size / 2; o > 0; o /= 2) {
          const unsigned y = __shfl_xor_sync(FULL, k, o), y2 = __shfl_xor_sync(FULL, k2, o);
          const bool large = ((lane & o) == 0) == ((lane & size) == 0);
          k = large ? max(k, y) : min(k, y);
          k2 = large ? max(k2, y2) : min(k2, y2);
        }
      k = max(k, __shfl_sync(FULL, k2, 31 - lane));      // the largest 32 of both
#pragma unroll
      for (int o = 16; o > 0; o /= 2) {
        const unsigned y = __shfl_xor_sync(FULL, k, o);
        k = (lane & o) == 0 ? max(k, y) : min(k, y);
      }
      at = __shfl_sync(FULL, k, kw - 1);
    }
    if (lane == 0) {
      s_max[warp] = top;
      s_thr[warp] = at;
    }
  }
  __syncthreads();
  const unsigned wm = lane < W ? s_max[lane] : 0u, M = __reduce_max_sync(FULL, wm);
  const unsigned thr = __reduce_min_sync(FULL, lane < W ? s_thr[lane] : 0xffffffffu);
  const int holder = __ffs(__ballot_sync(FULL, wm == M)) - 1;
  const float xm = ord2f(M), hi = xm * c, lo = fmaf(xm, c, -hi);
  bool fast = M != 0 && a.low > -INFINITY && fabsf(hi) < SC_FAR;
  const bool owner = warp == holder && lane == __ffs(__ballot_sync(FULL, key == M)) - 1;
  if (fast) {
    // ---- the units that reach the threshold, and the largest's without its own 1
    const bool wanted = a.top > 0 && key >= thr && iu != -2;
    if (wanted) {
      // logits that reach the threshold; a unit of -inf alone is not looked at again, so none is collected
      const float low = fmaxf(ord2f(max(thr, 0x007fffffu)), -FLT_MAX);
      auto reach = [&](const ScoreUnit& u) {             // which of them do
        unsigned m = 0;
        pairs(u, [&](float p, float q, int i) { m |= (p >= low ? 1u << i : 0u) | (q >= low ? 2u << i : 0u); });
        return m;
      };
      auto collect = [&](unsigned m, int v1, int v2) {   // of unit v1, and 16 bits up of v2
        int n = atomicAdd(&s_n, __popc(m));
        for (; m; m &= m - 1, ++n) {
          const int i = __ffs(m) - 1, v = i < 16 ? v1 : v2, id = v < 0 ? mine : head + v * N + (i & 15);
          if (n < SC_CAP) s_key[n] = score_key(score_at(x, id), id);
        }
      };
      const bool two = tm2 >= low;
      const ScoreUnit u1 = unit(iu), u2 = unit(two ? iu2 : iu);
      collect(reach(u1) | (two ? reach(u2) << 16 : 0u), iu, iu2);
      if (tm3 >= low) {
        for (int v = mine >= 0 ? -1 : tid; v < nu; v = v < 0 ? tid : v + step) {
          if (v == iu || v == iu2) continue;
          const ScoreUnit u = unit(v);
          if (score_max<T>(u) >= low) collect(reach(u), v, v);
        }
      }
    }
    if (owner) {
      bool skip = true;
      bs = bd = 0.f;
      pairs(clamped(unit(iu)), [&](float p, float q, int) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float f = i ? q : p, y = fmaf(f, c, -R), e = skip && f == xm ? 0.f : ex2(y);
          skip = skip && f != xm;
          bs += e;
          bd = fmaf(e, y, bd);
        }
      });
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
    rest = warp_sum(lane < W ? s_sum[lane] : 0.f);
    ent = warp_sum(lane < W ? s_dot[lane] : 0.f);
    before = __reduce_add_sync(FULL, lane < W ? s_cnt[lane] : 0);
    fast = rest == rest && s_n <= SC_CAP && s_n >= a.top;   // fewer: -inf among the alternatives
  }
  if (!fast) {
    scores_slow<T>(a, r);
    return;
  }
  const float logz = log1pf(rest);
  if (tid == 0) {
    a.logprob[r] = known ? score_below(xt, xm, a.inv) - logz : -INFINITY;
    a.entropy[r] = logz + SC_LN2 * ent / (1.f + rest);
    a.rank[r] = known ? before : a.V;
  }
  int n = s_n;
  // More than two a thread (rows of few units, whose maxima say little): the first warp finds the last logit that counts, by
  // halves of the ordered numbers between, and keeps what reaches it.
  if (n > 2 * step && n <= 32 * SC_EACH) {
    if (warp == 0) {
      unsigned v[SC_EACH];
#pragma unroll
      for (int i = 0; i < SC_EACH; ++i) v[i] = 32 * i + lane < n ? (unsigned)(s_key[32 * i + lane] >> 32) : 0u;
      unsigned low = thr, high = M + 1;                  // as many as wanted reach `low`, fewer `high`
      while (high - low > 1) {
        const unsigned mid = low + (high - low) / 2;
        int c = 0;
#pragma unroll
        for (int i = 0; i < SC_EACH; ++i) c += v[i] >= mid;
        c = __reduce_add_sync(FULL, c);
        if (c >= a.top) low = mid;
        else high = mid;
        if (c == a.top) break;
      }
      int m = 0;
      for (int i = 0; i < n; i += 32) {
        const unsigned long long k = i + lane < n ? s_key[i + lane] : 0ull;
        const unsigned keep = __ballot_sync(FULL, i + lane < n && (unsigned)(k >> 32) >= low);
        __syncwarp();
        if ((keep >> lane) & 1u) s_key[m + __popc(keep & ((1u << lane) - 1))] = k;
        m += __popc(keep);
        __syncwarp();
      }
      if (lane == 0) s_kept = m;                         // not s_n: other warps may still be on their way to this branch
    }
    __syncthreads();
    n = s_kept;
  }
  for (int i = tid; i < n; i += step) {
    const unsigned long long k = s_key[i];
    int at = 0;
    for (int j = 0; j < n; ++j) at += s_key[j] > k;
    if (at < a.top) {
      a.top_id[(long long)r * a.top + at] = (int)(0xffffffffu - (unsigned)k);
      a.top_logprob[(long long)r * a.top + at] = score_below(ord2f((unsigned)(k >> 32)), xm, a.inv) - logz;
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
  int e = 0;
  std::frexp(a.c, &e);                                   // c in [2^(e - 1), 2^e): low c in (2 SC_START, SC_START]
  a.low = std::isfinite(a.c) && 31 - e <= 127 ? -std::ldexp(1.f, 31 - e) : -INFINITY;
  a.logprob = logprob, a.entropy = entropy, a.top_logprob = top_logprob;
  a.rank = (long long*)rank, a.top_id = (long long*)top_id;
  // Threads of a row.  While the rows leave SMs half empty, up to 512, of four units and more (500 rows of 65536 in fp32: 68
  // us with 128, 38 with 256).  Else up to 128 (4095 rows of 32003 in bf16: 88, 73 and 81 us with 64, 128 and 256), of
  // sixteen units and more (12000 rows of 8200 in bf16, 8 alternatives: 63 us with 64, 73 with 128; of 2149 31 with 32, 39
  // with 64), or eight where a warp would have to yield more than 24 alternatives (32 of them, rows of 4100: 59 with 64, 65
  // with 32).
  const int units = V / (is_bf16 ? 16 : 8);
  int threads = 32;
  for (; threads < SC_MAX; threads *= 2) {
    const bool full = (int64_t)rows * threads * 2 > 1024ll * fbh::num_sms();
    if (full && threads == 128) break;
    if (threads * (!full ? 4 : top > threads * 3 / 4 ? 8 : 16) > units) break;
  }
  void* args[] = {(void*)&a};
  return fbh::launch_pdl(is_bf16 ? (const void*)scores_kernel<uint16_t> : (const void*)scores_kernel<float>, dim3(rows),
                         dim3(threads), 0, (cudaStream_t)stream, args, true);
}
