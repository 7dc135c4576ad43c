// flashb: attention of a run of tokens over a long cache with a sliding window and first tokens that stay visible, on
// the 5th-generation tensor cores.
//
// q [B, NH, L, 128] holds the tokens at slots q_start .. q_start + L - 1 of k / v [B, NKV, S, 128].  The token at slot
// p of row b sees slot j when start_b <= j <= p and (j > p - window or j < start_b + sinks);
//   out = softmax(scaling q k^T over those) v in fp32, rounded once; a token without a visible key (p < start_b) gives 0.
//
// A CTA computes 128 rows: the G query heads of a KV head for 128 / G tokens.  Packing the group makes the keys that a
// tile must visit window + 128 / G instead of window + 128, and reads each K and V tile once for the group.  Those keys
// are cut into segments of 32: the sinks that the window of the CTA's first token does not reach, then the slots from
// that window's beginning to the CTA's last token.  Two segments are a tile (the last one may be half a tile, and costs
// as many MMAs); no tile is spent on a handful of sinks alone.
//
// Per tile: S = Q K^T (64 fp32 TMEM columns); warps 0-3 (a thread per row) read their row into registers, which frees S
// for the next tile, subtract the running maximum, take exponentials and write P as bf16 pairs (32 columns, twice); O +=
// P V with P as the MMA's TMEM operand (128 columns); a warp each issues the copies, S and P V.  So S of the next tile
// and P V of the last one run while exponentials are taken, and two CTAs share an SM (96 KB of shared memory, 256 TMEM
// columns each).  The running maximum moves only when a tile's exceeds it by 2^8 (the sums are exact either way), so O is
// hardly ever rescaled.  Masks are applied to the segments that need one for some row of the CTA.
//
// Measured on a B200: 8192 tokens, 16 heads over 4, window 1024: 80 us in a CUDA graph, 808 TFLOP/s, and 90 us a call among
// others (717; clocks fall under the sustained load); windows of 512 and 2048 55 and 123 us, so about 1150 TFLOP/s and 25 us
// that do not grow with the window (beginning and ending 3.5 waves of CTAs).  What bounds it is the chain of one softmax
// warp (wait, TMEM read, maximum, exponentials, TMEM write; about 1700 cycles a tile, two CTAs side by side): with three
// quarters of P V, seven eighths of S, the exponential unit's share or the copies' traffic left out, the time moved by 5%
// at most.  Tried, against 83 us then: P over S's columns with S twice (88 us: S waits for P V),
// two threads per row (93), alternate tiles to two groups of warps (93 to 132), one warp issuing everything (113), CTAs
// that go on to further units (85, and 301 instead of 257 us with a causal mask alone), part of the exponentials as
// polynomials on the FMA pipe (98 to 106), 128-key tiles with S and P V in turn (127).
//
// Rounding: fp32 scores, statistics and sums; P goes to bf16, the type of V's operand, unnormalised: one part, where the
// decode takes two.  Its error against 64 bits (relative, root mean square) is 2.0e-3 to 2.1e-3 at 197 and 8192 tokens where
// fp32 weights have 1.6e-3, the output's own rounding.  A second part would double P V and P's TMEM columns.
//
// A slot that a row does not see gets weight 0, and 0 times an infinity or a NaN in V is NaN.  Slots past the tokens
// read as zeros (the tensor maps end there), sink segments are zeroed past the sinks; what is left are slots that other
// rows of the CTA see.  So a row whose output is not finite is computed again, one visible key at a time
// (a token before its row's start sees none and gives 0).
#include <type_traits>

#include "fb_long.cuh"
#include "fb_tc.cuh"

namespace fb {

constexpr int LP_ROWS = 128;                      // rows of a CTA (TMEM lanes)
constexpr int LP_SEG = 32, LP_TILE = 64;          // keys per segment and tile
constexpr int LP_THREADS = 224;                   // 4 softmax warps; one each for copies, S and P V
constexpr int LP_Q = LP_ROWS * LG_D * 2;          // bytes of the Q tile
constexpr int LP_KV = LP_TILE * LG_D * 2;         // ... of a K or V tile
constexpr int LP_SMEM = LP_Q + 4 * LP_KV + 1024;  // Q, K and V twice, at a 1024-byte boundary
constexpr uint32_t LP_COLS = 256;                 // TMEM: S in columns 0-63, P twice in 64-127, O in 128-255
constexpr float LP_SLACK = 8.f;
// P x 2^-24: the unnormalised sums of 2^16 keys stay in fp32's range for every finite V
constexpr float LP_SHIFT = -24.f;

struct alignas(64) LongPrefillArgs {
  CUtensorMap tq, to, tk, tv, tk32, tv32;         // Q and out tiles; K, V: boxes of 64 and of 32 slots
  const bf16 *q, *k, *v;
  long long q_sb, q_sh, q_sl, k_sb, k_sh, k_sl, v_sb, v_sh, v_sl;
  const long long* starts;
  int B, NH, NKV, G, nq, L, q_start, window, sinks;  // nq = 128 / G tokens a CTA; window 0: none
  float scale;                                    // scaling x log2(e)
  bf16* out;
  long long o_sb, o_sl, o_sh;
  unsigned* err;
};

__device__ __forceinline__ void lp_load(void* dst, const CUtensorMap* m, int c1, int c2, int c3, int c4, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
      "%6}], [%7];" ::"r"(smem_u32(dst)),
      "l"(m), "r"(0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar))
      : "memory");
}
// D (+)= P V: P in TMEM (row = lane, two bf16 per column), V in shared memory with the dims contiguous
__device__ __forceinline__ void lp_mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void lp_ld32(uint32_t taddr, float* f) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r[i]);
}
// 64 consecutive fp32 columns of this thread's TMEM lane.
__device__ __forceinline__ void lp_ld64(uint32_t taddr, float* f) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 64; ++i) f[i] = __uint_as_float(r[i]);
}
// Bits [lo, hi) of 32, whatever the two are.
__device__ __forceinline__ uint32_t lp_bits(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  return lo < hi ? (0xffffffffu >> (32 - hi)) & (0xffffffffu << lo) : 0u;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void lp_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};\n\t"
      "tcgen05.wait::st.sync.aligned;" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}

// One row over its visible keys, one at a time (the case of a non-finite output; see the header): a warp, four dims a
// lane.  d: the row in the output tile (its halves LP_Q / 2 apart), x: the swizzle of its 16-byte units.
__device__ __noinline__ void long_row_again(const LongPrefillArgs& a, int b, int hq, int l, long long start, unsigned char* d,
                                            int x) {
  const int lane = threadIdx.x & 31, p = a.q_start + l, h = hq / a.G;
  const LongRow row = long_row(p + 1, start, p + 1, a.window, a.sinks);
  const bf16* kb = a.k + b * a.k_sb + h * a.k_sh + 4 * lane;
  const bf16* vb = a.v + b * a.v_sb + h * a.v_sh + 4 * lane;
  const uint2 qw = *reinterpret_cast<const uint2*>(a.q + b * a.q_sb + hq * a.q_sh + l * a.q_sl + 4 * lane);
  float m = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = 0; i < row.n; ++i) {
    const long long j = row.slot(i);
    const uint2 kw = *reinterpret_cast<const uint2*>(kb + j * a.k_sl), vw = *reinterpret_cast<const uint2*>(vb + j * a.v_sl);
    const float s = a.scale * warp_sum(lo_f(qw.x) * lo_f(kw.x) + hi_f(qw.x) * hi_f(kw.x) + lo_f(qw.y) * lo_f(kw.y) +
                                       hi_f(qw.y) * hi_f(kw.y));
    const float mn = fmaxf(m, s), f = m > -INFINITY ? ex2(m - mn) : 0.f;
    const float w = mn > -INFINITY ? ex2(s - mn + LP_SHIFT) : (s == -INFINITY ? 0.f : s);
    m = mn;
    sum = sum * f + w;
    o[0] = o[0] * f + w * lo_f(vw.x);
    o[1] = o[1] * f + w * hi_f(vw.x);
    o[2] = o[2] * f + w * lo_f(vw.y);
    o[3] = o[3] * f + w * hi_f(vw.y);
  }
  // scores of -inf alone: 0 / 0, as softmax has it; nothing visible (a padded token that shares its tile with tokens that
  // see the odd value): 0
  const float inv = row.n == 0 ? 0.f : 1.f / sum;
  d += (lane >> 4) * (LP_Q / 2) + ((((lane & 15) >> 1) ^ x) << 4) + (lane & 1) * 8;
  *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
}

// Bounded wait; the clock is read only after a long stretch of polling.
__device__ __forceinline__ bool lp_wait(uint64_t* bar, unsigned parity, unsigned* err) {
#pragma unroll 1
  for (int i = 0; i < 256; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait(bar, parity, err);
}
__device__ __forceinline__ bool lp_wait_warp(uint64_t* bar, unsigned parity, unsigned* err) {
  return __all_sync(FULL, lp_wait(bar, parity, err));
}

__global__ void __launch_bounds__(LP_THREADS, 2) long_prefill_kernel(const __grid_constant__ LongPrefillArgs a) {
  extern __shared__ __align__(16) unsigned char raw[];
  unsigned char* sq = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);   // Q; the output tile at the end
  unsigned char* sk = sq + LP_Q;                                          // [2]
  unsigned char* sv = sk + 2 * LP_KV;                                     // [2]
  __shared__ __align__(8) uint64_t bar_k[2], bar_v[2], bar_s[2], bar_f, bar_p[2], bar_o[2];
  __shared__ uint32_t tslot;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // the latest tokens of every row and head first: they have the most keys, and the short ones end the launch (head after
  // head instead: 83.8 against 81.3 us at the size above, 70.3 against 65.7 at 4 rows of 2048; 16 rows of 8192, whose
  // windows pass the L2, 1305 against 1317)
  const int at = blockIdx.x / (a.B * a.NKV), bh = blockIdx.x - at * (a.B * a.NKV);
  const int b = bh / a.NKV, h = bh - b * a.NKV, q0 = ((a.L - 1) / a.nq - at) * a.nq;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_k[i], 1);
      mbar_init(&bar_v[i], 1);
      mbar_init(&bar_s[i], 1);
      mbar_init(&bar_p[i], LP_ROWS);
      mbar_init(&bar_o[i], 1);
    }
    mbar_init(&bar_f, LP_ROWS);
    fence_mbar_init();
    for (const CUtensorMap* m : {&a.tq, &a.tk, &a.tv, &a.tk32, &a.tv32, &a.to})
      asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tslot)), "r"(LP_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tslot, t_o = tmem + 128;
  pdl_wait();
  pdl_trigger();

  // ---- the CTA's keys: nss segments of sinks from st, then segments from lo to the last token
  const int p_lo = a.q_start + q0, p_hi = a.q_start + min(q0 + a.nq, a.L) - 1;
  const long long start = a.starts ? a.starts[b] : 0;
  const int st = (int)(start < 0 ? 0 : (start > p_hi + 1 ? p_hi + 1 : start));
  const int lo = a.window > 0 && p_lo - a.window + 1 > st ? p_lo - a.window + 1 : st;
  const int ns = min(a.sinks, lo - st), nss = (ns + LP_SEG - 1) / LP_SEG;
  const int segs = nss + (p_hi + 1 - lo + LP_SEG - 1) / LP_SEG;
  const int tiles = (segs + 1) >> 1;
  auto seg_base = [&](int s) { return s < nss ? st + LP_SEG * s : lo + LP_SEG * (s - nss); };

  if (warp == 4) {                                 // copies: one thread
    auto load = [&](bool is_v, int t) {
      const int n = min(2, segs - 2 * t);
      uint64_t* bar = is_v ? &bar_v[t & 1] : &bar_k[t & 1];
      unsigned char* dst = (is_v ? sv : sk) + (t & 1) * LP_KV;
      mbar_arrive_expect_tx(bar, (unsigned)(n * (LP_KV / 2) + (!is_v && t == 0 ? LP_Q : 0)));
      if (n == 2 && 2 * t >= nss) {
        lp_load(dst, is_v ? &a.tv : &a.tk, seg_base(2 * t), 0, h, b, bar);
      } else {
        for (int s = 0; s < n; ++s)
          for (int half = 0; half < 2; ++half)
            lp_load(dst + half * (LP_KV / 2) + s * (LP_KV / 4), is_v ? &a.tv32 : &a.tk32, seg_base(2 * t + s), half, h, b,
                    bar);
      }
    };
    if (lane == 0) {
      // K and V each as soon as their buffer is free (S of t - 2 has read its K, P V of t - 2 its V): waited for in one
      // order, a V that is still in use holds up the next K
      int nk = 0, nv = 0;                          // tiles copied
      uint64_t since = 0;
      while (nk < tiles || nv < tiles) {
        const bool k = nk < tiles && (nk < 2 || mbar_test(&bar_s[nk & 1], ((nk - 2) >> 1) & 1));
        if (k) {
          load(false, nk);
          if (nk == 0) lp_load(sq, &a.tq, q0, h * a.G, 0, b, &bar_k[0]);
          ++nk;
        }
        const bool v = nv < tiles && (nv < 2 || mbar_test(&bar_o[nv & 1], ((nv - 2) >> 1) & 1));
        if (v) load(true, nv++);
        if (k || v) {
          since = 0;
        } else if (since == 0) {
          since = globaltimer();
        } else if (globaltimer() - since > WAIT_LIMIT_NS) {
          set_error(a.err, FB_ERR_TIMEOUT);
          break;
        }
      }
      // no copy may be in flight when the CTA ends (after a wait that gave up: nobody else waits for them)
      for (int t = max(0, nk - 2); t < nk; ++t) lp_wait(&bar_k[t & 1], (t >> 1) & 1, a.err);
      for (int t = max(0, nv - 2); t < nv; ++t) lp_wait(&bar_v[t & 1], (t >> 1) & 1, a.err);
    }
    __syncwarp();
  } else if (warp == 5) {                          // S: one thread
    // descriptors are constants plus compile-time offsets: built in the loop they cost the issuing thread more than
    // twice an MMA's 64 cycles
    const uint64_t dq = tc_desc_sw128(smem_u32(sq)), dk = tc_desc_sw128(smem_u32(sk));
    auto step = [&](auto buf, int t) -> bool {
      constexpr int B = decltype(buf)::value;
      if (!lp_wait(&bar_k[B], (t >> 1) & 1, a.err)) return false;
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
    if (lane == 0)
      for (int t = 0; t < tiles; t += 2)
        if (!step(std::integral_constant<int, 0>(), t) ||
            (t + 1 < tiles && !step(std::integral_constant<int, 1>(), t + 1)))
          break;
    __syncwarp();
  } else if (warp == 6) {                          // P V
    const uint64_t dv = tc_desc(smem_u32(sv), LP_KV / 2, 1024, 2);   // dims contiguous: two halves of 64, 8-key groups
    auto step = [&](auto buf, int t) -> bool {
      constexpr int B = decltype(buf)::value;
      if (!lp_wait_warp(&bar_v[B], (t >> 1) & 1, a.err)) return false;
      if ((ns & 31) && (nss - 1) >> 1 == t) {      // the last sink segment: zero past the sinks
        unsigned char* z = sv + B * LP_KV + ((nss - 1) & 1) * (LP_KV / 4);
        for (int i = (ns & 31) * 8 + lane; i < LP_SEG * 8; i += 32)
          for (int half = 0; half < 2; ++half)
            *reinterpret_cast<uint4*>(z + half * (LP_KV / 2) + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async();
        __syncwarp();
      }
      if (!lp_wait_warp(&bar_p[B], (t >> 1) & 1, a.err)) return false;
      tc_after();
      if (lane == 0) {
        constexpr uint32_t idesc = tc_idesc(LG_D) | (1u << 16);   // V: dims contiguous
        const bool half = segs - 2 * t < 2;
#pragma unroll
        for (int s = 0; s < 4; ++s)
          if (s < 2 || !half)
            lp_mma_ts(t_o, tmem + 64 + 32 * B + 8 * s, dv + ((B * LP_KV + 2048 * s) >> 4), idesc, s > 0 || t > 0);
        tc_commit(&bar_o[B]);
      }
      __syncwarp();
      return true;
    };
    for (int t = 0; t < tiles; t += 2)
      if (!step(std::integral_constant<int, 0>(), t) || (t + 1 < tiles && !step(std::integral_constant<int, 1>(), t + 1)))
        break;
  } else {
    const int r = tid, g = r / a.nq, l = q0 + r - g * a.nq, p = a.q_start + l, hq = h * a.G + g;
    const uint32_t my = (uint32_t)(warp * 32) << 16;
    const int wnd = a.window > 0 ? a.window : 0x40000000;   // none: more than any cache has
    const uint64_t scale2 = f2(a.scale, a.scale);
    float m = -INFINITY;
    uint64_t sum2[2] = {0, 0};
    bool ok = true;
    for (int t = 0; t < tiles; ++t) {
      ok = lp_wait_warp(&bar_s[t & 1], (t >> 1) & 1, a.err);
      if (!ok) break;
      tc_after();
      float s[LP_TILE];
      lp_ld64(tmem + my, s);                       // half a tile: the rest is old scores, past every p and masked below
      tc_before();
      mbar_arrive(&bar_f);
#pragma unroll
      for (int sg = 0; sg < 2; ++sg) {
        const int j0 = seg_base(2 * t + sg);
        const bool sink = 2 * t + sg < nss;
        if (sink || j0 + LP_SEG - 1 > p_lo || p_hi - j0 >= wnd) {
          // the row's keys of the segment as bits: sinks, those of the segment; else slots p - window + 1 .. p and the
          // sinks that the window has reached
          const uint32_t see = p < st ? 0u : sink ? lp_bits(0, st + ns - j0)
                                                  : lp_bits(p - wnd + 1 - j0, p + 1 - j0) | lp_bits(0, min(p + 1, st + a.sinks) - j0);
#pragma unroll
          for (int c = 0; c < LP_SEG; ++c) s[LP_SEG * sg + c] = (see >> c) & 1u ? s[LP_SEG * sg + c] : -INFINITY;
        }
      }
      float x[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int c = 4; c < 64; c += 4) {
        x[(c >> 2) & 3] = max3(x[(c >> 2) & 3], s[c], s[c + 1]);
        x[((c >> 2) + 2) & 3] = max3(x[((c >> 2) + 2) & 3], s[c + 2], s[c + 3]);
      }
      // scale > 0 (checked): the maximum of the scaled scores
      const float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * a.scale;
      const bool up = mx > m + LP_SLACK;
      if (__any_sync(FULL, up)) {
        const float mn = up ? mx : m, f = up ? (m > -INFINITY ? ex2(m - mn) : 0.f) : 1.f;
        m = mn;
        const float2 u = f2_get(f2_add(sum2[0], sum2[1]));
        sum2[0] = f2(u.x * f, u.y * f);
        sum2[1] = 0;
        if (t > 0) {
          ok = lp_wait_warp(&bar_o[(t - 1) & 1], ((t - 1) >> 1) & 1, a.err);
          if (!ok) break;
          tc_after();
#pragma unroll 1
          for (int c = 0; c < LG_D; c += 32) {
            float o[32];
            lp_ld32(t_o + my + c, o);
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(o[i] * f);
            lp_st32(t_o + my + c, w);
          }
        }
      }
      // P's buffer: free once P V of t - 2 is done (asked here, needed after the exponentials)
      const bool free = t < 2 || mbar_test(&bar_o[t & 1], ((t - 2) >> 1) & 1);
      const float off = m > -INFINITY ? LP_SHIFT - m : 0.f;
      const uint64_t off2 = f2(off, off);
      uint32_t w[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        const float2 e = f2_get(f2_fma(f2(s[2 * c], s[2 * c + 1]), scale2, off2));
        const float p0 = ex2(e.x), p1 = ex2(e.y);
        sum2[c & 1] = f2_add(sum2[c & 1], f2(p0, p1));
        w[c] = pack_bf16(p0, p1);
      }
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
    // ---- the row, in the layout of the output's tensor map (128-byte swizzle), over Q
    const float2 u = f2_get(f2_add(sum2[0], sum2[1]));
    const float sum = u.x + u.y, inv = sum == 0.f ? 0.f : 1.f / sum;
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
    const bool bad = !isfinite(sum) || !(od.x + od.y == 0.f) || (sum == 0.f && p >= st);   // the last: -inf scores alone
    // rows that are not finite, again: the warp, a row at a time
    __syncwarp();
    for (unsigned todo = __ballot_sync(FULL, bad && ok && l < a.L); todo; todo &= todo - 1) {
      const int i = warp * 32 + __ffs(todo) - 1, gi = i / a.nq;
      long_row_again(a, b, h * a.G + gi, q0 + i - gi * a.nq, start, sq + i * 128, i & 7);
    }
    fence_proxy_async();
    named_sync(1, LP_ROWS);
    if (tid == 0) {                                // tokens past L are outside the map and not written
      asm volatile("cp.async.bulk.tensor.5d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4, %5}], [%6];" ::"l"(&a.to),
                   "r"(0), "r"(q0), "r"(h * a.G), "r"(0), "r"(b), "r"(smem_u32(sq))
                   : "memory");
      asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");   // shared memory is read
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 4) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(LP_COLS));
  }
}

}  // namespace fb

namespace {
using namespace fb;

// [B][heads][slots][128] as (64 dims, slots, half, heads, B); boxes of `box` slots x both halves, or 32 x one half
int lp_map(CUtensorMap* m, const void* base, long long n, int heads, int B, long long sl, long long sh, long long sb,
           int box) {
  const unsigned long long dims[5] = {64, (unsigned long long)n, 2, (unsigned long long)heads, (unsigned long long)B};
  const unsigned long long st[4] = {(unsigned long long)sl * 2, 128, (unsigned long long)(heads > 1 ? sh : LG_D) * 2,
                                    (unsigned long long)(B > 1 ? sb : LG_D) * 2};
  const unsigned bx[5] = {64, (unsigned)box, box == LP_SEG ? 1u : 2u, 1, 1};
  return fbh::tmap_bf16(m, base, 5, dims, st, bx);
}

// [B][L][heads][128] (any strides) as (64 dims, L, heads, half, B); boxes of nq tokens of G heads
int lp_map_rows(CUtensorMap* m, const void* base, int L, int heads, int B, long long sl, long long sh, long long sb, int nq,
                int G) {
  const unsigned long long dims[5] = {64, (unsigned long long)L, (unsigned long long)heads, 2, (unsigned long long)B};
  const unsigned long long st[4] = {(unsigned long long)(L > 1 ? sl : LG_D) * 2, (unsigned long long)(heads > 1 ? sh : LG_D) * 2,
                                    128, (unsigned long long)(B > 1 ? sb : LG_D) * 2};
  const unsigned bx[5] = {64, (unsigned)nq, (unsigned)G, 2, 1};
  return fbh::tmap_bf16(m, base, 5, dims, st, bx);
}

}  // namespace

extern "C" int flashb_long_prefill(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_sl, const void* k, int64_t k_sb,
                                   int64_t k_sh, int64_t k_sl, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_sl,
                                   int B, int NH, int NKV, int L, int S, int q_start, const int64_t* starts, int window,
                                   int sinks, float scaling, void* out, int64_t o_sb, int64_t o_sl, int64_t o_sh,
                                   void* stream) {
  FB_CHECK_ARG(q && k && v && out, "long_prefill: null pointer argument");
  FB_CHECK_ARG(B >= 1 && L >= 1 && NKV >= 1 && NH >= NKV && NH % NKV == 0, "long_prefill: bad shape B=%d NH=%d NKV=%d L=%d",
               B, NH, NKV, L);
  const int G = NH / NKV;
  if (G != 1 && G != 2 && G != 4 && G != 8) {
    fbh::set_msg("long_prefill: GQA group %d not built (1, 2, 4, 8)", G);
    return FB_ERR_UNSUPPORTED;
  }
  FB_CHECK_ARG(q_start >= 0 && (int64_t)q_start + L <= S, "long_prefill: tokens at slots %d .. of a cache of %d", q_start, S);
  FB_CHECK_ARG(S <= 0x3fffff00, "long_prefill: %d slots", S);
  FB_CHECK_ARG(sinks >= 0, "long_prefill: sinks %d", sinks);
  FB_CHECK_ARG(scaling > 0.f, "long_prefill: scaling must be positive");
  FB_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) == 0 &&
                   (q_sb | q_sh | q_sl | k_sb | k_sh | k_sl | v_sb | v_sh | v_sl | o_sb | o_sl | o_sh) % 8 == 0,
               "long_prefill: tensors must be 16-byte aligned with strides multiple of 8 elements");
  FB_CHECK_ARG(q_sl >= LG_D && k_sl >= LG_D && v_sl >= LG_D, "long_prefill: position strides below the row");
  FB_CHECK_ARG((q_sb | q_sh | k_sb | k_sh | v_sb | v_sh) >= 0 && (B == 1 || (q_sb > 0 && k_sb > 0 && v_sb > 0)) &&
                   (NH == 1 || (q_sh > 0 && o_sh > 0)) && (NKV == 1 || (k_sh > 0 && v_sh > 0)) && (B == 1 || o_sb > 0) &&
                   (L == 1 || o_sl > 0),
               "long_prefill: batch and head strides must be positive");
  FB_CHECK_ARG(!fbh::long_box_folds(fbh::long_box(out, B, NH, L, 2 * o_sb, 2 * o_sh, 2 * o_sl, 2 * LG_D)),
               "long_prefill: rows of out share memory");
  LongPrefillArgs a{};
  const int nq = LP_ROWS / G;
  const int64_t pairs = (int64_t)B * NKV, ctas = pairs <= 0x7fffffff ? (L + nq - 1) / nq * pairs : pairs;
  FB_CHECK_ARG(ctas <= 0x7fffffff, "long_prefill: too many rows, heads and tokens");
  int rc = lp_map_rows(&a.tq, q, L, NH, B, q_sl, q_sh, q_sb, nq, G);
  if (!rc) rc = lp_map_rows(&a.to, out, L, NH, B, o_sl, o_sh, o_sb, nq, G);
  const long long n = (long long)q_start + L;     // later slots read as zeros
  if (!rc) rc = lp_map(&a.tk, k, n, NKV, B, k_sl, k_sh, k_sb, LP_TILE);
  if (!rc) rc = lp_map(&a.tk32, k, n, NKV, B, k_sl, k_sh, k_sb, LP_SEG);
  if (!rc) rc = lp_map(&a.tv, v, n, NKV, B, v_sl, v_sh, v_sb, LP_TILE);
  if (!rc) rc = lp_map(&a.tv32, v, n, NKV, B, v_sl, v_sh, v_sb, LP_SEG);
  if (rc) return rc;
  a.q = (const bf16*)q, a.k = (const bf16*)k, a.v = (const bf16*)v;
  a.q_sb = q_sb, a.q_sh = q_sh, a.q_sl = q_sl, a.k_sb = k_sb, a.k_sh = k_sh, a.k_sl = k_sl;
  a.v_sb = v_sb, a.v_sh = v_sh, a.v_sl = v_sl;
  a.starts = (const long long*)starts;
  a.B = B, a.NH = NH, a.NKV = NKV, a.G = G, a.nq = nq, a.L = L, a.q_start = q_start;
  a.window = window > 0 && window < S ? window : 0;
  a.sinks = sinks < S ? sinks : S;                 // slot + sinks stays an int
  a.scale = scaling * LG_LOG2E, a.out = (bf16*)out, a.o_sb = o_sb, a.o_sl = o_sl, a.o_sh = o_sh;
  a.err = fbh::device_err_ptr();
  static int attr_done[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(long_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LP_SMEM);
    if (e != cudaSuccess) {
      fbh::set_msg("long_prefill: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
      return FB_ERR_CUDA;
    }
    if (dev < 64) attr_done[dev] = 1;
  }
  void* args[] = {(void*)&a};
  return fbh::launch_pdl((const void*)long_prefill_kernel, dim3((unsigned)ctas), dim3(LP_THREADS), LP_SMEM,
                         (cudaStream_t)stream, args, true);
}
