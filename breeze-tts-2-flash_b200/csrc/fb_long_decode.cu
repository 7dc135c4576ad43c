// flashb: single-token attention over a long cache, with a sliding window and first tokens that stay visible
// ("sinks"), over bf16 or 4-bit keys and values, optionally adding each slot's attention weight to an accumulator.
//
//   s_j = scaling (q . k_j),  p = softmax(s) over the visible slots,  out = sum_j p_j v_j        (0 without any)
//   acc_out[j] = decay acc[j] + sum over the q heads of the group of p_j   (every slot; p_j = 0 where not visible)
//
// Measured on a B200 (in a CUDA graph): 128 rows of 4 KV heads over a window of 2048 (404 MB) 66 us, 0.94 of the measured
// copy bandwidth; 64 ragged rows of up to 8192 slots in 4 bits (152 MB) 36 to 38 us, 0.60 to 0.64; weights wanted, up to
// 4096 slots (277 MB), 51 to 54 us, 0.80; one stream over some hundred keys 5 to 8 us.  K and V through rings of cp.async in
// shared memory instead of straight to registers took 85 us at the first of these.
//
// Bound: the visible K and V are read once (512 bytes a key and KV head in bf16, 144 in 4 bits) and do 2 G flops per
// value, so HBM bounds bf16; below some megabytes the launch and one memory round trip do.  In 4 bits nothing is saturated:
// DRAM at 46% of its nominal rate, issue slots at 54%, the ALU pipe at 46%.  A warp runs 590 instructions on 32 keys, waits
// for its own loads 38% of the time (128 registers a thread leave no room for the next tile's) and shares its scheduler
// with three others; a sixth of the (profiled) launch is its beginning and end.
//
// Few short rows: long_cluster_kernel, one launch (below).  Else two launches.  long_decode_kernel: the visible keys of
// every (row, KV head), in chunks, form one list; CTA c of N takes the c-th N-th of it whatever the rows' lengths are, so
// ragged batches leave no CTA idle.  A CTA's share is one or more pieces (a contiguous run of one row's keys); each leaves
// (max, sum, unnormalised out) in a slot of the workspace.  long_merge_kernel joins a row's pieces in a fixed order (no
// atomics: the same inputs give the same bits) and, when weights are wanted, turns the scores that the first kernel left
// in the workspace into weights.
//
// In a piece each of the 4 warps takes tiles of 16 keys (4-bit: 32) on its own, straight from global memory into the
// fragments of mma.m16n8k16 (no shared memory, no barrier until the piece ends):
//   S^T[keys x heads] = K Q^T : a lane's 16-byte loads hold 8 dims of a key; the contraction takes dims in that order
//     for K and q alike, so no shuffle is needed
//   O^T[dims x heads] += V^T P^T : a lane loads 16 dims of 4 keys and pairs neighbouring keys by byte permutes; P^T
//     comes from S^T by movmatrix.
// fp32 scores, statistics and sums.  The tensor cores take P in the type of V's operand.  fp16 for the 4-bit cache
// (its values are exact in fp16): 11 bits, below the bf16 output's 8.  For a bf16 cache P is the sum of two bf16
// values, 16 bits: with G <= 4 the eight columns of the product hold each head twice (q is loaded so), the upper four
// take the second part, and a shuffle at the piece's end adds them -- no instruction more on the tensor cores; with
// G = 8 the second part is a second product.  One bf16 part alone measured 1.3 times the error of fp32 weights.
// The maximum moves only when a tile's exceeds it by 2^8: the sums are exact either way, and the 32 accumulators are
// rescaled a few times a piece instead of every tile, and the lanes that share a head compare maxima only then (with the
// scale and the subtraction in one multiply-add, two scores an instruction: 40.4 to 39.3 us at the 4-bit case above).
//
// PAGED: slot j of a row lies in page table[j >> shift] of a pool.  A warp's tile of 16 keys is in one page (pages have 16
// slots at least, and a window's numbering begins at a multiple of 16), whose entry is read a tile ahead; a tile whose entry is
// no page is left out.  128 ragged rows of up
// to 8192 slots (1.07 GB) 179 us in a CUDA graph and 166 a call among others, 0.92 to 0.98 of the measured copy bandwidth, in
// pages of 16 as of 64, in order or not; over a window of 2048 (484 MB) 80 to 82 us; 2 rows of 2049 slots 7.7 us, in a table
// of 16384, by whose width the form is chosen, 10.3.
#include <cooperative_groups.h>

#include <cfloat>
#include <cmath>
#include <type_traits>

#include "fb_paged.cuh"

namespace cg = cooperative_groups;

namespace fb {

constexpr int LD_WARPS = 4;
constexpr int LD_THREADS = 32 * LD_WARPS;
constexpr int LM_THREADS = 128;         // the merge
constexpr int LC_MAX = 16;              // CTAs of a cluster
constexpr int LC_CHUNKS = 8;            // chunks a cluster's CTA may have (4 when the cluster is not a full one)
constexpr int LD_SLICE = 512;           // slots per accumulator CTA of the merge

struct LongDecodeArgs {
  LongCache c;
  const bf16* q;
  long long q_sb, q_sh;
  const long long *lengths, *starts;
  int B, NH, NKV, G, S, window, sinks;
  int ncta, per, slices;                // CTAs, batch rows per lane of the plan, accumulator CTAs per row
  int dense;                            // position strides are the row's own bytes
  float scale;                          // |scaling| x log2(e) (x the cache's key scale), > 0
  uint32_t flip;                        // sign bits of a pair of q's values, when scaling is negative
  float v_scale;
  const float* acc;
  float* acc_out;
  float decay, shift;                   // shift: LongTile's SHIFT
  long long acc_sb, acc_sh, acco_sb, acco_sh;
  float* po;                            // pieces: unnormalised out [slot][G][128],
  float2* ml;                           //   maximum and sum [slot][G]
  int2* own;                            // [row] first and last CTA with a piece of it
  float* sc;                            // scores [row][cap][G] in log2 units (weights wanted), else null
  int cap;                              // visible keys a row can have
  bf16* out;
  PagedTable t;                         // a paged cache: c.k_sb and c.v_sb are the pages' strides
};

// Paged: the visible keys' numbering begins at a multiple of 16 slots (sinks end at one), so that a warp's tile of 16 lies
// in one page; what it holds beside visible keys gets no weight.
struct LongPagedRow : LongRow {
  int vlo, vns;                         // visible: slots below vns, and from vlo on
  __device__ __forceinline__ bool sees(int j) const { return (j >= vlo || j < vns) && index(j) >= 0; }
};
template <bool PAGED>
using LongRowOf = std::conditional_t<PAGED, LongPagedRow, LongRow>;

template <int BITS>
struct LongTile {
  // per SM: 168 registers a thread, and 128 (64 ragged rows of up to 8192 slots: 44.2 us with three, 41.9 with four; later
  // 38.9 with four and 46.2 with five, whose 96 registers spill)
  static constexpr int CTAS = BITS == 16 ? 3 : 4;
  static constexpr int KEYS = BITS == 16 ? 16 : 32;      // keys per warp and step
  static constexpr int CHUNK = KEYS * LD_WARPS;
  static constexpr int EXTRA = 1;                        // empty chunks before a row's own (see LongPlace)
  // P x 2^SHIFT.  fp16: 2^6, with the 2^8 of slack below its 65504.  bf16: 2^-24, so that the unnormalised sums of 2^16 keys
  // stay in fp32's range for every finite V (from 0 on they left it past 1e34); what falls below the range instead is 2^-125
  // of the output at most, a bf16 step at its smallest normal values.
  static constexpr float SHIFT = BITS == 16 ? -24.f : 6.f;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// One half twice, from its 16-bit register: the multiply takes it as it is (a byte permute first: 39.3 instead of 38.9 us).
__device__ __forceinline__ uint32_t both_lo(uint32_t x) {
  uint32_t r;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tmov.b32 %0, {a, a};\n\t}" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t both_hi(uint32_t x) {
  uint32_t r;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tmov.b32 %0, {b, b};\n\t}" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint2 ld_nc_v2(const void* p) {
  uint2 r;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}

// The list of chunks: row b's NKV heads in turn, ceil(visible / chunk) chunks each after EXTRA empty ones.  Beginning a
// row costs a CTA some microseconds (q, the first loads, its part of the output), and the empty chunks stand for that:
// with ragged rows the CTAs of many short ones came out last by a quarter of the time without them (the 4-bit case above,
// one to four of them: 38.4, 38.7, 39.2, 40.1 us).  Every warp works the
// list out for itself (no barrier): lane i counts the chunks of rows [i per, i per + per).
template <bool PAGED>
struct LongPlace {
  int b, before;                        // batch row, chunks of one KV head of all rows before it
  LongRowOf<PAGED> row;
};
template <bool PAGED>
__device__ __forceinline__ LongRowOf<PAGED> long_row_of(const LongDecodeArgs& a, int b) {
  if constexpr (PAGED) {
    LongPagedRow r;
    const LongRow x = long_row(a.lengths[b], 0, a.S, a.window, a.sinks);
    const int lo = x.lo & ~15, ns = (x.ns + 15) & ~15, end = x.lo + x.n - x.ns;
    r.st = 0, r.vlo = x.lo, r.vns = x.ns;
    r.ns = ns < lo ? ns : 0;
    r.lo = ns < lo ? lo : 0;
    r.n = r.ns + end - r.lo;
    return r;
  } else {
    return long_row(a.lengths[b], a.starts ? a.starts[b] : 0, a.S, a.window, a.sinks);
  }
}
template <int BITS>
__device__ __forceinline__ int long_chunks(const LongRow& row) {
  using T = LongTile<BITS>;
  return row.n > 0 ? (row.n + T::CHUNK - 1) / T::CHUNK + T::EXTRA : 0;
}
template <int BITS, bool PAGED>
__device__ __forceinline__ int long_count(const LongDecodeArgs& a, int per, int lane, int& upto) {   // total; upto: inclusive
  int n = 0;
#pragma unroll 4
  for (int i = 0; i < per; ++i) {
    const int b = lane * per + i;
    if (b < a.B) n += long_chunks<BITS>(long_row_of<PAGED>(a, b));
  }
  upto = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(FULL, upto, o);
    if (lane >= o) upto += y;
  }
  const int total = __shfl_sync(FULL, upto, 31);
  upto -= n;                            // exclusive
  return total;
}
// The batch row whose chunks hold number x of one KV head's list (x < total).
template <int BITS, bool PAGED>
__device__ __forceinline__ LongPlace<PAGED> long_find(const LongDecodeArgs& a, int per, int lane, int before, int x) {
  const int owner = 31 - __clz(__ballot_sync(FULL, before <= x));     // empty lanes share a count: the last of them
  LongPlace<PAGED> p;
  p.b = owner * per;
  p.before = __shfl_sync(FULL, before, owner);
  while (true) {
    p.row = long_row_of<PAGED>(a, p.b);
    const int n = long_chunks<BITS>(p.row);
    if (x < p.before + n) return p;
    p.before += n;
    ++p.b;
  }
}
// CTA c of n takes chunks [share(c), share(c + 1)); the inverse.
__device__ __forceinline__ int long_share(int total, int n, int c) { return total / n * c + min(c, total % n); }
__device__ __forceinline__ int long_owner(int total, int n, int x) {
  const int q = total / n, big = total % n * (q + 1);
  return x < big ? x / (q + 1) : total % n + (x - big) / q;
}

// Paged: head hq of batch row b again, a key at a time, where an output is not finite (a weight's two parts, and the places
// of hidden keys, make a NaN of an infinity in a visible slot) though the weights' sum L is a number above 0.  Without one the
// output is NaN whatever V holds, and a row that has gone bad does not hold up the others.
__device__ __noinline__ uint2 long_paged_again(const LongDecodeArgs& a, int b, int hq) {
  const PagedPool pool{const_cast<unsigned char*>(a.c.k), const_cast<unsigned char*>(a.c.v), a.c.k_sb, a.c.k_sh, a.c.k_sp,
                       a.c.v_sb, a.c.v_sh, a.c.v_sp, a.t.pages, a.NKV, a.t.page, a.t.shift};
  const LongRow row = long_row(a.lengths[b], 0, a.S, a.window, a.sinks);
  return paged_one(pool, a.t, row, a.scale, b, hq / a.G, a.q + b * a.q_sb + (long long)hq * a.q_sh);
}

struct LongStat {
  float mA, mB;           // heads 2t, 2t + 1: the subtracted maximum (the same in the eight lanes of a t)
  uint64_t l;             // the two partial sums
};

// hide (paged): bits 0 and 1, this lane's keys that get no weight.
// Scores of a step (rows g, g + 8 of each 16-key tile, heads 2t, 2t + 1) -> weights as the B fragments of P^T; bf16:
// the second parts of the weights in the upper columns (G <= 4) or in pl (G = 8).
template <int BITS, bool SCORED, bool PAGED, int NT>
__device__ __forceinline__ void long_softmax(float (&s)[NT][4], uint32_t (&pf)[NT][2], uint32_t (&pl)[2], LongStat& st,
                                             float (&o)[8][4], int i0, int n, bool whole, uint32_t hide, float scA, float scB,
                                             float* scp, int G, int g, int t) {
  constexpr float SHIFT = LongTile<BITS>::SHIFT;
  if (!whole) {
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (PAGED ? (hide >> e) & 1u : i0 + 16 * k + g + 8 * e >= n) s[k][2 * e] = s[k][2 * e + 1] = -INFINITY;
  }
  const uint64_t sc = f2(scA, scB);
  float xA = s[0][0], xB = s[0][1];
#pragma unroll
  for (int k = 0; k < NT; ++k) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (SCORED) {
        const int i = i0 + 16 * k + g + 8 * e;
        const float2 y = f2_get(f2_mul(f2(s[k][2 * e], s[k][2 * e + 1]), sc));
        if (whole || i < n) {
          if (2 * t + 1 < G) *reinterpret_cast<float2*>(scp + (long long)i * G + 2 * t) = y;
          else if (2 * t < G) scp[(long long)i * G + 2 * t] = y.x;
        }
      }
      xA = fmaxf(xA, s[k][2 * e]);
      xB = fmaxf(xB, s[k][2 * e + 1]);
    }
  }
  xA = xA * scA - SHIFT;                // scA, scB > 0
  xB = xB * scB - SHIFT;
  // the eight lanes of a t compare their own scores; the maximum over all is worked out only when it moves (also in the
  // first tile: it is -inf)
  if (__any_sync(FULL, xA > st.mA + 8.f || xB > st.mB + 8.f)) {
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      xA = fmaxf(xA, __shfl_xor_sync(FULL, xA, x));
      xB = fmaxf(xB, __shfl_xor_sync(FULL, xB, x));
    }
    const float nA = fmaxf(st.mA, xA), nB = fmaxf(st.mB, xB);
    const float fA = st.mA > -INFINITY ? ex2(st.mA - nA) : 0.f, fB = st.mB > -INFINITY ? ex2(st.mB - nB) : 0.f;
    st.mA = nA;
    st.mB = nB;
    const uint64_t f = f2(fA, fB);
    st.l = f2_mul(st.l, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i][0] *= fA;
      o[i][1] *= fB;
      o[i][2] *= fA;
      o[i][3] *= fB;
    }
  }
  const uint64_t off = f2(st.mA > -INFINITY ? -st.mA : 0.f, st.mB > -INFINITY ? -st.mB : 0.f);
#pragma unroll
  for (int k = 0; k < NT; ++k) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float2 y = f2_get(f2_fma(f2(s[k][2 * e], s[k][2 * e + 1]), sc, off));
      const float pA = ex2(y.x), pB = ex2(y.y);
      st.l = f2_add(st.l, f2(pA, pB));
      if (BITS == 16) {
        const uint32_t hi = pack_bf16(pA, pB), lo = pack_bf16(pA - lo_f(hi), pB - hi_f(hi));
        pf[k][e] = movmatrix(G <= 4 && t >= 2 ? lo : hi);
        if (G == 8) pl[e] = movmatrix(lo);
      } else {
        pf[k][e] = movmatrix(pack_h2(pA, pB));
      }
    }
  }
}

// Keys [i_first, i_end) of row (b, h) by the CTA's four warps; each leaves its (max, sum, unnormalised out) in shared
// memory.  scp: score i of head g goes to scp[i G + g].
template <int BITS, bool SCORED, bool PAGED>
__device__ __forceinline__ void long_piece(const LongDecodeArgs& a, int b, int h, const LongRowOf<PAGED>& row, int i_first, int i_end,
                                           float* scp, float (*s_o)[8][LG_D], float (*s_m)[8], float (*s_l)[8]) {
  using T = LongTile<BITS>;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int G = a.G;
  // ---- q of the group, column g: the head's values at the dims this lane's keys hold, zero beyond the group
  uint32_t qf[8][2];
  const int qh = BITS == 16 && G <= 4 ? g & 3 : g;
  float scA = a.scale, scB = a.scale;
  {
    const bf16* qp = a.q + b * a.q_sb + (long long)(h * G + qh) * a.q_sh;
    uint4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = make_uint4(0, 0, 0, 0);
      // 16-bit keys: dims 32 i + 8 t .. + 7;  4-bit keys: dims 32 t + 8 i .. + 7
      if (qh < G) w[i] = *reinterpret_cast<const uint4*>(qp + (BITS == 16 ? 32 * i + 8 * t : 32 * t + 8 * i));
      w[i].x ^= a.flip, w[i].y ^= a.flip, w[i].z ^= a.flip, w[i].w ^= a.flip;
    }
    if (BITS == 16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        qf[2 * i][0] = w[i].x;
        qf[2 * i][1] = w[i].y;
        qf[2 * i + 1][0] = w[i].z;
        qf[2 * i + 1][1] = w[i].w;
      }
    } else {
      // fp16 operands: the head is scaled by a power of two to a largest value in [8, 16), so that values down to
      // 2^-18 of it stay exact and none overflows; the score takes the power back
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[8];
        cvt8(w[i], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(f[e]));
      }
      amax = fmaxf(amax, __shfl_xor_sync(FULL, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(FULL, amax, 2));
      int ex = (int)(__float_as_uint(amax) >> 23) - 127 - 3;
      if (amax == 0.f || ex > 120 || ex < -120) ex = ex > 120 ? 120 : (amax == 0.f ? 0 : -120);
      const float down = __uint_as_float((uint32_t)(127 - ex) << 23);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[8];
        cvt8(w[i], f);
        qf[2 * i][0] = pack_h2(f[0] * down, f[1] * down);
        qf[2 * i][1] = pack_h2(f[2] * down, f[3] * down);
        qf[2 * i + 1][0] = pack_h2(f[4] * down, f[5] * down);
        qf[2 * i + 1][1] = pack_h2(f[6] * down, f[7] * down);
      }
      const float up = __uint_as_float((uint32_t)(127 + ex) << 23);
      scA = a.scale * __shfl_sync(FULL, up, 8 * t);          // head 2t lives in lanes 4 (2t) ..
      scB = a.scale * __shfl_sync(FULL, up, 8 * t + 4);
      if (scA == 0.f) scA = FLT_MIN;                         // a masked score stays -inf
      if (scB == 0.f) scB = FLT_MIN;
    }
  }

  float o[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  LongStat st{-INFINITY, -INFINITY, 0};

  const unsigned char* kb = a.c.k + (PAGED ? 0 : b * a.c.k_sb) + h * a.c.k_sh;
  const unsigned char* vb = a.c.v + (PAGED ? 0 : b * a.c.v_sb) + h * a.c.v_sh;
  // the tile's page, one tile ahead of its keys
  const int* table = PAGED ? a.t.table + b * a.t.table_sb : nullptr;
  int next = 0;
  bool some = false;                                         // a visible key in a page of the pool
  if (PAGED && i_first + warp * T::KEYS < i_end) next = table[row.slot(i_first + warp * T::KEYS) >> a.t.shift];
  for (int i0 = i_first + warp * T::KEYS; i0 < i_end; i0 += T::CHUNK) {
    float s[T::KEYS / 16][4];
    uint32_t pf[T::KEYS / 16][2], pl[2];
    // a tile of consecutive slots: with rows of the dense stride every load is one address and a constant
    bool whole = i0 + T::KEYS <= row.n && (i0 >= row.ns || i0 + T::KEYS <= row.ns);
    long long slot0 = row.slot(i0);
    uint32_t hide = 0;
    int pick[2], vpick[4];                                   // paged: offsets in the tile of the keys that are read
    const unsigned char *kt = kb, *vt = vb;
    if constexpr (PAGED) {
      const int j0 = (int)slot0, page = next;
      if (i0 + T::CHUNK < i_end) next = table[row.slot(i0 + T::CHUNK) >> a.t.shift];
      if ((unsigned)page >= (unsigned)a.t.pages) continue;   // not in the pool: not visible
      some = true;
      slot0 = j0 & (a.t.page - 1);
      kt += page * a.c.k_sb;
      vt += page * a.c.v_sb;
      whole = whole && (j0 >= row.vlo || j0 + T::KEYS <= row.vns);
      if (!whole || !a.dense) {
        // the place of a key that is not visible is read as the tile's first visible key
        const int first = j0 < row.vns ? 0 : max(row.vlo - j0, 0);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int x = g + 8 * e;
          const bool see = row.sees(j0 + x);
          pick[e] = see ? x : first;
          hide |= see ? 0u : 1u << e;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int x = 2 * t + (e & 1) + 8 * (e >> 1);
          vpick[e] = row.sees(j0 + x) ? x : first;
        }
      }
    }
    const bool fast = whole && a.dense;
    if constexpr (BITS == 16) {
      __align__(16) uint32_t kw[2][16], vw[4][8];
      if (fast) {
        const unsigned char* pk = kt + (slot0 + g) * 256 + 16 * t;
        const unsigned char* pv = vt + (slot0 + 2 * t) * 256 + 16 * g;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(&kw[e][4 * i]) = ld_nc_v4(pk + 2048 * e + 64 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint4*>(&vw[e][4 * i]) = ld_nc_v4(pv + 256 * ((e & 1) + 8 * (e >> 1)) + 128 * i);
      } else {
        // keys past the row's end read its last key (a visible one) and get no weight
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const unsigned char* p =
              kt + (PAGED ? slot0 + pick[e] : row.slot(min(i0 + g + 8 * e, row.n - 1))) * a.c.k_sp + 16 * t;
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(&kw[e][4 * i]) = ld_nc_v4(p + 64 * i);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned char* p =
              vt + (PAGED ? slot0 + vpick[e] : row.slot(min(i0 + 2 * t + (e & 1) + 8 * (e >> 1), row.n - 1))) * a.c.v_sp +
              16 * g;
#pragma unroll
          for (int i = 0; i < 2; ++i) *reinterpret_cast<uint4*>(&vw[e][4 * i]) = ld_nc_v4(p + 128 * i);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[0][e] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        mma_bf16(s[0], kw[0][2 * i], kw[1][2 * i], kw[0][2 * i + 1], kw[1][2 * i + 1], qf[i][0], qf[i][1]);
      long_softmax<BITS, SCORED, PAGED>(s, pf, pl, st, o, i0, row.n, whole, hide, scA, scB, scp, G, g, t);
      // dims: row g of tile i is 8 g + i, row g + 8 is 64 + 8 g + i
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int w = i >> 1;
        const uint32_t sel = (i & 1) ? 0x7632u : 0x5410u;
        const uint32_t a0 = __byte_perm(vw[0][w], vw[1][w], sel), a1 = __byte_perm(vw[0][4 + w], vw[1][4 + w], sel);
        const uint32_t a2 = __byte_perm(vw[2][w], vw[3][w], sel), a3 = __byte_perm(vw[2][4 + w], vw[3][4 + w], sel);
        mma_bf16(o[i], a0, a1, a2, a3, pf[0][0], pf[0][1]);
        if (G == 8) mma_bf16(o[i], a0, a1, a2, a3, pl[0], pl[1]);
      }
    } else {
      const unsigned char* ksb = a.c.ks + b * a.c.ks_sb + h * a.c.ks_sh;
      const unsigned char* vsb = a.c.vs + b * a.c.vs_sb + h * a.c.vs_sh;
      __align__(16) uint32_t kw[2][2][4], vw[2][4][2];
      uint16_t ksc[2][2];
      unsigned char vsc[2][4];
      if (fast) {
        const unsigned char* pk = kb + (slot0 + g) * 64 + 16 * t;
        const unsigned char* pv = vb + (slot0 + 2 * t) * 64 + 8 * g;
        const unsigned char* pks = ksb + (slot0 + g) * 8 + 2 * t;
        const unsigned char* pvs = vsb + (slot0 + 2 * t) * 8 + g;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            *reinterpret_cast<uint4*>(&kw[n][e][0]) = ld_nc_v4(pk + 64 * (16 * n + 8 * e));
            ksc[n][e] = __ldg(reinterpret_cast<const uint16_t*>(pks + 8 * (16 * n + 8 * e)));
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row_off = 16 * n + (e & 1) + 8 * (e >> 1);
            *reinterpret_cast<uint2*>(&vw[n][e][0]) = ld_nc_v2(pv + 64 * row_off);
            vsc[n][e] = __ldg(pvs + 8 * row_off);
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const long long sl = row.slot(min(i0 + 16 * n + g + 8 * e, row.n - 1));
            *reinterpret_cast<uint4*>(&kw[n][e][0]) = ld_nc_v4(kb + sl * a.c.k_sp + 16 * t);
            ksc[n][e] = __ldg(reinterpret_cast<const uint16_t*>(ksb + sl * a.c.ks_sp + 2 * t));
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const long long sl = row.slot(min(i0 + 16 * n + 2 * t + (e & 1) + 8 * (e >> 1), row.n - 1));
            *reinterpret_cast<uint2*>(&vw[n][e][0]) = ld_nc_v2(vb + sl * a.c.v_sp + 8 * g);
            vsc[n][e] = __ldg(vsb + sl * a.c.vs_sp + g);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
        const uint32_t sg = e4m3x2_to_h2(ksc[n][0]), sh = e4m3x2_to_h2(ksc[n][1]);   // blocks 2t, 2t + 1
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t x[4], y[4];
          e2m1x8_to_h2(kw[n][0][w], x);
          e2m1x8_to_h2(kw[n][1][w], y);
          const uint32_t fx = w < 2 ? both_lo(sg) : both_hi(sg), fy = w < 2 ? both_lo(sh) : both_hi(sh);
          mma_f16(s[n], hmul2(x[0], fx), hmul2(y[0], fy), hmul2(x[1], fx), hmul2(y[1], fy), qf[2 * w][0],
                  qf[2 * w][1]);
          mma_f16(s[n], hmul2(x[2], fx), hmul2(y[2], fy), hmul2(x[3], fx), hmul2(y[3], fy), qf[2 * w + 1][0],
                  qf[2 * w + 1][1]);
        }
      }
      long_softmax<BITS, SCORED, PAGED>(s, pf, pl, st, o, i0, row.n, whole, hide, scA, scB, scp, G, g, t);
      // dims: row g of tile i is 16 g + i (first code word), row g + 8 is 16 g + 8 + i (second)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint32_t f0 = e4m3x2_to_h2((uint16_t)(vsc[n][0] | (vsc[n][1] << 8)));   // scales of keys 2t, 2t + 1
        const uint32_t f1 = e4m3x2_to_h2((uint16_t)(vsc[n][2] | (vsc[n][3] << 8)));
        uint32_t lo[4][4], hi[4][4];   // [2 word + key pair][byte]: even dims, odd dims, (first key, second key)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t x = vw[n][2 * e][w], y = vw[n][2 * e + 1][w];
            e2m1x8_to_h2((x & 0x0f0f0f0fu) | ((y << 4) & 0xf0f0f0f0u), lo[2 * w + e]);
            e2m1x8_to_h2(((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u), hi[2 * w + e]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          mma_f16(o[2 * i], hmul2(lo[0][i], f0), hmul2(lo[2][i], f0), hmul2(lo[1][i], f1), hmul2(lo[3][i], f1),
                  pf[n][0], pf[n][1]);
          mma_f16(o[2 * i + 1], hmul2(hi[0][i], f0), hmul2(hi[2][i], f0), hmul2(hi[1][i], f1), hmul2(hi[3][i], f1),
                  pf[n][0], pf[n][1]);
        }
      }
    }
  }

  if (BITS == 16 && G <= 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] += __shfl_down_sync(FULL, o[i][e], 2);
  }
  // ---- the four warps' parts of the piece, joined in warp order
  float2 l = f2_get(st.l);
#pragma unroll
  for (int x = 4; x < 32; x <<= 1) {
    l.x += __shfl_xor_sync(FULL, l.x, x);
    l.y += __shfl_xor_sync(FULL, l.y, x);
  }
  // a NaN score is in the sum and not in the maximum: as the largest part it cannot be lost in the joins
  if (l.x != l.x) st.mA = FLT_MAX;
  if (l.y != l.y) st.mB = FLT_MAX;
  // paged: visible scores of -inf alone are told from no visible key, whose maximum stays -inf
  if (PAGED && some) {
    st.mA = fmaxf(st.mA, -FLT_MAX);
    st.mB = fmaxf(st.mB, -FLT_MAX);
  }
  if (g == 0) {
    s_m[warp][2 * t] = st.mA;
    s_m[warp][2 * t + 1] = st.mB;
    s_l[warp][2 * t] = l.x;
    s_l[warp][2 * t + 1] = l.y;
  }
  {
    const int d0 = BITS == 16 ? 8 * g : 16 * g, d1 = d0 + (BITS == 16 ? 64 : 8);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (2 * t + e < G) {
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          *reinterpret_cast<float4*>(&s_o[warp][2 * t + e][d0 + i]) =
              make_float4(o[i][e], o[i + 1][e], o[i + 2][e], o[i + 3][e]);
          *reinterpret_cast<float4*>(&s_o[warp][2 * t + e][d1 + i]) =
              make_float4(o[i][2 + e], o[i + 1][2 + e], o[i + 2][2 + e], o[i + 3][2 + e]);
        }
      }
    }
  }
}

// Joins the four warps' parts in warp order: head gg's maximum, sum and this thread's dim.
__device__ __forceinline__ void long_join(const float (*s_o)[8][LG_D], const float (*s_m)[8], const float (*s_l)[8], int gg,
                                          float& M, float& L, float& O) {
  M = s_m[0][gg];
#pragma unroll
  for (int w = 1; w < LD_WARPS; ++w) M = fmaxf(M, s_m[w][gg]);
  L = O = 0.f;
#pragma unroll
  for (int w = 0; w < LD_WARPS; ++w) {
    const float f = s_m[w][gg] > -INFINITY ? ex2(s_m[w][gg] - M) : 0.f;
    L += f * s_l[w][gg];
    O += f * s_o[w][gg][threadIdx.x];                    // a warp without a tile: 0
  }
}

template <int BITS, bool SCORED, bool PAGED>
__global__ void __launch_bounds__(LD_THREADS, LongTile<BITS>::CTAS) long_decode_kernel(const __grid_constant__ LongDecodeArgs a) {
  using T = LongTile<BITS>;
  __shared__ __align__(16) float s_o[LD_WARPS][8][LG_D];
  __shared__ float s_m[LD_WARPS][8], s_l[LD_WARPS][8];
  const int tid = threadIdx.x, lane = tid & 31, G = a.G;
  pdl_wait();
  pdl_trigger();
  int before;
  const int total = long_count<BITS, PAGED>(a, a.per, lane, before) * a.NKV;
  const int ncta = min(a.ncta, total);                    // every CTA below it has a chunk at least
  const int cta = blockIdx.x;
  if (cta >= ncta) return;
  int pos = long_share(total, ncta, cta);
  const int end = long_share(total, ncta, cta + 1);
  LongPlace<PAGED> at = long_find<BITS, PAGED>(a, a.per, lane, before, pos / a.NKV);
  while (true) {
    const int nb = long_chunks<BITS>(at.row), rem = pos - at.before * a.NKV;
    const int h = rem / nb, e0 = rem - h * nb, e1 = min(nb, e0 + (end - pos));
    const int ch0 = max(0, e0 - T::EXTRA), ch1 = e1 - T::EXTRA;      // the row's own chunks
    const int r = at.b * a.NKV + h;
    if (ch1 > ch0) {
      long_piece<BITS, SCORED, PAGED>(a, at.b, h, at.row, ch0 * T::CHUNK, min(at.row.n, ch1 * T::CHUNK),
                               SCORED ? a.sc + (long long)r * a.cap * G : nullptr, s_o, s_m, s_l);
      __syncthreads();
      const long long piece = (long long)cta + r;         // pieces in list order have increasing CTA or row: unique
      for (int gg = 0; gg < G; ++gg) {
        float M, L, O;
        long_join(s_o, s_m, s_l, gg, M, L, O);
        a.po[(piece * G + gg) * LG_D + tid] = O;
        if (tid == 0) a.ml[piece * G + gg] = make_float2(M, L);
      }
      if (ch0 == 0 && tid == 0) a.own[r] = make_int2(cta, long_owner(total, ncta, pos - e0 + nb - 1));
    }
    pos += e1 - e0;
    if (pos == end) return;
    if (h == a.NKV - 1 && e1 == nb) {                     // the next row that has keys
      at.before += nb;
      do at.row = long_row_of<PAGED>(a, ++at.b);
      while (at.row.n == 0);
    }
    __syncthreads();
  }
}

// Few rows: a thread-block cluster per (row, KV head), its CTAs on equal runs of chunks; one launch, no workspace.  The
// parts are joined through distributed shared memory in rank order.  Scores stay in shared memory until the row's
// maximum and sum are known.
template <int BITS, bool SCORED, bool PAGED>
__global__ void __launch_bounds__(LD_THREADS, LongTile<BITS>::CTAS) long_cluster_kernel(const __grid_constant__ LongDecodeArgs a) {
  using T = LongTile<BITS>;
  extern __shared__ __align__(16) unsigned char smem[];
  float* s_sc = reinterpret_cast<float*>(smem);          // [its chunks x CHUNK][G] (weights wanted)
  __shared__ __align__(16) float s_o[LD_WARPS][8][LG_D];
  __shared__ float s_m[LD_WARPS][8], s_l[LD_WARPS][8];
  __shared__ float c_o[8][LG_D], c_m[8], c_l[8];         // this CTA's part, read by its peers
  __shared__ float s_max[8], s_inv[8];
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, split = blockIdx.x, ns = gridDim.x;
  const int r = blockIdx.y, b = r / a.NKV, h = r - b * a.NKV, G = a.G;
  pdl_wait();
  pdl_trigger();
  const auto row = long_row_of<PAGED>(a, b);
  const int nb = (row.n + T::CHUNK - 1) / T::CHUNK;
  const int i_first = nb * split / ns * T::CHUNK, i_end = min(row.n, nb * (split + 1) / ns * T::CHUNK);
  long_piece<BITS, SCORED, PAGED>(a, b, h, row, i_first, i_end, SCORED ? s_sc - (long long)i_first * G : nullptr, s_o, s_m, s_l);
  __syncthreads();
  for (int gg = 0; gg < G; ++gg) {
    float M, L, O;
    long_join(s_o, s_m, s_l, gg, M, L, O);
    c_o[gg][tid] = O;
    if (tid == 0) {
      c_m[gg] = M;
      c_l[gg] = L;
    }
  }
  cluster.sync();
  for (int gg = split; gg < G; gg += ns) {
    float mv[LC_MAX], lv[LC_MAX], ov[LC_MAX];
#pragma unroll
    for (int c = 0; c < LC_MAX; ++c)
      if (c < ns) {                                      // all peers' loads together
        mv[c] = *cluster.map_shared_rank(&c_m[gg], c);
        lv[c] = *cluster.map_shared_rank(&c_l[gg], c);
        ov[c] = *cluster.map_shared_rank(&c_o[gg][tid], c);
      }
    float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
    for (int c = 0; c < LC_MAX; ++c)
      if (c < ns) M = fmaxf(M, mv[c]);
#pragma unroll
    for (int c = 0; c < LC_MAX; ++c)
      if (c < ns) {
        const float f = mv[c] > -INFINITY ? ex2(mv[c] - M) : 0.f;
        L += f * lv[c];
        O += f * ov[c];
      }
    const bool none = PAGED ? M == -INFINITY : row.n == 0;
    const float y = none ? 0.f : O / L * a.v_scale;
    bf16* out = a.out + ((long long)b * a.NH + h * G + gg) * LG_D;
    if (PAGED && L > 0.f && __any_sync(FULL, !isfinite(y))) {       // the warp's own 32 dims: lanes 8 warp .. of the head
      const uint2 w = long_paged_again(a, b, h * G + gg);
      if ((tid & 31) >> 3 == tid >> 5) *reinterpret_cast<uint2*>(out + 4 * (tid & 31)) = w;
    } else {
      out[tid] = __float2bfloat16_rn(y);
    }
  }
  if constexpr (SCORED) {
    if (tid < G) {
      float M = -INFINITY, L = 0.f;
      for (int c = 0; c < ns; ++c) M = fmaxf(M, *cluster.map_shared_rank(&c_m[tid], c));
      for (int c = 0; c < ns; ++c) {
        const float m = *cluster.map_shared_rank(&c_m[tid], c);
        if (m > -INFINITY) L += ex2(m - M) * *cluster.map_shared_rank(&c_l[tid], c);
      }
      s_max[tid] = M + T::SHIFT;                         // scores near the maximum: a difference near 0 keeps its bits
      s_inv[tid] = ex2(T::SHIFT) / L;
    }
    __syncthreads();
    const float* ap = a.acc + b * a.acc_sb + h * a.acc_sh;
    float* op = a.acc_out + b * a.acco_sb + h * a.acco_sh;
    for (int i = i_first + tid; i < i_end; i += LD_THREADS) {
      float w = 0.f;
      for (int gg = 0; gg < G; ++gg) w += ex2(s_sc[(i - i_first) * G + gg] - s_max[gg]) * s_inv[gg];
      const long long j = row.slot(i);
      op[j] = a.decay * ap[j] + w;
    }
    if (ap != op || a.decay != 1.f)                      // slots that are not visible
      for (int j = (int)((long long)a.S * split / ns) + tid; j < (int)((long long)a.S * (split + 1) / ns); j += LD_THREADS)
        if (row.index(j) < 0) op[j] = a.decay * ap[j];
  }
  cluster.sync();                                        // a peer may still be reading this CTA's part
}

// Slots j0, j0 + LM_THREADS, .. of a slice: the scores of the group's heads -> weights, added to the accumulator.  The loads
// of N slots a thread are under way while the heads' maxima and sums are worked out.
template <int G, class Stats>
__device__ __forceinline__ void long_weights(const LongDecodeArgs& a, const LongRow& row, int b, int h, int r, int j0,
                                             Stats stats, float* s_m, float* s_inv) {
  constexpr int ALL = LD_SLICE / LM_THREADS, N = G == 8 ? ALL / 2 : ALL;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float* ap = a.acc + b * a.acc_sb + h * a.acc_sh;
  float* op = a.acc_out + b * a.acco_sb + h * a.acco_sh;
  const float* scp = a.sc + (long long)r * a.cap * G;
#pragma unroll 1
  for (int k0 = 0; k0 < ALL; k0 += N, j0 += N * LM_THREADS) {
    float acc[N], s[N][G];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int j = j0 + k * LM_THREADS, i = j < a.S ? row.index(j) : -1;
      acc[k] = j < a.S ? ap[j] : 0.f;
#pragma unroll
      for (int g = 0; g < G; g += G < 4 ? G : 4) {
        const float* p = scp + (long long)i * G + g;
        if constexpr (G >= 4) {
          const float4 x = i >= 0 ? *reinterpret_cast<const float4*>(p) : make_float4(0.f, 0.f, 0.f, 0.f);
          s[k][g] = x.x, s[k][g + 1] = x.y, s[k][g + 2] = x.z, s[k][g + 3] = x.w;
        } else if constexpr (G == 2) {
          const float2 x = i >= 0 ? *reinterpret_cast<const float2*>(p) : make_float2(0.f, 0.f);
          s[k][0] = x.x, s[k][1] = x.y;
        } else {
          s[k][0] = i >= 0 ? *p : 0.f;
        }
      }
    }
    if (k0 == 0) {
      for (int gg = warp; gg < G; gg += LM_THREADS / 32) {
        float M, L;
        stats(gg, M, L);
        if (lane == 0) {
          s_m[gg] = M + a.shift;                 // scores near the maximum: a difference near 0 keeps its bits
          s_inv[gg] = ex2(a.shift) / L;          // not used for a row without a visible slot
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int j = j0 + k * LM_THREADS;
      if (j >= a.S) return;
      const bool seen = row.index(j) >= 0;
      if (!seen && ap == op && a.decay == 1.f) continue;
      float w = 0.f;
      if (seen) {
#pragma unroll
        for (int g = 0; g < G; ++g) w += ex2(s[k][g] - s_m[g]) * s_inv[g];
      }
      op[j] = a.decay * acc[k] + w;
    }
  }
}

// Joins the pieces of every row: a warp per (row, head), in CTA order, or WIDE (few rows of many pieces each) a CTA, its
// warps on every fourth piece and joined in warp order; past those, CTAs of LD_SLICE slots turn scores into weights.
// Eight CTAs an SM: the weights of 64 rows of up to 4096 slots and 4 heads 54.2 us in all, with the 96 registers of five
// CTAs 57.1, with the 48 of ten 55.9; slices of 256 or 1024 slots 58.5 and 57.6.
template <bool SCORED, bool WIDE, bool PAGED>
__global__ void __launch_bounds__(LM_THREADS, 8) long_merge_kernel(const __grid_constant__ LongDecodeArgs a) {
  __shared__ float s_m[8], s_inv[8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = a.G;
  constexpr int W = LM_THREADS / 32;
  const int heads = a.B * a.NKV * G, joins = WIDE ? heads : (heads + W - 1) / W;
  const bool join = (int)blockIdx.x < joins;
  const int item = join && !WIDE ? blockIdx.x * W + warp : blockIdx.x - (join ? 0 : joins);
  const int r = join ? min(item, heads - 1) / G : item / a.slices, b = r / a.NKV, h = r - b * a.NKV;
  const auto row = long_row_of<PAGED>(a, b);    // written at least two launches back
  pdl_wait();
  pdl_trigger();
  const int2 own = row.n > 0 ? a.own[r] : make_int2(0, -1);   // CTAs [x, y] hold pieces of this row
  // a head's maximum and sum over the pieces (every lane)
  auto stats = [&](int gg, float& M, float& L) {
    M = -INFINITY;
    L = 0.f;
    for (int c = own.x + lane; c <= own.y; c += 32) M = fmaxf(M, a.ml[(long long)(c + r) * G + gg].x);
    M = warp_max(M);
    for (int c = own.x + lane; c <= own.y; c += 32) {
      const float2 x = a.ml[(long long)(c + r) * G + gg];
      if (x.x > -INFINITY) L += ex2(x.x - M) * x.y;
    }
    L = warp_sum(L);
  };
  if (join) {
    if (item >= heads) return;
    const int gg = item - r * G;
    float M, L;
    stats(gg, M, L);
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = own.x + (WIDE ? warp : 0); c <= own.y; c += WIDE ? W : 1) {
      const long long at = (long long)(c + r) * G + gg;
      const float m = a.ml[at].x;
      const float4 x = *reinterpret_cast<const float4*>(a.po + at * LG_D + 4 * lane);
      const float f = m > -INFINITY ? ex2(m - M) : 0.f;
      O.x += f * x.x;
      O.y += f * x.y;
      O.z += f * x.z;
      O.w += f * x.w;
    }
    if constexpr (WIDE) {
      __shared__ __align__(16) float4 s_o[W][32];
      s_o[warp][lane] = O;
      __syncthreads();
      if (warp > 0) return;
#pragma unroll
      for (int w = 1; w < W; ++w) {
        const float4 x = s_o[w][lane];
        O.x += x.x;
        O.y += x.y;
        O.z += x.z;
        O.w += x.w;
      }
    }
    // visible keys with scores of -inf alone: 0 / 0, as softmax has it
    const float f = a.v_scale / L;
    const bool none = PAGED ? M == -INFINITY : row.n == 0;
    uint2 y = make_uint2(none ? 0u : pack_bf16(O.x * f, O.y * f), none ? 0u : pack_bf16(O.z * f, O.w * f));
    if (PAGED && L > 0.f && __any_sync(FULL, !isfinite(O.x) || !isfinite(O.y) || !isfinite(O.z) || !isfinite(O.w)))
      y = long_paged_again(a, b, h * G + gg);
    *reinterpret_cast<uint2*>(a.out + ((long long)b * a.NH + h * G + gg) * LG_D + 4 * lane) = y;
    return;
  }
  if constexpr (SCORED) {
    const int j0 = (item - r * a.slices) * LD_SLICE + tid;
    switch (G) {
      case 1: long_weights<1>(a, row, b, h, r, j0, stats, s_m, s_inv); break;
      case 2: long_weights<2>(a, row, b, h, r, j0, stats, s_m, s_inv); break;
      case 4: long_weights<4>(a, row, b, h, r, j0, stats, s_m, s_inv); break;
      default: long_weights<8>(a, row, b, h, r, j0, stats, s_m, s_inv);
    }
  }
}

}  // namespace fb

namespace fbh {

int long_cache(const fb_kv_cache* c, fb::LongCache* out) {
  FB_CHECK_ARG(c, "long cache: null descriptor");
  FB_CHECK_ARG(c->bits == 16 || c->bits == 4, "long cache: bits %d (16 or 4)", c->bits);
  FB_CHECK_ARG(c->B >= 1 && c->NKV >= 1 && c->S >= 1, "long cache: bad shape B=%d NKV=%d S=%d", c->B, c->NKV, c->S);
  FB_CHECK_ARG(c->k && c->v, "long cache: null keys or values");
  const bool four = c->bits == 4;
  const int64_t es = four ? 1 : 2, row = four ? fb::LG_D / 2 : fb::LG_D;
  const int64_t st[6] = {c->k_sb, c->k_sh, c->k_sp, c->v_sb, c->v_sh, c->v_sp};
  for (int64_t x : st)
    FB_CHECK_ARG(x >= 0 && x * es % 16 == 0, "long cache: strides must be multiples of 16 bytes");
  FB_CHECK_ARG(c->k_sp >= row && c->v_sp >= row, "long cache: position strides below the row (%lld)", (long long)row);
  FB_CHECK_ARG(((uintptr_t)c->k & 15) == 0 && ((uintptr_t)c->v & 15) == 0, "long cache: keys and values 16-byte aligned");
  out->k = (const unsigned char*)c->k;
  out->v = (const unsigned char*)c->v;
  out->k_sb = c->k_sb * es, out->k_sh = c->k_sh * es, out->k_sp = c->k_sp * es;
  out->v_sb = c->v_sb * es, out->v_sh = c->v_sh * es, out->v_sp = c->v_sp * es;
  out->ks = out->vs = nullptr;
  out->ks_sb = out->ks_sh = out->ks_sp = out->vs_sb = out->vs_sh = out->vs_sp = 0;
  if (four) {
    FB_CHECK_ARG(c->ks && c->vs, "long cache: null scales");
    const int64_t ss[6] = {c->ks_sb, c->ks_sh, c->ks_sp, c->vs_sb, c->vs_sh, c->vs_sp};
    for (int64_t x : ss) FB_CHECK_ARG(x >= 0 && x % 8 == 0, "long cache: scale strides must be multiples of 8 bytes");
    FB_CHECK_ARG(c->ks_sp >= 8 && c->vs_sp >= 8, "long cache: scale position strides below 8");
    FB_CHECK_ARG(((uintptr_t)c->ks & 7) == 0 && ((uintptr_t)c->vs & 7) == 0, "long cache: scales 8-byte aligned");
    out->ks = (const unsigned char*)c->ks;
    out->vs = (const unsigned char*)c->vs;
    out->ks_sb = c->ks_sb, out->ks_sh = c->ks_sh, out->ks_sp = c->ks_sp;
    out->vs_sb = c->vs_sb, out->vs_sh = c->vs_sh, out->vs_sp = c->vs_sp;
    const float sc[2] = {c->k_scale, c->v_scale};
    for (float x : sc) {
      int e;
      FB_CHECK_ARG(x > 0.f && std::isfinite(x) && std::frexp(x, &e) == 0.5f && e > -60 && e < 60,
                   "long cache: the tensor scales must be powers of two between 2^-60 and 2^58");
    }
  }
  return FB_OK;
}

LongBox long_box(const void* p, int B, int NKV, long long S, long long sb, long long sh, long long sp, long long row) {
  LongBox x{p, {B, NKV, S}, {sb, sh, sp}, row};
  for (int i = 0; i < 3; ++i)
    if (x.s[i] < 0) {                             // the same bytes, counted from the other end
      x.p = (const unsigned char*)x.p + (x.n[i] - 1) * x.s[i];
      x.s[i] = -x.s[i];
    }
  return x;
}

namespace {
// An axis along which the distance of two rows changes by s a step, from lo to hi steps.
struct BoxAxis {
  long long s, lo, hi;
};
// Whether a choice of steps on axes [i, n) brings the distance d into (-rb, ra).
bool boxes_reach(const BoxAxis* ax, int n, int i, long long d, long long ra, long long rb, int& budget) {
  if (i == n) return d < rb && d > -ra;
  if (--budget < 0) return true;
  long long lo = -ra + 1, hi = rb - 1;            // what the axes after this one can make up for
  for (int j = i + 1; j < n; ++j) {
    lo -= ax[j].s * ax[j].hi;
    hi -= ax[j].s * ax[j].lo;
  }
  // steps x with lo <= d + s x <= hi
  const long long s = ax[i].s, a = lo - d, b = hi - d;
  long long x0 = a >= 0 ? (a + s - 1) / s : -(-a / s), x1 = b >= 0 ? b / s : -((-b + s - 1) / s);
  if (x0 < ax[i].lo) x0 = ax[i].lo;
  if (x1 > ax[i].hi) x1 = ax[i].hi;
  for (long long x = x0; x <= x1; ++x)
    if (boxes_reach(ax, n, i + 1, d + s * x, ra, rb, budget)) return true;
  return false;
}
}  // namespace

bool long_boxes_meet(const LongBox& a, const LongBox& b) {
  const auto span = [](const LongBox& x) {
    long long e = x.row;
    for (int i = 0; i < 3; ++i) e += (x.n[i] - 1) * x.s[i];
    return e;
  };
  const long long d = (const unsigned char*)a.p - (const unsigned char*)b.p;
  if (d >= span(b) || -d >= span(a)) return false;
  // views of one buffer, or interleaved tensors: the axes with the largest stride first; strides that both have make one
  // axis of differences, so that rows that nest leave a step or two to try on each
  BoxAxis ax[6];
  int n = 0;
  const auto add = [&](long long s, long long lo, long long hi) {
    if (s == 0 || lo == hi) return;
    for (int i = 0; i < n; ++i)
      if (ax[i].s == s) {
        ax[i].lo += lo;
        ax[i].hi += hi;
        return;
      }
    int i = n++;
    for (; i > 0 && ax[i - 1].s < s; --i) ax[i] = ax[i - 1];
    ax[i] = {s, lo, hi};
  };
  for (int i = 0; i < 3; ++i) {
    add(a.s[i], 0, a.n[i] - 1);
    add(b.s[i], 1 - b.n[i], 0);
  }
  int budget = 4096;
  return boxes_reach(ax, n, 0, d, a.row, b.row, budget);
}

bool long_box_folds(const LongBox& x) {
  int o[3] = {0, 1, 2};
  for (int i = 1; i < 3; ++i)
    for (int j = i; j > 0 && x.s[o[j]] < x.s[o[j - 1]]; --j) {
      const int t = o[j];
      o[j] = o[j - 1];
      o[j - 1] = t;
    }
  long long e = x.row;                            // bytes from the first to the last row so far
  for (int i : o) {
    if (x.n[i] == 1) continue;
    if (x.s[i] < e) return true;
    e += (x.n[i] - 1) * x.s[i];
  }
  return false;
}

int long_cache_boxes(const fb_kv_cache* c, const fb::LongCache& x, LongBox (&out)[4]) {
  const int row = c->bits == 16 ? 2 * fb::LG_D : fb::LG_D / 2;
  out[0] = long_box(x.k, c->B, c->NKV, c->S, x.k_sb, x.k_sh, x.k_sp, row);
  out[1] = long_box(x.v, c->B, c->NKV, c->S, x.v_sb, x.v_sh, x.v_sp, row);
  if (c->bits == 16) return 2;
  out[2] = long_box(x.ks, c->B, c->NKV, c->S, x.ks_sb, x.ks_sh, x.ks_sp, fb::LG_D / 16);
  out[3] = long_box(x.vs, c->B, c->NKV, c->S, x.vs_sb, x.vs_sh, x.vs_sp, fb::LG_D / 16);
  return 4;
}

int long_cache_written(const fb_kv_cache* c, const fb::LongCache& x, const char* who) {
  LongBox box[4];
  const int n = long_cache_boxes(c, x, box);
  for (int i = 0; i < n; ++i) {
    FB_CHECK_ARG(!long_box_folds(box[i]), "%s: slots of the cache that is written share memory", who);
    for (int j = 0; j < i; ++j)
      FB_CHECK_ARG(!long_boxes_meet(box[i], box[j]), "%s: keys, values and scales of the cache that is written share memory", who);
  }
  return FB_OK;
}

}  // namespace fbh

namespace {
using namespace fb;

struct LongPlan {
  int split;                                       // CTAs of a row's cluster, 0: the two launches
  int ncta, cap, slices;
  size_t smem;
  int64_t slots, ws_floats, off_ml, off_own, off_s;   // float offsets of the workspace's parts
};

// edges: slots beside the visible ones that a row's numbering can hold
int long_plan_host(const fb_kv_cache* c, int NH, int window, int sinks, bool scored, LongPlan* p, int edges = 0) {
  FB_CHECK_ARG(NH >= c->NKV && NH % c->NKV == 0, "long_decode: %d query heads over %d key/value heads", NH, c->NKV);
  const int G = NH / c->NKV;
  if (G != 1 && G != 2 && G != 4 && G != 8) {
    fbh::set_msg("long_decode: GQA group %d not built (1, 2, 4, 8)", G);
    return FB_ERR_UNSUPPORTED;
  }
  FB_CHECK_ARG(sinks >= 0, "long_decode: sinks %d", sinks);
  p->cap = window > 0 && (int64_t)window + sinks + edges < c->S ? window + sinks + edges : c->S;
  const int chunk = c->bits == 16 ? LongTile<16>::CHUNK : LongTile<4>::CHUNK;
  const int64_t most = (int64_t)c->B * c->NKV * ((p->cap + chunk - 1) / chunk);
  const int ctas = c->bits == 16 ? LongTile<16>::CTAS : LongTile<4>::CTAS;
  const int64_t all = (int64_t)fbh::num_sms() * ctas, want = (int64_t)fbh::grid_sms() * ctas;
  // One cluster per row, of up to two CTAs an SM in all, while its CTAs have few chunks; else the list.  Measured, cluster
  // against list, bf16: 4 rows of 16384 slots 18.1 / 19.0 us (16 chunks a CTA); 8 of 8192 13.6 / 15.2 (8), of 16384 24.9 /
  // 19.6; 32 of 2048 11.6 / 12.1 (4), of 4096 18.2 / 16.2; 64 of 1024 11.5 / 12.9 (4), of 2048 18.5 / 17.0; 128 of 512 12.1 /
  // 12.2 (4), of 1024 19.3 / 16.3; one chunk a CTA 5 to 8 / 7 to 11.  (Clusters that fill three CTAs an SM do not all fit:
  // 32 of 1024 took 13.5 us against 8.2.)  That choice and the workspace's size go by the device's SMs, so that they do
  // not change with the calling thread's budget.
  const int64_t rows = (int64_t)c->B * c->NKV, chunks = (p->cap + chunk - 1) / chunk;
  int64_t split = 2 * (int64_t)fbh::num_sms() / rows;
  if (split > LC_MAX) split = LC_MAX;
  if (split > chunks) split = chunks;
  const int64_t most_chunks = split == LC_MAX ? LC_CHUNKS : LC_CHUNKS / 2;
  p->split = split >= 1 && chunks <= most_chunks * split && rows <= 65535 ? (int)split : 0;
  if (p->split) {
    p->ncta = p->slices = 0;
    p->smem = scored ? (size_t)((chunks + split - 1) / split) * chunk * G * sizeof(float) : 0;
    p->ws_floats = 0;
    return FB_OK;
  }
  p->ncta = (int)(most < want ? most : want);
  FB_CHECK_ARG(rows * (chunks + 4) <= (1ll << 30), "long_decode: too many keys");
  p->slots = (most < all ? most : all) + rows;
  p->slices = scored ? (c->S + LD_SLICE - 1) / LD_SLICE : 0;
  FB_CHECK_ARG(rows * (G + p->slices) <= 0x7fffffff, "long_decode: too many rows");
  p->smem = 0;
  p->off_ml = p->slots * G * LG_D;
  p->off_own = p->off_ml + p->slots * G * 2;
  p->off_s = (p->off_own + rows * 2 + 3) / 4 * 4;
  p->ws_floats = p->off_s + (scored ? rows * p->cap * G : 0);
  return FB_OK;
}

template <int BITS, bool SCORED, bool PAGED = false>
int long_launch(LongDecodeArgs& a, const LongPlan& p, cudaStream_t st) {
  void* args[] = {(void*)&a};
  if (p.split) {
    static int attr_done[64] = {0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !attr_done[dev]) {
      cudaError_t e = cudaFuncSetAttribute(long_cluster_kernel<BITS, SCORED, PAGED>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e == cudaSuccess && SCORED)
        e = cudaFuncSetAttribute(long_cluster_kernel<BITS, SCORED, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 LC_CHUNKS * LongTile<BITS>::CHUNK * 8 * (int)sizeof(float));
      if (e != cudaSuccess) {
        fbh::set_msg("long_decode: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
        return FB_ERR_CUDA;
      }
      if (dev < 64) attr_done[dev] = 1;
    }
    return fbh::launch_pdl((const void*)long_cluster_kernel<BITS, SCORED, PAGED>, dim3(p.split, a.B * a.NKV), dim3(LD_THREADS),
                           p.smem, st, args, true, p.split);
  }
  int rc = fbh::launch_pdl((const void*)long_decode_kernel<BITS, SCORED, PAGED>, dim3(p.ncta), dim3(LD_THREADS), p.smem, st,
                           args, true);
  if (rc) return rc;
  const int rows = a.B * a.NKV, heads = rows * a.G, per = LM_THREADS / 32;
  if (p.ncta > 8 * rows)                                 // more than eight pieces a row
    return fbh::launch_pdl((const void*)long_merge_kernel<SCORED, true, PAGED>, dim3(heads + rows * p.slices), dim3(LM_THREADS), 0, st,
                           args, true);
  return fbh::launch_pdl((const void*)long_merge_kernel<SCORED, false, PAGED>, dim3((heads + per - 1) / per + rows * p.slices),
                         dim3(LM_THREADS), 0, st, args, true);
}

}  // namespace

extern "C" int64_t flashb_long_decode_ws_floats(const fb_kv_cache* cache, int NH, int window, int sinks, int scored) {
  fb::LongCache lc;
  LongPlan p{};
  if (fbh::long_cache(cache, &lc) != FB_OK || long_plan_host(cache, NH, window, sinks, scored != 0, &p) != FB_OK)
    return -1;
  return p.ws_floats;
}

extern "C" int flashb_long_decode(const fb_kv_cache* cache, const void* q, int64_t q_sb, int64_t q_sh, int NH,
                                  const int64_t* lengths, const int64_t* starts, int window, int sinks, float scaling,
                                  const float* acc, int64_t acc_sb, int64_t acc_sh, float* acc_out, int64_t acco_sb,
                                  int64_t acco_sh, float decay, float* ws, int64_t ws_floats, void* out, void* stream) {
  LongDecodeArgs a{};
  int rc = fbh::long_cache(cache, &a.c);
  if (rc) return rc;
  FB_CHECK_ARG(q && lengths && out, "long_decode: null pointer argument");
  FB_CHECK_ARG((acc == nullptr) == (acc_out == nullptr), "long_decode: acc and acc_out come together");
  if (acc) {
    const auto weights = [&](const float* w, int64_t sb, int64_t sh) {
      return fbh::long_box(w, cache->B, cache->NKV, 1, 4 * sb, 4 * sh, 0, 4ll * cache->S);
    };
    const bool in_place = acc == acc_out && (cache->B == 1 || acc_sb == acco_sb) && (cache->NKV == 1 || acc_sh == acco_sh);
    FB_CHECK_ARG(in_place || !fbh::long_boxes_meet(weights(acc, acc_sb, acc_sh), weights(acc_out, acco_sb, acco_sh)),
                 "long_decode: acc and acc_out share memory and are not the same");
    FB_CHECK_ARG(!fbh::long_box_folds(weights(acc_out, acco_sb, acco_sh)), "long_decode: rows of acc_out share memory");
  }
  LongPlan p{};
  rc = long_plan_host(cache, NH, window, sinks, acc != nullptr, &p);
  if (rc) return rc;
  FB_CHECK_ARG(((uintptr_t)q & 15) == 0 && q_sb % 8 == 0 && q_sh % 8 == 0,
               "long_decode: q must be 16-byte aligned with strides multiple of 8 elements");
  FB_CHECK_ARG(((uintptr_t)out & 7) == 0, "long_decode: out must be 8-byte aligned");   // the merge stores four values at once
  FB_CHECK_ARG(p.ws_floats == 0 || (ws && ((uintptr_t)ws & 15) == 0 && ws_floats >= p.ws_floats),
               "long_decode: workspace of %lld floats, %lld needed", (long long)ws_floats, (long long)p.ws_floats);
  a.q = (const bf16*)q, a.q_sb = q_sb, a.q_sh = q_sh;
  a.lengths = (const long long*)lengths, a.starts = (const long long*)starts;
  a.B = cache->B, a.NH = NH, a.NKV = cache->NKV, a.G = NH / cache->NKV, a.S = cache->S;
  a.window = window > 0 ? window : 0, a.sinks = sinks, a.ncta = p.ncta;
  const bool four = cache->bits == 4;
  a.scale = std::fabs(scaling) * LG_LOG2E * (four ? cache->k_scale : 1.f);
  if (a.scale == 0.f) a.scale = FLT_MIN;                 // a masked score stays -inf
  a.flip = scaling < 0.f ? 0x80008000u : 0u;
  a.dense = a.c.k_sp == (four ? 64 : 256) && a.c.v_sp == a.c.k_sp && (!four || (a.c.ks_sp == 8 && a.c.vs_sp == 8));
  a.v_scale = four ? cache->v_scale : 1.f;
  a.shift = four ? LongTile<4>::SHIFT : LongTile<16>::SHIFT;
  a.acc = acc, a.acc_out = acc_out, a.decay = decay;
  a.acc_sb = acc_sb, a.acc_sh = acc_sh, a.acco_sb = acco_sb, a.acco_sh = acco_sh;
  a.po = ws, a.ml = (float2*)(ws + p.off_ml), a.own = (int2*)(ws + p.off_own), a.sc = ws + p.off_s;
  a.per = (a.B + 31) / 32, a.slices = p.slices, a.cap = p.cap, a.out = (bf16*)out;
  const cudaStream_t s = (cudaStream_t)stream;
  if (four) return acc ? long_launch<4, true>(a, p, s) : long_launch<4, false>(a, p, s);
  return acc ? long_launch<16, true>(a, p, s) : long_launch<16, false>(a, p, s);
}

namespace {
// The list of rows as the contiguous form's host code takes it: `rows` rows of width x page slots.
fb_kv_cache paged_shape(const fb_paged_cache* c, int rows, int width) {
  fb_kv_cache s{};
  s.bits = 16, s.B = rows, s.NKV = c->NKV, s.S = width * c->page;
  return s;
}
constexpr int PAGED_EDGES = 30;        // a window's first tile and the sinks' last, at most 15 slots each
}  // namespace

extern "C" int64_t flashb_paged_decode_ws_floats(const fb_paged_cache* cache, int rows, int width, int NH, int window,
                                                 int sinks) {
  fb::PagedPool pool;
  LongPlan p{};
  if (fbh::paged_pool(cache, &pool) != FB_OK || fbh::paged_width(cache, rows, width) != FB_OK) return -1;
  const fb_kv_cache shape = paged_shape(cache, rows, width);
  if (long_plan_host(&shape, NH, window, sinks, false, &p, PAGED_EDGES) != FB_OK) return -1;
  return p.ws_floats;
}

extern "C" int flashb_paged_decode(const fb_paged_cache* cache, const int32_t* table, int64_t table_sb, int rows, int width,
                                   const int64_t* lengths, const void* q, int64_t q_st, int64_t q_sh, int NH, int window,
                                   int sinks, float scaling, float* ws, int64_t ws_floats, void* out, void* stream) {
  fb::PagedPool pool;
  int rc = fbh::paged_pool(cache, &pool);
  if (!rc) rc = fbh::paged_width(cache, rows, width);
  if (rc) return rc;
  FB_CHECK_ARG(q && lengths && out && table, "paged_decode: null pointer argument");
  FB_CHECK_ARG(table_sb >= 0, "paged_decode: table stride %lld", (long long)table_sb);
  LongDecodeArgs a{};
  LongPlan p{};
  const fb_kv_cache shape = paged_shape(cache, rows, width);
  rc = long_plan_host(&shape, NH, window, sinks, false, &p, PAGED_EDGES);
  if (rc) return rc;
  FB_CHECK_ARG(((uintptr_t)q & 15) == 0 && q_st % 8 == 0 && q_sh % 8 == 0,
               "paged_decode: q must be 16-byte aligned with strides multiple of 8 elements");
  FB_CHECK_ARG(((uintptr_t)out & 7) == 0, "paged_decode: out must be 8-byte aligned");
  FB_CHECK_ARG(scaling > 0.f && scaling * LG_LOG2E < INFINITY, "paged_decode: scaling must be positive, and finite times log2(e)");
  rc = fbh::paged_apart(pool, rows, NH, q, q_st, q_sh, out, (int64_t)NH * LG_D, LG_D);
  if (rc) return rc;
  FB_CHECK_ARG(p.ws_floats == 0 || (ws && ((uintptr_t)ws & 15) == 0 && ws_floats >= p.ws_floats),
               "paged_decode: workspace of %lld floats, %lld needed", (long long)ws_floats, (long long)p.ws_floats);
  a.c.k = pool.k, a.c.v = pool.v;
  a.c.k_sb = pool.k_sb, a.c.k_sh = pool.k_sh, a.c.k_sp = pool.k_sl;
  a.c.v_sb = pool.v_sb, a.c.v_sh = pool.v_sh, a.c.v_sp = pool.v_sl;
  a.t = fb::PagedTable{table, table_sb, pool.pages, pool.page, pool.shift};
  a.q = (const bf16*)q, a.q_sb = q_st, a.q_sh = q_sh, a.lengths = (const long long*)lengths;
  a.B = rows, a.NH = NH, a.NKV = cache->NKV, a.G = NH / cache->NKV, a.S = shape.S;
  a.window = window > 0 ? window : 0, a.sinks = sinks, a.ncta = p.ncta;
  a.scale = std::fmax(scaling * LG_LOG2E, FLT_MIN);
  a.dense = pool.k_sl == 256 && pool.v_sl == 256;
  a.v_scale = 1.f, a.shift = LongTile<16>::SHIFT, a.decay = 1.f;
  a.po = ws, a.ml = (float2*)(ws + p.off_ml), a.own = (int2*)(ws + p.off_own);
  a.per = (a.B + 31) / 32, a.cap = p.cap, a.out = (bf16*)out;
  return long_launch<16, false, true>(a, p, (cudaStream_t)stream);
}
