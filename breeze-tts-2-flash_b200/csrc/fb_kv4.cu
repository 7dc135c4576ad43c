// flashb: a KV cache held in 4 bits -- storing bf16 heads into it and reading them back.
//
// A head's 128 values are 8 blocks of 16.  With x the block divided by the tensor scale (a power of two):
//   s = e4m3(max |x| / 6),  code = e2m1(x / s) (values 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign),  value = code s
// both to nearest, ties to even; s saturates at 448 (values beyond 6 s at 6 s), s = 0 gives zeros, and a block with a
// NaN or an infinity gets s = NaN.  64 bytes of codes and 8 of scales stand for 256 bytes of bf16.
//
// The quotients are formed as products with an fp32 reciprocal, off by less than 2^-22 of themselves.  A bf16 x over an
// e4m3 s lies on a rounding tie of the target (0.25 .. 5) or at least 2^-9 of itself away from it (8 + 4 significant bits
// against the tie's 3): rounding the product to a multiple of 2^-15 puts every tie exactly on the tie and leaves all
// others on their side, so the codes are those of exact arithmetic.  That rounding is the addition of 384 in the same
// fused multiply-add, and its subtraction, two values an instruction.  max / 6 is rounded to 16 fraction bits in the same
// way (8 significant bits against the tie's 7).
//
// Bound: HBM, 328 bytes a head and token.  Measured on a B200: 8 x 4097 tokens of 4 heads, K and V, 28.2 us stored and read
// back (0.93 of the measured copy bandwidth; the read finds the codes in L2); a token of 128 rows 3.7 us.  A thread owns a
// block (two 16-byte loads, 8 bytes of codes, one scale), so the block's maximum, scale and reciprocal are its own; the
// maximum is taken on the bf16 bit patterns, two at a time, where a NaN or an infinity shows as the largest.
#include "fb_long.cuh"

namespace fb {

struct KV4Args {
  unsigned char *kq, *vq, *ks, *vs;
  long long k_sb, k_sh, k_sp, v_sb, v_sh, v_sp, ks_sb, ks_sh, ks_sp, vs_sb, vs_sh, vs_sp;
  const bf16 *k, *v;                       // store: the heads to store
  long long xk_sb, xk_sh, xk_sl, xv_sb, xv_sh, xv_sl;
  bf16 *ko, *vo;                           // read: [B, NKV, L, 128] contiguous
  const long long* slots;
  long long slot_sb;
  int NKV, L, S;
  float k_scale, v_scale, k_inv, v_inv;    // powers of two and their inverses
};

// x to 16 fraction bits, nearest (see the header); an infinity stays one
__device__ __forceinline__ float snap16(float x) { return __uint_as_float((__float_as_uint(x) + 0x40u) & 0xffffff80u); }
__device__ __forceinline__ unsigned char f_to_e4m3(float x) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(x));
  return (unsigned char)(r & 0xff);
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A thread's two 16-byte units of a row and its neighbour's are four in a row, (0, 1) and (2, 3).  Written as (0, 2) and
// (1, 3) each store of the two covers whole 32-byte sectors: the read kernel takes 15.2 us instead of 20.8 at 8 x 4097
// tokens.  (Loads come through the cache either way; the exchange made the store kernel 2 us slower.)
__device__ __forceinline__ void swap_units(uint4& a, uint4& b) {
  const bool second = threadIdx.x & 1;
  uint4 x = second ? a : b;                                     // what the neighbour is to have
  x.x = __shfl_xor_sync(FULL, x.x, 1);
  x.y = __shfl_xor_sync(FULL, x.y, 1);
  x.z = __shfl_xor_sync(FULL, x.z, 1);
  x.w = __shfl_xor_sync(FULL, x.w, 1);
  if (second) a = x;
  else b = x;
}

// Eight threads per head, KV4_ROWS tokens each (their loads together): grid (tokens, B * NKV, K | V)
constexpr int KV4_ROWS = 2;

__global__ void __launch_bounds__(256) kv4_store_kernel(const __grid_constant__ KV4Args a) {
  pdl_wait();
  pdl_trigger();
  const int per = blockDim.x >> 3, l0 = blockIdx.x * per * KV4_ROWS + (threadIdx.x >> 3), j = threadIdx.x & 7;
  const int b = blockIdx.y / a.NKV, h = blockIdx.y - b * a.NKV;
  const bool is_v = blockIdx.z != 0;
  const bf16* x = (is_v ? a.v + b * a.xv_sb + h * a.xv_sh : a.k + b * a.xk_sb + h * a.xk_sh) + 16 * j;
  const long long sl = is_v ? a.xv_sl : a.xk_sl;
  uint32_t w[KV4_ROWS][8];
  long long slot[KV4_ROWS];
#pragma unroll
  for (int i = 0; i < KV4_ROWS; ++i) {
    const int l = l0 + i * per;
    slot[i] = -1;
    uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
    if (l < a.L) {
      lo = ld_nc_v4(x + l * sl);
      hi = ld_nc_v4(x + l * sl + 8);
      slot[i] = a.slots[b * a.slot_sb + l];
    }
    w[i][0] = lo.x, w[i][1] = lo.y, w[i][2] = lo.z, w[i][3] = lo.w;
    w[i][4] = hi.x, w[i][5] = hi.y, w[i][6] = hi.z, w[i][7] = hi.w;
  }
  const float down = is_v ? a.v_inv : a.k_inv;
  unsigned char* qp = (is_v ? a.vq + b * a.v_sb + h * a.v_sh : a.kq + b * a.k_sb + h * a.k_sh) + 8 * j;
  unsigned char* sc = (is_v ? a.vs + b * a.vs_sb + h * a.vs_sh : a.ks + b * a.ks_sb + h * a.ks_sh) + j;
  const long long sp = is_v ? a.v_sp : a.k_sp, ssp = is_v ? a.vs_sp : a.ks_sp;
#pragma unroll
  for (int i = 0; i < KV4_ROWS; ++i) {
    if (slot[i] < 0 || slot[i] >= a.S) continue;
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = __vmaxu2(top, w[i][e] & 0x7fff7fffu);
    top = max(top & 0xffffu, top >> 16);
    const bool odd = top >= 0x7f80u;                            // a NaN or an infinity
    unsigned char sb = f_to_e4m3(snap16(__uint_as_float(top << 16) * down * (1.0f / 6.0f)));   // overflow saturates
    const float s = __half2float(__ushort_as_half((unsigned short)(e4m3x2_to_h2(sb) & 0xffffu)));
    const float inv = odd || s == 0.f ? 0.f : rcp(s) * down;
    uint32_t q[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float f[8];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float2 y = f2_get(f2_add(f2_fma(f2(lo_f(w[i][4 * e + c]), hi_f(w[i][4 * e + c])), f2(inv, inv), f2(384.f, 384.f)),
                                       f2(-384.f, -384.f)));
        f[2 * c] = y.x;
        f[2 * c + 1] = y.y;
      }
      q[e] = inv == 0.f ? 0u : f8_to_e2m1(f);
    }
    if (odd) sb = 0x7f;
    *reinterpret_cast<uint2*>(qp + slot[i] * sp) = make_uint2(q[0], q[1]);
    sc[slot[i] * ssp] = sb;
  }
}

__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ KV4Args a) {
  pdl_wait();
  pdl_trigger();
  const int per = blockDim.x >> 3, l0 = blockIdx.x * per * KV4_ROWS + (threadIdx.x >> 3), j = threadIdx.x & 7;
  const int b = blockIdx.y / a.NKV, h = blockIdx.y - b * a.NKV;
  const bool is_v = blockIdx.z != 0;
  const unsigned char* qp = (is_v ? a.vq + b * a.v_sb + h * a.v_sh : a.kq + b * a.k_sb + h * a.k_sh) + 8 * j;
  const unsigned char* sc = (is_v ? a.vs + b * a.vs_sb + h * a.vs_sh : a.ks + b * a.ks_sb + h * a.ks_sh) + j;
  const long long sp = is_v ? a.v_sp : a.k_sp, ssp = is_v ? a.vs_sp : a.ks_sp;
  long long slot[KV4_ROWS];
  uint2 w[KV4_ROWS];
  unsigned char sb[KV4_ROWS];
#pragma unroll
  for (int i = 0; i < KV4_ROWS; ++i) slot[i] = l0 + i * per < a.L ? a.slots[b * a.slot_sb + l0 + i * per] : -1;
#pragma unroll
  for (int i = 0; i < KV4_ROWS; ++i) {
    w[i] = make_uint2(0u, 0u);
    sb[i] = 0;
    if (slot[i] >= 0 && slot[i] < a.S) {
      w[i] = *reinterpret_cast<const uint2*>(qp + slot[i] * sp);
      sb[i] = sc[slot[i] * ssp];
    }
  }
  const float up = is_v ? a.v_scale : a.k_scale;
  bf16* op = (is_v ? a.vo : a.ko) + (long long)blockIdx.y * a.L * LG_D + 32 * (j >> 1) + 8 * (j & 1);
#pragma unroll
  for (int i = 0; i < KV4_ROWS; ++i) {
    const int l = l0 + i * per;
    const float s = __half2float(__ushort_as_half((unsigned short)(e4m3x2_to_h2(sb[i]) & 0xffffu))) * up;
    uint32_t o[8];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint32_t x[4];
      e2m1x8_to_h2(e ? w[i].y : w[i].x, x);
#pragma unroll
      for (int c = 0; c < 4; ++c) {                           // 2 + 4 significant bits: exact in bf16
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[c]));
        const float2 y = f2_get(f2_mul(f2(f.x, f.y), f2(s, s)));
        o[4 * e + c] = pack_bf16(y.x, y.y);
      }
    }
    uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
    swap_units(lo, hi);
    if (l < a.L) {
      *reinterpret_cast<uint4*>(op + (long long)l * LG_D) = lo;
      *reinterpret_cast<uint4*>(op + (long long)l * LG_D + 16) = hi;
    }
  }
}

}  // namespace fb

namespace {
using namespace fb;

int kv4_fill(const fb_kv_cache* c, const int64_t* slots, int64_t slot_sb, int L, KV4Args* a) {
  LongCache lc;
  const int rc = fbh::long_cache(c, &lc);
  if (rc) return rc;
  FB_CHECK_ARG(c->bits == 4, "kv4: the cache holds %d bits", c->bits);
  FB_CHECK_ARG(slots, "kv4: null slots");
  FB_CHECK_ARG(L >= 1 && slot_sb >= 0, "kv4: bad slots L=%d", L);
  FB_CHECK_ARG((int64_t)c->B * c->NKV <= 65535, "kv4: more than 65535 rows and heads");
  a->kq = (unsigned char*)c->k, a->vq = (unsigned char*)c->v, a->ks = (unsigned char*)c->ks, a->vs = (unsigned char*)c->vs;
  a->k_sb = lc.k_sb, a->k_sh = lc.k_sh, a->k_sp = lc.k_sp, a->v_sb = lc.v_sb, a->v_sh = lc.v_sh, a->v_sp = lc.v_sp;
  a->ks_sb = lc.ks_sb, a->ks_sh = lc.ks_sh, a->ks_sp = lc.ks_sp;
  a->vs_sb = lc.vs_sb, a->vs_sh = lc.vs_sh, a->vs_sp = lc.vs_sp;
  a->slots = (const long long*)slots, a->slot_sb = slot_sb;
  a->NKV = c->NKV, a->L = L, a->S = c->S, a->k_scale = c->k_scale, a->v_scale = c->v_scale;
  a->k_inv = 1.0f / c->k_scale, a->v_inv = 1.0f / c->v_scale;
  return FB_OK;
}

int kv4_launch(const void* kern, KV4Args& a, int rows, cudaStream_t st) {
  int per = 4;                                   // heads per CTA: a warp at least, 32 at most
  while (per < 32 && per < a.L) per *= 2;
  void* args[] = {(void*)&a};
  return fbh::launch_pdl(kern, dim3((a.L + per * KV4_ROWS - 1) / (per * KV4_ROWS), rows, 2), dim3(8 * per), 0, st, args, true);
}

}  // namespace

extern "C" int flashb_kv4_store(const fb_kv_cache* cache, const void* k, int64_t k_sb, int64_t k_sh, int64_t k_sl,
                                const void* v, int64_t v_sb, int64_t v_sh, int64_t v_sl, const int64_t* slots,
                                int64_t slot_sb, int L, void* stream) {
  KV4Args a{};
  int rc = kv4_fill(cache, slots, slot_sb, L, &a);
  if (rc) return rc;
  FB_CHECK_ARG(k && v, "kv4_store: null pointer argument");
  LongCache lc;
  fbh::long_cache(cache, &lc);
  rc = fbh::long_cache_written(cache, lc, "kv4_store");
  if (rc) return rc;
  FB_CHECK_ARG((((uintptr_t)k | (uintptr_t)v) & 15) == 0 && (k_sb | k_sh | k_sl | v_sb | v_sh | v_sl) % 8 == 0,
               "kv4_store: keys and values must be 16-byte aligned with strides multiple of 8 elements");
  a.k = (const bf16*)k, a.xk_sb = k_sb, a.xk_sh = k_sh, a.xk_sl = k_sl;
  a.v = (const bf16*)v, a.xv_sb = v_sb, a.xv_sh = v_sh, a.xv_sl = v_sl;
  return kv4_launch((const void*)kv4_store_kernel, a, cache->B * cache->NKV, (cudaStream_t)stream);
}

extern "C" int flashb_kv4_read(const fb_kv_cache* cache, const int64_t* slots, int64_t slot_sb, int L, void* k_out,
                               void* v_out, void* stream) {
  KV4Args a{};
  const int rc = kv4_fill(cache, slots, slot_sb, L, &a);
  if (rc) return rc;
  FB_CHECK_ARG(k_out && v_out && (((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0,
               "kv4_read: outputs null or not 16-byte aligned");
  a.ko = (bf16*)k_out, a.vo = (bf16*)v_out;
  return kv4_launch((const void*)kv4_read_kernel, a, cache->B * cache->NKV, (cudaStream_t)stream);
}
