// flashb: a KV cache held in 4 bits -- storing bf16 heads into it and reading them back.
//
// A head's 128 values are 8 blocks of 16.  With x the block divided by the tensor scale (a power of two):
//   s = e4m3(max |x| / 6),  code = e2m1(x / s) (values 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign),  value = code s
// both to nearest, ties to even; s saturates at 448 (values beyond 6 s at 6 s), s = 0 gives zeros, and a block with a
// NaN or an infinity gets s = NaN.  64 bytes of codes and 8 of scales stand for 256 bytes of bf16.
//
// The quotients are formed as products with an fp32 reciprocal.  A bf16 x over an e4m3 s lies on a rounding tie of
// the target or at least 2^-9 of itself away from it (8 + 4 significant bits against the tie's 3; the same for
// max / 6 with 8 against 7), while the product is off by less than 2^-22: rounding it to 16 fraction bits puts every
// tie exactly on the tie and leaves all others on their side, so the codes are those of exact arithmetic.
//
// Bound: HBM, 328 bytes a head and token.  A thread owns 8 values (one 16-byte load, 4 bytes of codes); its block's
// maximum is one shuffle away.
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
  float k_scale, v_scale;
};

// x to 16 fraction bits, nearest (see the header); NaN and infinity pass
__device__ __forceinline__ float snap16(float x) {
  return isfinite(x) ? __uint_as_float((__float_as_uint(x) + 0x40u) & 0xffffff80u) : x;
}
__device__ __forceinline__ unsigned char f_to_e4m3(float x) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(x));
  return (unsigned char)(r & 0xff);
}

// Block of 16 threads per head: grid (tokens / rows per CTA, B * NKV, K | V)
__global__ void __launch_bounds__(256) kv4_store_kernel(const __grid_constant__ KV4Args a) {
  pdl_wait();
  pdl_trigger();
  const int l = blockIdx.x * (blockDim.x >> 4) + (threadIdx.x >> 4), j = threadIdx.x & 15;
  const int b = blockIdx.y / a.NKV, h = blockIdx.y - b * a.NKV;
  const bool is_v = blockIdx.z != 0;
  const long long slot = l < a.L ? a.slots[b * a.slot_sb + l] : -1;
  const bool ok = slot >= 0 && slot < a.S;
  float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (ok) {
    const bf16* x = is_v ? a.v + b * a.xv_sb + h * a.xv_sh + l * a.xv_sl : a.k + b * a.xk_sb + h * a.xk_sh + l * a.xk_sl;
    cvt8(ld_nc_v4(x + 8 * j), f);
  }
  const float down = 1.0f / (is_v ? a.v_scale : a.k_scale);   // a power of two: exact
  float amax = 0.f;
  bool odd = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    odd |= !isfinite(f[e]);
    f[e] *= down;                                             // may overflow: saturates below
    amax = fmaxf(amax, fabsf(f[e]));
  }
  amax = fmaxf(amax, __shfl_xor_sync(FULL, amax, 1));
  odd |= __shfl_xor_sync(FULL, (int)odd, 1) != 0;
  unsigned char sb = f_to_e4m3(snap16(amax * (1.0f / 6.0f)));
  const float s = __half2float(__ushort_as_half((unsigned short)(e4m3x2_to_h2(sb) & 0xffffu)));
  const float inv = s > 0.f ? 1.0f / s : 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = odd || s == 0.f ? 0.f : snap16(f[e] * inv);
  if (odd) sb = 0x7f;
  if (!ok) return;
  unsigned char* q = is_v ? a.vq + b * a.v_sb + h * a.v_sh + slot * a.v_sp : a.kq + b * a.k_sb + h * a.k_sh + slot * a.k_sp;
  unsigned char* sc =
      is_v ? a.vs + b * a.vs_sb + h * a.vs_sh + slot * a.vs_sp : a.ks + b * a.ks_sb + h * a.ks_sh + slot * a.ks_sp;
  *reinterpret_cast<uint32_t*>(q + 4 * j) = f8_to_e2m1(f);
  if ((j & 1) == 0) sc[j >> 1] = sb;
}

__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ KV4Args a) {
  pdl_wait();
  pdl_trigger();
  const int l = blockIdx.x * (blockDim.x >> 4) + (threadIdx.x >> 4), j = threadIdx.x & 15;
  if (l >= a.L) return;
  const int b = blockIdx.y / a.NKV, h = blockIdx.y - b * a.NKV;
  const bool is_v = blockIdx.z != 0;
  const long long slot = a.slots[b * a.slot_sb + l];
  uint4 w = make_uint4(0, 0, 0, 0);
  if (slot >= 0 && slot < a.S) {
    const unsigned char* q =
        is_v ? a.vq + b * a.v_sb + h * a.v_sh + slot * a.v_sp : a.kq + b * a.k_sb + h * a.k_sh + slot * a.k_sp;
    const unsigned char* sc =
        is_v ? a.vs + b * a.vs_sb + h * a.vs_sh + slot * a.vs_sp : a.ks + b * a.ks_sb + h * a.ks_sh + slot * a.ks_sp;
    const float up = is_v ? a.v_scale : a.k_scale;
    uint32_t x[4];
    e2m1x8_to_h2(*reinterpret_cast<const uint32_t*>(q + 4 * j), x);
    const uint32_t s2 = e4m3x2_to_h2((uint16_t)(sc[j >> 1] * 0x0101u));
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t p = hmul2(x[e], s2);   // exact in fp16: 2 + 4 significant bits, 2^-10 .. 2688
      o[e] = pack2(__half2float(__ushort_as_half((unsigned short)(p & 0xffffu))) * up,
                   __half2float(__ushort_as_half((unsigned short)(p >> 16))) * up);
    }
    w = make_uint4(o[0], o[1], o[2], o[3]);
  }
  bf16* out = (is_v ? a.vo : a.ko) + ((long long)blockIdx.y * a.L + l) * LG_D + 8 * j;
  *reinterpret_cast<uint4*>(out) = w;
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
  return FB_OK;
}

int kv4_launch(const void* kern, KV4Args& a, int rows, cudaStream_t st) {
  int per = 2;                                   // heads per CTA: a warp at least, 16 at most
  while (per < 16 && per < a.L) per *= 2;
  void* args[] = {(void*)&a};
  return fbh::launch_pdl(kern, dim3((a.L + per - 1) / per, rows, 2), dim3(16 * per), 0, st, args, true);
}

}  // namespace

extern "C" int flashb_kv4_store(const fb_kv_cache* cache, const void* k, int64_t k_sb, int64_t k_sh, int64_t k_sl,
                                const void* v, int64_t v_sb, int64_t v_sh, int64_t v_sl, const int64_t* slots,
                                int64_t slot_sb, int L, void* stream) {
  KV4Args a{};
  const int rc = kv4_fill(cache, slots, slot_sb, L, &a);
  if (rc) return rc;
  FB_CHECK_ARG(k && v, "kv4_store: null pointer argument");
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
