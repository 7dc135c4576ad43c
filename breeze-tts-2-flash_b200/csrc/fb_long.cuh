// flashb: what the long-speech kernels share (fb_long_decode.cu, fb_long_prefill.cu, fb_kv4.cu, fb_evict.cu): the
// visible keys of a cache row, the arguments of a cache, conversions between 4-bit blocks and fp16.
#pragma once
#include <cuda_fp16.h>

#include "fb_common.cuh"

namespace fb {

constexpr int LG_D = 128;        // head dim
constexpr float LG_LOG2E = 1.4426950408889634f;

// Keys of one row: slots [st, len); the token at slot len - 1 sees the first ns of them ("sinks", when the window
// does not cover them) and slots [lo, len).  Visible keys are numbered i = 0 .. n - 1 in slot order.
struct LongRow {
  int st, lo, ns, n;
  __device__ __forceinline__ long long slot(int i) const { return i < ns ? st + i : lo + (i - ns); }
  // the number of slot j, -1 if it is not visible
  __device__ __forceinline__ int index(int j) const {
    if (j >= lo) return ns + (j - lo) < n ? ns + (j - lo) : -1;
    return j >= st && j < st + ns ? j - st : -1;
  }
};
__device__ __forceinline__ LongRow long_row(long long len, long long start, int S, int window, int sinks) {
  const int e = (int)(len < 0 ? 0 : (len > S ? S : len));
  const int s = (int)(start < 0 ? 0 : (start > e ? e : start));
  LongRow r;
  r.st = s;
  r.lo = window > 0 && e - s > window ? e - window : s;   // window <= 0: no window
  r.ns = min(sinks, r.lo - s);
  r.n = r.ns + (e - r.lo);
  return r;
}

// A cache as the kernels see it: byte strides per batch row, head and position.  bits 16: rows of 128 bf16 values;
// bits 4: rows of 64 code bytes (two e2m1 codes each, the even element in the low half) and rows of 8 e4m3 scales.
struct LongCache {
  const unsigned char *k, *v, *ks, *vs;
  long long k_sb, k_sh, k_sp, v_sb, v_sh, v_sp;
  long long ks_sb, ks_sh, ks_sp, vs_sb, vs_sh, vs_sp;
};

// Two e2m1 codes per byte of w -> four half2 (byte j: low code in the low half).
__device__ __forceinline__ void e2m1x8_to_h2(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// Eight floats, already exact at rounding ties -> eight e2m1 codes (nearest, ties to even, saturated at 6).
__device__ __forceinline__ uint32_t f8_to_e2m1(const float (&f)[8]) {
  uint32_t w;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(w)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return w;
}
// Two e4m3 scales (low byte -> low half), exact in fp16; the NaN code stays NaN.
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint16_t s) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(s));
  return h;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {   // one instruction
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 f2_get(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace fb

namespace fbh {
// Checks a public cache descriptor (NULL, shapes, alignment, strides) and fills the kernels' form.
int long_cache(const fb_kv_cache* c, fb::LongCache* out);
// Rows of `row` bytes at p + i s[0] + j s[1] + k s[2], i < n[0] and so on (byte strides; long_box makes them >= 0).
struct LongBox {
  const void* p;
  long long n[3], s[3], row;
};
LongBox long_box(const void* p, int B, int NKV, long long S, long long sb, long long sh, long long sp, long long row);
// Whether two share a byte (true also where that would take too long to find out: layouts that no tensor of either has).
bool long_boxes_meet(const LongBox& a, const LongBox& b);
// Whether rows of one share a byte: a stride of 0 (an expanded tensor), or rows that do not nest.
bool long_box_folds(const LongBox& x);
// The keys, values and (4 bits) scales of a cache: how many boxes.
int long_cache_boxes(const fb_kv_cache* c, const fb::LongCache& x, LongBox (&out)[4]);
// A cache that a kernel writes: FB_OK, or a refusal where two of its slots share memory.
int long_cache_written(const fb_kv_cache* c, const fb::LongCache& x, const char* who);
}  // namespace fbh
