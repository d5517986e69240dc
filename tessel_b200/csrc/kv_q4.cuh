// The 4-bit KV cache's format, shared by the kernels that write it (kv_q4.cu) and attend over it
// (decode_attention_q4.cu, chunk_attention_q4.cu).
//
// A cache is u8 [NP, G, P, RB] with RB = D/2 + 2 ceil(D/64) bytes per token and KV head. The P * RB
// bytes of one (page, head) hold first the P tokens' codes, D/2 bytes each, then their headers,
// ceil(D/64) 16-bit words each, one for every 64 elements (the last group may be shorter).
//
// Header: an f16 scale of seven significant bits, its low four mantissa bits replaced by the zero
// point zp. value = scale * (code - zp) with code in 0..15: |code - zp| has four bits, so the
// product has at most eleven and an f16 holds it exactly. Every kernel can therefore choose where
// it multiplies (in f16 tiles, or in f32 after the dot product) and still compute on the same numbers.
//
// Codes: eight elements e0..e7 take one 32-bit word, nibbles e0 e2 e4 e6 e1 e3 e5 e7 from the low
// end, so that masking a word with 0x000f000f << 4k leaves a pair of neighbours in the two halves.
//
// Quantising 64 f16 numbers x: lo = min(0, min x), hi = max(0, max x); scale = (hi - lo) / 15 rounded
// UP to seven significant bits (below 2^-14: to a multiple of 2^-20), so 15 steps reach across;
// zp = rint(-lo / scale), code = clamp(rint(x / scale) + zp, 0, 15), where rint(x / scale) is kept to
// floor(65504 / scale) steps, so that no value passes the largest f16 number. All zeros: scale 0. A
// group that holds an infinity or a NaN gets a NaN scale and stands for NaN throughout.
#pragma once

#include "common.cuh"

namespace tb {

constexpr int Q4_GROUP = 64;

struct Q4Shape {
  int NP, G, P, D;
  __host__ __device__ int ng() const { return (D + Q4_GROUP - 1) / Q4_GROUP; }
  __host__ __device__ int row_bytes() const { return D / 2 + 2 * ng(); }
  __host__ __device__ int record() const { return P * row_bytes(); }
};

// The cache shape of an op (array `i`) whose head_dim is `D`; null, or what is wrong with it.
inline const char* q4_shape(const Op& op, int i, int64_t D, Q4Shape* out) {
  const auto& s = op.shapes[i];
  if (s.size() != 4 || op.shapes[i + 1] != s) return "the caches are two arrays [NP,G,P,D/2 + 2*ceil(D/64)]";
  if (D < 16 || D % 16 || D > 256) return "head_dim must be a multiple of 16, at most 256";
  if (s[3] != D / 2 + 2 * ((D + Q4_GROUP - 1) / Q4_GROUP)) return "a cache row has D/2 + 2*ceil(D/64) bytes";
  if (s[2] < 2 || s[2] % 2 || s[2] > 1024) return "the page size must be even, at most 1024";
  if (s[1] < 1) return "at least one kv head";
  if (s[0] > 0x7fffffffLL / s[1] || s[0] > 0x7fffffffLL / s[2]) return "the cache has too many pages";
  if (s[1] > 0x7fffffffLL / (s[2] * s[3])) return "a page is too large";
  *out = Q4Shape{(int)s[0], (int)s[1], (int)s[2], (int)D};
  return nullptr;
}

inline bool aligned_to(uint64_t p, uint64_t n) { return (p & (n - 1)) == 0; }

int make_kv_q4(Ctx* c, Op& op);
int launch_kv_q4(Ctx* c, Op& op, const uint64_t* a);
// The tensor-core kernels behind decode_attention_q4 (decode_attention_q4.cu), for the shapes they take.
bool decode_q4_takes(const Q4Shape& q, int B, int MP);
size_t decode_q4_workspace(const Ctx* c, int D);  // bytes that a launch of any size needs at most
int make_decode_q4(Ctx* c, Op& op, const Q4Shape& q);
int launch_decode_q4(Ctx* c, Op& op, const uint64_t* a, const Q4Shape& q);
// And behind chunk_attention_q4 (chunk_attention_q4.cu).
bool chunk_q4_takes(const Q4Shape& q, int T, int H, int C, int MP);
size_t chunk_q4_workspace(const Ctx* c, int D);
int make_chunk_q4(Ctx* c, Op& op, const Q4Shape& q);
int launch_chunk_q4(Ctx* c, Op& op, const uint64_t* a, const Q4Shape& q);

#ifdef __CUDACC__

__device__ __forceinline__ float q4_scale(uint32_t head) { return __half2float(__ushort_as_half((unsigned short)(head & 0xfff0u))); }
__device__ __forceinline__ float q4_zero(uint32_t head) { return (float)(head & 15u); }

// Two f32 at a time: one instruction where issue slots are short. (Each half rounds as the plain operation does.)
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void split2(uint64_t d, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"((uint64_t)src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Element `i` (0..7) of a word of codes.
__device__ __forceinline__ int q4_code(uint32_t word, int i) { return (word >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15; }

// The header for a group whose bounds are -down <= 0 <= up. The division is a product with the rounded reciprocal,
// corrected by its exact remainder: with a correctly rounded reciprocal that is the rounded quotient (Markstein; `range`
// is 0 or at least 2^-24, nothing underflows). `rest` is what the sum lost (two f16 numbers may need 41 bits): it matters
// only where the sum is 15 steps to the bit and the range is larger, which takes the next step.
__device__ __forceinline__ uint32_t q4_scale_bits(float up, float down) {
  const float range = up + down, part = range - up, rest = (up - (range - part)) + (down - part);
  const float q = range * (1.0f / 15.0f), r = fmaf(fmaf(-q, 15.0f, range), 1.0f / 15.0f, q);
  float s;
  if (r < 6.103515625e-05f)  // 2^-14: f16 subnormals, four low bits of 2^-24 units kept free (and the sum is exact)
    s = ceilf(r * 1048576.0f) * 9.5367431640625e-07f;
  else {
    s = __uint_as_float((__float_as_uint(r) + 0x1ffffu) & ~0x1ffffu);
    if (fmaf(-15.0f, s, range) + rest > 0.f) s = __uint_as_float(__float_as_uint(s) + 0x20000u);
  }
  return __half_as_ushort(__float2half_rn(s));  // exact: seven bits, at most 2 * 65504 / 15 rounded up
}

#endif  // __CUDACC__

}  // namespace tb
