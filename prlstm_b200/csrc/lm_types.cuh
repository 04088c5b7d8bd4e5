// Element types of the language-model operators (gated_recurrence.cu,
// embedding.cu, token_logprobs.cu): float32, bfloat16 and float16 tensors,
// float32 arithmetic.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "hs_common.cuh"

namespace hs {

inline bool dtype_ok(int dtype) { return dtype == HS_F32 || dtype == HS_BF16 || dtype == HS_F16; }
inline size_t dtype_bytes(int dtype) { return dtype == HS_F32 ? 4 : 2; }

// Records a failure in a status word that may lie in pinned host memory (a
// call writes one code only, so a plain store will do).
HS_DEV void report(int *p, int code) { *reinterpret_cast<volatile int *>(p) = code; }

template <typename T> HS_DEV float to_f32(T v);
template <> HS_DEV float to_f32<float>(float v) { return v; }
template <> HS_DEV float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> HS_DEV float to_f32<__half>(__half v) { return __half2float(v); }

template <typename T> HS_DEV T from_f32(float v);
template <> HS_DEV float from_f32<float>(float v) { return v; }
template <> HS_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> HS_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }

// The values held by one 32-bit word: one float32 or two 16-bit values.
template <typename T> HS_DEV void unpack_word(unsigned w, float *v);
template <> HS_DEV void unpack_word<float>(unsigned w, float *v) { v[0] = __uint_as_float(w); }
template <> HS_DEV void unpack_word<__nv_bfloat16>(unsigned w, float *v) {
  v[0] = __uint_as_float(w << 16);
  v[1] = __uint_as_float(w & 0xffff0000u);
}
template <> HS_DEV void unpack_word<__half>(unsigned w, float *v) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
  v[0] = f.x;
  v[1] = f.y;
}

template <typename T> HS_DEV unsigned pack_word(const float *v);
template <> HS_DEV unsigned pack_word<float>(const float *v) { return __float_as_uint(v[0]); }
template <> HS_DEV unsigned pack_word<__nv_bfloat16>(const float *v) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(v[0], v[1]);
  return *reinterpret_cast<const unsigned *>(&p);
}
template <> HS_DEV unsigned pack_word<__half>(const float *v) {
  const __half2 p = __floats2half2_rn(v[0], v[1]);
  return *reinterpret_cast<const unsigned *>(&p);
}

// The larger of each value of two words of 16-bit values, NaN left out.
template <typename T> HS_DEV unsigned word_max(unsigned a, unsigned b);
template <> HS_DEV unsigned word_max<__nv_bfloat16>(unsigned a, unsigned b) {
  unsigned r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <> HS_DEV unsigned word_max<__half>(unsigned a, unsigned b) {
  unsigned r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// A word of -inf.
template <typename T> __host__ __device__ constexpr unsigned minus_inf_word();
template <> __host__ __device__ constexpr unsigned minus_inf_word<float>() { return 0xff800000u; }
template <> __host__ __device__ constexpr unsigned minus_inf_word<__nv_bfloat16>() { return 0xff80ff80u; }
template <> __host__ __device__ constexpr unsigned minus_inf_word<__half>() { return 0xfc00fc00u; }

template <typename T> struct PerWord { static constexpr int value = 4 / (int)sizeof(T); };

// One float32, or two as one pair of registers that sm_100a's packed float32
// instructions take at once.
template <int VEC> struct Cols;
template <> struct Cols<1> {
  float v;
  HS_DEV static Cols all(float a) { return {a}; }
  HS_DEV static Cols of(const float *a) { return {a[0]}; }
  HS_DEV void get(float *a) const { a[0] = v; }
};
template <> struct Cols<2> {
  unsigned long long v;
  HS_DEV static Cols of(const float *a) {
    Cols r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a[0]), "f"(a[1]));
    return r;
  }
  HS_DEV static Cols all(float a) {
    const float t[2] = {a, a};
    return of(t);
  }
  HS_DEV void get(float *a) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a[0]), "=f"(a[1]) : "l"(v)); }
};
HS_DEV Cols<1> operator+(Cols<1> a, Cols<1> b) { return {a.v + b.v}; }
HS_DEV Cols<1> operator-(Cols<1> a, Cols<1> b) { return {a.v - b.v}; }
HS_DEV Cols<1> operator*(Cols<1> a, Cols<1> b) { return {__fmul_rn(a.v, b.v)}; }
HS_DEV Cols<1> fma(Cols<1> a, Cols<1> b, Cols<1> c) { return {fmaf(a.v, b.v, c.v)}; }
HS_DEV Cols<2> fma(Cols<2> a, Cols<2> b, Cols<2> c) {
  Cols<2> r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
HS_DEV Cols<2> operator+(Cols<2> a, Cols<2> b) {
  Cols<2> r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
HS_DEV Cols<2> operator*(Cols<2> a, Cols<2> b) {
  Cols<2> r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
HS_DEV Cols<2> operator-(Cols<2> a, Cols<2> b) { return fma(b, Cols<2>::all(-1.f), a); }

}  // namespace hs
