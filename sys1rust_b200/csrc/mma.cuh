// Warp-level f16 products and their operands from 16-bit and 8-bit values.
#pragma once
#include <utility>

#include "common.cuh"

namespace s1c {

// A 16-bit value of type T in the bits of v.
template <typename T>
S1C_DEV float bits_f32(uint16_t v) { return to_f32(*reinterpret_cast<T*>(&v)); }

// Two values in one word, the first in the low half, each rounded once.
template <typename T>
S1C_DEV uint32_t pack2(float lo, float hi);
template <>
S1C_DEV uint32_t pack2<__half>(float lo, float hi) { return pack_f16x2(lo, hi); }
template <>
S1C_DEV uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }

// The larger of two; NaN where one is.
S1C_DEV float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// 16 bytes that are read once.
S1C_DEV uint4 ld_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// 32 bytes at a 32-byte boundary, in one access: a warp's stores fill whole sectors.
S1C_DEV void st_32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// D += A B, f16 in, fp32 sums: a 16 x 16 (row), b 16 x 8 (column).
S1C_DEV void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Loads from shared memory at an address and a constant offset.
template <int OFF>
S1C_DEV uint32_t lds_u32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(v) : "r"(at), "n"(OFF));
  return v;
}
template <int OFF>
S1C_DEV float lds_f32(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1 + %2];" : "=f"(v) : "r"(at), "n"(OFF));
  return v;
}
template <int OFF>
S1C_DEV uint2 lds_v2(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2 + %3];" : "=r"(v.x), "=r"(v.y) : "r"(at), "n"(OFF));
  return v;
}
template <int OFF>
S1C_DEV uint4 lds_v4(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at), "n"(OFF));
  return v;
}
// f(integral_constant 0), ..., f(integral_constant N - 1).
template <typename F, int... I>
S1C_DEV void static_for_(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
S1C_DEV void static_for(F&& f) {
  static_for_(f, std::make_integer_sequence<int, N>{});
}

// Two codes + 128 under the exponent of 1024 (1024 + 128 + code) to two f16 codes.
S1C_DEV uint32_t code_pair(uint32_t v) {
  const uint32_t base = 0x64806480u;  // 1152
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&base));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// 2^x to about 2^-22; 0 for -inf.
S1C_DEV float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace s1c
