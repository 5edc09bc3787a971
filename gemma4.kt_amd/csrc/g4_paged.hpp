// g4_paged.hpp -- what the attention kernels over a paged cache share: rows and what
// they see, cached elements, and operands of the matrix cores.
#pragma once

#include "g4_device.hpp"
#include "g4_internal.hpp"

namespace g4 {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.4426950408889634f;

// What a row sees: visible index j < ns is token j, later ones are token j + skip.
struct Seen {
  int count;
  int ns;
  int skip;
};

G4_DEV Seen seen_by(int pos, int window, int sinks) {
  Seen s;
  const int from = window > 0 ? max(0, pos - window + 1) : 0;
  s.ns = min(sinks, from);
  s.skip = from - s.ns;
  s.count = pos + 1 - s.skip;
  return s;
}

G4_DEV bool page_ok(int page, const KvArgs &kv) { return (unsigned)page < (unsigned)kv.n_pages; }

// Eight elements of a cached row as they are loaded, and as fp32.
template <int TYPE>
struct Raw8 {
  u32x4 w[TYPE == T_F32 ? 2 : 1];
  G4_DEV void load(const char *base, int64_t elem) {
    const u32x4 *p = (const u32x4 *)(base + elem * (TYPE == T_F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (TYPE == T_F32 ? 2 : 1); ++i) w[i] = p[i];
  }
  G4_DEV void zero() {
#pragma unroll
    for (int i = 0; i < (TYPE == T_F32 ? 2 : 1); ++i) w[i] = u32x4{0, 0, 0, 0};
  }
  G4_DEV void floats(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (TYPE == T_F32) f[i] = __uint_as_float(w[i >> 2][i & 3]);
      else if constexpr (TYPE == T_F16) f[i] = i & 1 ? f16hi(w[0][i >> 1]) : f16lo(w[0][i >> 1]);
      else f[i] = __uint_as_float(i & 1 ? w[0][i >> 1] & 0xFFFF0000u : w[0][i >> 1] << 16);
    }
  }
};

// a / b for a >= 0, b > 0; long division only where the numbers are long
G4_DEV int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// count up to a multiple of pad
G4_DEV int padded(int count, int pad) { return pad == 1 ? count : (count + pad - 1) / pad * pad; }

// v + the value of lane ^ S; for S = 16 and 32 one swap gives both sides in every lane
template <int S>
G4_DEV float add_partner(float v, int lane) {
  if constexpr (S == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else if constexpr (S == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else {
    return v + __uint_as_float(partner_u32<S>(__float_as_uint(v), lane));
  }
}

template <int N>
G4_DEV float lanes_sum(float s, int lane) {  // over each aligned group of N lanes, in every lane of it
  if constexpr (N > 1) s = add_partner<1>(s, lane);
  if constexpr (N > 2) s = add_partner<2>(s, lane);
  if constexpr (N > 4) s = add_partner<4>(s, lane);
  if constexpr (N > 8) s = add_partner<8>(s, lane);
  if constexpr (N > 16) s = add_partner<16>(s, lane);
  if constexpr (N > 32) s = add_partner<32>(s, lane);
  return s;
}

// 2^(a - b), b >= a, where both may be -infinity (nothing seen yet, or a hidden token)
G4_DEV float shrink(float a, float b) { return a == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(a - b); }

template <int TYPE>
struct Mfma;
template <>
struct Mfma<T_F32> {
  static constexpr int STEP = 16;  // dims of a step: 4 adjacent ones per lane
  G4_DEV static f32x4 step(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
};
template <>
struct Mfma<T_F16> {
  static constexpr int STEP = 32;  // 8 adjacent ones per lane
  G4_DEV static f32x4 step(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mfma<T_BF16> {
  static constexpr int STEP = 32;
  G4_DEV static f32x4 step(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

// Two fp32 values' next 16-bit parts, in one word; the values become the remainders.
// BF16 truncates: three parts hold the 24 bits of a finite value.  F16 rounds to
// nearest, 11 bits and a sign a part, on steps of 2^-24 at least.
template <int TYPE>
G4_DEV uint32_t take_part(float &x, float &y) {
  if constexpr (TYPE == T_BF16) {
    const uint32_t a = __float_as_uint(x) & 0xFFFF0000u, b = __float_as_uint(y) & 0xFFFF0000u;
    x -= __uint_as_float(a);
    y -= __uint_as_float(b);
    return (a >> 16) | b;
  } else {
    const _Float16 a = (_Float16)x, b = (_Float16)y;
    x -= (float)a;
    y -= (float)b;
    return (uint32_t)__builtin_bit_cast(uint16_t, a) | (uint32_t)__builtin_bit_cast(uint16_t, b) << 16;
  }
}

// The power of two that a query of this size (its largest element's) is multiplied by
// before it is split, and its inverse.  F16: to [2^14, 2^15), the highest that no part
// overflows, since parts stand on steps of 2^-24: what they leave out of an element is at
// most 2^-39 of the largest one (2^-25 with that at 1), or 2^-22 of itself with two parts, none with
// three.  An F16 key is at most 65504, so sums stay below 2^40.  BF16: only queries so
// small that their parts would be subnormal.  1 where nothing is split.
template <int TYPE>
G4_DEV void split_scale(float size, float &to, float &back) {
  to = back = 1.f;
  if constexpr (TYPE == T_F16) {
    const uint32_t e = max(__float_as_uint(size) >> 23 & 255, 15u);  // the inverse stays normal
    to = __uint_as_float((268u - e) << 23), back = __uint_as_float((e - 14u) << 23);
  } else if constexpr (TYPE == T_BF16) {
    if (size < 0x1p-80f) to = 0x1p40f, back = 0x1p-40f;
  }
}

G4_DEV float lanes16_max(float v, int lane) {
  v = fmaxf(v, __uint_as_float(partner_u32<1>(__float_as_uint(v), lane)));
  v = fmaxf(v, __uint_as_float(partner_u32<2>(__float_as_uint(v), lane)));
  v = fmaxf(v, __uint_as_float(partner_u32<4>(__float_as_uint(v), lane)));
  return fmaxf(v, __uint_as_float(partner_u32<8>(__float_as_uint(v), lane)));
}

// An offset that is the same in all lanes, in scalar registers: loads then take a scalar
// base and 32 bits of offset a lane.
G4_DEV int64_t uniform(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// Values that are formed here, before what follows: loads into the registers of their
// operands would otherwise be moved ahead, and the operands copied.
template <int N>
G4_DEV void formed(float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i]));
}

}  // namespace g4
