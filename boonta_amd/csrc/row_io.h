// Units of 8 columns of a row stored as float32 or bf16, moved 16 bytes at a
// time from any element's address (the hardware takes unaligned vector loads
// and stores), and a row's sequence and step from its number.
#pragma once
#include "split_f32.h"

namespace ppo {

constexpr int UNIT = 8;  // columns

// 8 values as stored.
template <typename S> struct Unit8;
template <> struct Unit8<uint16_t> { uint32_t w[4]; };
template <> struct Unit8<float> { uint32_t w[8]; };

// The unit at p of which `left` columns (of any number) exist; the others are zeros.
__device__ __forceinline__ void load_unit(const uint16_t* p, int left, Unit8<uint16_t>& u) {
  if (left >= UNIT) {
    __builtin_memcpy(u.w, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = 2 * i < left ? p[2 * i] : 0, hi = 2 * i + 1 < left ? p[2 * i + 1] : 0;
      u.w[i] = lo | hi << 16;
    }
  }
}
__device__ __forceinline__ void load_unit(const float* p, int left, Unit8<float>& u) {
  if (left >= UNIT) {
    __builtin_memcpy(u.w, p, 32);
  } else {
#pragma unroll
    for (int j = 0; j < UNIT; ++j) u.w[j] = j < left ? __float_as_uint(p[j]) : 0;
  }
}
// A whole unit that is read once: kept out of the caches' way (7.0 TB/s for 6.2 reading 1 GB).
typedef uint32_t uintx4u __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ void load_unit_once(const uint16_t* p, Unit8<uint16_t>& u) {
  const uintx4u v = __builtin_nontemporal_load(reinterpret_cast<const uintx4u*>(p));
  u.w[0] = v[0]; u.w[1] = v[1]; u.w[2] = v[2]; u.w[3] = v[3];
}
__device__ __forceinline__ void load_unit_once(const float* p, Unit8<float>& u) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uintx4u v = __builtin_nontemporal_load(reinterpret_cast<const uintx4u*>(p + 4 * h));
#pragma unroll
    for (int j = 0; j < 4; ++j) u.w[4 * h + j] = v[j];
  }
}
__device__ __forceinline__ float value(const Unit8<uint16_t>& u, int j) {
  return __uint_as_float(j & 1 ? u.w[j / 2] & 0xffff0000u : u.w[j / 2] << 16);
}
__device__ __forceinline__ float value(const Unit8<float>& u, int j) { return __uint_as_float(u.w[j]); }

// Rounded to nearest even where the storage is bf16; columns past `left` are not written.
__device__ __forceinline__ void store_unit(uint16_t* p, int left, const float (&v)[UNIT]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
  if (left >= UNIT) {
    __builtin_memcpy(p, w, 16);
  } else {
#pragma unroll
    for (int j = 0; j < UNIT; ++j)
      if (j < left) p[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
  }
}
__device__ __forceinline__ void store_unit(float* p, int left, const float (&v)[UNIT]) {
  if (left >= UNIT) {
    __builtin_memcpy(p, v, 32);
  } else {
#pragma unroll
    for (int j = 0; j < UNIT; ++j)
      if (j < left) p[j] = v[j];
  }
}

// The columns from `from` to `left` of the unit at p; the others are zeros.
template <typename S> __device__ __forceinline__ void load_between(const S* p, int from, int left, Unit8<S>& u) {
#pragma unroll
  for (int j = 0; j < UNIT; ++j) {
    const bool in = j >= from && j < left;
    if constexpr (sizeof(S) == 2) {
      const uint32_t v = in ? p[j] : 0;
      u.w[j / 2] = j & 1 ? u.w[j / 2] | v << 16 : v;
    } else {
      u.w[j] = in ? __float_as_uint(p[j]) : 0;
    }
  }
}
__device__ __forceinline__ void store_between(uint16_t* p, int from, int left, const float (&v)[UNIT]) {
#pragma unroll
  for (int j = 0; j < UNIT; ++j)
    if (j >= from && j < left) p[j] = (uint16_t)pack_bf16(v[j], v[j]);
}
__device__ __forceinline__ void store_between(float* p, int from, int left, const float (&v)[UNIT]) {
#pragma unroll
  for (int j = 0; j < UNIT; ++j)
    if (j >= from && j < left) p[j] = v[j];
}

// Division of n < 2^31 by a number of 1 .. 2^31 - 1 known on the host: with
// s = ceil(log2 d) and m = floor(2^(31+s) / d) + 1, m d exceeds 2^(31+s) by at
// most d <= 2^s, so that n (m d - 2^(31+s)) < 2^(31+s) and the quotient is exact.
struct Divisor {
  uint32_t d, m, s;
};
inline Divisor divisor(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return Divisor{d, (uint32_t)((1ull << (31 + s)) / d + 1), s};
}
__device__ __forceinline__ uint32_t quotient(uint32_t n, const Divisor& d) {
  return (uint32_t)(((uint64_t)n * d.m) >> 31 >> d.s);
}

// Element offset of row r of [batch, steps, ...] with the strides of (batch, step).
struct RowStride {
  int64_t batch, step;
};
__device__ __forceinline__ int64_t row_offset(uint32_t row, const Divisor& steps, const RowStride& s) {
  const uint32_t b = quotient(row, steps);
  return (int64_t)b * s.batch + (int64_t)(row - b * steps.d) * s.step;
}

// Sum over neighbouring lanes, 2^log2 of them (all active).
__device__ __forceinline__ float lanes_sum(float v, int log2) {
  if (log2 > 0) v += xor16<1>(v);
  if (log2 > 1) v += xor16<2>(v);
  if (log2 > 2) v += xor16<4>(v);
  if (log2 > 3) v += xor16<8>(v);
  if (log2 > 4) v = add_xor16(v);
  if (log2 > 5) v = add_xor32(v);
  return v;
}

// The largest of them (a NaN is none).
__device__ __forceinline__ float lanes_max(float v, int log2) {
  if (log2 > 0) v = fmaxf(v, xor16<1>(v));
  if (log2 > 1) v = fmaxf(v, xor16<2>(v));
  if (log2 > 2) v = fmaxf(v, xor16<4>(v));
  if (log2 > 3) v = fmaxf(v, xor16<8>(v));
  if (log2 > 4) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if (log2 > 5) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}

// A sigmoid from the hardware's exponential and reciprocal (1 ulp each): 0 and
// 1 at the infinities, NaN of NaN.  And 1 - sigmoid, e / (1 + e) where the
// difference would cancel (elsewhere e may be infinite).
__device__ __forceinline__ float sigmoid(float x, float& rest) {
  const float e = __builtin_amdgcn_exp2f(-1.4426950408889634f * x), s = __builtin_amdgcn_rcpf(1.f + e);
  rest = s > 0.5f ? e * s : 1.f - s;
  return s;
}
__device__ __forceinline__ float sigmoid(float x) {
  float rest;
  return sigmoid(x, rest);
}

}  // namespace ppo
