// Device helpers that the attention kernels share (gfx950): the softmax's constants, exchanges
// between the lane rows of a wave, and the 16-bit element types with their matrix instructions.
#pragma once

#include <initializer_list>
#include <type_traits>

#include "common.h"

// copy_to_lds sets M0 and names it as clobbered; clang warns that M0 is a reserved register.
#pragma clang diagnostic ignored "-Winline-asm"

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr float kNegInf = -__builtin_huge_valf();
// Where a unit's running maximum starts: below every finite score, so that the first tile replaces it,
// and finite, so that keys scoring -inf weigh exp2(-inf - m) = 0 also where nothing else has been seen
// (-inf - -inf would be NaN). Such a unit's state is (kLowest, 0, 0), which adds 0 to any merge.
constexpr float kLowest = -3.402823466e38f;  // -FLT_MAX
// Weights are 2^(score - m) with a reference m near the running maximum. m stays until a weight would pass 2^reach, and is then
// set so that the weight of that score is 2^(reach - kSlack): a tile seldom asks for it, so the accumulators are seldom
// rescaled. A wave rescales where any of its rows' scores pass, but only those rows move: a row's bits do not depend on its
// neighbours. The reach is the element type's (BF16, FP16 below).
constexpr float kSlack = 8.0f;

// The product of sizes, or 2^62 where it would be beyond that.
inline int64_t product(std::initializer_list<int64_t> sizes) {
  int64_t n = 1;
  for (int64_t s : sizes)
    if (__builtin_mul_overflow(n, s, &n) || n > 1LL << 62) return 1LL << 62;
  return n;
}
// Whether a launch may have so many workgroups of `threads`: the threads of all are a 32-bit number.
inline bool launchable(int64_t blocks, int threads) { return blocks <= 0xFFFFFFFFLL / threads; }

// x / d for 0 <= x < 2^31 and 1 <= d < 2^31: (2 x mul >> 32) >> shift with 2^shift >= d and mul = 2^(31 + shift) / d rounded
// up. The excess of mul is below 1, so times 2 x it stays below 2^32 <= 2^(32 + shift) / d: the quotient is exact.
struct Divisor {
  uint32_t mul, shift;
};
inline Divisor make_divisor(int64_t d) {
  uint32_t s = 0;
  while ((1LL << s) < d) ++s;
  return Divisor{(uint32_t)(((1ULL << (31 + s)) + (uint64_t)d - 1) / (uint64_t)d), s};
}
__device__ inline int divide(int x, const Divisor& d) { return (int)(__umulhi(2u * (uint32_t)x, d.mul) >> d.shift); }

__device__ inline float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Exchanges between the four 16-lane rows of a wave on the vector ALU (gfx950 lane swaps), in
// place of ds_bpermute round trips through the LDS pipe. The fp32 pairs come back as
// {x of the lower row or half, x of the upper}, for both sides.
__device__ inline void swap32(float& a, float& b) {  // a's upper half <-> b's lower half
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  a = __uint_as_float(r[0]);
  b = __uint_as_float(r[1]);
}
__device__ inline void swap16(float& a, float& b) {  // a's odd rows <-> b's even rows
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  a = __uint_as_float(r[0]);
  b = __uint_as_float(r[1]);
}
__device__ inline float rows_max(float v) {
  float a = v, b = v;
  swap16(a, b);
  v = fmaxf(a, b);
  a = v, b = v;
  swap32(a, b);
  return fmaxf(a, b);
}
__device__ inline float rows_sum(float v) {
  float a = v, b = v;
  swap16(a, b);
  v = a + b;
  a = v, b = v;
  swap32(a, b);
  return a + b;
}
// Running sums or maxima of values >= 0 over the lanes of a wave, this lane's included; wave_reduce: over all of them.
template <int CTRL, int ROWS>
__device__ inline int from_row(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
template <typename F>
__device__ inline int wave_scan(int x, F&& f) {
  x = f(x, from_row<0x111, 0xF>(x));  // the lanes 1, 2, 4 and 8 before, in rows of 16
  x = f(x, from_row<0x112, 0xF>(x));
  x = f(x, from_row<0x114, 0xF>(x));
  x = f(x, from_row<0x118, 0xF>(x));
  x = f(x, from_row<0x142, 0xA>(x));  // row 0's and 2's last lane to rows 1 and 3
  return f(x, from_row<0x143, 0xC>(x));  // row 1's last lane to rows 2 and 3
}
template <typename F>
__device__ inline int wave_reduce(int x, F&& f) {
  return __builtin_amdgcn_readlane(wave_scan(x, f), 63);
}

template <int N, typename F, int I = 0>
__device__ inline void static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<N, F, I + 1>(static_cast<F&&>(f));
  }
}

// The two 16-bit element types. Operands of the matrix instructions are held as four dwords of
// two elements each; products of two such elements are exact in fp32.
struct BF16 {
  static constexpr uint32_t kExpMask = 0x7F80u, kOne = 0x3F80u;
  // Values may be as large as floats are: a row's weights stay below one over the number of its keys, so that its sums stay below
  // the largest value. (Values below some 2^-100 lose bits in turn.)
  static __device__ inline float reach(int keys) { return keys <= 1 << 12 ? -12.0f : keys <= 1 << 18 ? -18.0f : -30.0f; }
  static __device__ inline float to_f32(uint16_t b) { return bf16_to_f32(b); }
  static __device__ inline uint32_t pack(float a, float b) {  // round to nearest even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2bf));
  }
  static __device__ inline v2f unpack(uint32_t w) {
    return v2f{__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)};
  }
  static __device__ inline v4f mfma16(v4u32 a, v4u32 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
  static __device__ inline v16f mfma32(v4u32 a, v4u32 b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
};
struct FP16 {
  static constexpr uint32_t kExpMask = 0x7C00u, kOne = 0x3C00u;
  // Values end at 65504, so weights may be as large as the type holds: many small ones count down to 2^-32 of a row's largest.
  static __device__ inline float reach(int) { return 15.0f; }
  static __device__ inline float to_f32(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }
  static __device__ inline uint32_t pack(float a, float b) {  // round to nearest even
    return __builtin_bit_cast(uint32_t, v2h{(_Float16)a, (_Float16)b});
  }
  static __device__ inline v2f unpack(uint32_t w) { return __builtin_convertvector(__builtin_bit_cast(v2h, w), v2f); }
  static __device__ inline v4f mfma16(v4u32 a, v4u32 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
  static __device__ inline v16f mfma32(v4u32 a, v4u32 b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};

// a * x of a sum a that may be an infinity or NaN and then stays what it is, also times 0: a value counts however small its weight.
__device__ inline float scaled(float a, float x) { return __builtin_isfinite(a) ? a * x : a; }
// Four elements' infinities and NaN, added to `sum`.
template <typename T>
__device__ inline void add_specials(v4f& sum, v2u32 w) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float f = T::to_f32((uint16_t)(w[e / 2] >> (16 * (e % 2))));
    if (!__builtin_isfinite(f)) sum[e] += f;
  }
}
// The elements of four dims whose values hold an infinity or NaN that the row attends to, in place of what was stored there. Such
// a value counts however small its weight; in the sums it has met weights of 0, or negative second parts of one, and become NaN.
__device__ inline void store_specials(void* out, int dtype, int64_t at, v4f special) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (!__builtin_isfinite(special[e])) store_f32_as(out, dtype, at + e, special[e]);
}
// The dword with its infinities and NaN replaced by 0, and which of its elements add +inf (SIGN = 0: +inf
// and NaN) or -inf (SIGN = 1: -inf and NaN), as elements 1 and 0.
template <typename T>
__device__ inline uint32_t only_finite(uint32_t w) {
  constexpr uint32_t m = T::kExpMask;
  return ((w & m) == m ? 0u : w & 0xFFFFu) | (((w >> 16) & m) == m ? 0u : w & 0xFFFF0000u);
}
template <typename T>
__device__ inline uint32_t only_special(uint32_t w) {  // the infinities and NaN, 0 elsewhere
  return w ^ only_finite<T>(w);
}
template <typename T, int SIGN>
__device__ inline uint32_t special_flags(uint32_t w) {
  constexpr uint32_t m = T::kExpMask, other = m | (SIGN ? 0u : 0x8000u);  // the infinity that does not count
  const uint32_t lo = w & 0xFFFFu, hi = w >> 16;
  return ((lo & m) == m && lo != other ? T::kOne : 0u) | ((hi & m) == m && hi != other ? T::kOne << 16 : 0u);
}

// Four 16-bit elements of one column, from four rows that the 16 lanes of a group address together (8 bytes a lane,
// four lanes a row): gfx950's transposing LDS read.
__device__ inline v2u32 read_transposed(const char* lds) {
  typedef short v4s __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4s lds_v4s;
  return __builtin_bit_cast(v2u32, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)lds));
}

typedef __attribute__((address_space(3))) void lds_void_t;

// 16 bytes a lane straight from memory into LDS: lane i's land at dst + 16 i. From inline asm: with the builtin the
// compiler, which cannot tell one buffer from another, waits for copies in flight before it reads any. Explicit waits order
// them. M0 needs one wait state before the load that uses it; the build checks that only this code uses it.
__device__ inline void copy_to_lds(const char* src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(dst) : "memory", "m0");
}

// Tiles of 16-bit keys and values in LDS, a key after the other in 16-byte chunks: chunk c of a key lies at
// c ^ swizzle(key), so that 16 lanes that read one chunk of 16 keys (K), or four chunks of four keys (V, transposed), meet
// 16 different 16-byte columns of the 256 bytes that the banks deliver.
template <int D>
__device__ inline int key_swizzle(int key) { return D == 64 ? (key >> 1) & 7 : key & 15; }
template <int D>
__device__ inline int value_swizzle(int key) { return D == 64 ? 4 * ((key >> 1) & 1) : 4 * (key & 3); }
