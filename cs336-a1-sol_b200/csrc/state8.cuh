// The 8-bit form of an optimizer state (device side).
//
// A state is cut into blocks of 128 consecutive elements of the flattened
// tensor, each with one fp32 scale s:
//   signed (first moments, momentum):  s = max |x|,      code q = sgn(x) floor(127 sqrt(|x| / s) + u)
//                                      value s q |q| / 127^2
//   root (second moments, x >= 0):     s = max sqrt(x),  code q = floor(255 sqrt(sqrt(x) / s) + u), >= 1 where x > 0
//                                      value (s (q / 255)^2)^2
//
// Why codes of the square root: the spacing of the values grows with their
// size, so an element is off by a part of itself (1/q) and not of its block's
// largest. A second moment that is not zero never becomes zero: the update
// would divide a live first moment by eps alone.
//
// Why u: with u = 1/2 (nearest) a change below half a code step is lost every
// time. At beta2 = 0.999 an element's second moment would then never decay
// but with its block, and at beta = 0.9 a first moment whose gradient has
// become zero would stay at 9 of 127 codes for good. In a step, u therefore
// runs evenly over [0, 1): u = h / 2^32 to 23 bits, h = A i + B t (+ 2^31 for
// signed) mod 2^32 for element i of the tensor and step t, A = 2^32 / golden
// ratio, B = 2^32 (sqrt 2 - 1): turns that leave no wide gap. The rounding is then right on average over steps, with no random
// state to keep. Simulated updates (128-element blocks, lognormal scales of
// the elements with sigma 0.3, betas 0.9 / 0.95, .99, .999) are off by 3.2, 3.5
// and 3.8 % rms against 2.9, 6.3 and 5.4 % to nearest. A conversion (encode)
// uses u = 1/2, so that what was decoded encodes to the same codes.
//
// A code is exact: it depends on nothing but the fp32 state, its block's fp32
// scale and u. The fast path computes y = levels sqrt(x / s) with approximate
// instructions (error below 1e-4); where y + u lands within 1e-4 of an
// integer K, the side is decided by comparing x levels^2 with s (K - u)^2 in
// 64 bits.
//
// Special blocks: a value that is not finite makes the scale NaN and every
// code 0 (the whole block reads as NaN); s = 0 (for signed also s < 2^-126,
// whose reciprocal overflows) makes every code 0.
#pragma once

#include "b2o_common.cuh"

namespace b2o {

constexpr int kQ8Block = 128;              // elements per scale: 16 lanes x 8
constexpr int kQ8Tile = 256;               // elements per warp step: two blocks
constexpr float kQ8Signed = 1.0f / 16129;  // 1 / 127^2
constexpr float kQ8Root = 1.0f / 65025;    // 1 / 255^2

__device__ __forceinline__ float sqrt_approx(float x) {  // relative error 2^-23, subnormals kept
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float sqrt_approx_ftz(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Byte k of four packed codes as a float: 2^23 + byte by its bits, minus 2^23
// (the integer conversion would take the pipe that the square roots need).
__device__ __forceinline__ float byte_f32(uint32_t word, int k, float bias) {
  return __uint_as_float(__byte_perm(word, 0x4B000000u, 0x7540u + k)) - bias;
}

// value of a signed code (as a float): s q |q| / 127^2, two roundings
__device__ __forceinline__ float signed_value(float q, float s) {
  return __fmul_rn(__fmul_rn(q * fabsf(q), kQ8Signed), s);
}
// value of a root code: the root, then its square
__device__ __forceinline__ float root_value(float q, float s) {
  const float r = __fmul_rn(__fmul_rn(q * q, kQ8Root), s);
  return __fmul_rn(r, r);
}

__device__ __forceinline__ void unpack_signed(uint2 c, float s, float* x) {
  c.x ^= 0x80808080u;
  c.y ^= 0x80808080u;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[k] = signed_value(byte_f32(c.x, k, 8388608.0f + 128.0f), s);
    x[4 + k] = signed_value(byte_f32(c.y, k, 8388608.0f + 128.0f), s);
  }
}
__device__ __forceinline__ void unpack_root(uint2 c, float s, float* x) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[k] = root_value(byte_f32(c.x, k, 8388608.0f), s);
    x[4 + k] = root_value(byte_f32(c.y, k, 8388608.0f), s);
  }
}

// Largest bit pattern over the 16 lanes of a block: for values that are not
// negative the order of the patterns is the order of the values, infinity and
// NaN above them all. Every lane of the warp calls it.
__device__ __forceinline__ uint32_t block_max(uint32_t bits) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
  return bits;
}

struct BlockScale {
  float s, inv;  // the scale that is stored, and 1 / s (0 where every code is 0)
};
__device__ __forceinline__ BlockScale signed_scale(uint32_t bits) {
  BlockScale b;
  b.s = bits >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : bits < 0x00800000u ? 0.0f : __uint_as_float(bits);
  b.inv = b.s > 0.0f ? __frcp_rn(b.s) : 0.0f;
  return b;
}
__device__ __forceinline__ BlockScale root_scale(uint32_t bits) {
  BlockScale b;
  b.s = bits >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __fsqrt_rn(__uint_as_float(bits));
  b.inv = b.s > 0.0f ? __frcp_rn(b.s) : 0.0f;
  return b;
}

// h of element i in step t; the other elements of a lane add kQ8Turn each.
constexpr uint32_t kQ8Turn = 0x9E3779B9u, kQ8StepTurn = 0x6A09E667u, kQ8SignedPhase = 0x80000000u;
__device__ __forceinline__ uint32_t dither_of(int64_t i, uint32_t t) {
  return static_cast<uint32_t>(i) * kQ8Turn + t * kQ8StepTurn;
}
// u - 1/2 from the top 23 bits of h
__device__ __forceinline__ float dither_f32(uint32_t h) { return __uint_as_float((h >> 9) | 0x3f800000u) - 1.5f; }

// The exact code for a size x in [0, s], given z = levels sqrt(x / s) + u - 1/2
// to within 1e-4 and near the middle between two integers.
__device__ __forceinline__ uint32_t near_code(float x, float s, float z, double levels, double u) {
  const double k = rint(static_cast<double>(z) + 0.5);
  const double c = k - u;
  const bool reached = c <= 0.0 || static_cast<double>(x) * (levels * levels) >= static_cast<double>(s) * (c * c);
  return static_cast<uint32_t>(static_cast<int>(reached ? k : k - 1.0));
}

constexpr float kQ8Magic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer, which its low byte holds
constexpr float kQ8Near = 0.4999f;

__device__ __forceinline__ uint32_t pack4(const uint32_t* t) {
  return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}

// Codes (low byte of q[k]) of eight sizes; exact(k) gives the fp32 size that
// the definition compares, rough[k] is that size to within 2^-23.
template <bool DITHER, int LEVELS, typename Exact>
__device__ __forceinline__ void size_codes(const float* rough, BlockScale b, uint32_t h, uint32_t* q, Exact exact) {
  bool close = false;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float y = static_cast<float>(LEVELS) * sqrt_approx_ftz(rough[k] * b.inv);
    const float z = DITHER ? y + dither_f32(h + k * kQ8Turn) : y;
    const float m = z + kQ8Magic;
    q[k] = __float_as_uint(m);
    close |= fabsf(z - (m - kQ8Magic)) > kQ8Near;
  }
  if (close) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t hk = h + k * kQ8Turn;
      const float y = static_cast<float>(LEVELS) * sqrt_approx_ftz(rough[k] * b.inv);
      const float z = DITHER ? y + dither_f32(hk) : y;
      if (fabsf(z - rintf(z)) > kQ8Near)
        q[k] = near_code(exact(k), b.s, z, LEVELS, DITHER ? (hk >> 9) * (1.0 / 8388608.0) : 0.5);
    }
  }
}

template <bool DITHER>
__device__ __forceinline__ uint2 pack_signed(const float* x, BlockScale b, uint32_t h) {
  uint32_t q[8];
  float size[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) size[k] = fabsf(x[k]);
  size_codes<DITHER, 127>(size, b, h + kQ8SignedPhase, q, [&](int k) { return size[k]; });
#pragma unroll
  for (int k = 0; k < 8; ++k) q[k] = x[k] < 0.0f ? 0u - q[k] : q[k];
  return b.inv > 0.0f ? make_uint2(pack4(q), pack4(q + 4)) : make_uint2(0u, 0u);
}

// x: the states, r: their square roots to within 2^-23
template <bool DITHER>
__device__ __forceinline__ uint2 pack_root(const float* x, const float* r, BlockScale b, uint32_t h) {
  uint32_t q[8];
  size_codes<DITHER, 255>(r, b, h, q, [&](int k) { return __fsqrt_rn(x[k]); });
  // a live state keeps a code
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (x[k] > 0.0f && (q[k] & 0xffu) == 0) q[k] |= 1u;
  return b.inv > 0.0f ? make_uint2(pack4(q), pack4(q + 4)) : make_uint2(0u, 0u);
}

__device__ __forceinline__ uint32_t max_abs_bits(const float* x) {
  uint32_t b = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) b = max(b, __float_as_uint(x[k]) & 0x7fffffffu);
  return b;
}

// Eight codes at p (element i of a list that ends at `end`): one 8-byte access
// where `vec`, else the bytes inside the list.
__device__ __forceinline__ uint2 load_codes(const void* p, int64_t i, int64_t end, bool vec) {
  const uint8_t* c = static_cast<const uint8_t*>(p) + i;
  if (vec) return *reinterpret_cast<const uint2*>(c);
  uint32_t w[2] = {0u, 0u};
  for (int k = 0; k < 8; ++k)
    if (i + k < end) w[k >> 2] |= static_cast<uint32_t>(c[k]) << (8 * (k & 3));
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store_codes(void* p, int64_t i, int64_t end, bool vec, uint2 v) {
  uint8_t* c = static_cast<uint8_t*>(p) + i;
  if (vec) {
    *reinterpret_cast<uint2*>(c) = v;
    return;
  }
  for (int k = 0; k < 8; ++k)
    if (i + k < end) c[k] = static_cast<uint8_t>((k < 4 ? v.x : v.y) >> (8 * (k & 3)));
}

}  // namespace b2o
