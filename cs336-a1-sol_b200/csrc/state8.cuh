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
// ratio, B = 2^32 (sqrt 2 - 1): turns that leave no wide gap. The code is then
// right on average over steps, with no random state to keep. A conversion
// (encode) uses u = 1/2, so that what was decoded encodes to the same codes.
//
// What it costs (oracle/state8_accuracy.py, betas 0.9 / 0.95, standard deviations
// of a block's elements lognormal with sigma 0.3, 1.0, 1.5): updates are off by
// 2.2, 6.5 and 21 % rms; to nearest by 2.0, 5.7 and 15 %, so in a steady run u is
// a little worse. At beta2 = 0.999: 4.3, 9.9, 22 % against 3.6, 8.8, 20 %. Elements
// whose gradient stops move on by 2.3 to 2.5 lr in 600 steps (64-bit moments: 2.3;
// to nearest 12 to 22). The code is right on average, its value is not: that is
// the code's square (second moments: fourth power), so second moments lie 1 to 2 %
// high where their root is 0.003 to 0.03 of the block's largest, 13 % below that
// (beta2 = 0.999: 4 to 6 %, 20 %).
//
// A code is exact: it depends on nothing but the fp32 state, its block's fp32
// scale and u. The fast path computes y = levels sqrt(x / s) with approximate
// instructions (error below 1e-4) as a fixed-point number with 16 bits behind
// the point, so that adding the top 16 bits of h leaves the code in one byte.
// Where y + u lands within 8 (signed: 4) / 65536 of an integer K, the side is
// decided by comparing x levels^2 with s (K - u)^2 in 64 bits.
//
// What bounds the passes that write codes is instruction issue, not memory: a
// first form with scalar arithmetic and u added in floating point took 208 us
// for a step of 33.5 M bf16 weights (10.1 bytes an element, 52 us at copy
// bandwidth) at 103 instructions an element. Hence the fixed point, packed pairs
// of floats (two roundings an instruction, each as the scalar one), the block
// maximum in reduction instructions, one kernel for each set of options, and
// the next step's loads ahead of this one's work: 70 us at 58 instructions.
//
// These times are for blocks without zeros. A second moment that is 0 or has sunk
// to code 1 in a live block is settled one by one in 64 bits (size_codes): with 1,
// 10 and 50 % of such elements, scattered, a bf16 step takes 83 to 89, 100 to 116
// and 133 to 172 us, and an encode of second moments 44, 62 and 97 us against 29.
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
__device__ __forceinline__ float rsqrt_approx_ftz(float x) {  // relative error 2^-22.9
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx_ftz(float x) {  // relative error 2^-23
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// ------------------------------------------------- pairs of fp32 in a register ---
typedef unsigned long long F2;
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 f2(float x) { return f2(x, x); }
__device__ __forceinline__ float2 f2_split(F2 x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// with subnormal operands and results taken as 0
__device__ __forceinline__ F2 fma2_ftz(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// a b + c with the product and the sum each rounded by itself. The sum is a
// fused product one + c with one = 1 from the kernel's arguments: a packed
// product and a packed sum are contracted into one rounding, although both say
// .rn, and so is the form with a literal 1.
__device__ __forceinline__ F2 mul_add2(F2 a, F2 b, F2 c, float one) { return fma2(mul2(a, b), f2(one), c); }
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {  // the sign mode too
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}

// Eight consecutive elements as four pairs.
struct V8 { F2 p[4]; };

// Eight consecutive elements as they lie in memory. load: of a list that ends
// at `end`, elements behind it as 0; one or two 16-byte accesses where `vec`.
template <typename T> struct Raw8;
template <> struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p, int64_t i, int64_t end, bool vec) {
    if (vec) {
      a = *reinterpret_cast<const float4*>(p + i);
      b = *reinterpret_cast<const float4*>(p + i + 4);
      return;
    }
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = i + k < end ? p[i + k] : 0.0f;
    a = make_float4(x[0], x[1], x[2], x[3]);
    b = make_float4(x[4], x[5], x[6], x[7]);
  }
  __device__ __forceinline__ void store(float* p, int64_t i, int64_t end, bool vec) const {
    if (vec) {
      *reinterpret_cast<float4*>(p + i) = a;
      *reinterpret_cast<float4*>(p + i + 4) = b;
      return;
    }
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < end) p[i + k] = x[k];
  }
  __device__ __forceinline__ V8 get() const { return V8{{f2(a.x, a.y), f2(a.z, a.w), f2(b.x, b.y), f2(b.z, b.w)}}; }
  __device__ __forceinline__ void set(const V8& v) {
    const float2 x = f2_split(v.p[0]), y = f2_split(v.p[1]), z = f2_split(v.p[2]), w = f2_split(v.p[3]);
    a = make_float4(x.x, x.y, y.x, y.y);
    b = make_float4(z.x, z.y, w.x, w.y);
  }
};
template <> struct Raw8<uint16_t> {  // bf16
  uint4 a;
  __device__ __forceinline__ void load(const uint16_t* p, int64_t i, int64_t end, bool vec) {
    if (vec) {
      a = *reinterpret_cast<const uint4*>(p + i);
      return;
    }
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < end) w[k >> 1] |= static_cast<uint32_t>(p[i + k]) << (16 * (k & 1));
    a = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void store(uint16_t* p, int64_t i, int64_t end, bool vec) const {
    if (vec) {
      *reinterpret_cast<uint4*>(p + i) = a;
      return;
    }
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < end) p[i + k] = static_cast<uint16_t>(w[k >> 1] >> (16 * (k & 1)));
  }
  static __device__ __forceinline__ F2 pair(uint32_t w) {
    return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t round(F2 v) {  // to nearest even
    const float2 x = f2_split(v);
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x.y), "f"(x.x));
    return r;
  }
  __device__ __forceinline__ V8 get() const { return V8{{pair(a.x), pair(a.y), pair(a.z), pair(a.w)}}; }
  __device__ __forceinline__ void set(const V8& v) {
    a = make_uint4(round(v.p[0]), round(v.p[1]), round(v.p[2]), round(v.p[3]));
  }
};

// ------------------------------------------------------------------ reading ---
// Bytes k and k + 1 of four packed codes as floats: 2^23 + byte by its bits,
// minus 2^23 + bias (the integer conversion would take the pipe that the square
// roots need).
__device__ __forceinline__ F2 bytes_f2(uint32_t word, int k, float bias) {
  return add2(f2(__uint_as_float(__byte_perm(word, 0x4B000000u, 0x7540u + k)),
                 __uint_as_float(__byte_perm(word, 0x4B000000u, 0x7541u + k))), f2(-8388608.0f - bias));
}

// s q |q| / 127^2, two roundings (q |q| is exact)
__device__ __forceinline__ V8 unpack_signed(uint2 c, float s) {
  V8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = (j < 2 ? c.x : c.y) ^ 0x80808080u;
    const float2 q = f2_split(bytes_f2(w, 2 * (j & 1), 128.0f));
    v.p[j] = mul2(mul2(f2(q.x * fabsf(q.x), q.y * fabsf(q.y)), f2(kQ8Signed)), f2(s));
  }
  return v;
}
// (s (q / 255)^2)^2, three roundings
__device__ __forceinline__ V8 unpack_root(uint2 c, float s) {
  V8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const F2 q = bytes_f2(j < 2 ? c.x : c.y, 2 * (j & 1), 0.0f);
    const F2 r = mul2(mul2(mul2(q, q), f2(kQ8Root)), f2(s));
    v.p[j] = mul2(r, r);
  }
  return v;
}

// the same for four codes
__device__ __forceinline__ float4 unpack4(uint32_t w, float s, bool root) {
  F2 v[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (root) {
      const F2 q = bytes_f2(w, 2 * j, 0.0f);
      const F2 r = mul2(mul2(mul2(q, q), f2(kQ8Root)), f2(s));
      v[j] = mul2(r, r);
    } else {
      const float2 q = f2_split(bytes_f2(w ^ 0x80808080u, 2 * j, 128.0f));
      v[j] = mul2(mul2(f2(q.x * fabsf(q.x), q.y * fabsf(q.y)), f2(kQ8Signed)), f2(s));
    }
  }
  const float2 a = f2_split(v[0]), b = f2_split(v[1]);
  return make_float4(a.x, a.y, b.x, b.y);
}

// ------------------------------------------------------------------ scaling ---
// A lane holds N vectors of 8 elements of one block, so a block is 16 / N lanes
// and a warp step 256 N elements. Vector k of a lane starts at this offset.
template <int N>
__device__ __forceinline__ int lane_offset(int lane, int k) {
  constexpr int kLanes = 16 / N;
  return (lane / kLanes) * kQ8Block + (lane % kLanes) * 8 + k * (8 * kLanes);
}

// Largest magnitude of a block; NaN if one is NaN. Every lane of the warp calls it.
template <int N>
__device__ __forceinline__ float block_max(const V8* v) {
  float m = 0.0f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = f2_split(v[k].p[j]);
      asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(x.x), "f"(x.y));
    }
  }
  if (N == 1) {
    // one reduction of the whole warp for each half: half masks would run one after the other
    const bool upper = (threadIdx.x & 16) != 0;
    float lo, hi;
    // (volatile: every lane has to execute them, so they stay ahead of any branch)
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(lo) : "f"(upper ? 0.0f : m));
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(hi) : "f"(upper ? m : 0.0f));
    return upper ? hi : lo;
  }
#pragma unroll
  for (int o = 8 / N; o > 0; o >>= 1) {
    const float x = __shfl_xor_sync(0xffffffffu, m, o);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(x));
  }
  return m;
}

struct BlockScale {
  float s;      // the scale that is stored
  float inv;    // 1 / s (signed, from s = 1 on: 4 / s, since 1 / s may be subnormal); 0 where every code is 0
  float half;   // 1, or 1/2 to go with 4 / s: sqrt(x / s) = half sqrt(x inv)
  float tie;    // the state whose size is exactly s / 4, midway between the two middle codes (-1: none that small)
};
__device__ __forceinline__ BlockScale signed_scale(float top) {
  BlockScale b;
  b.s = !(top < __int_as_float(0x7f800000)) ? __int_as_float(0x7fffffff) : top < 1.17549435e-38f ? 0.0f : top;
  const bool big = b.s >= 1.0f;
  b.inv = b.s > 0.0f ? rcp_approx_ftz(big ? 0.25f * b.s : b.s) : 0.0f;
  b.half = big ? 0.5f : 1.0f;
  b.tie = b.s >= 1e-36f ? 0.25f * b.s : -1.0f;
  return b;
}
__device__ __forceinline__ BlockScale root_scale(float top) {  // roots lie between 2^-75 and 2^64
  BlockScale b;
  b.s = !(top < __int_as_float(0x7f800000)) ? __int_as_float(0x7fffffff) : __fsqrt_rn(top);
  b.inv = b.s > 0.0f ? rcp_approx_ftz(b.s) : 0.0f;
  b.half = 1.0f;
  b.tie = top >= 1e-36f ? 0.0625f * top : -1.0f;
  return b;
}

// ------------------------------------------------------------------ writing ---
// h of element i in step t; the other elements of a lane add kQ8Turn each.
constexpr uint32_t kQ8Turn = 0x9E3779B9u, kQ8StepTurn = 0x6A09E667u, kQ8SignedPhase = 0x80000000u;
__device__ __forceinline__ uint32_t dither_of(int64_t i, uint32_t t) {
  return static_cast<uint32_t>(i) * kQ8Turn + t * kQ8StepTurn;
}

// The exact code of a size x in [0, s] where levels sqrt(x / s) + u is near the
// integer k: k if it reaches it, else k - 1.
__device__ __forceinline__ uint32_t near_code(float x, float s, int k, double levels, double u) {
  const double c = k - u;
  const bool reached = c <= 0.0 || static_cast<double>(x) * (levels * levels) >= static_cast<double>(s) * (c * c);
  return static_cast<uint32_t>(reached ? k : k - 1);
}

__device__ __forceinline__ uint32_t pack4(const uint32_t* t) {  // byte 2 of each
  return prmt(prmt(t[0], t[1], 0x0062), prmt(t[2], t[3], 0x0062), 0x5410);
}
__device__ __forceinline__ float pick8(const V8& v, int k) {
  float r = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = f2_split(v.p[j]);
    r = k == 2 * j ? x.x : k == 2 * j + 1 ? x.y : r;
  }
  return r;
}

// Codes of the sizes of one lane's eight states (their magnitudes, or for ROOT
// their square roots). rough: the sizes to within 2^-23, signs ignored.
// y's fixed point comes from adding 2^7 (2^8 for 255 levels, whose last place
// is 2^-15) and kSlack / 65536: a sum within kSlack / 65536 of an integer on
// either side then has the high bits of its fraction clear. kSlack covers, in
// units of 2^-16: levels x 2^-24 x ((2 of a rough root, none of a size, + 2 of
// 1 / s + 1 of their product) / 2 + 2 of the root), half a place of the sum (1/2;
// ROOT 1), and 1 of cutting u to 16 bits: 3.3 of 4 and 6.5 of 8.
template <bool DITHER, bool ROOT>
__device__ __forceinline__ uint2 size_codes(const V8& x, const V8& rough, BlockScale b, uint32_t h) {
  constexpr uint32_t kSlack = ROOT ? 8 : 4;
  constexpr float kLevels = ROOT ? 255.0f : 127.0f;
  constexpr float kPoint = (ROOT ? 256.0f : 128.0f) + kSlack / 65536.0f;
  constexpr float kOne = kPoint + 1.0f;
  const float levels = kLevels * b.half;
  uint32_t q[8];
  float small = kOne;  // ROOT: sizes below one code step
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 y = f2_split(mul2(rough.p[j], f2(b.inv)));
    const F2 ys = f2(sqrt_approx_ftz(ROOT ? y.x : fabsf(y.x)), sqrt_approx_ftz(ROOT ? y.y : fabsf(y.y)));
    const float2 t = f2_split(fma2(ys, f2(levels), f2(kPoint)));
    if (ROOT) asm("min.f32 %0, %0, %1, %2;" : "+f"(small) : "f"(t.x), "f"(t.y));
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int k = 2 * j + e;
      const uint32_t w = __float_as_uint(e ? t.y : t.x);
      const uint32_t w16 = ROOT ? w + w : w;
      q[k] = DITHER ? w16 + ((h + k * kQ8Turn) >> 16) : w16 + 0x8000u;
    }
  }
  uint2 out = make_uint2(pack4(q), pack4(q + 4));
  // the smallest fraction, two to a register
  const uint32_t least2 = __vminu2(
      __vimin3_u16x2(prmt(q[0], q[1], 0x5410), prmt(q[2], q[3], 0x5410), prmt(q[4], q[5], 0x5410)),
      prmt(q[6], q[7], 0x5410));
  const uint32_t least = min(least2 & 0xffffu, least2 >> 16);
  if ((least < 2 * kSlack || (ROOT && small < kOne)) && b.inv > 0.0f) {
    uint32_t todo = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t at = q[k] & 0xffffffu;
      const float2 pair = f2_split(x.p[k / 2]);
      // u = 1/2: a size of exactly s / 4 lies on the border and has the integer
      // part already (levels / 2 + 1/2, rounded up). Among bf16 states one in
      // 700 is such a tie.
      const bool tie = !DITHER && fabsf(k & 1 ? pair.y : pair.x) == b.tie;
      if (((at & 0xffffu) < 2 * kSlack && !tie) || (ROOT && at < 0x20000u)) todo |= 1u << k;
    }
    while (todo) {
      const int k = __ffs(todo) - 1;
      todo &= todo - 1;
      const int shift = 8 * (k & 3);
      const uint32_t word = k < 4 ? out.x : out.y;
      const double u = DITHER ? ((h + k * kQ8Turn) >> 9) * (1.0 / 8388608.0) : 0.5;
      const float v = pick8(x, k);
      const int near = static_cast<int>((word >> shift) & 0xffu);
      uint32_t code = near;
      if (ROOT && near < 2) {
        // A live state keeps a code. One this small may have lost its rough
        // size to 0, and the largest's sum may have wrapped past 2^24 to here.
        const double y = 255.0 * sqrt(static_cast<double>(__fsqrt_rn(v)) / static_cast<double>(b.s));
        code = v > 0.0f ? max(1, static_cast<int>(y + u)) : 0;
      } else {
        code = near_code(ROOT ? __fsqrt_rn(v) : fabsf(v), b.s, near, kLevels, u);
      }
      const uint32_t fixed = (word & ~(0xffu << shift)) | code << shift;
      if (k < 4) out.x = fixed; else out.y = fixed;
    }
  }
  return out;
}

template <bool DITHER>
__device__ __forceinline__ uint2 pack_signed(const V8& v, BlockScale b, uint32_t h) {
  const uint2 c = size_codes<DITHER, false>(v, v, b, h + kQ8SignedPhase);
  uint32_t w[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const float2 x = f2_split(v.p[2 * half]), y = f2_split(v.p[2 * half + 1]);
    // bytes 0xff where the state is negative; then two's complement byte by
    // byte: the sum of the low seven bits carries into the eighth at most
    const uint32_t m = prmt(prmt(__float_as_uint(x.x), __float_as_uint(x.y), 0x00fb),
                            prmt(__float_as_uint(y.x), __float_as_uint(y.y), 0x00fb), 0x5410);
    const uint32_t n = (half ? c.y : c.x) ^ m;
    w[half] = ((n & 0x7f7f7f7fu) + (m & 0x01010101u)) ^ (n & 0x80808080u);
  }
  return b.inv > 0.0f ? make_uint2(w[0], w[1]) : make_uint2(0u, 0u);
}

// v: the states, r: their square roots to within 2^-23 (0 for a subnormal state is fine)
template <bool DITHER>
__device__ __forceinline__ uint2 pack_root(const V8& v, const V8& r, BlockScale b, uint32_t h) {
  const uint2 c = size_codes<DITHER, true>(v, r, b, h);
  return b.inv > 0.0f ? c : make_uint2(0u, 0u);
}

// Eight codes at p + i of a list that ends at `end`: one 8-byte access where
// `vec`, else the bytes inside the list.
__device__ __forceinline__ uint2 load_codes(const void* p, int64_t i, int64_t end, bool vec) {
  const uint8_t* c = static_cast<const uint8_t*>(p) + i;
  if (vec) return *reinterpret_cast<const uint2*>(c);
  uint32_t w[2] = {0u, 0u};
#pragma unroll
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
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (i + k < end) c[k] = static_cast<uint8_t>((k < 4 ? v.x : v.y) >> (8 * (k & 3)));
}

}  // namespace b2o
