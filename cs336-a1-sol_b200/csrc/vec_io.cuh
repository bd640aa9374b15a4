// 16-byte vector loads and stores of fp32 and bf16 elements.
#pragma once

#include "b2o_common.cuh"

namespace b2o {

// ------------------------------------------------------------ vector I/O ---
struct alignas(16) U16x8 { uint16_t v[8]; };
struct alignas(16) F32x4 { float v[4]; };

template <typename T> struct Elem;
template <> struct Elem<float> {
  __device__ static void load8(const float* p, float* o) {
    F32x4 a = *reinterpret_cast<const F32x4*>(p);
    F32x4 b = *reinterpret_cast<const F32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { o[i] = a.v[i]; o[4 + i] = b.v[i]; }
  }
  __device__ static void store8(float* p, const float* x) {
    F32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) { a.v[i] = x[i]; b.v[i] = x[4 + i]; }
    *reinterpret_cast<F32x4*>(p) = a;
    *reinterpret_cast<F32x4*>(p + 4) = b;
  }
  __device__ static float load1(const float* p) { return *p; }
  __device__ static void store1(float* p, float x) { *p = x; }
  // value after rounding to the storage type
  __device__ static float rnd(float x) { return x; }
};
template <> struct Elem<uint16_t> {  // bf16 stored as raw bits
  __device__ static void load8(const uint16_t* p, float* o) {
    U16x8 a = *reinterpret_cast<const U16x8*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = bf16_to_f32(a.v[i]);
  }
  __device__ static void store8(uint16_t* p, const float* x) {
    U16x8 a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a.v[i] = f32_to_bf16(x[i]);
    *reinterpret_cast<U16x8*>(p) = a;
  }
  __device__ static float load1(const uint16_t* p) { return bf16_to_f32(*p); }
  __device__ static void store1(uint16_t* p, float x) { *p = f32_to_bf16(x); }
  __device__ static float rnd(float x) { return round_bf16(x); }
};

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace b2o
