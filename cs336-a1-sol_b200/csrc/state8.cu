// Optimizer state held in 8 bits (format in state8.cuh):
//   * AdamW step with both moments in 8 bits (+ EMA), over many tensors
//   * encode / decode of many states between 8 bits (or bf16 pairs) and fp32 / bf16
// Tensor lists go by value as kernel parameters, like the other streaming
// passes. One warp step covers 256 consecutive elements of one tensor, 8 a
// lane, so a scale's block is half a warp.
#include "b2o_common.cuh"
#include "b2o_internal.h"
#include "state8.cuh"
#include "vec_io.cuh"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

namespace b2o {

constexpr int kS8Threads = 256;
constexpr int kS8Tensors = 96;
constexpr int kS8Groups = 8;
constexpr int kS8Chunk = (kS8Threads / 32) * kQ8Tile * 4;  // elements per CTA step: four tiles a warp

static inline bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

// Eight elements at p + i of a list that ends at `end`; elements behind it read as 0.
template <typename T>
__device__ __forceinline__ void load_some(const T* p, int64_t i, int64_t end, bool vec, float* x) {
  if (vec) {
    Elem<T>::load8(p + i, x);
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = i + k < end ? Elem<T>::load1(p + i + k) : 0.0f;
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, int64_t i, int64_t end, bool vec, const float* x) {
  if (vec) {
    Elem<T>::store8(p + i, x);
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (i + k < end) Elem<T>::store1(p + i + k, x[k]);
}

// ================================================================ AdamW ===
// Coefficients of one group: bias corrections and 1 - beta from double on the
// host, rounded once.
struct Adam8Coef {
  float b1, w1, b2, w2;          // m = b1 m + w1 g, v = b2 v + w2 g^2
  float step_size, inv_bc2, eps;  // w -= step_size m / (sqrt(v) inv_bc2 + eps)
  float lr_wd;
  float step;                     // torch's state["step"]
  uint32_t turn;                  // the step count that the codes' offsets run with
  int wd_on, cautious;
  const float* grad_scale;
};

struct Adam8Table {
  b2o_adamw8_tensor t[kS8Tensors];
  Adam8Coef g[kS8Groups];
  int chunk_start[kS8Tensors + 1];
  int vec_ok[kS8Tensors];
  int ntensors;
  float ema_weight;
};

template <typename Table>
__device__ __forceinline__ int find_tensor(const Table& tab, int chunk) {
  int lo = 0, hi = tab.ntensors - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.chunk_start[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <typename PT>
__global__ void __launch_bounds__(kS8Threads) adamw8_kernel(const __grid_constant__ Adam8Table tab) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int total = tab.chunk_start[tab.ntensors];
  for (int chunk = blockIdx.x; chunk < total; chunk += gridDim.x) {
    const int ti = find_tensor(tab, chunk);
    const b2o_adamw8_tensor& T = tab.t[ti];
    const Adam8Coef& c = tab.g[T.group];
    if (T.step_out && chunk == tab.chunk_start[ti] && threadIdx.x == 0) *T.step_out = c.step;
    const int64_t base = static_cast<int64_t>(chunk - tab.chunk_start[ti]) * kS8Chunk;
    const int64_t end = min(T.numel, base + kS8Chunk);
    PT* __restrict__ P = static_cast<PT*>(T.param);
    const PT* __restrict__ G = static_cast<const PT*>(T.grad);
    const bool aligned = tab.vec_ok[ti] != 0;
    const float gs = c.grad_scale ? *c.grad_scale : 1.0f;
    for (int64_t tile = base + (threadIdx.x >> 5) * kQ8Tile; tile < end; tile += (kS8Threads / 32) * kQ8Tile) {
      const int64_t i = tile + lane * 8;
      const bool vec = aligned && i + 8 <= end;
      const int64_t blk = i / kQ8Block;
      float g[8], w[8], m[8], v[8];
      load_some(G, i, end, vec, g);
      load_some(P, i, end, vec, w);
      const float ms = i < end ? T.exp_avg_scale[blk] : 0.0f;
      const float vs = i < end ? T.exp_avg_sq_scale[blk] : 0.0f;
      unpack_signed(load_codes(T.exp_avg, i, end, vec), ms, m);
      unpack_root(load_codes(T.exp_avg_sq, i, end, vec), vs, v);
      if (T.rem) {
        float r[8];
        load_some(T.rem, i, end, vec, r);
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] += r[k];
      }
      if (c.grad_scale) {
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] = Elem<PT>::rnd(g[k] * gs);
      }
      // Each product and sum of the moments rounds by itself: what is stored
      // depends on their fp32 values alone, whatever the compiler contracts.
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        m[k] = __fadd_rn(__fmul_rn(c.b1, m[k]), __fmul_rn(c.w1, g[k]));
        v[k] = __fadd_rn(__fmul_rn(c.b2, v[k]), __fmul_rn(c.w2, __fmul_rn(g[k], g[k])));
      }
      const BlockScale sm = signed_scale(block_max(max_abs_bits(m)));
      const BlockScale sv = root_scale(block_max(max_abs_bits(v)));
      float r[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] = sqrt_approx(v[k]);
      const uint32_t h = dither_of(T.first + i, c.turn);
      if (i < end) {
        store_codes(T.exp_avg, i, end, vec, pack_signed<true>(m, sm, h));
        store_codes(T.exp_avg_sq, i, end, vec, pack_root<true>(v, r, sv, h));
        if ((lane & 15) == 0) {
          T.exp_avg_scale[blk] = sm.s;
          T.exp_avg_sq_scale[blk] = sv.s;
        }
      }
      float p[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (c.wd_on) w[k] -= (!c.cautious || m[k] * w[k] > 0.0f) ? c.lr_wd * w[k] : 0.0f;
        w[k] -= __fdividef(c.step_size * m[k], fmaf(r[k], c.inv_bc2, c.eps));
        p[k] = Elem<PT>::rnd(w[k]);
      }
      if (i < end) {
        store_some(P, i, end, vec, p);
        if (T.rem) {
          float q[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) q[k] = w[k] - p[k];
          store_some(T.rem, i, end, vec, q);
        }
        if (T.ema) {
          float e[8];
          load_some(T.ema, i, end, vec, e);
#pragma unroll
          for (int k = 0; k < 8; ++k) e[k] = torch_lerp(e[k], p[k], tab.ema_weight);
          store_some(T.ema, i, end, vec, e);
        }
      }
    }
  }
}

int adamw8_step(const b2o_adamw8_tensor* tensors, int ntensors, const b2o_adamw8_group* groups, int ngroups,
                int param_dtype, float ema_weight, cudaStream_t stream) {
  if (ntensors < 0 || (ntensors > 0 && !tensors)) { set_error("adamw8: bad tensor list"); return -1; }
  if (ngroups <= 0 || ngroups > kS8Groups || !groups) { set_error("adamw8: 1..8 groups required"); return -1; }
  if (param_dtype != B2O_F32 && param_dtype != B2O_BF16) { set_error("adamw8: bad param dtype"); return -1; }
  Adam8Table tab;
  memset(&tab, 0, sizeof(tab));
  for (int i = 0; i < ngroups; ++i) {
    const b2o_adamw8_group& g = groups[i];
    // (written so that NaN fails too)
    if (!(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0 && g.eps >= 0.0 && g.step >= 1.0 && g.step < 9e15)) {
      set_error("adamw8: group " + std::to_string(i) + " needs betas in [0, 1), eps >= 0 and step in [1, 9e15)");
      return -1;
    }
    Adam8Coef& c = tab.g[i];
    c.b1 = static_cast<float>(g.beta1); c.w1 = static_cast<float>(1.0 - g.beta1);
    c.b2 = static_cast<float>(g.beta2); c.w2 = static_cast<float>(1.0 - g.beta2);
    c.step_size = static_cast<float>(g.lr / (1.0 - std::pow(g.beta1, g.step)));
    c.inv_bc2 = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(g.beta2, g.step)));
    c.eps = static_cast<float>(g.eps);
    c.lr_wd = static_cast<float>(g.lr * g.weight_decay);
    c.step = static_cast<float>(g.step);
    c.turn = static_cast<uint32_t>(static_cast<int64_t>(g.step));
    c.wd_on = g.weight_decay != 0.0;
    c.cautious = g.cautious;
    c.grad_scale = g.grad_scale;
  }
  tab.ema_weight = ema_weight;
  for (int i = 0; i < ntensors; ++i) {
    const b2o_adamw8_tensor& t = tensors[i];
    if (t.numel < 0 || t.first < 0 || (t.numel > 0 && (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || !t.exp_avg_scale ||
                                        !t.exp_avg_sq_scale))) {
      set_error("adamw8: tensor " + std::to_string(i) + " has a null pointer or a negative size"); return -1;
    }
    if (t.first % kQ8Block) { set_error("adamw8: a slice starts at a multiple of 128 elements"); return -1; }
    if (t.group < 0 || t.group >= ngroups) { set_error("adamw8: tensor group out of range"); return -1; }
    if (t.rem && param_dtype != B2O_BF16) { set_error("adamw8: remainder needs bf16 params"); return -1; }
    if ((t.numel + kS8Chunk - 1) / kS8Chunk > (1ll << 30)) { set_error("adamw8: tensor too large"); return -1; }
  }
  for (int done = 0; done < ntensors;) {
    int n = 0, chunks = 0;
    for (; done + n < ntensors && n < kS8Tensors; ++n) {
      const b2o_adamw8_tensor& t = tensors[done + n];
      const int ch = static_cast<int>((t.numel + kS8Chunk - 1) / kS8Chunk);
      if (n > 0 && chunks + static_cast<int64_t>(ch) > (1ll << 30)) break;
      tab.t[n] = t;
      tab.chunk_start[n] = chunks;
      tab.vec_ok[n] = aligned16(t.param) && aligned16(t.grad) && aligned8(t.exp_avg) && aligned8(t.exp_avg_sq) &&
                      (!t.rem || aligned16(t.rem)) && (!t.ema || aligned16(t.ema));
      chunks += ch;
    }
    tab.chunk_start[n] = chunks;
    tab.ntensors = n;
    if (chunks > 0) {
      const int grid = std::min(chunks, num_sms() * 8);
      if (param_dtype == B2O_F32)
        launch_pdl(adamw8_kernel<float>, dim3(grid), dim3(kS8Threads), 0, stream, tab);
      else
        launch_pdl(adamw8_kernel<uint16_t>, dim3(grid), dim3(kS8Threads), 0, stream, tab);
      count_launch();
      if (int e = check_launch("adamw8")) return e;
    }
    done += n;
  }
  return 0;
}

// ====================================================== encode / decode ===
struct StateTable {
  b2o_state_tensor t[kS8Tensors];
  int chunk_start[kS8Tensors + 1];
  int vec_ok[kS8Tensors];
  int ntensors;
};

template <typename VT>
__device__ __forceinline__ void encode_tile(const b2o_state_tensor& T, int64_t i, int64_t end, bool vec, int lane) {
  float x[8];
  load_some(static_cast<const VT*>(T.value), i, end, vec, x);
  if (T.kind == B2O_STATE_PAIR) {
    if (i >= end) return;
    float r[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float p = round_bf16(x[k]);
      r[k] = x[k] - p;
      x[k] = p;
    }
    store_some(static_cast<uint16_t*>(T.codes), i, end, vec, x);
    store_some(static_cast<uint16_t*>(T.scales), i, end, vec, r);
    return;
  }
  const bool root = T.kind == B2O_STATE_ROOT;
  BlockScale b;
  uint2 codes;
  if (root) {
    // a second moment is not negative: a negative value counts as one that is not a number
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = x[k] < 0.0f ? __uint_as_float(0x7fffffffu) : x[k];
    b = root_scale(block_max(max_abs_bits(x)));
    float r[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) r[k] = sqrt_approx(x[k]);
    codes = pack_root<false>(x, r, b, 0);
  } else {
    b = signed_scale(block_max(max_abs_bits(x)));
    codes = pack_signed<false>(x, b, 0);
  }
  if (i >= end) return;
  store_codes(T.codes, i, end, vec, codes);
  if ((lane & 15) == 0) static_cast<float*>(T.scales)[i / kQ8Block] = b.s;
}

template <typename VT>
__device__ __forceinline__ void decode_tile(const b2o_state_tensor& T, int64_t i, int64_t end, bool vec) {
  if (i >= end) return;
  float x[8];
  if (T.kind == B2O_STATE_PAIR) {
    float r[8];
    load_some(static_cast<const uint16_t*>(T.codes), i, end, vec, x);
    load_some(static_cast<const uint16_t*>(T.scales), i, end, vec, r);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] += r[k];
  } else {
    const float s = static_cast<const float*>(T.scales)[i / kQ8Block];
    const uint2 codes = load_codes(T.codes, i, end, vec);
    if (T.kind == B2O_STATE_ROOT) unpack_root(codes, s, x);
    else unpack_signed(codes, s, x);
  }
  store_some(static_cast<VT*>(T.value), i, end, vec, x);
}

template <bool ENCODE>
__global__ void __launch_bounds__(kS8Threads) state_kernel(const __grid_constant__ StateTable tab) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int total = tab.chunk_start[tab.ntensors];
  for (int chunk = blockIdx.x; chunk < total; chunk += gridDim.x) {
    const int ti = find_tensor(tab, chunk);
    const b2o_state_tensor& T = tab.t[ti];
    const int64_t base = static_cast<int64_t>(chunk - tab.chunk_start[ti]) * kS8Chunk;
    const int64_t end = min(T.numel, base + kS8Chunk);
    for (int64_t tile = base + (threadIdx.x >> 5) * kQ8Tile; tile < end; tile += (kS8Threads / 32) * kQ8Tile) {
      const int64_t i = tile + lane * 8;
      const bool vec = tab.vec_ok[ti] && i + 8 <= end;
      if (T.value_dtype == B2O_F32) {
        if (ENCODE) encode_tile<float>(T, i, end, vec, lane);
        else decode_tile<float>(T, i, end, vec);
      } else {
        if (ENCODE) encode_tile<uint16_t>(T, i, end, vec, lane);
        else decode_tile<uint16_t>(T, i, end, vec);
      }
    }
  }
}

template <bool ENCODE>
static int state_launch(const b2o_state_tensor* tensors, int ntensors, cudaStream_t stream) {
  const std::string what = ENCODE ? "state_encode" : "state_decode";
  if (ntensors < 0 || (ntensors > 0 && !tensors)) { set_error(what + ": bad tensor list"); return -1; }
  for (int i = 0; i < ntensors; ++i) {
    const b2o_state_tensor& t = tensors[i];
    if (t.numel < 0 || (t.numel > 0 && (!t.value || !t.codes || !t.scales))) {
      set_error(what + ": tensor " + std::to_string(i) + " has a null pointer"); return -1;
    }
    if (t.kind != B2O_STATE_SIGNED && t.kind != B2O_STATE_ROOT && t.kind != B2O_STATE_PAIR) {
      set_error(what + ": tensor " + std::to_string(i) + " has an unknown kind"); return -1;
    }
    if (t.value_dtype != B2O_F32 && t.value_dtype != B2O_BF16) {
      set_error(what + ": values are fp32 or bf16"); return -1;
    }
    if ((t.numel + kS8Chunk - 1) / kS8Chunk > (1ll << 30)) { set_error(what + ": tensor too large"); return -1; }
  }
  StateTable tab;
  memset(&tab, 0, sizeof(tab));
  for (int done = 0; done < ntensors;) {
    int n = 0, chunks = 0;
    for (; done + n < ntensors && n < kS8Tensors; ++n) {
      const b2o_state_tensor& t = tensors[done + n];
      const int ch = static_cast<int>((t.numel + kS8Chunk - 1) / kS8Chunk);
      if (n > 0 && chunks + static_cast<int64_t>(ch) > (1ll << 30)) break;
      tab.t[n] = t;
      tab.chunk_start[n] = chunks;
      const bool pair = t.kind == B2O_STATE_PAIR;
      tab.vec_ok[n] = aligned16(t.value) && (pair ? aligned16(t.codes) && aligned16(t.scales) : aligned8(t.codes));
      chunks += ch;
    }
    tab.chunk_start[n] = chunks;
    tab.ntensors = n;
    if (chunks > 0) {
      const int grid = std::min(chunks, num_sms() * 8);
      launch_pdl(state_kernel<ENCODE>, dim3(grid), dim3(kS8Threads), 0, stream, tab);
      count_launch();
      if (int e = check_launch(what.c_str())) return e;
    }
    done += n;
  }
  return 0;
}

int64_t state_blocks(int64_t numel) { return numel <= 0 ? 0 : (numel + kQ8Block - 1) / kQ8Block; }

int state_encode(const b2o_state_tensor* tensors, int ntensors, cudaStream_t stream) {
  return state_launch<true>(tensors, ntensors, stream);
}
int state_decode(const b2o_state_tensor* tensors, int ntensors, cudaStream_t stream) {
  return state_launch<false>(tensors, ntensors, stream);
}

}  // namespace b2o
