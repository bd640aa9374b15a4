// Optimizer state held in 8 bits (format in state8.cuh):
//   * AdamW step with both moments in 8 bits (+ EMA), over many tensors
//   * encode / decode of many states between 8 bits (or bf16 pairs) and fp32 / bf16
// Tensor lists go by value as kernel parameters, like the other streaming
// passes. One warp step covers 256 consecutive elements of one tensor, 8 a
// lane, so a scale's block is half a warp.
#include "b2o_common.cuh"
#include "b2o_internal.h"
#include "state8.cuh"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

namespace b2o {

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int kS8Threads = 256;
constexpr int kS8Tensors = 96;
constexpr int kS8Groups = 8;
constexpr int kS8Chunk = (kS8Threads / 32) * kQ8Tile * 4;  // elements per CTA step: four tiles a warp

static inline bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

// ================================================================ AdamW ===
// Coefficients of one group: bias corrections and 1 - beta from double on the
// host, rounded once.
struct Adam8Coef {
  float b1, w1, b2, w2;          // m = b1 m + w1 g, v = b2 v + w2 g^2
  float step_size, inv_bc2, eps;  // w -= step_size m / (sqrt(v) inv_bc2 + eps)
  float lr_wd;
  float step;                     // torch's state["step"]
  uint32_t turn;                  // the step count that the codes' offsets run with
  float one;                      // 1 (see mul_add2)
  float far;                      // a root whose denominator is finite and has the reciprocal 0
  int wd_on, cautious;
  // 1: the roots of subnormal second moments may read as anything below 2^-63 in
  // the update (eps is more than 2^25 times that, so the denominator rounds to
  // eps); 0: they are computed, and root and quotient are IEEE's
  int plain_roots;
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

// One warp step: 256 elements, 8 a lane, blocks of 16 lanes.
// FULL: all of them exist and every pointer takes vector accesses. EXTRA 1: a
// group may have a clip coefficient or weight decay; 2: also an eps that does not
// cover the roots of subnormal second moments (see plain_roots): a launch of its own.
// `mine` are the step's first inputs, loaded during the step before.
template <typename PT>
struct Adam8In {
  Raw8<PT> g;
  uint2 mc, vc;
  float ms, vs;
  __device__ __forceinline__ void load(const b2o_adamw8_tensor& T, int64_t i, int64_t end, bool vec, bool in) {
    g.load(static_cast<const PT*>(T.grad), i, end, vec);
    mc = load_codes(T.exp_avg, i, end, vec);
    vc = load_codes(T.exp_avg_sq, i, end, vec);
    ms = in ? T.exp_avg_scale[i / kQ8Block] : 0.0f;
    vs = in ? T.exp_avg_sq_scale[i / kQ8Block] : 0.0f;
  }
};

template <typename PT, bool REM, bool EMA, int EXTRA, bool FULL>
__device__ __forceinline__ void adamw8_tile(const b2o_adamw8_tensor& T, const Adam8Coef& c, float ema_weight,
                                            const Adam8In<PT>& mine, int64_t i, int64_t end, bool aligned, float gs) {
  const bool vec = FULL || (aligned && i + 8 <= end);
  const bool in = FULL || i < end;
  const int64_t blk = i / kQ8Block;
  PT* const P = static_cast<PT*>(T.param);
  Raw8<PT> graw = mine.g, praw;
  Raw8<uint16_t> rraw;
  Raw8<float> eraw;
  praw.load(P, i, end, vec);
  if (REM) rraw.load(T.rem, i, end, vec);
  if (EMA) eraw.load(T.ema, i, end, vec);
  V8 g = graw.get();
  if (EXTRA && c.grad_scale) {
#pragma unroll
    for (int j = 0; j < 4; ++j) g.p[j] = mul2(g.p[j], f2(gs));
    graw.set(g);  // clipped gradient g = dtype(g * coef)
    g = graw.get();
  }
  // Each product and sum of the moments rounds by itself: what is stored
  // depends on their fp32 values alone, whatever the compiler contracts.
  V8 m = unpack_signed(mine.mc, mine.ms), v = unpack_root(mine.vc, mine.vs);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m.p[j] = mul_add2(f2(c.b1), m.p[j], mul2(f2(c.w1), g.p[j]), c.one);
    v.p[j] = mul_add2(f2(c.b2), v.p[j], mul2(f2(c.w2), mul2(g.p[j], g.p[j])), c.one);
  }
  const BlockScale sm = signed_scale(block_max<1>(&m));
  const BlockScale sv = root_scale(block_max<1>(&v));
  // Roots for the update and the codes. With a remainder the stored weight has
  // twice the bits, and the root gets a residual step (Newton: s + (v - s^2) /
  // (2 s)). Its remainder v - s^2 takes subnormal numbers as 0: 0 and subnormal v
  // keep the root 0, which sends their codes to the exact path, and a v below
  // 2^-103 keeps s, of which eps covers the last places.
  V8 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = f2_split(v.p[j]);
    if (EXTRA < 2) r.p[j] = f2(sqrt_approx_ftz(x.x), sqrt_approx_ftz(x.y));
    else if (REM) r.p[j] = f2(__fsqrt_rn(x.x), __fsqrt_rn(x.y));
    else r.p[j] = f2(sqrt_approx(x.x), sqrt_approx(x.y));
    if (REM && EXTRA < 2) {
      const F2 inv = f2(fminf(rsqrt_approx_ftz(x.x), 9.2233720e18f), fminf(rsqrt_approx_ftz(x.y), 9.2233720e18f));
      const F2 rest = fma2_ftz(mul2(r.p[j], f2(-1.0f)), r.p[j], v.p[j]);
      r.p[j] = fma2(rest, mul2(inv, f2(0.5f)), r.p[j]);
    }
  }
  // A second moment that has overflowed (its block's scale is then NaN and its
  // codes 0): the quotient is m / inf, 0 for a finite m, but the residual steps
  // would make it inf * 0. Its root is set so that the denominator is finite and
  // its reciprocal 0. One test for 8 elements costs nothing that shows (69.7 us
  // for 33.5 M bf16 weights); a test at each pair's quotient took 72.8.
  if (EXTRA < 2 && isnan(sv.s)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = f2_split(v.p[j]), y = f2_split(r.p[j]);
      r.p[j] = f2(isinf(x.x) ? c.far : y.x, isinf(x.y) ? c.far : y.y);
    }
  }
  if (!in) return;
  V8 w = praw.get();
  if (REM) {
    const V8 q = rraw.get();
#pragma unroll
    for (int j = 0; j < 4; ++j) w.p[j] = add2(w.p[j], q.p[j]);
  }
  if (EXTRA && c.wd_on) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (c.cautious) {
        const float2 x = f2_split(w.p[j]), y = f2_split(m.p[j]);
        w.p[j] = mul2(w.p[j], f2(x.x * y.x > 0.0f ? 1.0f - c.lr_wd : 1.0f, x.y * y.y > 0.0f ? 1.0f - c.lr_wd : 1.0f));
      } else {
        w.p[j] = mul_add2(w.p[j], f2(-c.lr_wd), w.p[j], c.one);
      }
    }
  }
  // w -= step_size m / (sqrt(v) inv_bc2 + eps), each operation rounded by itself.
  // The quotient is corrected by its residual (Markstein's step: q + (a - d q) /
  // d), so it is the rounded one: where a second moment is 0 the denominator is
  // eps alone, and an update that much larger than the weight would show the
  // approximation in the stored bf16 bits.
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const F2 minus_d = mul_add2(r.p[j], f2(-c.inv_bc2), f2(-c.eps), c.one);
    const F2 a = mul2(m.p[j], f2(-c.step_size));
    const float2 d = f2_split(minus_d);
    F2 q;
    if (EXTRA < 2) {
      const F2 inv = f2(rcp_approx_ftz(-d.x), rcp_approx_ftz(-d.y));
      q = mul2(a, inv);
      q = fma2(fma2(minus_d, q, a), inv, q);
    } else {  // (eps may be 0, and with it the denominator)
      const float2 x = f2_split(a);
      q = f2(__fdiv_rn(x.x, -d.x), __fdiv_rn(x.y, -d.y));
    }
    w.p[j] = add2(w.p[j], q);
  }
  praw.set(w);
  praw.store(P, i, end, vec);
  const V8 p = praw.get();  // the weight as it is stored
  if (REM) {
    V8 q;
#pragma unroll
    for (int j = 0; j < 4; ++j) q.p[j] = fma2(p.p[j], f2(-1.0f), w.p[j]);
    rraw.set(q);
    rraw.store(T.rem, i, end, vec);
  }
  if (EMA) {
    V8 e = eraw.get();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = f2_split(e.p[j]), y = f2_split(p.p[j]);
      e.p[j] = f2(torch_lerp(x.x, y.x, ema_weight), torch_lerp(x.y, y.y, ema_weight));
    }
    eraw.set(e);
    eraw.store(T.ema, i, end, vec);
  }
  const uint32_t h = dither_of(T.first + i, c.turn);
  store_codes(T.exp_avg, i, end, vec, pack_signed<true>(m, sm, h));
  store_codes(T.exp_avg_sq, i, end, vec, pack_root<true>(v, r, sv, h));
  if ((threadIdx.x & 15) == 0) {
    T.exp_avg_scale[blk] = sm.s;
    T.exp_avg_sq_scale[blk] = sv.s;
  }
}

// 256 threads, a chunk of 8192 elements a CTA, 3 or 4 CTAs an SM (80 or 64
// registers). Measured on 33.5 M elements (a 32768 x 1024 table) without zeros,
// against copy bandwidth: bf16 weights 70 us (74 %, bound by instruction issue: 58
// an element), with weight decay 78 us (66 %; 65 instructions, no two-step unroll),
// with a remainder 83 us (87 %), with a remainder and cautious decay 97 us (74 %; 82
// instructions), with remainder and EMA 118 us (96 %); fp32 83 us (99 %), with decay
// 88 us (94 %), with the EMA 123 us (100 %). The residual steps of quotient and
// root cost 2 and 4 us where issue binds. Without the loads a step ahead the
// first of these took 102 us; with 2 CTAs an SM 145; 16 elements a lane instead
// of 8 took 19 % fewer instructions and the same time (fewer warps).
template <typename PT, bool REM, bool EMA, int EXTRA>
__global__ void __launch_bounds__(kS8Threads, EMA || EXTRA == 2 ? 3 : 4)
    adamw8_kernel(const __grid_constant__ Adam8Table tab) {
  pdl_wait();
  const int ti = find_tensor(tab, blockIdx.x);
  const b2o_adamw8_tensor& T = tab.t[ti];
  const Adam8Coef& c = tab.g[T.group];
  const int first = tab.chunk_start[ti];
  if (T.step_out && blockIdx.x == first && threadIdx.x == 0) *T.step_out = c.step;
  const int64_t base = static_cast<int64_t>(blockIdx.x - first) * kS8Chunk;
  const int64_t end = min(T.numel, base + kS8Chunk);
  const float gs = EXTRA && c.grad_scale ? *c.grad_scale : 1.0f;
  const int64_t i0 = base + (threadIdx.x >> 5) * kQ8Tile + (threadIdx.x & 31) * 8;
  constexpr int kStride = (kS8Threads / 32) * kQ8Tile;
  // two steps where the registers suffice: fewer moves
  constexpr int kUnroll = sizeof(PT) == 2 && !EMA && !EXTRA ? 2 : 1;
  if (tab.vec_ok[ti] && base + kS8Chunk <= T.numel) {
    Adam8In<PT> next;
    next.load(T, i0, end, true, true);
#pragma unroll kUnroll
    for (int n = 0; n < kS8Chunk / kStride; ++n) {
      const Adam8In<PT> mine = next;
      if (n + 1 < kS8Chunk / kStride) next.load(T, i0 + (n + 1) * kStride, end, true, true);
      adamw8_tile<PT, REM, EMA, EXTRA, true>(T, c, tab.ema_weight, mine, i0 + n * kStride, end, true, gs);
    }
  } else {
#pragma unroll 1
    for (int64_t i = i0; i - (threadIdx.x & 31) * 8 < end; i += kStride) {
      Adam8In<PT> mine;
      mine.load(T, i, end, tab.vec_ok[ti] && i + 8 <= end, i < end);
      adamw8_tile<PT, REM, EMA, EXTRA, false>(T, c, tab.ema_weight, mine, i, end, tab.vec_ok[ti] != 0, gs);
    }
  }
}

template <typename PT, bool REM, bool EMA>
static void adamw8_launch(const Adam8Table& tab, int chunks, int extra, cudaStream_t stream) {
  launch_pdl(extra == 2   ? adamw8_kernel<PT, REM, EMA, 2>
             : extra == 1 ? adamw8_kernel<PT, REM, EMA, 1>
                          : adamw8_kernel<PT, REM, EMA, 0>,
             dim3(chunks), dim3(kS8Threads), 0, stream, tab);
}
template <typename PT, bool REM>
static void adamw8_launch(const Adam8Table& tab, int chunks, bool ema, int extra, cudaStream_t stream) {
  if (ema) adamw8_launch<PT, REM, true>(tab, chunks, extra, stream);
  else adamw8_launch<PT, REM, false>(tab, chunks, extra, stream);
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
    c.inv_bc2 = 1.0f / static_cast<float>(std::sqrt(1.0 - std::pow(g.beta2, g.step)));
    c.eps = static_cast<float>(g.eps);
    c.lr_wd = static_cast<float>(g.lr * g.weight_decay);
    c.step = static_cast<float>(g.step);
    c.turn = static_cast<uint32_t>(static_cast<int64_t>(g.step));
    c.one = 1.0f;
    c.far = 3e38f / c.inv_bc2;
    c.wd_on = g.weight_decay != 0.0;
    c.cautious = g.cautious;
    // eps 2^-25 >= 2^-63 inv_bc2 (and below the numbers whose reciprocal is subnormal)
    c.plain_roots = c.eps * 2.9802322e-8f >= 1.0842022e-19f * c.inv_bc2 && c.eps < 1e37f;
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
  // One launch for each mix of remainder, EMA and eps (one in all, as a rule): the
  // passes without them are then without their branches too, and a tensor's
  // result depends on its own group alone, not on what shares its launch.
  for (int mix = 0; mix < 8; ++mix) {
    const bool rem = (mix & 1) != 0, ema = (mix & 2) != 0, exact = (mix & 4) != 0;
    for (int at = 0; at < ntensors;) {
      int n = 0, chunks = 0;
      int extra = 0;
      for (; at < ntensors && n < kS8Tensors; ++at) {
        const b2o_adamw8_tensor& t = tensors[at];
        const Adam8Coef& c = tab.g[t.group];
        if (t.numel == 0 || (t.rem != nullptr) != rem || (t.ema != nullptr) != ema || (c.plain_roots == 0) != exact) continue;
        const int ch = static_cast<int>((t.numel + kS8Chunk - 1) / kS8Chunk);
        if (n > 0 && chunks + static_cast<int64_t>(ch) > (1ll << 30)) break;
        tab.t[n] = t;
        tab.chunk_start[n] = chunks;
        tab.vec_ok[n] = aligned16(t.param) && aligned16(t.grad) && aligned8(t.exp_avg) && aligned8(t.exp_avg_sq) &&
                        (!t.rem || aligned16(t.rem)) && (!t.ema || aligned16(t.ema));
        extra = std::max(extra, exact ? 2 : c.grad_scale || c.wd_on ? 1 : 0);
        chunks += ch;
        ++n;
      }
      if (n == 0) break;
      tab.chunk_start[n] = chunks;
      tab.ntensors = n;
      if (param_dtype == B2O_F32) adamw8_launch<float, false>(tab, chunks, ema, extra, stream);
      else if (rem) adamw8_launch<uint16_t, true>(tab, chunks, ema, extra, stream);
      else adamw8_launch<uint16_t, false>(tab, chunks, ema, extra, stream);
      count_launch();
      if (int e = check_launch("adamw8")) return e;
    }
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

// Two tiles a step, loads of both before the work of either.
constexpr int kS8Two = 2;

template <typename VT, int KIND, bool FULL>
__device__ __forceinline__ void encode_tiles(const b2o_state_tensor& T, int64_t tile, int64_t end, bool aligned,
                                             int lane) {
  Raw8<VT> raw[kS8Two];
  int64_t i[kS8Two];
  bool vec[kS8Two];
#pragma unroll
  for (int n = 0; n < kS8Two; ++n) {
    i[n] = tile + n * kQ8Tile + lane * 8;
    vec[n] = FULL || (aligned && i[n] + 8 <= end);
    raw[n].load(static_cast<const VT*>(T.value), i[n], end, vec[n]);
  }
#pragma unroll
  for (int n = 0; n < kS8Two; ++n) {
    V8 x = raw[n].get();
    if (KIND == B2O_STATE_PAIR) {
      if (!FULL && i[n] >= end) continue;
      Raw8<uint16_t> p, r;
      p.set(x);
      const V8 y = p.get();
#pragma unroll
      for (int j = 0; j < 4; ++j) x.p[j] = fma2(y.p[j], f2(-1.0f), x.p[j]);
      r.set(x);
      p.store(static_cast<uint16_t*>(T.codes), i[n], end, vec[n]);
      r.store(static_cast<uint16_t*>(T.scales), i[n], end, vec[n]);
      continue;
    }
    BlockScale b;
    uint2 codes;
    if (KIND == B2O_STATE_ROOT) {
      // a second moment is not negative: a negative value counts as one that is not a number
      V8 r;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 y = f2_split(x.p[j]);
        y.x = y.x < 0.0f ? __int_as_float(0x7fffffff) : y.x;
        y.y = y.y < 0.0f ? __int_as_float(0x7fffffff) : y.y;
        x.p[j] = f2(y.x, y.y);
        r.p[j] = f2(sqrt_approx_ftz(y.x), sqrt_approx_ftz(y.y));
      }
      b = root_scale(block_max<1>(&x));
      codes = pack_root<false>(x, r, b, 0);
    } else {
      b = signed_scale(block_max<1>(&x));
      codes = pack_signed<false>(x, b, 0);
    }
    if (!FULL && i[n] >= end) continue;
    store_codes(T.codes, i[n], end, vec[n], codes);
    if ((lane & 15) == 0) static_cast<float*>(T.scales)[i[n] / kQ8Block] = b.s;
  }
}

template <typename VT>
__device__ __forceinline__ void decode_tiles(const b2o_state_tensor& T, int64_t tile, int64_t end, bool aligned,
                                             int lane) {
  int64_t i[kS8Two];
  bool vec[kS8Two];
#pragma unroll
  for (int n = 0; n < kS8Two; ++n) {
    i[n] = tile + n * kQ8Tile + lane * 8;
    vec[n] = aligned && i[n] + 8 <= end;
  }
  V8 x[kS8Two];
  if (T.kind == B2O_STATE_PAIR) {
    Raw8<uint16_t> p[kS8Two], r[kS8Two];
#pragma unroll
    for (int n = 0; n < kS8Two; ++n) {
      p[n].load(static_cast<const uint16_t*>(T.codes), i[n], end, vec[n]);
      r[n].load(static_cast<const uint16_t*>(T.scales), i[n], end, vec[n]);
    }
#pragma unroll
    for (int n = 0; n < kS8Two; ++n) {
      x[n] = p[n].get();
      const V8 y = r[n].get();
#pragma unroll
      for (int j = 0; j < 4; ++j) x[n].p[j] = add2(x[n].p[j], y.p[j]);
    }
  } else {
    float s[kS8Two];
    uint2 codes[kS8Two];
#pragma unroll
    for (int n = 0; n < kS8Two; ++n) {
      codes[n] = load_codes(T.codes, i[n], end, vec[n]);
      s[n] = i[n] < end ? static_cast<const float*>(T.scales)[i[n] / kQ8Block] : 0.0f;
    }
#pragma unroll
    for (int n = 0; n < kS8Two; ++n)
      x[n] = T.kind == B2O_STATE_ROOT ? unpack_root(codes[n], s[n]) : unpack_signed(codes[n], s[n]);
  }
#pragma unroll
  for (int n = 0; n < kS8Two; ++n) {
    if (i[n] >= end) continue;
    Raw8<VT> raw;
    raw.set(x[n]);
    raw.store(static_cast<VT*>(T.value), i[n], end, vec[n]);
  }
}

// A whole chunk decoded, vector accesses: a warp takes 1024 elements in a row.
// fp32 values are written 4 a lane, so that a store covers 512 bytes in a row:
// with 8 a lane, in two halves 32 bytes apart, 33.5 M codes took 37 us instead
// of 26. Stores are streaming ones: nothing here reads them again.
constexpr int kS8Warp = kS8Chunk / (kS8Threads / 32);

__device__ __forceinline__ void decode_whole(const b2o_state_tensor& T, int64_t at, int lane, float) {
  constexpr int kN = kS8Warp / kQ8Block;
  float* const out = static_cast<float*>(T.value) + at + lane * 4;
  if (T.kind == B2O_STATE_PAIR) {
    uint2 p[kN], r[kN];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      p[n] = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(T.codes) + at + n * kQ8Block + lane * 4);
      r[n] = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(T.scales) + at + n * kQ8Block + lane * 4);
    }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const float2 x = f2_split(add2(Raw8<uint16_t>::pair(p[n].x), Raw8<uint16_t>::pair(r[n].x)));
      const float2 y = f2_split(add2(Raw8<uint16_t>::pair(p[n].y), Raw8<uint16_t>::pair(r[n].y)));
      __stcs(reinterpret_cast<float4*>(out + n * kQ8Block), make_float4(x.x, x.y, y.x, y.y));
    }
    return;
  }
  const float* const sc = static_cast<const float*>(T.scales) + at / kQ8Block;
  uint32_t w[kN];
  float s[kN];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    w[n] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(T.codes) + at + n * kQ8Block + lane * 4);
    s[n] = sc[n];
  }
  const bool root = T.kind == B2O_STATE_ROOT;
#pragma unroll
  for (int n = 0; n < kN; ++n) __stcs(reinterpret_cast<float4*>(out + n * kQ8Block), unpack4(w[n], s[n], root));
}

__device__ __forceinline__ void decode_whole(const b2o_state_tensor& T, int64_t at, int lane, uint16_t) {
  constexpr int kN = kS8Warp / kQ8Tile;
  const int64_t i = at + lane * 8;
  uint4* const out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(T.value) + i);
  if (T.kind == B2O_STATE_PAIR) {
    Raw8<uint16_t> p[kN], r[kN];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      p[n].load(static_cast<const uint16_t*>(T.codes), i + n * kQ8Tile, 0, true);
      r[n].load(static_cast<const uint16_t*>(T.scales), i + n * kQ8Tile, 0, true);
    }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      V8 x = p[n].get();
      const V8 y = r[n].get();
#pragma unroll
      for (int j = 0; j < 4; ++j) x.p[j] = add2(x.p[j], y.p[j]);
      p[n].set(x);
      __stcs(out + n * (kQ8Tile / 8), p[n].a);
    }
    return;
  }
  uint2 w[kN];
  float s[kN];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    w[n] = load_codes(T.codes, i + n * kQ8Tile, 0, true);
    s[n] = static_cast<const float*>(T.scales)[i / kQ8Block + 2 * n];
  }
  const bool root = T.kind == B2O_STATE_ROOT;
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    Raw8<uint16_t> v;
    v.set(root ? unpack_root(w[n], s[n]) : unpack_signed(w[n], s[n]));
    __stcs(out + n * (kQ8Tile / 8), v.a);
  }
}

template <typename VT, int KIND>
__device__ __forceinline__ void encode_chunk(const b2o_state_tensor& T, int64_t base, int64_t end, bool aligned,
                                             int lane, int warp) {
  constexpr int kStep = kS8Two * kQ8Tile, kStride = (kS8Threads / 32) * kStep;
  if (aligned && end - base == kS8Chunk) {
#pragma unroll
    for (int n = 0; n < kS8Chunk / kStride; ++n)
      encode_tiles<VT, KIND, true>(T, base + warp * kStep + n * kStride, end, true, lane);
    return;
  }
#pragma unroll 1
  for (int64_t tile = base + warp * kStep; tile < end; tile += kStride)
    encode_tiles<VT, KIND, false>(T, tile, end, aligned, lane);
}

template <bool ENCODE, typename VT>
__device__ __forceinline__ void state_chunk(const b2o_state_tensor& T, int64_t base, bool aligned) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t end = min(T.numel, base + kS8Chunk);
  if (!ENCODE && aligned && base + kS8Chunk <= T.numel) {
    decode_whole(T, base + warp * kS8Warp, lane, VT());
    return;
  }
  if (ENCODE) {
    if (T.kind == B2O_STATE_SIGNED) encode_chunk<VT, B2O_STATE_SIGNED>(T, base, end, aligned, lane, warp);
    else if (T.kind == B2O_STATE_ROOT) encode_chunk<VT, B2O_STATE_ROOT>(T, base, end, aligned, lane, warp);
    else encode_chunk<VT, B2O_STATE_PAIR>(T, base, end, aligned, lane, warp);
    return;
  }
  for (int64_t tile = base + warp * (kS8Two * kQ8Tile); tile < end; tile += (kS8Threads / 32) * (kS8Two * kQ8Tile))
    decode_tiles<VT>(T, tile, end, aligned, lane);
}

// 5 CTAs an SM (48 registers): the writing of codes is issue-bound and needs the
// warps (33.5 M elements, signed: bf16 25.9 us against 30.8 with 3, fp32 26.7
// against 31.5; with one tile a step instead of two 28.4 and 30.2). From bf16 it is
// at 60 % (signed) and 53 % (root) of copy bandwidth with the ALU pipe 74 and 69 %
// busy and issue slots 64 and 63 %: neither is full, so latency has a part.
template <bool ENCODE>
__global__ void __launch_bounds__(kS8Threads, 5) state_kernel(const __grid_constant__ StateTable tab) {
  pdl_wait();
  const int ti = find_tensor(tab, blockIdx.x);
  const b2o_state_tensor& T = tab.t[ti];
  const int64_t base = static_cast<int64_t>(blockIdx.x - tab.chunk_start[ti]) * kS8Chunk;
  if (T.value_dtype == B2O_F32) state_chunk<ENCODE, float>(T, base, tab.vec_ok[ti] != 0);
  else state_chunk<ENCODE, uint16_t>(T, base, tab.vec_ok[ti] != 0);
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
      launch_pdl(state_kernel<ENCODE>, dim3(chunks), dim3(kS8Threads), 0, stream, tab);
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
