// linear.cuh -- device pieces shared by the fused linear operators (linear.cu)
// and the 8-bit activation checkpoints (ckpt8.cu): element types, activations
// and their slopes, the checkpoint's group code, and the epilogue.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace orca {
namespace lin {

// ---------------------------------------------------------------- element types
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// V consecutive elements at p as f32.  `vec` (uniform): p is aligned to
// min(16, V * sizeof(T)) bytes and all V elements are inside.
template <typename T, int V>
__device__ __forceinline__ void load_row(const T* p, int valid, bool vec, float (&v)[V]) {
  constexpr int BYTES = V * (int)sizeof(T);
  if (vec) {
    union { uint4 q[(BYTES + 15) / 16]; uint2 d; T e[V]; } u;
    if (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) u.q[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      u.d = *reinterpret_cast<const uint2*>(p);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32(u.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < valid ? to_f32(p[i]) : 0.0f;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, int valid, bool vec, const float (&v)[V]) {
  constexpr int BYTES = V * (int)sizeof(T);
  if (vec) {
    union { uint4 q[(BYTES + 15) / 16]; uint2 d; T e[V]; } u;
#pragma unroll
    for (int i = 0; i < V; ++i) u.e[i] = from_f32<T>(v[i]);
    if (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(p)[i] = u.q[i];
    } else {
      *reinterpret_cast<uint2*>(p) = u.d;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < valid) p[i] = from_f32<T>(v[i]);
  }
}

// ---------------------------------------------------------------- activations
// f(z) and f'(z) in f32.  f is off by up to 2^-21.5 of |z| (GELU; 2^-22.5 the others),
// f' by up to 2^-21.5 of 1 + |z|, measured over |z| <= 12; both 2^-24 rms, where the sums of
// F32 products are off by 2^-22.5 rms.  Relative to f itself GELU's tail is off by 5e-4 at -4
// and 4e-3, half a BF16 step, at -6.  erf, expf and divisions would be off by 2^-23 of |z|
// and take several times the instructions.  They run in epilogues and
// in passes bound by HBM, so they take two values at a time (packed f32 arithmetic
// issues once for both), are built from the fast exponential and reciprocal and
// have no branches.  ReLU is z > 0 ? z : 0, as the F32 path's.
struct F2 {
  uint64_t u;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.u) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ void split(F2 x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.u));
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.u) : "l"(a.u), "l"(b.u), "l"(c.u));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <typename F> __device__ __forceinline__ F2 each(F2 x, F f) {
  float a, b;
  split(x, a, b);
  return f2(f(a), f(b));
}
__device__ __forceinline__ F2 rcp2(F2 x) { return each(x, [](float v) { return rcp(v); }); }
__device__ __forceinline__ F2 exp2_2(F2 x) { return each(x, [](float v) { return exp2_fast(v); }); }
constexpr float LOG2_E = 1.44269504f;

// -Q(|z|), Q the normal upper tail erfc(|z| / sqrt 2) / 2, by formula 7.1.26 of
// Abramowitz and Stegun (|error| of erf <= 1.5e-7): a polynomial in
// t = 1 / (1 + p x) times e^(-x^2), x = |z| / sqrt 2.  x2 = |z|, bounded so that
// an infinity times 0 does not become a NaN (a NaN stays one through e);
// e = e^(-z^2 / 2).
__device__ __forceinline__ F2 normal_tail(F2 z, F2& x2, F2& e) {
  x2 = each(z, [](float v) { return fminf(fabsf(v), 1e38f); });
  const F2 t = rcp2(fma2(f2(0.3275911f * 0.70710678f), x2, f2(1.0f)));
  F2 q = fma2(t, f2(-0.5f * 1.061405429f), f2(0.5f * 1.453152027f));
  q = fma2(t, q, f2(-0.5f * 1.421413741f));
  q = fma2(t, q, f2(0.5f * 0.284496736f));
  q = fma2(t, q, f2(-0.5f * 0.254829592f));
  e = exp2_2(mul2(mul2(z, z), f2(-0.5f * LOG2_E)));
  return mul2(mul2(q, t), e);
}
// 1 / (1 + e^-x); 0 below about -88, where e^-x is infinite.
__device__ __forceinline__ F2 sigmoid2(F2 x) {
  return rcp2(add2(exp2_2(mul2(x, f2(-LOG2_E))), f2(1.0f)));
}
// 2 sqrt(2 / pi) (z + 0.044715 z^3): (1 + tanh(half of it)) / 2 is its sigmoid.
__device__ __forceinline__ F2 tanh_arg(F2 z) {
  return mul2(z, fma2(mul2(z, z), f2(0.0713548163f), f2(1.59576912f)));
}

template <int ACT> __device__ __forceinline__ F2 act_value(F2 z) {
  if (ACT == ORCA_ACT_RELU) return each(z, [](float v) { return v > 0.0f ? v : 0.0f; });
  if (ACT == ORCA_ACT_GELU) {
    // z (1 - Q) above 0, z Q below: z or 0, less |z| Q.
    F2 x, e;
    const F2 q = normal_tail(z, x, e);
    return fma2(x, q, each(z, [](float v) { return fmaxf(v, 0.0f); }));
  }
  if (ACT == ORCA_ACT_GELU_TANH) return mul2(z, sigmoid2(tanh_arg(z)));
  return mul2(z, sigmoid2(z));   // SiLU
}
template <int ACT> __device__ __forceinline__ F2 act_slope(F2 z) {
  if (ACT == ORCA_ACT_RELU) return each(z, [](float v) { return v > 0.0f ? 1.0f : 0.0f; });
  if (ACT == ORCA_ACT_GELU) {
    // Phi(z) = 1/2 + sign(z) (1/2 - Q), and z times the density.
    F2 x, e;
    const F2 h = add2(normal_tail(z, x, e), f2(0.5f));
    float a, b, ha, hb;
    split(z, a, b);
    split(h, ha, hb);
    return fma2(mul2(z, f2(0.39894228f)), e, add2(f2(copysignf(ha, a), copysignf(hb, b)), f2(0.5f)));
  }
  if (ACT == ORCA_ACT_GELU_TANH) {
    // Beyond |z| = 10 the sigmoid is 0 or 1 in f32 and the second term 0; the
    // bound keeps z * z finite there.  A NaN stays one through z - z.
    const F2 y = each(z, [](float v) { return fminf(fmaxf(v, -10.0f), 10.0f); });
    const F2 s = sigmoid2(tanh_arg(y));
    const F2 up = fma2(mul2(y, y), f2(0.2140644489f), f2(1.59576912f));
    const F2 r = fma2(mul2(mul2(y, s), fma2(s, f2(-1.0f), f2(1.0f))), up, s);
    return add2(r, fma2(z, f2(-1.0f), z));
  }
  const F2 s = sigmoid2(z);      // SiLU
  return mul2(s, fma2(z, fma2(s, f2(-1.0f), f2(1.0f)), f2(1.0f)));
}

// v = f(v), or v *= f'(z), for V values with one uniform branch for all.
template <int ACT, int V> __device__ __forceinline__ void act_all(float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 2) split(act_value<ACT>(f2(v[i], v[i + 1])), v[i], v[i + 1]);
}
template <int ACT, int V> __device__ __forceinline__ void slope_all(const float (&z)[V], float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 2)
    split(mul2(f2(v[i], v[i + 1]), act_slope<ACT>(f2(z[i], z[i + 1]))), v[i], v[i + 1]);
}
template <int V> __device__ __forceinline__ void apply_act(int act, float (&v)[V]) {
  switch (act) {
    case ORCA_ACT_RELU: act_all<ORCA_ACT_RELU>(v); break;
    case ORCA_ACT_GELU: act_all<ORCA_ACT_GELU>(v); break;
    case ORCA_ACT_GELU_TANH: act_all<ORCA_ACT_GELU_TANH>(v); break;
    case ORCA_ACT_SILU: act_all<ORCA_ACT_SILU>(v); break;
    default: break;
  }
}
template <int V> __device__ __forceinline__ void mul_slope(int act, const float (&z)[V], float (&v)[V]) {
  switch (act) {
    case ORCA_ACT_RELU: slope_all<ORCA_ACT_RELU>(z, v); break;
    case ORCA_ACT_GELU: slope_all<ORCA_ACT_GELU>(z, v); break;
    case ORCA_ACT_GELU_TANH: slope_all<ORCA_ACT_GELU_TANH>(z, v); break;
    case ORCA_ACT_SILU: slope_all<ORCA_ACT_SILU>(z, v); break;
    default: break;
  }
}

// ---------------------------------------------------------------- 8-bit checkpoints
// A matrix [m, n] in 8 bits: codes [m * n], then at the next multiple of 16
// bytes one exponent byte per row and group of 32 columns.  value =
// code * 2^(E - 127); the power of two makes both the scaling and the decoded
// value exact (7 bits and a sign fit BF16), so rounding to the code is the only
// error: at most half a step, one step where 127.5 and above saturate.  A
// step is 2^-6 of the power of two at or below the group's largest value.
constexpr int GROUP = 32;
constexpr uint32_t E_NONFINITE = 255;

__host__ __device__ inline int64_t ckpt_groups(int64_t n) { return (n + GROUP - 1) / GROUP; }
__host__ __device__ inline int64_t ckpt_exps_at(int64_t m, int64_t n) { return (m * n + 15) / 16 * 16; }

// The largest magnitude of a, |v|, |w|; a NaN among them stays.
__device__ __forceinline__ float ckpt_max(float a, float v, float w) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(v), "f"(w));
  return r;
}
__device__ __forceinline__ uint32_t ckpt_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);       // a NaN is above an infinity
  if (bits >= 0x7f800000u) return E_NONFINITE;
  const int e = (int)(bits >> 23) - 6;
  return (uint32_t)(e < 1 ? 1 : e);
}
__device__ __forceinline__ float ckpt_up(uint32_t e) {      // 2^(127 - E); 0 for a marked group
  return e == E_NONFINITE ? 0.0f : __uint_as_float((254u - e) << 23);
}
__device__ __forceinline__ float ckpt_down(uint32_t e) {    // 2^(E - 127); NaN for a marked group
  return e == E_NONFINITE ? __uint_as_float(0x7fffffffu) : __uint_as_float(e << 23);
}
// Codes of N values, four to a word.  v * up is exact, and adding 1.5 * 2^23 rounds
// it to the nearest whole number, ties to even, into the low mantissa bits: no
// conversion instruction (those share a slow pipe with the exponentials).  Only
// a group whose largest value reaches 127.5 (one in 256) needs the bounds.
template <int N>
__device__ __forceinline__ void ckpt_words(const float* v, float amax, float up, uint32_t* w) {
  const F2 scale = f2(up), magic = f2(12582912.0f);
  const bool bound = amax * up >= 127.5f;
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    float q[4];
    if (!bound) {
      split(fma2(f2(v[i], v[i + 1]), scale, magic), q[0], q[1]);
      split(fma2(f2(v[i + 2], v[i + 3]), scale, magic), q[2], q[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = fminf(fmaxf(v[i + j] * up, -127.0f), 127.0f) + 12582912.0f;
    }
    const uint32_t a = __byte_perm(__float_as_uint(q[0]), __float_as_uint(q[1]), 0x0040);
    const uint32_t b = __byte_perm(__float_as_uint(q[2]), __float_as_uint(q[3]), 0x0040);
    w[i / 4] = up == 0.0f ? 0u : __byte_perm(a, b, 0x5410);
  }
}

// Values of the four codes of a word: a code plus 128 as the low mantissa byte of
// 2^23, less 2^23 + 128 (exact; again no conversion instruction).
__device__ __forceinline__ void ckpt_values(uint32_t word, float down, float* v) {
  const uint32_t w = word ^ 0x80808080u;
  const F2 scale = f2(down), less = f2(-8388736.0f);
  const auto at = [&](int sel) { return __uint_as_float(__byte_perm(w, 0x4B000000u, sel)); };
  split(mul2(add2(f2(at(0x7440), at(0x7441)), less), scale), v[0], v[1]);
  split(mul2(add2(f2(at(0x7442), at(0x7443)), less), scale), v[2], v[3]);
}

// Codes the V values of one lane, 32 / V adjacent lanes sharing a group (all
// of them call this), and stores codes and exponent.  Columns from `valid` on
// are outside.  V is 4 or 8; `align`: of the rows of codes, in bytes (16, 8, 4, 1).
template <int V>
__device__ __forceinline__ void ckpt_store(uint8_t* codes, uint8_t* exps, int64_t row, int64_t n,
                                           int64_t col, int valid, bool row_ok, int align,
                                           const float (&v)[V]) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < V; i += 2)
    amax = ckpt_max(amax, i < valid ? v[i] : 0.0f, i + 1 < valid ? v[i + 1] : 0.0f);
#pragma unroll
  for (int o = 1; o < GROUP / V; o <<= 1) amax = ckpt_max(amax, amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (!row_ok || valid <= 0) return;
  const uint32_t e = ckpt_exponent(amax);
  const float up = ckpt_up(e);
  if (col % GROUP == 0) exps[row * ckpt_groups(n) + col / GROUP] = (uint8_t)e;
  uint8_t* p = codes + row * n + col;
  uint32_t w[V / 4];
  ckpt_words<V>(v, amax, up, w);
  if (valid >= V && align >= 4) {
    if (V == 8 && align >= 8) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[V / 4 - 1]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) reinterpret_cast<uint32_t*>(p)[i] = w[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < valid) p[i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
  }
}

// The V (4 or 8) values at (row, col .. col + V) of a checkpoint; col is a multiple of
// V, so they share one exponent.
template <int V>
__device__ __forceinline__ void ckpt_load(const uint8_t* codes, const uint8_t* exps, int64_t row,
                                          int64_t n, int64_t col, int valid, int align,
                                          float (&v)[V]) {
  const float down = valid > 0 ? ckpt_down(exps[row * ckpt_groups(n) + col / GROUP]) : 0.0f;
  const uint8_t* p = codes + row * n + col;
  if (valid >= V && align >= 4) {
    uint32_t w[V / 4];
    if (V == 8 && align >= 8) {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      w[0] = q.x;
      w[V / 4 - 1] = q.y;
    } else {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
#pragma unroll
    for (int i = 0; i < V / 4; ++i) ckpt_values(w[i], down, v + 4 * i);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < valid ? (float)(int8_t)p[i] * down : 0.0f;
  }
}

// Largest of 16, 8, 4, 1 that divides both the pointer and the row stride.
inline int byte_alignment(const void* p, int64_t stride) {
  const uint64_t v = reinterpret_cast<uintptr_t>(p) | (uint64_t)stride;
  return v % 16 == 0 ? 16 : (v % 8 == 0 ? 8 : (v % 4 == 0 ? 4 : 1));
}

// ---------------------------------------------------------------- epilogue
enum Mode : int { FWD = 0, DX = 1, DW = 2 };

// What becomes of the f32 sums D[rows, cols]; every matrix is row-major with
// `cols` columns.
struct Epilogue {
  int64_t rows = 0, cols = 0;
  int act = ORCA_ACT_NONE;
  int align = 1;                      // of the rows of every T matrix below, in bytes (16, 8, 4, 1)
  int bias_vec = 0;                   // 16-byte loads of the bias are aligned
  int ckpt_align = 1;                 // of a checkpoint's rows, in bytes
  void* out = nullptr;                // T; DW with out_f32: float
  int out_f32 = 0;
  const void* bias = nullptr;         // FWD: T [cols]
  const void* residual = nullptr;     // FWD, DX: T
  void* z = nullptr;                  // FWD: the pre-activation in T, kept
  uint8_t* codes = nullptr;           // FWD: kept in 8 bits; DX: x in 8 bits
  uint8_t* exps = nullptr;
  const void* x = nullptr;            // DX: x in T (with an activation only)
  void* a = nullptr;                  // DX: act(x) in T, the operand of dW, is written here
};

// For 4 fixed columns of up to 2 rows, in two steps: load what the rows'
// epilogues read, then finish them; the bias is loaded once.  All lanes of a warp
// call it together, each with its 4 columns of the same rows.
template <typename T, int MODE> struct ColumnEpilogue {
  const Epilogue& e;
  int64_t col;
  int cols;                  // columns inside, 0..4
  bool vec;
  float bias[4], res[2][4], x[2][4];
  __device__ ColumnEpilogue(const Epilogue& e_, int64_t col_) : e(e_), col(col_) {
    cols = col >= e.cols ? 0 : (e.cols - col < 4 ? (int)(e.cols - col) : 4);
    vec = e.align == 16 && cols == 4;
    if (MODE == FWD) {
#pragma unroll
      for (int i = 0; i < 4; ++i) bias[i] = 0.0f;
      if (e.bias && cols > 0) load_row<T, 4>((const T*)e.bias + col, cols, e.bias_vec && cols == 4, bias);
    }
  }
  __device__ __forceinline__ void load(int u, int64_t row) {
    if (MODE == DW || row >= e.rows || cols == 0) return;
    const int64_t at = row * e.cols + col;
    if (MODE == DX && (e.codes || e.x)) {
      if (e.codes) ckpt_load<4>(e.codes, e.exps, row, e.cols, col, cols, e.ckpt_align, x[u]);
      else load_row<T, 4>((const T*)e.x + at, cols, vec, x[u]);
    }
    if (e.residual) load_row<T, 4>((const T*)e.residual + at, cols, vec, res[u]);
  }
  __device__ __forceinline__ void store(int u, int64_t row, float (&v)[4]) {
    const bool ok = row < e.rows;
    const int valid = ok ? cols : 0;
    const int64_t at = row * e.cols + col;
    if (MODE == DW) {
      if (valid <= 0) return;
      if (e.out_f32) store_row<float, 4>((float*)e.out + at, valid, vec, v);
      else store_row<T, 4>((T*)e.out + at, valid, vec, v);
      return;
    }
    if (MODE == FWD) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += bias[i];
      if (e.z && valid > 0) store_row<T, 4>((T*)e.z + at, valid, vec, v);
      if (e.codes) ckpt_store<4>(e.codes, e.exps, row, e.cols, col, valid, ok, e.ckpt_align, v);
      if (valid <= 0) return;
      apply_act<4>(e.act, v);
    } else {
      if (valid <= 0) return;
      if (e.codes || e.x) {
        mul_slope<4>(e.act, x[u], v);
        if (e.a) {
          apply_act<4>(e.act, x[u]);
          store_row<T, 4>((T*)e.a + at, valid, vec, x[u]);
        }
      }
    }
    if (e.residual) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += res[u][i];
    }
    store_row<T, 4>((T*)e.out + at, valid, vec, v);
  }
};

// ---------------------------------------------------------------- 32 x 32 blocks
// A warp's 32 rows x 32 columns, a row per lane (as TMEM gives them), and
// row-major memory: the block goes through the warp's 4 KB of shared memory so
// that the 16-byte accesses of a warp cover whole rows of the block (64 or 128
// bytes, full sectors) instead of one piece in each of 32 rows.  16-byte pieces
// are placed at (piece ^ f(row)), free of bank conflicts both ways.
constexpr int BLOCK_SMEM = 32 * 32 * 4;       // 16-bit types need half

__device__ __forceinline__ uint4 lds_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void sts_v4(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// P pieces of 16 bytes a row.
template <int P> __device__ __forceinline__ uint32_t piece_at(uint32_t smem, int row, int piece) {
  const int f = P == 8 ? row & 7 : (P == 4 ? (row >> 1) & 3 : (row >> 2) & 1);
  return smem + (uint32_t)(row * P + (piece ^ f)) * 16;
}
// What of a block is inside the matrix: rows, and bytes of each row; and the largest
// power of two, as a shift, that row starts and row lengths share (16 bytes at most).
struct Inside {
  int rows, bytes, shift;
};
__device__ __forceinline__ int align_shift(int align) { return 31 - __clz(align); }

__device__ __forceinline__ void lds_unit(uint32_t a, uint4& v) { v = lds_v4(a); }
__device__ __forceinline__ void lds_unit(uint32_t a, uint2& v) {
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
}
__device__ __forceinline__ void lds_unit(uint32_t a, uint32_t& v) {
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
}
__device__ __forceinline__ void lds_unit(uint32_t a, uint16_t& v) {
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(a));
}
__device__ __forceinline__ void lds_unit(uint32_t a, uint8_t& v) {
  uint32_t w;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(w) : "r"(a));
  v = (uint8_t)w;
}
__device__ __forceinline__ void sts_unit(uint32_t a, uint4 v) { sts_v4(a, v); }
__device__ __forceinline__ void sts_unit(uint32_t a, uint2 v) {
  asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(a), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ void sts_unit(uint32_t a, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void sts_unit(uint32_t a, uint16_t v) {
  asm volatile("st.shared.b16 [%0], %1;" ::"r"(a), "h"(v) : "memory");
}
__device__ __forceinline__ void sts_unit(uint32_t a, uint8_t v) {
  asm volatile("st.shared.u8 [%0], %1;" ::"r"(a), "r"((uint32_t)v) : "memory");
}

// Moves the block between shared memory and rows of the matrix in units of type U:
// adjacent lanes take adjacent units, up to 8 of a lane's in flight.
template <int P, bool STORE, typename U>
__device__ __forceinline__ void block_move(uint8_t* p, int64_t stride, const Inside& in, uint32_t smem, int lane) {
  constexpr int N = 32 * P * 16 / (int)sizeof(U), PER_ROW = P * 16 / (int)sizeof(U);
  constexpr int AT_ONCE = N / 32 < 8 ? N / 32 : 8;
#pragma unroll 1
  for (int i0 = 0; i0 < N; i0 += 32 * AT_ONCE) {
    U v[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = i0 + u * 32 + lane, r = i / PER_ROW, off = i % PER_ROW * (int)sizeof(U);
      if (STORE) lds_unit(piece_at<P>(smem, r, off >> 4) + (uint32_t)(off & 15), v[u]);
      else v[u] = r < in.rows && off < in.bytes ? *reinterpret_cast<const U*>(p + r * stride + off) : U{};
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = i0 + u * 32 + lane, r = i / PER_ROW, off = i % PER_ROW * (int)sizeof(U);
      if (!STORE) sts_unit(piece_at<P>(smem, r, off >> 4) + (uint32_t)(off & 15), v[u]);
      else if (r < in.rows && off < in.bytes) *reinterpret_cast<U*>(p + r * stride + off) = v[u];
    }
  }
}
// UNIT: bytes known to be aligned; 0: by in.shift.
template <int P, bool STORE, int UNIT>
__device__ __forceinline__ void block_move(uint8_t* p, int64_t stride, const Inside& in, uint32_t smem, int lane) {
  if constexpr (UNIT == 16) {
    block_move<P, STORE, uint4>(p, stride, in, smem, lane);
  } else if constexpr (UNIT == 8) {
    block_move<P, STORE, uint2>(p, stride, in, smem, lane);
  } else {
    switch (in.shift) {
      case 4: block_move<P, STORE, uint4>(p, stride, in, smem, lane); break;
      case 3: block_move<P, STORE, uint2>(p, stride, in, smem, lane); break;
      case 2: block_move<P, STORE, uint32_t>(p, stride, in, smem, lane); break;
      case 1: block_move<P, STORE, uint16_t>(p, stride, in, smem, lane); break;
      default: block_move<P, STORE, uint8_t>(p, stride, in, smem, lane);
    }
  }
}

// u: this lane's row, P pieces.
template <int P, int UNIT>
__device__ __forceinline__ void block_store(uint8_t* p, int64_t stride, const Inside& in, const uint4 (&u)[P],
                                            uint32_t smem, int lane) {
#pragma unroll
  for (int i = 0; i < P; ++i) sts_v4(piece_at<P>(smem, lane, i), u[i]);
  __syncwarp();
  block_move<P, true, UNIT>(p, stride, in, smem, lane);
  __syncwarp();
}
template <int P, int UNIT>
__device__ __forceinline__ void block_load(const uint8_t* p, int64_t stride, const Inside& in, uint4 (&u)[P],
                                           uint32_t smem, int lane) {
  block_move<P, false, UNIT>(const_cast<uint8_t*>(p), stride, in, smem, lane);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < P; ++i) u[i] = lds_v4(piece_at<P>(smem, lane, i));
  __syncwarp();
}
template <typename T, int UNIT>
__device__ __forceinline__ void block_store_f32(T* p, int64_t ld, const Inside& in, const float (&v)[32],
                                                uint32_t smem, int lane) {
  constexpr int P = 2 * (int)sizeof(T);
  union { uint4 q[P]; T e[32]; } u;
#pragma unroll
  for (int i = 0; i < 32; ++i) u.e[i] = from_f32<T>(v[i]);
  block_store<P, UNIT>(reinterpret_cast<uint8_t*>(p), ld * (int64_t)sizeof(T), in, u.q, smem, lane);
}
template <typename T, int UNIT>
__device__ __forceinline__ void block_load_f32(const T* p, int64_t ld, const Inside& in, float (&v)[32],
                                               uint32_t smem, int lane) {
  constexpr int P = 2 * (int)sizeof(T);
  union { uint4 q[P]; T e[32]; } u;
  block_load<P, UNIT>(reinterpret_cast<const uint8_t*>(p), ld * (int64_t)sizeof(T), in, u.q, smem, lane);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = to_f32(u.e[i]);
}

// Elements as 32-bit words: 4 columns of T in 2 words (F32: 4).
template <typename T> __device__ __forceinline__ void words_to_f32(const uint32_t* w, float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(w[j]);
  } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __half2float(__ushort_as_half((unsigned short)(w[j / 2] >> (16 * (j % 2)))));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
  }
}
template <typename T> __device__ __forceinline__ void f32_to_words(const float (&v)[4], uint32_t* w) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(v[j]);
  } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      w[j] = (uint32_t)__half_as_ushort(__float2half_rn(v[2 * j])) |
             (uint32_t)__half_as_ushort(__float2half_rn(v[2 * j + 1])) << 16;
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      w[j] = (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v[2 * j])) |
             (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v[2 * j + 1])) << 16;
  }
}
// v *= act'(x) and x = act(x) in T, four columns at a time: x comes as codes or as
// the words of T, and is never 32 registers more.
template <typename T, int ACT>
__device__ __forceinline__ void slope_block(const uint32_t (&codes)[8], bool packed, float down,
                                            uint32_t (&x)[8 * sizeof(T)], float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float z[4];
    if (packed) ckpt_values(codes[i], down, z);
    else words_to_f32<T>(x + i * (int)sizeof(T), z);
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const F2 y = f2(z[j], z[j + 1]);
      split(mul2(f2(v[4 * i + j], v[4 * i + j + 1]), act_slope<ACT>(y)), v[4 * i + j], v[4 * i + j + 1]);
      split(act_value<ACT>(y), z[j], z[j + 1]);
    }
    f32_to_words<T>(z, x + i * (int)sizeof(T));
  }
}
template <int P> __device__ __forceinline__ void pieces_to_words(const uint4 (&q)[P], uint32_t* w) {
#pragma unroll
  for (int i = 0; i < P; ++i) { w[4 * i] = q[i].x; w[4 * i + 1] = q[i].y; w[4 * i + 2] = q[i].z; w[4 * i + 3] = q[i].w; }
}

// The epilogue of one block: rows row0 + lane, columns col .. col + 32, of which
// those inside the matrix are touched.  Sums beyond its columns are zeros.  ALIGNED:
// rows of T are 16-byte aligned and those of codes 8-byte; a kernel of its own,
// since the units of the other forms spill the registers of this one.
template <typename T, int MODE, bool ALIGNED>
__device__ __forceinline__ void block_epilogue(const Epilogue& e, int64_t row0, int64_t col, float (&v)[32],
                                               uint32_t smem, int lane) {
  constexpr int UNIT = ALIGNED ? 16 : 0, UNIT8 = ALIGNED ? 8 : 0;
  const bool packed = e.codes != nullptr;
  if (row0 >= e.rows) return;
  const int rows = e.rows - row0 < 32 ? (int)(e.rows - row0) : 32;
  const int cols = e.cols - col < 32 ? (int)(e.cols - col) : 32;
  const int64_t at = row0 * e.cols + col;
  // A T matrix without a wider alignment is aligned to its elements.
  const int shift = e.align > (int)sizeof(T) ? align_shift(e.align) : (sizeof(T) == 4 ? 2 : 1);
  const Inside in{rows, cols * (int)sizeof(T), shift};
  if (MODE == DW) {
    if (e.out_f32) {
      // 16 columns at a time: 2 KB of shared memory, as the 16-bit types have.
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        union { uint4 q[4]; float f[16]; } u;
#pragma unroll
        for (int i = 0; i < 16; ++i) u.f[i] = v[16 * h + i];
        const int left = cols - 16 * h;
        const Inside part{rows, left <= 0 ? 0 : (left < 16 ? left : 16) * 4, shift < 2 ? 2 : shift};
        block_store<4, UNIT>(reinterpret_cast<uint8_t*>((float*)e.out + at + 16 * h), e.cols * 4, part, u.q, smem, lane);
      }
    } else {
      block_store_f32<T, UNIT>((T*)e.out + at, e.cols, in, v, smem, lane);
    }
    return;
  }
  const Inside in8{rows, cols, align_shift(e.ckpt_align)};
  if (MODE == FWD) {
    if (e.bias) {
      float t[32];
      load_row<T, 32>((const T*)e.bias + col, cols, e.bias_vec && cols == 32, t);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] += t[i];
    }
    if (e.z) block_store_f32<T, UNIT>((T*)e.z + at, e.cols, in, v, smem, lane);
    if (packed) {
      float amax = 0.0f;
#pragma unroll
      for (int i = 0; i < 32; i += 2) amax = ckpt_max(amax, v[i], v[i + 1]);
      const uint32_t x = ckpt_exponent(amax);
      const float up = ckpt_up(x);
      if (lane < rows) e.exps[(row0 + lane) * ckpt_groups(e.cols) + col / GROUP] = (uint8_t)x;
      union { uint4 q[2]; uint32_t w[8]; } u;
      ckpt_words<32>(v, amax, up, u.w);
      block_store<2, UNIT8>(e.codes + at, e.cols, in8, u.q, smem, lane);
    }
    apply_act<32>(e.act, v);
  } else if (packed || e.x) {
    constexpr int P = 2 * (int)sizeof(T);
    uint32_t codes[8], x[4 * P];
    float down = 0.0f;
    if (packed) {
      if (lane < rows) down = ckpt_down(e.exps[(row0 + lane) * ckpt_groups(e.cols) + col / GROUP]);
      uint4 q[2];
      block_load<2, UNIT8>(e.codes + at, e.cols, in8, q, smem, lane);
      pieces_to_words<2>(q, codes);
    } else {
      uint4 q[P];
      block_load<P, UNIT>(reinterpret_cast<const uint8_t*>((const T*)e.x + at), e.cols * (int64_t)sizeof(T), in, q, smem, lane);
      pieces_to_words<P>(q, x);
    }
    switch (e.act) {
      case ORCA_ACT_RELU: slope_block<T, ORCA_ACT_RELU>(codes, packed, down, x, v); break;
      case ORCA_ACT_GELU: slope_block<T, ORCA_ACT_GELU>(codes, packed, down, x, v); break;
      case ORCA_ACT_GELU_TANH: slope_block<T, ORCA_ACT_GELU_TANH>(codes, packed, down, x, v); break;
      default: slope_block<T, ORCA_ACT_SILU>(codes, packed, down, x, v);   // x is there with an activation only
    }
    if (e.a) {
      uint4 q[P];
#pragma unroll
      for (int i = 0; i < P; ++i) q[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
      block_store<P, UNIT>(reinterpret_cast<uint8_t*>((T*)e.a + at), e.cols * (int64_t)sizeof(T), in, q, smem, lane);
    }
  }
  if (e.residual) {
    float t[32];
    block_load_f32<T, UNIT>((const T*)e.residual + at, e.cols, in, t, smem, lane);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] += t[i];
  }
  block_store_f32<T, UNIT>((T*)e.out + at, e.cols, in, v, smem, lane);
}

}  // namespace lin

// ckpt8.cu: enqueue on ctx->stream; checked arguments.
orca_status ckpt8_pack_launch(orca_ctx* ctx, const void* x, orca_dtype dtype, int64_t m, int64_t n,
                              uint8_t* ckpt);
orca_status ckpt8_unpack_launch(orca_ctx* ctx, const uint8_t* ckpt, int64_t m, int64_t n, int act,
                                void* out, orca_dtype dtype);
// out = act(x), rounded to the type once (the operand of dW from a plainly kept x).
orca_status act_launch(orca_ctx* ctx, const void* x, orca_dtype dtype, int64_t len, int act, void* out);

namespace lin {
// A matrix as the tensor cores take it: rows of `cols` contiguous 16-bit elements
// with 16-byte aligned row starts, in 1 plane (BF16, F16) or 3 (F32).  ld and
// plane count elements.
struct Planes {
  const void* p = nullptr;
  int64_t ld = 0, plane = 0;
  int64_t rows = 0, cols = 0;
};

// Stream-ordered scratch of one call; in a captured graph it becomes the
// graph's own allocation, so graphs share nothing.
struct Scratch {
  orca_ctx* ctx;
  void* p = nullptr;
  explicit Scratch(orca_ctx* c) : ctx(c) {}
  ~Scratch() { if (p) cudaFreeAsync(p, ctx->stream); }
  Scratch(const Scratch&) = delete;
  Scratch& operator=(const Scratch&) = delete;
  orca_status get(size_t bytes) {
    ORCA_CUDA_TRY(cudaMallocAsync(&p, bytes, ctx->stream));
    return ORCA_OK;
  }
};
}  // namespace lin

// linear_mma.cu.  mma_prepare: takes contiguous [rows, cols] matrices of any
// alignment (p, rows, cols set) and makes planes of them, in `scratch` where the
// matrix itself will not do.  mma_product: D[M, N] = A @ B through the epilogue,
// K > 0; an operand's matrix has the sum along its rows' elements, or with *_mn
// along its rows.
constexpr int MAX_OPERANDS = 2;
orca_status mma_prepare(orca_ctx* ctx, orca_dtype dtype, lin::Planes* const* x, int count,
                        lin::Scratch& scratch);
orca_status mma_product(orca_ctx* ctx, int mode, orca_dtype dtype, int64_t M, int64_t N, int64_t K,
                        const lin::Planes& a, int a_mn, const lin::Planes& b, int b_mn,
                        const lin::Epilogue& e);

// Checks of spans (linear.cu).
orca_status need_span(orca_ctx* ctx, const orca_span* s, int64_t len, const char* what);
// The memory of a span's first len elements: what a call touches of it.
struct Extent {
  uintptr_t at;
  size_t bytes;
};
Extent used(const orca_span* s, int64_t len);
orca_status need_apart(Extent out, Extent other, const char* what);
orca_status need_float(const orca_span* s, const char* what);
orca_status need_dim(int64_t v, const char* what);
constexpr int64_t MAX_DIM = INT32_MAX - 4096;   // sizes fit the TMA coordinates, products of two stay far from 2^63

}  // namespace orca
