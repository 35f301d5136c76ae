// ckpt8.cu -- 8-bit activation checkpoints: pack and unpack (layout and code in
// linear.cuh).
//
// Both directions are one pass over memory, bound by HBM: pack reads s bytes
// and writes 33/32 bytes per element, unpack the reverse, so the work per
// thread is laid out for wide accesses only.  The 32 columns of a group lie in
// 32 / V adjacent lanes, which agree on the group's largest value by shuffles;
// nothing goes through shared memory.
#include <algorithm>

#include "linear.cuh"

namespace orca {
namespace lin {

constexpr int THREADS = 256;

// Rows of whole groups, 16-byte aligned: the matrix, its codes and its exponents
// are three contiguous arrays.  A lane takes 8 values (pack) or 16 (unpack), with
// all its loads in flight before the first is used: HBM needs ~44 KB in flight
// per SM.  4096 x 16384 BF16: pack 31.6 us (6.5 TB/s; before its arithmetic
// shrank 39, with 2 steps 41, with 1 46), unpack 35 us, through GELU 43 (two operations of
// the exponential and reciprocal units a value; 49 with 4 steps).
constexpr int PACK_STEPS = 4, UNPACK_STEPS = 2;

template <typename T>
__global__ void __launch_bounds__(THREADS)
pack_flat_kernel(const T* __restrict__ x, int64_t vecs, uint8_t* __restrict__ codes,
                 uint8_t* __restrict__ exps) {
  constexpr int P = (int)sizeof(T) / 2;              // 16-byte pieces of 8 values
  const int64_t base = (int64_t)blockIdx.x * (THREADS * PACK_STEPS) + threadIdx.x;
  union { uint4 q[P]; T e[8]; } in[PACK_STEPS];
#pragma unroll
  for (int s = 0; s < PACK_STEPS; ++s) {
    const int64_t i = base + s * THREADS;
#pragma unroll
    for (int p = 0; p < P; ++p)
      in[s].q[p] = i < vecs ? __ldcs(reinterpret_cast<const uint4*>(x) + i * P + p) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int s = 0; s < PACK_STEPS; ++s) {
    const int64_t i = base + s * THREADS;
    float v[8], amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32(in[s].e[j]);
#pragma unroll
    for (int j = 0; j < 8; j += 2) amax = ckpt_max(amax, v[j], v[j + 1]);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1)                  // a group is 4 lanes (vecs is a multiple of 4)
      amax = ckpt_max(amax, amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (i >= vecs) continue;
    const uint32_t e = ckpt_exponent(amax);
    const float up = ckpt_up(e);
    uint32_t w[2];
    ckpt_words<8>(v, amax, up, w);
    reinterpret_cast<uint2*>(codes)[i] = make_uint2(w[0], w[1]);
    if (i % 4 == 0) exps[i / 4] = (uint8_t)e;
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
unpack_flat_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps, int64_t vecs,
                   int act, T* __restrict__ out) {
  const int64_t base = (int64_t)blockIdx.x * (THREADS * UNPACK_STEPS) + threadIdx.x;
  uint4 in[UNPACK_STEPS];
  uint32_t e[UNPACK_STEPS];
#pragma unroll
  for (int s = 0; s < UNPACK_STEPS; ++s) {
    const int64_t i = base + s * THREADS;
    in[s] = i < vecs ? __ldcs(reinterpret_cast<const uint4*>(codes) + i) : make_uint4(0, 0, 0, 0);
    e[s] = i < vecs ? __ldg(exps + i / 2) : 1u;
  }
#pragma unroll 1
  for (int s = 0; s < UNPACK_STEPS; ++s) {
    const int64_t i = base + s * THREADS;
    // (the loads' registers have no index: select)
    uint4 q = in[0];
    uint32_t x = e[0];
#pragma unroll
    for (int t = 1; t < UNPACK_STEPS; ++t)
      if (s == t) { q = in[t]; x = e[t]; }
    if (i >= vecs) break;
    const float down = ckpt_down(x);
    float v[16];
    ckpt_values(q.x, down, v);
    ckpt_values(q.y, down, v + 4);
    ckpt_values(q.z, down, v + 8);
    ckpt_values(q.w, down, v + 12);
    apply_act<16>(act, v);
    store_row<T, 16>(out + i * 16, 16, true, v);
  }
}

// Any other matrix.  A block covers `lanes_x` lanes of V columns and THREADS /
// lanes_x rows and walks the rows with the grid's stride.  Row ends are ragged:
// lanes past the last column stay for the shuffles.
template <typename T, int V>
__global__ void __launch_bounds__(THREADS)
pack_kernel(const T* __restrict__ x, int64_t m, int64_t n, uint8_t* __restrict__ codes,
            uint8_t* __restrict__ exps, int lanes_x, int vec, int align) {
  const int tx = threadIdx.x % lanes_x, ty = threadIdx.x / lanes_x;
  const int rows = THREADS / lanes_x;
  const int64_t col = ((int64_t)blockIdx.x * lanes_x + tx) * V;
  const int valid = col >= n ? 0 : (n - col < V ? (int)(n - col) : V);
  // Every lane of a warp takes the same number of steps (the shuffles).
  for (int64_t r0 = (int64_t)blockIdx.y * rows; r0 < m; r0 += (int64_t)gridDim.y * rows) {
    const int64_t row = r0 + ty;
    const bool ok = row < m;
    float v[V];
    load_row<T, V>(x + (ok ? row * n + col : 0), ok ? valid : 0, ok && vec && valid == V, v);
    ckpt_store<V>(codes, exps, row, n, col, valid, ok, align, v);
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(THREADS)
unpack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps, int64_t m,
              int64_t n, int act, T* __restrict__ out, int lanes_x, int vec, int align) {
  const int tx = threadIdx.x % lanes_x, ty = threadIdx.x / lanes_x;
  const int rows = THREADS / lanes_x;
  const int64_t col = ((int64_t)blockIdx.x * lanes_x + tx) * V;
  const int valid = col >= n ? 0 : (n - col < V ? (int)(n - col) : V);
  if (valid == 0) return;
  for (int64_t row = (int64_t)blockIdx.y * rows + ty; row < m; row += (int64_t)gridDim.y * rows) {
    float v[V];
    ckpt_load<V>(codes, exps, row, n, col, valid, align, v);
    apply_act<V>(act, v);
    store_row<T, V>(out + row * n + col, valid, vec && valid == V, v);
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
act_kernel(const T* __restrict__ x, T* __restrict__ out, int64_t len, int act) {
  constexpr int V = 8;
  const int64_t vecs = cdiv(len, V);
  const bool aligned = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < vecs;
       i += (int64_t)gridDim.x * THREADS) {
    const int valid = len - i * V < V ? (int)(len - i * V) : V;
    float v[V];
    load_row<T, V>(x + i * V, valid, aligned && valid == V, v);
    apply_act<V>(act, v);
    store_row<T, V>(out + i * V, valid, aligned && valid == V, v);
  }
}

// Blocks of the row walk: enough to fill the SMs several times over.
static dim3 walk_grid(orca_ctx* ctx, int64_t m, int64_t n, int v, int* lanes_x) {
  const int64_t lanes = cdiv(n, v);
  int lx = GROUP / v;                       // a group's lanes stay together
  while (lx < THREADS && lx < lanes) lx *= 2;
  *lanes_x = lx;
  const int64_t bx = cdiv(lanes, lx);
  const int64_t want = std::max<int64_t>(1, (int64_t)ctx->sm_count * 32 / bx);
  const int64_t by = std::min(std::min(cdiv(m, THREADS / lx), want), (int64_t)65535);
  return dim3((unsigned)bx, (unsigned)by);
}

template <typename T>
static void pack(orca_ctx* ctx, const T* x, int64_t m, int64_t n, uint8_t* ckpt) {
  uint8_t* exps = ckpt + ckpt_exps_at(m, n);
  const int align = byte_alignment(ckpt, n);
  const bool vec = byte_alignment(x, n * (int64_t)sizeof(T)) == 16;
  if (vec && align == 16 && n % GROUP == 0) {
    const int64_t vecs = m * n / 8;
    pack_flat_kernel<T><<<(unsigned)cdiv(vecs, THREADS * PACK_STEPS), THREADS, 0, ctx->stream>>>(x, vecs, ckpt, exps);
    return;
  }
  int lx;
  // 8 columns a lane where their 16-byte (F32: 32-byte) loads are aligned; 4 in
  // single elements otherwise.
  if (vec) {
    const dim3 g = walk_grid(ctx, m, n, 8, &lx);
    pack_kernel<T, 8><<<g, THREADS, 0, ctx->stream>>>(x, m, n, ckpt, exps, lx, 1, align);
  } else {
    const dim3 g = walk_grid(ctx, m, n, 4, &lx);
    pack_kernel<T, 4><<<g, THREADS, 0, ctx->stream>>>(x, m, n, ckpt, exps, lx, 0, align);
  }
}

template <typename T>
static void unpack(orca_ctx* ctx, const uint8_t* ckpt, int64_t m, int64_t n, int act, T* out) {
  const uint8_t* exps = ckpt + ckpt_exps_at(m, n);
  const int align = byte_alignment(ckpt, n);
  const bool vec = byte_alignment(out, n * (int64_t)sizeof(T)) == 16;
  if (vec && align == 16 && n % GROUP == 0) {
    const int64_t vecs = m * n / 16;
    unpack_flat_kernel<T><<<(unsigned)cdiv(vecs, THREADS * UNPACK_STEPS), THREADS, 0, ctx->stream>>>(
        ckpt, exps, vecs, act, out);
    return;
  }
  int lx;
  if (vec) {
    const dim3 g = walk_grid(ctx, m, n, 8, &lx);
    unpack_kernel<T, 8><<<g, THREADS, 0, ctx->stream>>>(ckpt, exps, m, n, act, out, lx, 1, align);
  } else {
    const dim3 g = walk_grid(ctx, m, n, 4, &lx);
    unpack_kernel<T, 4><<<g, THREADS, 0, ctx->stream>>>(ckpt, exps, m, n, act, out, lx, 0, align);
  }
}

}  // namespace lin

orca_status ckpt8_pack_launch(orca_ctx* ctx, const void* x, orca_dtype dtype, int64_t m, int64_t n,
                              uint8_t* ckpt) {
  if (m <= 0 || n <= 0) return ORCA_OK;
  if (dtype == ORCA_F32) lin::pack(ctx, (const float*)x, m, n, ckpt);
  else if (dtype == ORCA_F16) lin::pack(ctx, (const __half*)x, m, n, ckpt);
  else lin::pack(ctx, (const __nv_bfloat16*)x, m, n, ckpt);
  count_launch(ctx);
  ORCA_CUDA_TRY(cudaGetLastError());
  return ORCA_OK;
}

orca_status ckpt8_unpack_launch(orca_ctx* ctx, const uint8_t* ckpt, int64_t m, int64_t n, int act,
                                void* out, orca_dtype dtype) {
  if (m <= 0 || n <= 0) return ORCA_OK;
  if (dtype == ORCA_F32) lin::unpack(ctx, ckpt, m, n, act, (float*)out);
  else if (dtype == ORCA_F16) lin::unpack(ctx, ckpt, m, n, act, (__half*)out);
  else lin::unpack(ctx, ckpt, m, n, act, (__nv_bfloat16*)out);
  count_launch(ctx);
  ORCA_CUDA_TRY(cudaGetLastError());
  return ORCA_OK;
}

orca_status act_launch(orca_ctx* ctx, const void* x, orca_dtype dtype, int64_t len, int act,
                       void* out) {
  if (len <= 0) return ORCA_OK;
  const unsigned grid = (unsigned)std::min<int64_t>(cdiv(len, 8 * lin::THREADS), (int64_t)ctx->sm_count * 16);
#define ORCA_ACT(T) \
  lin::act_kernel<T><<<grid, lin::THREADS, 0, ctx->stream>>>((const T*)x, (T*)out, len, act)
  if (dtype == ORCA_F32) ORCA_ACT(float);
  else if (dtype == ORCA_F16) ORCA_ACT(__half);
  else ORCA_ACT(__nv_bfloat16);
#undef ORCA_ACT
  count_launch(ctx);
  ORCA_CUDA_TRY(cudaGetLastError());
  return ORCA_OK;
}

}  // namespace orca

using namespace orca;

static orca_status ckpt_bytes(int64_t m, int64_t n, int64_t* out, const char* what) {
  ORCA_TRY(need_dim(m, what));
  ORCA_TRY(need_dim(n, what));
  *out = (int64_t)orca_ckpt8_bytes(m, n);
  return ORCA_OK;
}

extern "C" {

size_t orca_ckpt8_bytes(int64_t m, int64_t n) {
  if (m <= 0 || n <= 0 || m > MAX_DIM || n > MAX_DIM) return 0;
  return (size_t)(lin::ckpt_exps_at(m, n) + m * lin::ckpt_groups(n));
}

orca_status orca_ckpt8_pack(orca_ctx* ctx, const orca_span* x, int64_t m, int64_t n,
                            const orca_span* ckpt) {
  ORCA_TRY(check_ctx(ctx));
  std::lock_guard<std::mutex> lk(ctx->mu);
  int64_t bytes = 0;
  ORCA_TRY(ckpt_bytes(m, n, &bytes, "ckpt8_pack"));
  ORCA_TRY(need_span(ctx, x, m * n, "ckpt8_pack: x"));
  ORCA_TRY(need_float(x, "ckpt8_pack: x"));
  ORCA_TRY(need_span(ctx, ckpt, bytes, "ckpt8_pack: ckpt"));
  if (ckpt->dtype != ORCA_U8) return fail(ORCA_DTYPE_MISMATCH, "ckpt8_pack: ckpt must be U8");
  ORCA_TRY(need_apart(used(ckpt, bytes), used(x, m * n), "ckpt8_pack: ckpt and x"));
  return ckpt8_pack_launch(ctx, x->data, x->dtype, m, n, (uint8_t*)ckpt->data);
}

orca_status orca_ckpt8_unpack(orca_ctx* ctx, const orca_span* ckpt, int64_t m, int64_t n,
                              orca_act act, const orca_span* out) {
  ORCA_TRY(check_ctx(ctx));
  std::lock_guard<std::mutex> lk(ctx->mu);
  int64_t bytes = 0;
  ORCA_TRY(ckpt_bytes(m, n, &bytes, "ckpt8_unpack"));
  if ((int)act < ORCA_ACT_NONE || (int)act > ORCA_ACT_SILU)
    return fail(ORCA_INVALID_ARGUMENT, "ckpt8_unpack: unknown activation %d", (int)act);
  ORCA_TRY(need_span(ctx, ckpt, bytes, "ckpt8_unpack: ckpt"));
  if (ckpt->dtype != ORCA_U8) return fail(ORCA_DTYPE_MISMATCH, "ckpt8_unpack: ckpt must be U8");
  ORCA_TRY(need_span(ctx, out, m * n, "ckpt8_unpack: out"));
  ORCA_TRY(need_float(out, "ckpt8_unpack: out"));
  ORCA_TRY(need_apart(used(out, m * n), used(ckpt, bytes), "ckpt8_unpack: out and ckpt"));
  return ckpt8_unpack_launch(ctx, (const uint8_t*)ckpt->data, m, n, act, out->data, out->dtype);
}

}  // extern "C"
