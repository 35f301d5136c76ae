// linear.cu -- fused linear operators: out = act(x @ w + b) + residual and its
// backward, in BF16, F16 and F32.
#include <algorithm>
#include <type_traits>

#include "linear.cuh"

namespace orca {

// ---------------------------------------------------------------- checks
orca_status need_dim(int64_t v, const char* what) {
  if (v < 0 || v > MAX_DIM)
    return fail(ORCA_INVALID_ARGUMENT, "%s: size %lld is out of range", what, (long long)v);
  return ORCA_OK;
}

orca_status need_float(const orca_span* s, const char* what) {
  if (s->dtype != ORCA_F32 && s->dtype != ORCA_F16 && s->dtype != ORCA_BF16)
    return fail(ORCA_UNSUPPORTED_DTYPE, "%s: dtype %d is none of F32, F16, BF16", what, (int)s->dtype);
  return ORCA_OK;
}

orca_status need_span(orca_ctx* ctx, const orca_span* s, int64_t len, const char* what) {
  if (!s) return fail(ORCA_INVALID_ARGUMENT, "%s: null span", what);
  const size_t es = dtype_size(s->dtype);
  if (!es) return fail(ORCA_UNSUPPORTED_DTYPE, "%s: unknown dtype %d", what, (int)s->dtype);
  if (s->len < (size_t)len)
    return fail(ORCA_SHAPE_MISMATCH, "%s: the span holds %zu elements, the sizes need %lld", what,
                s->len, (long long)len);
  if (len == 0) return ORCA_OK;
  if (!s->data) return fail(ORCA_INVALID_ARGUMENT, "%s: null data", what);
  if (reinterpret_cast<uintptr_t>(s->data) % es)
    return fail(ORCA_INVALID_ARGUMENT, "%s: data is not aligned to its elements", what);
  cudaPointerAttributes at;
  ORCA_CUDA_TRY(cudaPointerGetAttributes(&at, s->data));
  if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
    return fail(ORCA_DEVICE_MISMATCH, "%s: data is not device memory", what);
  if (at.type == cudaMemoryTypeDevice && at.device != ctx->device)
    return fail(ORCA_DEVICE_MISMATCH, "%s: data is on device %d, the context on %d", what, at.device,
                ctx->device);
  return ORCA_OK;
}

Extent used(const orca_span* s, int64_t len) {
  if (!s || len <= 0) return Extent{0, 0};
  return Extent{reinterpret_cast<uintptr_t>(s->data), (size_t)len * dtype_size(s->dtype)};
}

orca_status need_apart(Extent out, Extent other, const char* what) {
  if (!out.bytes || !other.bytes) return ORCA_OK;
  if (out.at < other.at + other.bytes && other.at < out.at + out.bytes)
    return fail(ORCA_INVALID_ARGUMENT, "%s overlap", what);
  return ORCA_OK;
}

namespace lin {

// ---------------------------------------------------------------- empty sums
// K = 0: the epilogue of zeros, 4 columns a lane.
template <typename T, int MODE>
__global__ void __launch_bounds__(256)
zero_kernel(Epilogue e) {
  const int64_t vecs = cdiv(e.cols, 128) * 32;       // whole warps per row (groups of columns)
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < e.rows * vecs; i += (int64_t)gridDim.x * 256) {
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    ColumnEpilogue<T, MODE> ce(e, i % vecs * 4);
    ce.load(0, i / vecs);
    ce.store(0, i / vecs, v);
  }
}

// ---------------------------------------------------------------- column sums
// db: a cluster of up to 8 CTAs per 64, 128 or 256 columns, each with a part of the
// rows: `lanes` lanes of 8 columns by 256 / lanes rows a CTA, F32 sums per lane,
// joined over the rows' lanes and then, through the cluster's shared memory, over
// the CTAs, always in the same order.  One pass over dy, bound by HBM, which wants
// long row pieces (4096 x 16384 BF16: 26 us with 512 bytes, 41 with 128) and enough
// CTAs: as many columns as leave 64 clusters.
constexpr int CS_RANKS = 8, CS_MAX_COLS = 256;

template <typename T, typename G>
__global__ void __launch_bounds__(256)
colsum_kernel(const T* __restrict__ x, int64_t m, int64_t n, int lanes, int ranks, int64_t rows, int vec,
              G* __restrict__ out) {
  __shared__ float s[32 * (64 + 8)];                 // [256 / lanes][8 * lanes + 8]
  __shared__ float part[CS_MAX_COLS];
  const int tx = threadIdx.x % lanes, ty = threadIdx.x / lanes, ys = 256 / lanes, cols = 8 * lanes;
  const uint32_t rank = cluster_ctarank();
  const int64_t col0 = (int64_t)(blockIdx.x / ranks) * cols, col = col0 + tx * 8;
  const int valid = col >= n ? 0 : (n - col < 8 ? (int)(n - col) : 8);
  const bool whole = vec && valid == 8;
  const int64_t r1 = std::min<int64_t>(m, (rank + 1) * rows);
  float acc[8] = {};
  if (valid > 0) {
    int64_t r = rank * rows + ty;
    for (; r + 3 * ys < r1; r += 4 * ys) {
      float v[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u) load_row<T, 8>(x + (r + u * ys) * n + col, valid, whole, v[u]);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += v[u][i];
    }
    for (; r < r1; r += ys) {
      float v[8];
      load_row<T, 8>(x + r * n + col, valid, whole, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += v[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) s[ty * (cols + 8) + tx * 8 + i] = acc[i];
  __syncthreads();
  if (threadIdx.x < cols) {
    float t = 0.0f;
    for (int y = 0; y < ys; ++y) t += s[y * (cols + 8) + threadIdx.x];
    part[threadIdx.x] = t;
  }
  cluster_sync_all();
  if (rank == 0 && threadIdx.x < cols && col0 + threadIdx.x < n) {
    float t = 0.0f;
    for (uint32_t r = 0; r < (uint32_t)ranks; ++r) {
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(part + threadIdx.x, r)) : "memory");
      t += v;
    }
    out[col0 + threadIdx.x] = from_f32<G>(t);
  }
  cluster_sync_all();   // no CTA leaves while its part may still be read
}

template <typename T, typename G>
static orca_status colsum_launch(orca_ctx* ctx, const T* x, int64_t m, int64_t n, G* out) {
  if (n <= 0) return ORCA_OK;
  const int ranks = m <= 64 ? 1 : CS_RANKS;
  const int lanes = n >= 64 * 256 ? 32 : (n >= 64 * 128 ? 16 : 8);
  const int64_t rows = std::max<int64_t>(1, cdiv(m, ranks));
  const int vec = byte_alignment(x, n * (int64_t)sizeof(T)) == 16;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(256);
  cfg.stream = ctx->stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)(cdiv(n, 8 * lanes) * ranks));
  ORCA_CUDA_TRY(cudaLaunchKernelEx(&cfg, colsum_kernel<T, G>, x, m, n, lanes, ranks, rows, vec, out));
  count_launch(ctx);
  return ORCA_OK;
}

template <typename T>
static orca_status colsum(orca_ctx* ctx, const T* x, int64_t m, int64_t n, const orca_span* out) {
  if (out->dtype == ORCA_F32) return colsum_launch(ctx, x, m, n, (float*)out->data);
  return colsum_launch(ctx, x, m, n, (T*)out->data);
}

// ---------------------------------------------------------------- products
template <typename T> constexpr orca_dtype dtype_of() {
  return std::is_same<T, float>::value ? ORCA_F32 : (std::is_same<T, __half>::value ? ORCA_F16 : ORCA_BF16);
}

template <typename T, int MODE>
static orca_status product(orca_ctx* ctx, int64_t M, int64_t N, int64_t K, const Planes& A, int a_mn,
                           const Planes& B, int b_mn, Epilogue e) {
  if (M <= 0 || N <= 0) return ORCA_OK;
  e.rows = M;
  e.cols = N;
  int al = 16;
  for (const void* p : {(const void*)e.out, e.residual, (const void*)e.z, e.x, (const void*)e.a})
    if (p) al = std::min(al, byte_alignment(p, N * (int64_t)sizeof(T)));
  e.align = al;
  if (e.out_f32) e.align = std::min(byte_alignment(e.out, N * 4), 16);
  e.bias_vec = e.bias && byte_alignment(e.bias, 0) == 16;
  if (e.codes) e.ckpt_align = byte_alignment(e.codes, N);
  if (K > 0) return mma_product(ctx, MODE, dtype_of<T>(), M, N, K, A, a_mn, B, b_mn, e);
  const unsigned grid = (unsigned)std::min<int64_t>(cdiv(M * cdiv(N, 128) * 32, 256), (int64_t)ctx->sm_count * 16);
  zero_kernel<T, MODE><<<grid, 256, 0, ctx->stream>>>(e);
  count_launch(ctx);
  ORCA_CUDA_TRY(cudaGetLastError());
  return ORCA_OK;
}

static Planes matrix(const void* p, int64_t rows, int64_t cols) {
  Planes x;
  x.p = p;
  x.rows = rows;
  x.cols = cols;
  return x;
}

template <typename T>
static orca_status forward(orca_ctx* ctx, const orca_span* x, const orca_span* w, int64_t m,
                           int64_t k, int64_t n, const Epilogue& e) {
  if (m <= 0 || n <= 0) return ORCA_OK;
  Scratch scratch(ctx);
  Planes px = matrix(x->data, m, k), pw = matrix(w->data, k, n);
  Planes* const both[] = {&px, &pw};
  ORCA_TRY(mma_prepare(ctx, dtype_of<T>(), both, 2, scratch));
  return product<T, FWD>(ctx, m, n, k, px, 0, pw, 1, e);
}

template <typename T>
static orca_status backward(orca_ctx* ctx, const orca_span* x, const orca_span* w,
                            const orca_span* dy, const orca_span* residual, int64_t m, int64_t k,
                            int64_t n, int act, const orca_span* dx, const orca_span* dw,
                            const orca_span* db) {
  constexpr orca_dtype dtype = dtype_of<T>();
  const bool packed = x && x->dtype == ORCA_U8;
  // dW's operand a = act(x), rounded to T as the forward pass rounded it (in more bits it
  // would take a second plane, twice the product): x itself, or a matrix that the epilogue of the dX
  // product writes on the way where it reads x for the slope (4096 x 16384 GELU:
  // 935 us against 963 with a pass of its own), or a pass of its own (without an
  // activation: 919 us against 931).
  Scratch act_x(ctx), scratch(ctx), scratch_a(ctx);
  const void* a = x ? x->data : nullptr;
  if (dw && m * k > 0 && (packed || act != ORCA_ACT_NONE)) {
    ORCA_TRY(act_x.get((size_t)(m * k) * sizeof(T)));
    a = act_x.p;
  }
  const bool emit = act_x.p && dx && n > 0 && act != ORCA_ACT_NONE;
  Planes pdy = matrix(dy->data, m, n), pw, pa;
  if (dx) pw = matrix(w->data, k, n);
  Planes* const first[] = {&pdy, &pw};
  if ((dx || dw) && k > 0) ORCA_TRY(mma_prepare(ctx, dtype, first, 2, scratch));
  if (dx) {
    Epilogue e;
    e.act = act;
    e.out = dx->data;
    if (residual) e.residual = residual->data;
    if (act != ORCA_ACT_NONE) {
      if (packed) {
        e.codes = (uint8_t*)x->data;
        e.exps = e.codes + ckpt_exps_at(m, k);
      } else {
        e.x = x->data;
      }
    }
    if (emit) e.a = act_x.p;
    ORCA_TRY((product<T, DX>(ctx, m, k, n, pdy, 0, pw, 0, e)));
  }
  if (dw) {
    if (act_x.p && !emit) {
      if (packed)
        ORCA_TRY(ckpt8_unpack_launch(ctx, (const uint8_t*)x->data, m, k, act, act_x.p, dtype));
      else
        ORCA_TRY(act_launch(ctx, x->data, dtype, m * k, act, act_x.p));
    }
    Epilogue e;
    e.out = dw->data;
    e.out_f32 = dw->dtype == ORCA_F32;
    pa = matrix(a, m, k);
    Planes* const second[] = {&pa};
    ORCA_TRY(mma_prepare(ctx, dtype, second, 1, scratch_a));
    ORCA_TRY((product<T, DW>(ctx, k, n, m, pa, 1, pdy, 1, e)));
  }
  if (db) ORCA_TRY(colsum<T>(ctx, (const T*)dy->data, m, n, db));
  return ORCA_OK;
}

}  // namespace lin
}  // namespace orca

using namespace orca;

static orca_status need_type(const orca_span* s, orca_dtype t, const char* what) {
  if (s->dtype != t) return fail(ORCA_DTYPE_MISMATCH, "%s: dtype %d, expected %d", what, (int)s->dtype, (int)t);
  return ORCA_OK;
}

static orca_status need_act(orca_act act, const char* what) {
  if ((int)act < ORCA_ACT_NONE || (int)act > ORCA_ACT_SILU)
    return fail(ORCA_INVALID_ARGUMENT, "%s: unknown activation %d", what, (int)act);
  return ORCA_OK;
}

// out may be the residual's memory itself: each element is read before the
// same thread writes it.
static orca_status need_apart_or_same(Extent out, Extent residual, const char* what) {
  if (out.at == residual.at) return ORCA_OK;
  return need_apart(out, residual, what);
}

extern "C" {

orca_status orca_linear_act_fwd(orca_ctx* ctx, const orca_span* x, const orca_span* w,
                                const orca_span* b, const orca_span* residual, int64_t m,
                                int64_t k, int64_t n, orca_act act, const orca_span* out,
                                orca_keep keep, const orca_span* z) {
  ORCA_TRY(check_ctx(ctx));
  std::lock_guard<std::mutex> lk(ctx->mu);
  ORCA_TRY(need_dim(m, "linear_act_fwd: m"));
  ORCA_TRY(need_dim(k, "linear_act_fwd: k"));
  ORCA_TRY(need_dim(n, "linear_act_fwd: n"));
  ORCA_TRY(need_act(act, "linear_act_fwd"));
  ORCA_TRY(need_span(ctx, x, m * k, "linear_act_fwd: x"));
  ORCA_TRY(need_float(x, "linear_act_fwd: x"));
  ORCA_TRY(need_span(ctx, w, k * n, "linear_act_fwd: w"));
  ORCA_TRY(need_type(w, x->dtype, "linear_act_fwd: w"));
  if (b) {
    ORCA_TRY(need_span(ctx, b, n, "linear_act_fwd: b"));
    ORCA_TRY(need_type(b, x->dtype, "linear_act_fwd: b"));
  }
  if (residual) {
    ORCA_TRY(need_span(ctx, residual, m * n, "linear_act_fwd: residual"));
    ORCA_TRY(need_type(residual, x->dtype, "linear_act_fwd: residual"));
  }
  ORCA_TRY(need_span(ctx, out, m * n, "linear_act_fwd: out"));
  ORCA_TRY(need_type(out, x->dtype, "linear_act_fwd: out"));
  if ((int)keep < ORCA_KEEP_NONE || (int)keep > ORCA_KEEP_CKPT8)
    return fail(ORCA_INVALID_ARGUMENT, "linear_act_fwd: unknown keep %d", (int)keep);
  if ((keep != ORCA_KEEP_NONE) != (z != nullptr))
    return fail(ORCA_INVALID_ARGUMENT, "linear_act_fwd: z is given exactly when something is kept");
  if (z) {
    const bool packed = keep == ORCA_KEEP_CKPT8;
    ORCA_TRY(need_span(ctx, z, packed ? (int64_t)orca_ckpt8_bytes(m, n) : m * n, "linear_act_fwd: z"));
    ORCA_TRY(need_type(z, packed ? ORCA_U8 : x->dtype, "linear_act_fwd: z"));
  }
  const Extent ux = used(x, m * k), uw = used(w, k * n), ub = used(b, n), ur = used(residual, m * n), uo = used(out, m * n);
  const Extent uz = used(z, keep == ORCA_KEEP_CKPT8 ? (int64_t)orca_ckpt8_bytes(m, n) : m * n);
  for (const Extent o : {uo, uz}) {
    ORCA_TRY(need_apart(o, ux, "linear_act_fwd: an output and x"));
    ORCA_TRY(need_apart(o, uw, "linear_act_fwd: an output and w"));
    ORCA_TRY(need_apart(o, ub, "linear_act_fwd: an output and b"));
  }
  ORCA_TRY(need_apart_or_same(uo, ur, "linear_act_fwd: out and residual"));
  ORCA_TRY(need_apart(uz, ur, "linear_act_fwd: z and residual"));
  ORCA_TRY(need_apart(uo, uz, "linear_act_fwd: out and z"));
  lin::Epilogue e;
  e.act = act;
  e.out = out->data;
  if (b) e.bias = b->data;
  if (residual) e.residual = residual->data;
  if (keep == ORCA_KEEP_Z) e.z = z->data;
  if (keep == ORCA_KEEP_CKPT8) {
    e.codes = (uint8_t*)z->data;
    e.exps = e.codes + lin::ckpt_exps_at(m, n);
  }
  if (x->dtype == ORCA_F32) return lin::forward<float>(ctx, x, w, m, k, n, e);
  if (x->dtype == ORCA_F16) return lin::forward<__half>(ctx, x, w, m, k, n, e);
  return lin::forward<__nv_bfloat16>(ctx, x, w, m, k, n, e);
}

orca_status orca_linear_act_bwd(orca_ctx* ctx, const orca_span* x, const orca_span* w,
                                const orca_span* dy, const orca_span* residual, int64_t m,
                                int64_t k, int64_t n, orca_act act, const orca_span* dx,
                                const orca_span* dw, const orca_span* db) {
  ORCA_TRY(check_ctx(ctx));
  std::lock_guard<std::mutex> lk(ctx->mu);
  ORCA_TRY(need_dim(m, "linear_act_bwd: m"));
  ORCA_TRY(need_dim(k, "linear_act_bwd: k"));
  ORCA_TRY(need_dim(n, "linear_act_bwd: n"));
  ORCA_TRY(need_act(act, "linear_act_bwd"));
  ORCA_TRY(need_span(ctx, dy, m * n, "linear_act_bwd: dy"));
  ORCA_TRY(need_float(dy, "linear_act_bwd: dy"));
  const orca_dtype t = dy->dtype;
  Extent ux{0, 0}, uw{0, 0}, ur{0, 0};        // of what is read
  if (dw || (dx && act != ORCA_ACT_NONE)) {
    if (!x) return fail(ORCA_INVALID_ARGUMENT, "linear_act_bwd: x: null span");
    const bool packed = x->dtype == ORCA_U8;
    const int64_t len = packed ? (int64_t)orca_ckpt8_bytes(m, k) : m * k;
    ORCA_TRY(need_span(ctx, x, len, "linear_act_bwd: x"));
    if (!packed) ORCA_TRY(need_type(x, t, "linear_act_bwd: x"));
    ux = used(x, len);
  }
  if (dx) {
    uw = used(w, k * n);
    ur = used(residual, m * k);
    ORCA_TRY(need_span(ctx, w, k * n, "linear_act_bwd: w"));
    ORCA_TRY(need_type(w, t, "linear_act_bwd: w"));
    if (residual) {
      ORCA_TRY(need_span(ctx, residual, m * k, "linear_act_bwd: residual"));
      ORCA_TRY(need_type(residual, t, "linear_act_bwd: residual"));
    }
    ORCA_TRY(need_span(ctx, dx, m * k, "linear_act_bwd: dx"));
    ORCA_TRY(need_type(dx, t, "linear_act_bwd: dx"));
  }
  if (dw) {
    ORCA_TRY(need_span(ctx, dw, k * n, "linear_act_bwd: dw"));
    if (dw->dtype != ORCA_F32) ORCA_TRY(need_type(dw, t, "linear_act_bwd: dw"));
  }
  if (db) {
    ORCA_TRY(need_span(ctx, db, n, "linear_act_bwd: db"));
    if (db->dtype != ORCA_F32) ORCA_TRY(need_type(db, t, "linear_act_bwd: db"));
  }
  const Extent uy = used(dy, m * n), ox = used(dx, m * k), ow = used(dw, k * n), ob = used(db, n);
  for (const Extent o : {ox, ow, ob}) {
    ORCA_TRY(need_apart(o, ux, "linear_act_bwd: an output and x"));
    ORCA_TRY(need_apart(o, uw, "linear_act_bwd: an output and w"));
    ORCA_TRY(need_apart(o, uy, "linear_act_bwd: an output and dy"));
  }
  ORCA_TRY(need_apart_or_same(ox, ur, "linear_act_bwd: dx and residual"));
  ORCA_TRY(need_apart(ow, ur, "linear_act_bwd: dw and residual"));
  ORCA_TRY(need_apart(ob, ur, "linear_act_bwd: db and residual"));
  ORCA_TRY(need_apart(ox, ow, "linear_act_bwd: dx and dw"));
  ORCA_TRY(need_apart(ox, ob, "linear_act_bwd: dx and db"));
  ORCA_TRY(need_apart(ow, ob, "linear_act_bwd: dw and db"));
  if (t == ORCA_F32) return lin::backward<float>(ctx, x, w, dy, residual, m, k, n, act, dx, dw, db);
  if (t == ORCA_F16) return lin::backward<__half>(ctx, x, w, dy, residual, m, k, n, act, dx, dw, db);
  return lin::backward<__nv_bfloat16>(ctx, x, w, dy, residual, m, k, n, act, dx, dw, db);
}

}  // extern "C"
