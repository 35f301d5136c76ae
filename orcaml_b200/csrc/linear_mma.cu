// linear_mma.cu -- the products of the fused linear operators on the 5th-generation
// tensor cores.
//
// BF16 and F16 operands go to tcgen05.mma kind::f16 as they are.  An F32 operand
// is split into three BF16 planes, x = x0 + x1 + x2 (8 significant bits each, by
// truncation; exact down to BF16's smallest step 2^-133, so all 24 bits of values
// from 2^-110 up), and the product is the sum of six plane products,
// x2*y0 + x0*y2 + x1*y1 + x1*y0 + x0*y1 + x0*y0; the three left out are below
// 2^-21 of |x||y| together.  Both kinds run through the same kernels.
//
//  * pair_kernel: 256 x 256 or 512 x 256 output tiles on clusters of two CTAs
//    (cta_group::2), persistent; for outputs with enough tiles.
//  * split_kernel: 128 columns x 16..128 rows of the output per cluster, the sum
//    split over the cluster's CTAs and joined through their shared memory; for
//    few rows, where the weights are read once at HBM speed, and for outputs
//    with few tiles.
#include <cudaTypedefs.h>

#include <algorithm>
#include <type_traits>

#include "linear.cuh"

namespace orca {
namespace lin {

constexpr int BK = 64;                       // 128 bytes of 16-bit elements: one swizzle row
constexpr int ROWS = 128;                    // rows of an operand tile
constexpr int TILE = ROWS * BK * 2;          // 16 KB

// F32 plane pairs in the order they are added, smallest first; 4 bits each.
constexpr uint32_t PAIR_A = 0x001102u, PAIR_B = 0x010120u;   // pair p: (x >> 4 * p) & 15
constexpr int F32_PAIRS = 6;

// Steps (of four MMAs) per accumulation chunk.  The tensor core adds with a few bits
// less than F32, at the scale of what the accumulator holds, so the accumulator of
// a result that is to be F32-accurate is emptied into F32 registers in between.
//  F32 operands: after each 64-deep block of six plane products, the small ones
//  first, so that only the last four MMAs add at full scale: off by 1.7e-7 of the
//  result's norm (4096 x 784 x 8192; FMAs in F32: 6e-7), against 1.2e-6 after three
//  blocks, which took 280 us instead of 298.
//  F32 gradients of 16-bit operands: after GRAD_CHUNK steps, off by 4.7e-7 of their norm
//  whatever the sum's length (16 steps: 1.0e-6; 4: 2.4e-7; FMAs in F32: 2.5e-7 over
//  1024 rows, 6.1e-7 over 4096, 1.5e-6 over 16384).  The backward of 4096 x 4096 x 16384
//  takes 884 to 905 us, 0 to 1 % more than with 16 steps; with 4 it takes 3 % more.
//  8-bit checkpoints, whose codes flip with the sums' errors: after CKPT_CHUNK steps,
//  5.9e-7, as many flips as after FMAs in F32 (values off by 1.11e-4 of the norm beside the
//  rounding to codes, after 16 steps 1.42e-4).  4096 x 4096 x 16384 with GELU and the checkpoint decoded
//  takes 506 us, 494 with 16 steps, 512 with 8: the drains of short chunks wait for the
//  epilogue of the tile before.
//  16-bit results: after F16_CHUNK or BF16_CHUNK steps, off by 3e-5 or 2.5e-4 of the norm, an
//  eighth of what rounding them is off by (2.1e-4 and 1.7e-3; over 2^20 rows one chain
//  was off by 2.5e-4 in either type).  Sums of up to 32768 and 262144 rows are one chain in any
//  case, which 512-row tiles need: dW of 2048 x 1024 over 2^20 rows takes 3.5 ms in BF16 and, from
//  smaller tiles, 4.6 in F16.
constexpr int GRAD_CHUNK = 8, CKPT_CHUNK = 10, F16_CHUNK = 512, BF16_CHUNK = 4096;

// Shared-memory matrix descriptors for the 128-byte swizzle (layout code 2).
//  K-major: row r at 128 * r bytes, 8-row groups 1024 bytes apart (stride
//    offset); the 16-deep step s starts 32 * s bytes further.
//  MN-major: boxes of 64 mn x 64 k, k row at 128 bytes, 8-row groups of k 1024
//    bytes apart (stride offset), boxes 8 KB apart (leading offset); step s
//    starts 16 rows = 2 KB further.
// The issuing thread has ~500 clocks per 64-deep step, so the descriptors are
// kept as a low word (address and leading offset) that is advanced by adds and a
// constant high word.
__device__ __forceinline__ uint32_t desc_lo(uint32_t base, int mn_major) {
  return ((base >> 4) & 0x3FFFu) | (uint32_t)((mn_major ? 8192 : 16) >> 4) << 16;
}
constexpr uint32_t DESC_HI = (1024 >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint64_t desc(uint32_t lo) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(DESC_HI));
  return d;
}
__device__ __forceinline__ uint32_t desc_step(int mn_major) { return (mn_major ? 2048u : 32u) >> 4; }

// kind::f16 instruction descriptor: F32 accumulator, operand types (1 = BF16,
// 0 = F16), orientations, N and M.
__device__ __forceinline__ uint32_t idesc(int bf16, int a_mn, int b_mn, int n, int m) {
  return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)a_mn << 15) |
         ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
      "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_f16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                             uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
      "r"(id), "r"(acc)
      : "memory");
}

// One lane of the (converged) warp.  The MMA warp runs its loop with all lanes, so
// that the compiler keeps descriptors and counters in uniform registers, which is
// where the instructions take them from; only the issue itself is one lane's.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// Arrive once on the mbarrier at this offset in both CTAs of the pair when the
// MMAs issued so far have completed.
__device__ __forceinline__ void commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

// 32 lanes x 32 columns from registers, the layout of tmem_ld_32x32b_x32.
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const float* v) {
  uint32_t r[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
      "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
      "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}

struct Params {
  int64_t M, N, K;
  int a_mn, b_mn;
  int bf16;
  int pairs;               // plane pairs: 1, or F32_PAIRS
  int chunk;               // steps per accumulation chunk
  int group_m;             // tile rows per raster group
  int full;                // pair_kernel: tiles [0, full) are whole, one cluster each
  int tail;                // ... the rest is shared by the first `tail` clusters (0: no rest)
  uint32_t shared;         // ... its steps, all tiles together
  float* parts;            // ... their partial sums and arrival counters
  int* arrived;
  int* dev_err;
  Epilogue e;
};

// Tile row 0 of `rows` (64 or 128, 16.. for K-major) of an operand: one box, or
// one box per 64 when MN-major.
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar,
                                          int mn_major, int rows, int64_t mn0, int64_t k0, int plane) {
  if (mn_major) {
    for (int c = 0; c < rows / 64; ++c)
      tma_load_3d(dst + c * 8192, map, bar, (int)(mn0 + 64 * c), (int)k0, plane);
  } else {
    tma_load_3d(dst, map, bar, (int)k0, (int)mn0, plane);
  }
}
__device__ __forceinline__ void load_tile_pair(uint8_t* dst, const CUtensorMap* map, uint32_t bar_cl,
                                               int mn_major, int rows, int64_t mn0, int64_t k0,
                                               int plane) {
  if (mn_major) {
    for (int c = 0; c < rows / 64; ++c)
      tma_load_3d_pair(dst + c * 8192, map, bar_cl, (int)(mn0 + 64 * c), (int)k0, plane);
  } else {
    tma_load_3d_pair(dst, map, bar_cl, (int)k0, (int)mn0, plane);
  }
}

__device__ __forceinline__ void tile_at(int tile, int num_m, int num_n, int group_m, int& tm, int& tn) {
  const int size = group_m * num_n;           // group_m <= num_m: at most the tiles, below 2^31
  const int first = tile / size * group_m;
  const int gm = num_m - first < group_m ? num_m - first : group_m;
  const int r = tile % size;
  tm = first + r % gm;
  tn = r / gm;
}

// The pieces of work of one cluster of pair_kernel, in order: whole tiles, then its
// equal share of the steps of the tiles that do not fill a last round, which
// may end one tile, cover some and begin another.
struct Work {
  int next, nclusters, full, steps;
  uint32_t pos, end;              // of the shared steps, counted through the tiles
  __device__ Work(const Params& p, int c, int n, int steps_)
      : next(c), nclusters(n), full(p.full), steps(steps_), pos(0), end(0) {
    if (c < p.tail) {
      pos = first_step(p, c);
      end = first_step(p, c + 1);
    }
  }
  static __device__ uint32_t first_step(const Params& p, int c) {
    return (uint32_t)((uint64_t)p.shared * (uint32_t)c / (uint32_t)p.tail);
  }
  __device__ bool get(int& tile, int& begin, int& stop) {
    if (next < full) {
      tile = next;
      next += nclusters;
      begin = 0;
      stop = steps;
      return true;
    }
    if (pos >= end) return false;
    const uint32_t t = pos / (uint32_t)steps;
    begin = (int)(pos - t * (uint32_t)steps);
    stop = end - pos < (uint32_t)(steps - begin) ? begin + (int)(end - pos) : steps;
    tile = full + (int)t;
    pos += (uint32_t)(stop - begin);
    return true;
  }
};

// ---------------------------------------------------------------- CTA pairs
// Tiles beyond whole rounds of the resident clusters are cut along the sum, so
// that all clusters finish together (4096 x 4096 outputs are 3.46 rounds of 74
// clusters).  A cluster leaves the sums of a piece in memory and counts itself in;
// the last to arrive at a tile adds the pieces in their order -- the same bits
// whoever is last -- and finishes it.  Nobody waits for anybody.  Each epilogue
// warp does this for its own 32 x 128 part.
//
// Roles: warp 0 loads, warp 1 (of the even CTA) issues the MMAs, the other warps
// drain the accumulators.  The even CTA's full barrier counts both CTAs' bytes;
// the MMA's commits free the stage and publish the accumulator in both.  Every
// wait is bounded; a role that gives up raises the abort flag of both CTAs, and
// both pass the same two cluster barriers in every case.
//
// HALVES = 1: 256 x 256 tiles, two accumulators of 256 columns, one filled while 8
// warps drain the other; for F32 results it is emptied every `chunk` steps into
// F32 registers.
// F32 operands: a stage holds the three planes of both operands for a 64-deep step
// and feeds the six plane products, so that each byte is fetched once, not twice.
// HALVES = 2: 512 x 256 tiles, both accumulators filled together from one tile of
// B: a quarter fewer bytes from L2 and through shared memory per product, which
// under the power limit are what is left to save.  The drain is not hidden, so 16
// warps do it, each half being refilled as soon as it is empty.
// TN = 128 (HALVES = 1): 256 x 128 tiles, for outputs with few tiles or an unlucky
// last round.
//
// Bound by the tensor pipe (84 % of the clocks active without an activation, 89 %
// without any epilogue) and in a loop by the power limit: BF16 4096 x 16384 x 4096
// with residual 349 us alone (1.58 PFLOP/s), 450 us in a loop; F32 4096 x 784 x 8192
// 226 us alone (232 TFLOP/s of F32, six BF16 products each).
template <int HALVES, int TN, int PLANES> struct Shape {
  static constexpr int EPI_WARPS = 8 * HALVES;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int B_TILE = TN / 2 * BK * 2;            // this CTA's half of B's columns
  static constexpr int STAGE = (HALVES * TILE + B_TILE) * PLANES;
  static constexpr int STAGES = 196608 / STAGE;
  static constexpr int BLOCK = BLOCK_SMEM / HALVES;
  static constexpr int SMEM = STAGES * STAGE + EPI_WARPS * BLOCK + 1024 + 256;
  static constexpr int M = 256 * HALVES;
  static constexpr int WARP_COLS = TN / (2 * HALVES);       // columns of a half per warp
  static constexpr int BLOCKS = WARP_COLS / 32;             // ... in blocks of 32
  static constexpr int ALL_BLOCKS = BLOCKS * HALVES;
  static constexpr int64_t PART_FLOATS = M * TN;            // one piece of a tile
  static constexpr int ARRIVALS = 2 * EPI_WARPS;            // counters of a tile
  static_assert(SMEM <= 232448, "shared memory of one CTA");
};
constexpr int ACC_COLS = 256;                               // TMEM columns between the accumulators

// mbar_wait by a whole warp: one answer for all lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* dev_err,
                                          unsigned sleep_ns = 0) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, dev_err, sleep_ns));
}

template <typename T> constexpr int plane_count() { return std::is_same<T, float>::value ? 3 : 1; }

template <typename T, int MODE, int HALVES, int TN, bool ALIGNED>
__global__ void __launch_bounds__(Shape<HALVES, TN, plane_count<T>()>::THREADS, 1)
pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
            const __grid_constant__ Params p) {
  constexpr int PLANES = plane_count<T>();
  using S = Shape<HALVES, TN, PLANES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::STAGES * S::STAGE + S::EPI_WARPS * S::BLOCK);
  uint64_t* full_bar = bars;                              // (even) both CTAs' bytes
  uint64_t* empty_bar = bars + S::STAGES;
  uint64_t* tfull_bar = bars + 2 * S::STAGES;           // [2]
  uint64_t* tempty_bar = bars + 2 * S::STAGES + 2;      // [2] (even)
  uint64_t* drain_bar = bars + 2 * S::STAGES + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S::STAGES + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const uint32_t rank = cluster_ctarank();
  const bool even = rank == 0;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int num_m = (int)cdiv(p.M, S::M), num_n = (int)cdiv(p.N, TN);
  const int cluster = blockIdx.x >> 1, nclusters = gridDim.x >> 1;
  const int steps = (int)cdiv(p.K, BK);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 2 * S::EPI_WARPS);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 2 * ACC_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t peer_abort = cluster_addr(const_cast<int*>(abort_flag), rank ^ 1u);
  auto raise_abort = [&]() {
    *abort_flag = 1;
    st_remote_u32(peer_abort, 1u);
  };

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued[S::STAGES];
      for (int s = 0; s < S::STAGES; ++s) issued[s] = -1;
      uint64_t last_issue = 0;
      bool ok = true;
      Work work(p, cluster, nclusters, steps);
      int tile;
      int begin, stop;
      while (ok && work.get(tile, begin, stop)) {
        int tm, tn;
        tile_at(tile, num_m, num_n, p.group_m, tm, tn);
        const int row = tm * S::M + (int)rank * 128, col = tn * TN + (int)rank * (TN / 2);
        for (int it = begin; it < stop; ++it) {
          const int k0 = it * BK;
          if (!mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, p.dev_err)) {
            ok = false;
            break;
          }
          uint8_t* a_dst = smem + stage * S::STAGE;
          if (even) {
            mbar_arrive_expect_tx(&full_bar[stage], 2 * S::STAGE);
#pragma unroll
            for (int l = 0; l < PLANES; ++l) {
#pragma unroll
              for (int h = 0; h < HALVES; ++h)
                load_tile(a_dst + (l * HALVES + h) * TILE, &map_a, &full_bar[stage], p.a_mn, ROWS, row + h * 256, k0, l);
              load_tile(a_dst + PLANES * HALVES * TILE + l * S::B_TILE, &map_b, &full_bar[stage], p.b_mn, TN / 2, col, k0, l);
            }
            issued[stage] = (int)phase;
          } else {
            const uint32_t bar = cluster_addr(&full_bar[stage], 0);
#pragma unroll
            for (int l = 0; l < PLANES; ++l) {
#pragma unroll
              for (int h = 0; h < HALVES; ++h)
                load_tile_pair(a_dst + (l * HALVES + h) * TILE, &map_a, bar, p.a_mn, ROWS, row + h * 256, k0, l);
              load_tile_pair(a_dst + PLANES * HALVES * TILE + l * S::B_TILE, &map_b, bar, p.b_mn, TN / 2, col, k0, l);
            }
            last_issue = global_ns();
          }
          if (++stage == S::STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) {
        raise_abort();
        // The odd CTA's copies count on the even CTA's barrier: after an abort
        // it cannot see them land and waits far longer than a copy takes.
        if (!even && last_issue)
          while (global_ns() - last_issue < 50000ull) {
          }
      }
      // Never leave with copies in flight into this CTA's shared memory.
      for (int s = 0; s < S::STAGES; ++s) {
        if (issued[s] < 0) continue;
        const uint64_t t0 = global_ns();
        while (!mbar_try_wait(&full_bar[s], (uint32_t)issued[s]) && global_ns() - t0 < kWaitLimitNs) {
        }
      }
    }
  } else if (warp == 1) {
    if (even) {
      const uint32_t id = idesc(p.bf16, p.a_mn, p.b_mn, TN, 256);
      const uint32_t a0 = desc_lo(smem_u32(smem), p.a_mn), b0 = desc_lo(smem_u32(smem) + PLANES * HALVES * TILE, p.b_mn);
      const uint32_t a_step = desc_step(p.a_mn), b_step = desc_step(p.b_mn);
      int stage = 0;
      uint32_t phase = 0, chunks = 0;
      bool ok = true;
      Work work(p, cluster, nclusters, steps);
      int tile;
      int begin, stop;
      while (ok && work.get(tile, begin, stop)) {
        int in_chunk = 0;
        for (int it = begin; it < stop; ++it) {
          // HALVES = 1: this chunk's accumulator; HALVES = 2: both, chunk = tile.
          const int buf = HALVES == 1 ? (int)(chunks & 1u) : 0;
          const uint32_t use = HALVES == 1 ? chunks >> 1 : chunks;
          if (in_chunk == 0) {
            if (!warp_wait(&tempty_bar[buf], (use & 1u) ^ 1u, abort_flag, p.dev_err)) { ok = false; break; }
            tc_fence_after();
          }
          if (!warp_wait(&full_bar[stage], phase, abort_flag, p.dev_err)) { ok = false; break; }
          tc_fence_after();
          const uint32_t at = (uint32_t)(stage * (S::STAGE >> 4));
          const bool last = in_chunk + 1 == p.chunk || it == stop - 1;
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            if (h == 1 && in_chunk == 0) {
              if (!warp_wait(&tempty_bar[1], (use & 1u) ^ 1u, abort_flag, p.dev_err)) { ok = false; break; }
              tc_fence_after();
            }
            const uint32_t d = tmem + (uint32_t)((buf + h) * ACC_COLS), ah = a0 + at + h * (TILE >> 4);
            if (elect_one()) {
#pragma unroll
              for (int l = 0; l < (PLANES == 3 ? F32_PAIRS : 1); ++l) {
                const uint32_t pa = PLANES == 3 ? (PAIR_A >> (4 * l)) & 15u : 0u, pb = PLANES == 3 ? (PAIR_B >> (4 * l)) & 15u : 0u;
#pragma unroll
                for (int s = 0; s < BK / 16; ++s)
                  mma_f16_pair(d, desc(ah + pa * (HALVES * TILE >> 4) + s * a_step),
                               desc(b0 + at + pb * (S::B_TILE >> 4) + s * b_step), id, (in_chunk | l | s) ? 1u : 0u);
              }
              if (h == HALVES - 1) {
                commit_both(&empty_bar[stage]);
                if (last) commit_both(&tfull_bar[buf]);
              }
            }
            __syncwarp();
          }
          if (!ok) break;
          if (++stage == S::STAGES) { stage = 0; phase ^= 1u; }
          ++in_chunk;
          if (last) {
            ++chunks;
            in_chunk = 0;
          }
        }
      }
      if (!ok) raise_abort();
      if (elect_one()) tc_commit_pair(cluster_addr(drain_bar, 0));
      const uint64_t t0 = global_ns();
      while (!mbar_try_wait(drain_bar, 0) && global_ns() - t0 < kWaitLimitNs) {
      }
    }
  } else {
    // Warp w reads TMEM lanes [32 * (w % 4), +32) and, of each half, the columns
    // [WARP_COLS * ((w - 2) / 4), +WARP_COLS).
    const int quarter = warp & 3, first_col = (warp - 2) / 4 * S::WARP_COLS;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)first_col;
    const uint32_t tempty[2] = {cluster_addr(&tempty_bar[0], 0), cluster_addr(&tempty_bar[1], 0)};
    const uint32_t block = smem_u32(smem + S::STAGES * S::STAGE + (warp - 2) * S::BLOCK);
    uint32_t chunks = 0;
    bool ok = true;
    Work work(p, cluster, nclusters, steps);
    int tile;
    int begin, stop;
    while (ok && work.get(tile, begin, stop)) {
      int tm, tn;
      tile_at(tile, num_m, num_n, p.group_m, tm, tn);
      const int row = tm * S::M + (int)rank * 128 + quarter * 32;
      const int col = tn * TN + first_col;
      const bool piece = stop - begin < steps;
      const int nchunks = (stop - begin + p.chunk - 1) / p.chunk;
      auto release = [&](int buf) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(tempty[buf]);
      };
      int buf = HALVES == 1 ? (int)(chunks & 1u) : 0;
      ok = warp_wait(&tfull_bar[buf], (HALVES == 1 ? chunks >> 1 : chunks) & 1u, abort_flag, p.dev_err, 64);
      tc_fence_after();
      ++chunks;
      if (HALVES == 1 && ok && nchunks > 1) {
        // The sums go back to the last chunk's accumulator, where the epilogue finds
        // them block by block as it finds those of a single chunk: holding its sums
        // in registers through the epilogue spilled them, and with this much
        // shared memory in use the spills went to L2.
        float acc[S::WARP_COLS];
#pragma unroll
        for (int j = 0; j < S::WARP_COLS; ++j) acc[j] = 0.0f;
        for (int c = 0;; ++c) {
#pragma unroll
          for (int q = 0; q < S::WARP_COLS / 16; ++q) {
            float v[16];
            tmem_ld_32x32b_x16(lanes + (uint32_t)(buf * ACC_COLS + q * 16), v);
#pragma unroll
            for (int j = 0; j < 16; j += 2)
              split(add2(f2(acc[q * 16 + j], acc[q * 16 + j + 1]), f2(v[j], v[j + 1])), acc[q * 16 + j],
                    acc[q * 16 + j + 1]);
          }
          if (c == nchunks - 1) break;
          release(buf);
          buf = (int)(chunks & 1u);
          ok = warp_wait(&tfull_bar[buf], (chunks >> 1) & 1u, abort_flag, p.dev_err, 64);
          if (!ok) break;
          tc_fence_after();
          ++chunks;
        }
        if (ok) {
#pragma unroll
          for (int q = 0; q < S::BLOCKS; ++q) tmem_st_32x32b_x32(lanes + (uint32_t)(buf * ACC_COLS + q * 32), acc + q * 32);
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
      }
      if (!ok) break;
      int first = 0, count = 0;
      // This warp's part of a piece: blocks of 32 columns, four columns of each lane
      // side by side.
      const int my_part = (int)(rank * S::EPI_WARPS + warp - 2) * (S::ALL_BLOCKS * 1024) + lane * 4;
      if (piece) {
        float* mine = p.parts + (int64_t)(cluster * 2 + (begin == 0)) * S::PART_FLOATS + my_part;
#pragma unroll 1
        for (int q = 0; q < S::ALL_BLOCKS; ++q) {
          float v[32];
          tmem_ld_32x32b_x32(lanes + (uint32_t)((buf + q / S::BLOCKS) * ACC_COLS + q % S::BLOCKS * 32), v);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            __stcg(reinterpret_cast<float4*>(mine + (q * 8 + j) * 128),
                   make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
        }
        release(buf);
        if (HALVES == 2) release(1);
        // Clusters first .. first + count - 1 share this tile.
        const int t = tile - p.full;
        const uint32_t t0 = (uint32_t)t * (uint32_t)steps, t1 = t0 + (uint32_t)steps;
        first = (int)((uint64_t)t0 * (uint32_t)p.tail / p.shared);
        while (Work::first_step(p, first + 1) <= t0) ++first;
        while (Work::first_step(p, first) > t0) --first;
        count = 1;
        while (Work::first_step(p, first + count) < t1) ++count;
        __threadfence();
        __syncwarp();
        int before = 0;
        if (lane == 0) before = atomicAdd(p.arrived + t * S::ARRIVALS + rank * S::EPI_WARPS + warp - 2, 1);
        before = __shfl_sync(0xffffffffu, before, 0);
        if (before != count - 1) continue;
        __threadfence();
      }
#pragma unroll 1
      for (int q = 0; q < S::ALL_BLOCKS; ++q) {
        // Blocks of half 0, then of half 1.
        const int h = q / S::BLOCKS;
        const int c0 = col + q % S::BLOCKS * 32;
        float v[32];
        if (piece) {
          // The pieces in their order, the next one's loads behind this one's adds.
          const float* part = p.parts + (int64_t)(first * 2 + 1) * S::PART_FLOATS + my_part + q * 1024;
          float4 x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = __ldcg(reinterpret_cast<const float4*>(part + j * 128));
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0.0f;
          part += S::PART_FLOATS;             // (first + 1, 0), then every second
          for (int c = 1;; ++c) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              v[4 * j] = __fadd_rn(v[4 * j], x[j].x);
              v[4 * j + 1] = __fadd_rn(v[4 * j + 1], x[j].y);
              v[4 * j + 2] = __fadd_rn(v[4 * j + 2], x[j].z);
              v[4 * j + 3] = __fadd_rn(v[4 * j + 3], x[j].w);
              if (c < count) x[j] = __ldcg(reinterpret_cast<const float4*>(part + j * 128));
            }
            if (c == count) break;
            part += 2 * S::PART_FLOATS;
          }
        } else {
          tmem_ld_32x32b_x32(lanes + (uint32_t)((buf + h) * ACC_COLS + q % S::BLOCKS * 32), v);
          if (q % S::BLOCKS == S::BLOCKS - 1) release(buf + h);     // read out: refill it
        }
        if (c0 < p.N) block_epilogue<T, MODE, ALIGNED>(p.e, row + h * 256, c0, v, block, lane);
      }
    }
    if (!ok) raise_abort();
  }

  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, 2 * ACC_COLS);
}

// ---------------------------------------------------------------- few rows, few tiles
// One output tile of 128 columns x NT rows per cluster: the columns (weights) are
// the MMA's 128 rows, so few rows of the output cost little.  The cluster's CTAs
// take equal parts of the sum; their F32 parts meet in shared memory and each CTA
// adds, in rank order, and stores a share of the rows.  Warp 0 loads, warp 1
// issues the MMAs, warps 2-5 (one TMEM lane quarter each) hold a column per
// thread.  With few rows the weights' bytes are all the work, and the stages
// keep 100 to 190 KB of them in flight per SM: one token through 4096 x 16384 BF16
// weights 23.6 us (5.7 TB/s).
constexpr int SPLIT_THREADS = 192;
template <int NT> constexpr int split_stage() { return TILE + NT * BK * 2; }
// With 16 rows two CTAs share an SM (108 KB each): one starts while the other ends
// (16384 columns of 4096: 23.9 us against 26.0 with one CTA of 10 stages).
template <int NT> constexpr int split_stages() { return NT == 16 ? 6 : 196608 / split_stage<NT>(); }
template <int NT> constexpr int split_smem() { return split_stages<NT>() * split_stage<NT>() + 1024 + 256; }

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

template <typename T, int MODE, int NT>
__global__ void __launch_bounds__(SPLIT_THREADS, 1)
split_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
             const __grid_constant__ Params p, int ranks) {
  constexpr int STAGES = split_stages<NT>(), STAGE = split_stage<NT>();
  constexpr uint32_t COLS = 2 * NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + STAGES;
  uint64_t* tfull_bar = bars + 2 * STAGES;        // [2]
  uint64_t* tempty_bar = bars + 2 * STAGES + 2;   // [2]
  uint64_t* drain_bar = bars + 2 * STAGES + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* part = reinterpret_cast<float*>(smem);   // [NT][128], once the stages are done with

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = (int)cluster_ctarank();
  const int64_t tile = blockIdx.x / ranks, num_n = cdiv(p.N, 128);
  const int64_t col0 = tile % num_n * 128, row0 = tile / num_n * NT;
  const int64_t blocks = cdiv(p.K, BK);
  const int begin = (int)(blocks * rank / ranks) * p.pairs, end = (int)(blocks * (rank + 1) / ranks) * p.pairs;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 4);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&map_p);
    prefetch_tmap(&map_q);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // Up to here the kernel may run beside the end of the one before it in the stream;
  // it touches memory only once that one is complete.  Its own successor may set up
  // from here on.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  float acc[NT];

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      int pair = begin % p.pairs;
      int64_t k0 = (int64_t)(begin / p.pairs) * BK;
      for (int it = begin; it < end; ++it) {
        const int pq = p.pairs == 1 ? 0 : (int)(PAIR_A >> (4 * pair)) & 15;
        const int pp = p.pairs == 1 ? 0 : (int)(PAIR_B >> (4 * pair)) & 15;
        if (!mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, p.dev_err)) break;
        uint8_t* dst = smem + stage * STAGE;
        mbar_arrive_expect_tx(&full_bar[stage], STAGE);
        load_tile(dst, &map_p, &full_bar[stage], p.b_mn, 128, col0, k0, pp);
        load_tile(dst + TILE, &map_q, &full_bar[stage], p.a_mn, NT, row0, k0, pq);
        ++issued;
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        if (++pair == p.pairs) { pair = 0; k0 += BK; }
      }
      // Never leave with copies in flight: every stage's last use has landed.
      for (int s = 0; s < STAGES && s < issued; ++s) {
        const uint32_t uses = (uint32_t)((issued - 1 - s) / STAGES);
        const uint64_t t0 = global_ns();
        while (!mbar_try_wait(&full_bar[s], uses & 1u) && global_ns() - t0 < kWaitLimitNs) {
        }
      }
    }
  } else if (warp == 1) {
    {
      const uint32_t id = idesc(p.bf16, p.b_mn, p.a_mn, NT, 128);
      const uint32_t a0 = desc_lo(smem_u32(smem), p.b_mn), b0 = desc_lo(smem_u32(smem) + TILE, p.a_mn);
      const uint32_t a_step = desc_step(p.b_mn), b_step = desc_step(p.a_mn);
      int stage = 0, in_chunk = 0;
      uint32_t phase = 0, chunks = 0;
      for (int it = begin; it < end; ++it) {
        const int buf = (int)(chunks & 1u);
        if (in_chunk == 0) {
          if (!warp_wait(&tempty_bar[buf], ((chunks >> 1) & 1u) ^ 1u, abort_flag, p.dev_err)) break;
          tc_fence_after();
        }
        if (!warp_wait(&full_bar[stage], phase, abort_flag, p.dev_err)) break;
        tc_fence_after();
        const uint32_t at = (uint32_t)(stage * (STAGE >> 4));
        const bool last = in_chunk + 1 == p.chunk || it == end - 1;
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < BK / 16; ++s)
            mma_f16(tmem + (uint32_t)(buf * NT), desc(a0 + at + s * a_step), desc(b0 + at + s * b_step), id,
                    (in_chunk | s) ? 1u : 0u);
          tc_commit(&empty_bar[stage]);
          if (last) tc_commit(&tfull_bar[buf]);
        }
        __syncwarp();
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        ++in_chunk;
        if (last) {
          ++chunks;
          in_chunk = 0;
        }
      }
      if (elect_one()) tc_commit(drain_bar);
      const uint64_t t0 = global_ns();
      while (!mbar_try_wait(drain_bar, 0) && global_ns() - t0 < kWaitLimitNs) {
      }
    }
  } else {
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int nchunks = (end - begin + p.chunk - 1) / p.chunk;
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = 0.0f;
    for (int c = 0; c < nchunks; ++c) {
      const int buf = c & 1;
      if (!warp_wait(&tfull_bar[buf], (uint32_t)(c >> 1) & 1u, abort_flag, p.dev_err)) break;
      tc_fence_after();
#pragma unroll
      for (int q = 0; q < NT / 16; ++q) {
        float v[16];
        tmem_ld_32x32b_x16(lanes + (uint32_t)(buf * NT + q * 16), v);
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[q * 16 + j] = __fadd_rn(acc[q * 16 + j], v[j]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty_bar[buf]);
    }
  }
  // All MMAs of this CTA are done (drain) and all copies have landed.
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, COLS);
  if (warp >= 2) {
#pragma unroll
    for (int j = 0; j < NT; ++j) part[j * 128 + (warp & 3) * 32 + lane] = acc[j];
  }
  if (ranks == 1) __syncthreads();
  else cluster_sync_all();
  // A CTA that gave up has no whole part, and none of its cluster stores sums with it.  The
  // lanes fetch the flags beside the first parts.
  uint32_t gave_up = (uint32_t)*abort_flag;
  if (ranks > 1 && lane < ranks) gave_up = ld_cluster_u32(cluster_addr(const_cast<int*>(abort_flag), (uint32_t)lane));
  // A warp per row, 4 columns per lane; the parts of two rows, and what their
  // epilogues read, are in flight at once.
  constexpr int U = 2;
  const int col = (int)col0 + lane * 4, j1 = NT * (rank + 1) / ranks;
  ColumnEpilogue<T, MODE> ce(p.e, col);
  for (int j = NT * rank / ranks + warp * U; j < j1 && row0 + j < p.M; j += SPLIT_THREADS / 32 * U) {
    float v[U][4];
    if (ranks == 1) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float4 x = *reinterpret_cast<const float4*>(part + (j + u < NT ? j + u : j) * 128 + lane * 4);
        v[u][0] = x.x; v[u][1] = x.y; v[u][2] = x.z; v[u][3] = x.w;
      }
    } else {
      float4 x[U][8];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < ranks)
            x[u][r] = ld_cluster_f32x4(cluster_addr(part + (j + u < NT ? j + u : j) * 128 + lane * 4, (uint32_t)r));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v[u][0] = x[u][0].x; v[u][1] = x[u][0].y; v[u][2] = x[u][0].z; v[u][3] = x[u][0].w;
#pragma unroll
        for (int r = 1; r < 8; ++r) {
          if (r < ranks) {
            v[u][0] = __fadd_rn(v[u][0], x[u][r].x);
            v[u][1] = __fadd_rn(v[u][1], x[u][r].y);
            v[u][2] = __fadd_rn(v[u][2], x[u][r].z);
            v[u][3] = __fadd_rn(v[u][3], x[u][r].w);
          }
        }
      }
    }
    if (__any_sync(0xffffffffu, gave_up != 0)) break;
    // Rows past this CTA's share or the matrix are outside for the epilogue.
    int64_t row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) row[u] = j + u < j1 ? row0 + j + u : p.M;
#pragma unroll
    for (int u = 0; u < U; ++u) ce.load(u, row[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) ce.store(u, row[u], v[u]);
  }
  __syncwarp();
  if (ranks == 1) return;
  cluster_sync_all();   // no CTA leaves while another still reads its part
}

// ---------------------------------------------------------------- operand preparation
// Contiguous [rows, cols] matrices -> planes of BF16 / F16 with row stride ldp (a
// multiple of 8): F32 is split, 16-bit types are copied.  The padding is outside
// the tensor map.  One launch for all operands of a call; bound by HBM (F32: 10
// bytes an element, 4096 x 4096 in 25 us, 6.8 TB/s).
struct Prepare {
  const void* x[MAX_OPERANDS];
  uint16_t* out[MAX_OPERANDS];
  int64_t rows[MAX_OPERANDS], cols[MAX_OPERANDS], ldp[MAX_OPERANDS];
  int64_t end[MAX_OPERANDS];      // of each matrix's 8-element pieces, counted through
  int count;
};

template <bool F32>
__global__ void __launch_bounds__(256)
prepare_kernel(const __grid_constant__ Prepare job) {
  const int64_t total = job.end[job.count - 1];
  for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < total; g += (int64_t)gridDim.x * 256) {
    int o = 0;
    while (g >= job.end[o]) ++o;
    const int64_t i = g - (o ? job.end[o - 1] : 0), cols = job.cols[o], ldp = job.ldp[o];
    const int64_t per_row = ldp / 8, plane = job.rows[o] * ldp;
    const int64_t r = total <= INT32_MAX ? (int64_t)((uint32_t)i / (uint32_t)per_row) : i / per_row;
    const int64_t c = (i - r * per_row) * 8;
    union { uint4 q; uint16_t e[8]; } u[3];
    if (F32) {
      const float* p = (const float*)job.x[o] + r * cols + c;
      const bool whole = (reinterpret_cast<uintptr_t>(p) & 15) == 0 && c + 8 <= cols;
      float v[8];
      load_row<float, 8>(p, cols - c < 8 ? (int)(cols - c) : 8, whole, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t bits = __float_as_uint(v[j]), b0 = bits & 0xffff0000u;
        const float r1 = v[j] - __uint_as_float(b0);
        const uint32_t b1 = __float_as_uint(r1) & 0xffff0000u;
        const float r2 = r1 - __uint_as_float(b1);
        u[0].e[j] = (uint16_t)(b0 >> 16);
        u[1].e[j] = (uint16_t)(b1 >> 16);
        u[2].e[j] = (uint16_t)(__float_as_uint(r2) >> 16);
        // Plane 2 meets only plane 0 of the other operand, so an infinity is carried there
        // (planes +-1, 0, +-inf): meeting planes 1 and 2, which are zero for values of few
        // bits, it would make NaN.  Plane 0 is zero for nothing but zero for the same reason:
        // values below the smallest BF16 become that.
        if ((bits & 0x7fffffffu) > 0x7f800000u) {
          u[0].e[j] = (uint16_t)((bits >> 16) | 0x40u);
          u[1].e[j] = u[2].e[j] = 0;
        } else if ((bits & 0x7fffffffu) == 0x7f800000u) {
          u[0].e[j] = (uint16_t)((bits >> 16 & 0x8000u) | 0x3f80u);
          u[1].e[j] = 0;
          u[2].e[j] = (uint16_t)(bits >> 16);
        } else if ((b0 & 0x7fffffffu) == 0 && bits != b0) {
          u[0].e[j] = (uint16_t)((b0 >> 16) | 1u);
          u[1].e[j] = u[2].e[j] = 0;
        }
      }
    } else {
      const uint16_t* p = (const uint16_t*)job.x[o] + r * cols + c;
#pragma unroll
      for (int j = 0; j < 8; ++j) u[0].e[j] = c + j < cols ? p[j] : (uint16_t)0;
    }
    uint4* out = reinterpret_cast<uint4*>(job.out[o] + r * ldp + c);
    out[0] = u[0].q;
    if (F32) {
      out[plane / 8] = u[1].q;
      out[plane / 4] = u[2].q;
    }
  }
}
}  // namespace lin

orca_status mma_prepare(orca_ctx* ctx, orca_dtype dtype, lin::Planes* const* x, int count,
                        lin::Scratch& scratch) {
  using namespace lin;
  Prepare job = {};
  const int planes = dtype == ORCA_F32 ? 3 : 1;
  size_t bytes = 0, at[MAX_OPERANDS];
  Planes* which[MAX_OPERANDS];
  for (int i = 0; i < count; ++i) {
    Planes& p = *x[i];
    p.ld = p.cols;
    p.plane = p.rows * p.cols;
    if (p.plane <= 0 || (dtype != ORCA_F32 && byte_alignment(p.p, p.cols * 2) == 16)) continue;
    const int o = job.count++;
    which[o] = &p;
    job.x[o] = p.p;
    job.rows[o] = p.rows;
    job.cols[o] = p.cols;
    p.ld = job.ldp[o] = cdiv(p.cols, 8) * 8;
    p.plane = p.rows * p.ld;
    job.end[o] = p.plane / 8 + (o ? job.end[o - 1] : 0);
    at[o] = bytes;
    bytes += (size_t)(planes * p.plane) * 2;      // a multiple of 16
  }
  if (!job.count) return ORCA_OK;
  ORCA_TRY(scratch.get(bytes));
  for (int o = 0; o < job.count; ++o) {
    job.out[o] = (uint16_t*)((uint8_t*)scratch.p + at[o]);
    which[o]->p = job.out[o];
  }
  const unsigned grid = (unsigned)std::min<int64_t>(cdiv(job.end[job.count - 1], 256), (int64_t)ctx->sm_count * 16);
  if (dtype == ORCA_F32) prepare_kernel<true><<<grid, 256, 0, ctx->stream>>>(job);
  else prepare_kernel<false><<<grid, 256, 0, ctx->stream>>>(job);
  count_launch(ctx);
  ORCA_CUDA_TRY(cudaGetLastError());
  return ORCA_OK;
}

namespace lin {

// ---------------------------------------------------------------- tensor maps
static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  return fn;
}

// Boxes of 64 columns (one 128-byte swizzle row) x box_rows rows of one plane.
static orca_status make_map(CUtensorMap* map, const Planes& x, int planes, int bf16, int box_rows) {
  auto encode = encode_fn();
  if (!encode) return fail(ORCA_CUDA_ERROR, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[3] = {(cuuint64_t)x.cols, (cuuint64_t)x.rows, (cuuint64_t)planes};
  cuuint64_t strides[2] = {(cuuint64_t)(x.ld * 2), (cuuint64_t)(x.plane * 2)};
  cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
  cuuint32_t step[3] = {1, 1, 1};
  const CUresult r = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                            3, const_cast<void*>(x.p), dims, strides, box, step,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(ORCA_CUDA_ERROR, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return ORCA_OK;
}

// ---------------------------------------------------------------- plans
// Times in microseconds that the choices below compare, measured: a step of each
// tile (512 rows save bytes: 8192 x 8192 x 8192 took 793 us against 834; 128 columns
// save part of a round: 4704 x 896 over 2208 24 us against 38), the drain that 512 rows do not hide, and what sharing a tile among `parts` clusters costs (each leaves its
// sums in L2, the last one adds them).
static double pair_step(int halves, int tn, int planes) {
  const double t = halves == 2 ? 0.77 : (tn == 256 ? 0.41 : 0.29);
  return planes == 3 ? t * F32_PAIRS : t;
}
static double drain_cost(int mode) { return mode == DW ? 2.0 : (mode == FWD ? 7.0 : 9.0); }
static double share_cost(int64_t parts) { return 8.0 + 2.5 * (double)parts; }

// The tiles beyond whole rounds of n clusters: how many clusters share them (0:
// none do, they are a last round of their own), and the steps that round takes.
struct Tail {
  int64_t clusters, steps;
};
static Tail share(int64_t rest, int64_t steps, int64_t n, double step, int halves, double* us) {
  Tail best{0, rest ? steps : 0};
  *us = rest ? (double)steps * step : 0.0;
  // An equal number of clusters per tile, or all of them with ranges that cross tiles.
  for (int64_t parts = 2; rest && parts <= 5; ++parts) {
    int64_t c = rest * parts, pieces = parts;
    if (c > n) {
      c = n;
      pieces = cdiv(n, rest) + 1;
    }
    const int64_t s = cdiv(rest * steps, c);
    const double t = (double)s * step + halves * share_cost(pieces);
    if (t < *us) {
      *us = t;
      best = Tail{c, s};
    }
    if (c == n) break;
  }
  return best;
}

// ---------------------------------------------------------------- launches
template <typename T, int MODE, int HALVES, int TN, bool ALIGNED>
static orca_status launch_pair(orca_ctx* ctx, const Planes& a, const Planes& b, Params p) {
  constexpr int PLANES = plane_count<T>();
  using S = Shape<HALVES, TN, PLANES>;
  const auto kernel = pair_kernel<T, MODE, HALVES, TN, ALIGNED>;
  CUtensorMap ma, mb;
  ORCA_TRY(make_map(&ma, a, PLANES, p.bf16, p.a_mn ? BK : ROWS));
  ORCA_TRY(make_map(&mb, b, PLANES, p.bf16, p.b_mn ? BK : TN / 2));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ctx->sm_count / 2 * 2));
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = ctx->stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static std::atomic<int> fits[64];      // clusters that are resident at once, per device
  std::atomic<int>& fit = fits[ctx->device & 63];
  if (fit.load() == 0) {
    ORCA_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    int n = 0;
    ORCA_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    if (n < 1) return fail(ORCA_CUDA_ERROR, "no cluster of two CTAs fits on the device");
    fit.store(n);
  }
  // Raster: 2048 rows by 9 tile columns are about what runs at once.  Where all of A
  // stays in L2 (48 MB of 126), all its rows form one group and B is read once
  // (4096 x 4096 x 16384: 404 us against 416).
  const int64_t a_bytes = p.M * p.K * 2 * (p.pairs == 1 ? 1 : 3);
  const int64_t num_m = cdiv(p.M, S::M), tiles = num_m * cdiv(p.N, TN), n = fit.load();
  p.group_m = (int)(a_bytes <= (int64_t)48 << 20 ? num_m : std::min<int64_t>(num_m, 2048 / S::M));
  const int64_t steps = cdiv(p.K, BK), rest = tiles % n;
  double us;
  const Tail tail = share(rest, steps, n, pair_step(HALVES, TN, PLANES), HALVES, &us);
  if (PLANES == 3) p.chunk = 1;            // in 64-deep blocks here
  if (HALVES == 2) p.chunk = (int)steps;   // one chain
  if (tiles > INT32_MAX - 4096) return fail(ORCA_INVALID_ARGUMENT, "linear: too many tiles");
  p.full = (int)tiles;
  p.tail = 0;
  p.shared = 0;
  p.parts = nullptr;
  p.arrived = nullptr;
  Scratch scratch(ctx);
  if (tail.clusters && rest * steps <= INT32_MAX) {
    p.full = (int)(tiles - rest);
    p.shared = (uint32_t)(rest * steps);
    p.tail = (int)tail.clusters;
    const size_t parts = (size_t)(tail.clusters * 2 * S::PART_FLOATS) * 4, counters = (size_t)(rest * S::ARRIVALS) * 4;
    ORCA_TRY(scratch.get(parts + counters));
    p.parts = (float*)scratch.p;
    p.arrived = (int*)((uint8_t*)scratch.p + parts);
    ORCA_CUDA_TRY(cudaMemsetAsync(p.arrived, 0, counters, ctx->stream));
  }
  cfg.gridDim = dim3((unsigned)(2 * (p.tail ? n : std::min(tiles, n))));
  ORCA_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, ma, mb, p));
  count_launch(ctx);
  return ORCA_OK;
}

// Clusters of 2^i CTAs of a split_kernel that are resident at once (asked once per
// device: clusters of 8 do not fill every GPC).
template <typename T, int MODE, int NT>
static orca_status split_fits(orca_ctx* ctx, int (&fits)[4]) {
  static std::atomic<int> known[64][4];
  const auto kernel = split_kernel<T, MODE, NT>;
  for (int i = 3; i >= 0; --i) {
    std::atomic<int>& fit = known[ctx->device & 63][i];
    if (fit.load() == 0) {
      if (i == 3)
        ORCA_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, split_smem<NT>()));
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1u << i;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1024);
      cfg.blockDim = dim3(SPLIT_THREADS);
      cfg.dynamicSmemBytes = split_smem<NT>();
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      ORCA_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
      fit.store(std::max(n, 1));
    }
    fits[i] = fit.load();
  }
  return ORCA_OK;
}

template <typename T, int MODE, int NT>
static orca_status launch_split(orca_ctx* ctx, const Planes& a, const Planes& b, int planes, const Params& p,
                                int ranks) {
  CUtensorMap ma, mb;
  ORCA_TRY(make_map(&ma, a, planes, p.bf16, p.a_mn ? BK : NT));
  ORCA_TRY(make_map(&mb, b, planes, p.bf16, p.b_mn ? BK : ROWS));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  const int64_t blocks = cdiv(p.N, 128) * cdiv(p.M, NT) * ranks;
  if (blocks > INT32_MAX) return fail(ORCA_INVALID_ARGUMENT, "linear: too many tiles");
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(SPLIT_THREADS);
  cfg.dynamicSmemBytes = split_smem<NT>();
  cfg.stream = ctx->stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  ORCA_CUDA_TRY(cudaLaunchKernelEx(&cfg, split_kernel<T, MODE, NT>, mb, ma, p, ranks));
  count_launch(ctx);
  return ORCA_OK;
}

struct Plan {
  int nt = 0;       // 0: pair_kernel
  int halves = 1;   // ... with 256 or 512 rows a tile
  int tn = 256;     // ... and 256 or 128 columns
  int ranks = 1;
  double us = 0;
};

// split_kernel with NT rows: as many CTAs per tile as still run at once, and the
// time that takes, fitted to 48..1024 rows through 512 x 784 to 16384 x 4096.
template <typename T, int MODE, int NT>
static orca_status consider(orca_ctx* ctx, const Params& p, int64_t steps, Plan* best) {
  int fits[4];
  ORCA_TRY((split_fits<T, MODE, NT>(ctx, fits)));
  constexpr double STEP = NT == 16 ? 0.27 : (NT == 32 ? 0.28 : (NT == 64 ? 0.29 : 0.31));
  const int64_t tiles = cdiv(p.N, 128) * cdiv(p.M, NT);
  const double hbm = (p.pairs == 1 ? 2.0 : 6.0) * ((double)p.M + (double)p.N) * (double)p.K / 5.5e6 + 3.0;
  for (int i = 0; i < 4 && (1 << i) * p.pairs <= steps; ++i) {
    const int ranks = 1 << i;
    // With 16 rows two CTAs fit an SM; that hides their ends, it does not add bandwidth.
    const int64_t at_once = std::min<int64_t>(fits[i], std::max(1, ctx->sm_count / ranks));
    const double us = std::max(
        hbm, (double)cdiv(tiles, at_once) * ((double)cdiv(steps, ranks) * STEP + (NT == 128 ? 3.0 : 1.0)) + 6.3 + 0.05 * ranks);
    if (us < best->us) *best = Plan{NT, 1, 256, ranks, us};
  }
  return ORCA_OK;
}

template <typename T, int MODE>
static orca_status choose(orca_ctx* ctx, const Params& p, int64_t steps, bool aligned, Plan* plan) {
  const int64_t n = ctx->sm_count / 2, blocks = cdiv(p.K, BK);
  plan->us = 1e30;
  for (int shape = 0; shape < (aligned ? 3 : 1); ++shape) {
    const int halves = shape == 2 ? 2 : 1, tn = shape == 0 ? 128 : 256;
    const int64_t tiles = cdiv(p.M, 256 * halves) * cdiv(p.N, tn);
    const double step = pair_step(halves, tn, plane_count<T>());
    double us;
    const Tail tail = share(tiles % n, blocks, n, step, halves, &us);
    // The two-accumulator tile has no chunks: a tile, or a cluster's share of one, is one chain.
    if (halves == 2 && (std::is_same<T, float>::value || p.chunk < (tiles < n ? tail.steps : blocks))) break;
    us += (double)(tiles / n * blocks) * step + (double)cdiv(tiles, n) * (halves == 2 ? drain_cost(MODE) : 0.0) +
          (tn == 256 ? 8.0 : 7.0);
    if (us < plan->us) *plan = Plan{0, halves, tn, 1, us};
  }
  if constexpr (MODE != DW) {
    if (p.M <= 16) return consider<T, MODE, 16>(ctx, p, steps, plan);
    if (p.M <= 32) return consider<T, MODE, 32>(ctx, p, steps, plan);
  }
  ORCA_TRY((consider<T, MODE, 64>(ctx, p, steps, plan)));
  return p.M > 64 ? consider<T, MODE, 128>(ctx, p, steps, plan) : ORCA_OK;
}

template <typename T, int MODE>
static orca_status dispatch(orca_ctx* ctx, orca_dtype dtype, const Planes& a, const Planes& b, Params& p) {
  const int planes = dtype == ORCA_F32 ? 3 : 1;
  const int64_t steps = cdiv(p.K, BK) * p.pairs;
  if (steps > INT32_MAX) return fail(ORCA_INVALID_ARGUMENT, "linear: the sum is too long");
  p.chunk = dtype == ORCA_F32 ? F32_PAIRS
            : (MODE == DW && p.e.out_f32 ? GRAD_CHUNK
            : (MODE == FWD && p.e.codes ? CKPT_CHUNK
            : (int)std::min<int64_t>(steps, dtype == ORCA_F16 ? F16_CHUNK : BF16_CHUNK)));
  Plan plan;
  // Outputs without aligned rows have one tile shape.
  const bool aligned = p.e.align == 16 && (!p.e.codes || p.e.ckpt_align >= 8);
  ORCA_TRY((choose<T, MODE>(ctx, p, steps, aligned, &plan)));
  if constexpr (MODE != DW) {
    if (plan.nt == 16) return launch_split<T, MODE, 16>(ctx, a, b, planes, p, plan.ranks);
    if (plan.nt == 32) return launch_split<T, MODE, 32>(ctx, a, b, planes, p, plan.ranks);
  }
  if (plan.nt == 64) return launch_split<T, MODE, 64>(ctx, a, b, planes, p, plan.ranks);
  if (plan.nt == 128) return launch_split<T, MODE, 128>(ctx, a, b, planes, p, plan.ranks);
  if (!aligned) return launch_pair<T, MODE, 1, 128, false>(ctx, a, b, p);
  if constexpr (!std::is_same<T, float>::value) {
    if (plan.halves == 2) return launch_pair<T, MODE, 2, 256, true>(ctx, a, b, p);
  }
  if (plan.tn == 128) return launch_pair<T, MODE, 1, 128, true>(ctx, a, b, p);
  return launch_pair<T, MODE, 1, 256, true>(ctx, a, b, p);
}

}  // namespace lin

orca_status mma_product(orca_ctx* ctx, int mode, orca_dtype dtype, int64_t M, int64_t N, int64_t K,
                        const lin::Planes& a, int a_mn, const lin::Planes& b, int b_mn,
                        const lin::Epilogue& e) {
  using namespace lin;
  Params p;
  p.M = M; p.N = N; p.K = K;
  p.a_mn = a_mn;
  p.b_mn = b_mn;
  p.bf16 = dtype != ORCA_F16;
  p.pairs = dtype == ORCA_F32 ? F32_PAIRS : 1;
  p.dev_err = ctx->dev_err;
  p.e = e;
#define ORCA_MODE(MODE)                                                            \
  if (dtype == ORCA_F32) return dispatch<float, MODE>(ctx, dtype, a, b, p);        \
  if (dtype == ORCA_F16) return dispatch<__half, MODE>(ctx, dtype, a, b, p);       \
  return dispatch<__nv_bfloat16, MODE>(ctx, dtype, a, b, p);
  switch (mode) {
    case FWD: { ORCA_MODE(FWD) }
    case DX: { ORCA_MODE(DX) }
    default: { ORCA_MODE(DW) }
  }
#undef ORCA_MODE
}

}  // namespace orca
