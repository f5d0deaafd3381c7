// Grouped expert GEMM in 8-bit floating point with a scale for each block of 128, for sm_100a
// tensor cores (tcgen05 + TMEM + TMA).
//
//   out[r, n] = act(sum over blocks b of rs[r, b] * ws[e, n / 128, b]
//                       * sum over k in block b of rows[r, k] * weights[e, n, k])
//
// rows    [L, K] e4m3: a dispatched buffer (path e starts at e * max_path_load when padded, else
//                      at sum(loads[0..e)); only the first loads[e] rows of a path count)
// weights [E, N, K] e4m3
// rs      fp32, one per row and block of 128 along K, any strides
// ws      fp32 [E, ceil(N / 128), ceil(K / 128)]
// out     [L, N] bf16
// loads   [E] int32 on the device
//
// K and N are multiples of 16; blocks at their ends are cut (the TMA fills with zero codes).
//
// The scales are any fp32 numbers, which the tensor cores cannot apply: each block of 128 along
// K is one fresh accumulation in tensor memory (4 MMAs of K = 32), which the epilogue warps
// multiply by rs * ws and add to fp32 registers while the next block is being multiplied into
// the other half of tensor memory.  As in the bf16 kernel the weights are the M operand (128
// features per CTA, exactly one scale block) and an expert's rows the N operand, cut into equal
// tiles of at most 256.  Roles inside a CTA (384 threads):
//   warp 0     one elected lane issues the TMA loads into a shared-memory ring (128 bytes of K
//              per slot and row, 128-byte swizzle);
//   warp 1     allocates tensor memory; one elected lane of the first CTA issues the MMAs of the
//              pair;
//   warps 4-11 scale and accumulate: four warps for each half of the tile's rows.  They read
//              tensor memory in the 16x256b form, where a thread holds two neighbouring columns
//              of each eight, in four lanes: a column's scale is loaded once for four values, so
//              that scales take 64 shared-memory wavefronts per block instead of the 256 that
//              one-lane-per-thread reads take (shared memory already carries the TMA's writes
//              and the MMA's reads at its full rate).  At the end: ReLU, bf16, stmatrix turned
//              so that a row's 32 features are stored together;
//   warps 2-3  multiply the two scales of the next blocks into a ring in shared memory.
// Every wait is bounded: after the limit the role records an error and leaves its loop, the
// copies in flight are given time to land, the CTAs meet, free tensor memory and return.
#include <cuda_fp8.h>

#include "expert_tiles.cuh"
#include "tensor_core.cuh"

namespace brt_b200 {
namespace {

constexpr int kBM = 128;        // weight rows (features) per CTA: one scale block
constexpr int kBK = 128;        // codes of K per ring slot: one scale block, one swizzle row
constexpr int kBN = 256;        // rows of an expert in one tile, at most
constexpr int kBoxStep = 32;    // the rows come in one box of 32, 64, 96 or 128
constexpr int kBoxSizes = 4;
constexpr int kMmaK = 32;
constexpr int kScaleSlots = 4;
constexpr int kAccWarps = 8;
constexpr int kFirstScaleWarp = 2;
constexpr int kScaleWarps = 2;
constexpr int kFirstAccWarp = 4;  // warps are given registers by fours
constexpr int kThreads = 32 * (kFirstAccWarp + kAccWarps);
// The block starts with 168 registers a thread.  The accumulators alone are 128 of an
// accumulating thread's, so the other four warps hand over what they do not need:
// 128 x 72 + 256 x 216 = 384 x 168.
constexpr int kFewRegisters = 72, kManyRegisters = 216;
static_assert(128 * kFewRegisters + 32 * kAccWarps * kManyRegisters == kThreads * 168, "registers");
constexpr uint32_t kTileBytes = kBM * kBK;
constexpr uint32_t kRowBytes = kBK;
template <int kPair>
constexpr int kStages = kPair == 2 ? 6 : 4;  // 32 KB each with a pair, 48 KB without

struct RowMaps {
  CUtensorMap box[kBoxSizes];  // box[i]: (i + 1) * kBoxStep rows
};

struct Fp8Args {
  const int* loads;
  const float* row_scales;
  const float* weight_scales;
  __nv_bfloat16* out;
  int* error;
  long long row_stride, block_stride;  // of row_scales
  long long total_rows;
  long long N;
  int experts;
  int max_path_load;
  int m_tiles;   // of 128 * kPair features
  int n_blocks;  // of 128 features
  int k_blocks;
  int relu;
  int zero_unused;
};

// kind::f8f6f4: fp32 accumulators, e4m3 x e4m3, both operands K-major.
template <int kPair>
__device__ __forceinline__ uint32_t fp8_idesc(int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kPair * kBM >> 4) << 24);
}
template <int kPair>
__device__ __forceinline__ void mma_fp8(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  if constexpr (kPair == 2)
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 16 lanes x 32 columns.  Register 4u + 2h + i of a thread: lane thread / 4 + 8h, column
// 8u + 2 * (thread % 4) + i.
__device__ __forceinline__ void tmem_load_16x32(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// acc += (lo, hi) * scale, two fp32 at a time
__device__ __forceinline__ void scaled_add(uint64_t& acc, uint32_t lo, uint32_t hi,
                                           uint64_t scale) {
  asm("{\n"
      ".reg .b64 v;\n"
      "mov.b64 v, {%1, %2};\n"
      "fma.rn.f32x2 %0, v, %3, %0;\n"
      "}\n"
      : "+l"(acc)
      : "r"(lo), "r"(hi), "l"(scale));
}
// Four 8x8 blocks of 16-bit values, each stored with rows and columns exchanged; lane 8m + i
// gives the address of row i of block m.
__device__ __forceinline__ void store_turned(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
               : "memory");
}

// Column c of a tile in a slot of the scale ring: the four scales that a thread needs of 16
// neighbouring columns (two of each eight) lie together.
__device__ __forceinline__ int scale_at(int c) {
  return (c & ~15) + ((c & 6) << 1) + ((c & 8) >> 2) + (c & 1);
}

template <int kPair>
struct alignas(1024) Fp8Smem {
  unsigned char a[kStages<kPair>][kTileBytes];
  unsigned char b[kStages<kPair>][kBN / kPair * kBK];
  unsigned char turn[kAccWarps][32 * 64];  // 32 rows of 32 features each
  float scale[kScaleSlots][kBN];
  uint64_t full[kStages<kPair>];
  uint64_t empty[kStages<kPair>];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t scale_full[kScaleSlots];
  uint64_t scale_empty[kScaleSlots];
  uint32_t tmem_base;
  ExpertTable table;
};

struct TileAt {
  int expert, m_tile;
  int row0, rows;  // within the expert
  int width;       // columns of the MMA: rows of a tile, rounded up to 32
};
__device__ __forceinline__ TileAt tile_at(const ExpertTable& table, int experts, int m_tiles,
                                          int t) {
  TileAt at;
  at.expert = expert_of_tile(table, experts, t);
  const int local = t - table.first_tile[at.expert];
  const int load = table.load[at.expert];
  const int parts = (load + kBN - 1) / kBN;
  const int each = ((load + parts - 1) / parts + 31) & ~31;
  const int part = local / m_tiles;
  at.m_tile = local - part * m_tiles;
  at.row0 = part * each;
  at.rows = load - at.row0 < each ? load - at.row0 : each;  // <= 0: rounding left none
  at.width = each;
  return at;
}

// Zeros in the rows of `out` that belong to no expert, a warp each.
__device__ __forceinline__ void zero_unused_rows(const ExpertTable& table, const Fp8Args& g,
                                                 int first, int step) {
  const int lane = threadIdx.x & 31;
  const int parts = g.max_path_load != 0 ? g.experts : 1;
  for (int e = 0; e < parts; e++) {
    const int last = g.max_path_load != 0 ? e : g.experts - 1;
    const long long from = (long long)table.row_base[last] + table.load[last];
    const long long until =
        g.max_path_load != 0 && e + 1 < parts ? table.row_base[e + 1] : g.total_rows;
    for (long long r = from + first; r < until; r += step)
      for (long long n = lane * 8; n < g.N; n += 256)
        *reinterpret_cast<uint4*>(g.out + r * g.N + n) = make_uint4(0u, 0u, 0u, 0u);
  }
}

template <int kPair>
__global__ void __launch_bounds__(kThreads, 1)
expert_gemm_fp8_kernel(const __grid_constant__ CUtensorMap map_w,
                       const __grid_constant__ RowMaps map_r, const Fp8Args g) {
  constexpr int kRing = kStages<kPair>;
  extern __shared__ __align__(1024) unsigned char s_raw[];
  Fp8Smem<kPair>& s = *reinterpret_cast<Fp8Smem<kPair>*>(
      (reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = kPair == 2 ? cluster_rank() : 0;
  const int group = blockIdx.x / kPair;
  const int groups = gridDim.x / kPair;

  if (warp == 0) {
    const int m_tiles = g.m_tiles;
    fill_expert_table(s.table, g.loads, g.experts, g.max_path_load, g.total_rows,
                      [m_tiles](int load) { return (load + kBN - 1) / kBN * m_tiles; });
    if (lane == 0) {
      for (int i = 0; i < kRing; i++) {
        mbar_init(&s.full[i], 1);
        mbar_init(&s.empty[i], 1);
      }
      for (int i = 0; i < 2; i++) {
        mbar_init(&s.acc_full[i], 1);
        mbar_init(&s.acc_empty[i], kAccWarps * kPair);
      }
      for (int i = 0; i < kScaleSlots; i++) {
        mbar_init(&s.scale_full[i], kScaleWarps);
        mbar_init(&s.scale_empty[i], kAccWarps);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  if (warp == 1) tmem_alloc<kPair>(&s.tmem_base);
  tcgen05_before_sync();
  __syncthreads();
  group_sync<kPair>();  // the peer's barriers exist
  tcgen05_after_sync();
  const uint32_t tmem = s.tmem_base;
  const int total_tiles = s.table.first_tile[g.experts];
  bool failed = false;
  if (warp < kFirstAccWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
    if (warp == 0) {
      int slot = 0;
      uint32_t phase = 0;
      for (int t = group; t < total_tiles && !failed; t += groups) {
        const TileAt at = tile_at(s.table, g.experts, g.m_tiles, t);
        const int half = at.width / kPair;  // rows this CTA stages
        const int boxes = half > kBoxSizes * kBoxStep ? 2 : 1;
        const int size = (half / boxes + kBoxStep - 1) / kBoxStep;
        const int box_rows = size * kBoxStep;
        const CUtensorMap* const map_box = &map_r.box[size - 1];
        const int row0 = s.table.row_base[at.expert] + at.row0 + (int)rank * half;
        const int feature0 = (at.m_tile * kPair + (int)rank) * kBM;
        const uint32_t bytes = kPair * (kTileBytes + (uint32_t)(boxes * box_rows) * kRowBytes);
        for (int kb = 0; kb < g.k_blocks; kb++) {
          if (!mbar_wait(&s.empty[slot], phase ^ 1)) { failed = true; break; }
          if (elect_one()) {
            if (rank == 0) mbar_expect_tx(&s.full[slot], bytes);
            const uint32_t bar =
                kPair == 2 ? map_to_cta(&s.full[slot], 0) : smem_u32(&s.full[slot]);
            tma_load_3d<kPair>(s.a[slot], &map_w, bar, kb * kBK, feature0, at.expert);
            tma_load_2d<kPair>(s.b[slot], map_box, bar, kb * kBK, row0);
            if (kPair == 1 && boxes == 2)
              tma_load_2d<kPair>(s.b[slot] + box_rows * kRowBytes, map_box, bar, kb * kBK,
                                 row0 + box_rows);
          }
          __syncwarp();
          if (++slot == kRing) { slot = 0; phase ^= 1; }
        }
      }
      // copies still in flight land before the CTA's shared memory is given back
      if (failed)
        for (int i = 0; i < 1024; i++) __nanosleep(1000);
    } else if (warp == 1) {
      if (rank == 0) {
        int slot = 0, buf = 0;
        uint32_t phase = 0, buf_phase = 0;
        for (int t = group; t < total_tiles && !failed; t += groups) {
          const TileAt at = tile_at(s.table, g.experts, g.m_tiles, t);
          const uint32_t idesc = fp8_idesc<kPair>(at.width);
          for (int kb = 0; kb < g.k_blocks; kb++) {
            if (!mbar_wait(&s.acc_empty[buf], buf_phase ^ 1) || !mbar_wait(&s.full[slot], phase)) {
              failed = true;
              break;
            }
            tcgen05_after_sync();
            if (elect_one()) {
              const uint64_t da = umma_desc(s.a[slot]);
              const uint64_t db = umma_desc(s.b[slot]);
              const uint32_t d = tmem + (uint32_t)buf * kBN;
#pragma unroll
              for (int k = 0; k < kBK / kMmaK; k++)  // 32 bytes further along the swizzled row
                mma_fp8<kPair>(d, da + 2 * k, db + 2 * k, idesc, k != 0);
              umma_commit<kPair>(&s.empty[slot]);
              umma_commit<kPair>(&s.acc_full[buf]);
            }
            __syncwarp();
            if (++slot == kRing) { slot = 0; phase ^= 1; }
            buf ^= 1;
            if (buf == 0) buf_phase ^= 1;
          }
        }
      }
    } else {
      // two warps, half of a tile's columns each; the scales of the next kAhead blocks are on
      // their way while those of the last ones are handed over
      const int half = warp - kFirstScaleWarp;
      constexpr int kAhead = 4;
      constexpr int kPer = kBN / 2 / 32;
      float r[kAhead][kPer], w[kAhead];
      int slot = 0;
      uint32_t phase = 0;
      TileAt at;
      const auto fetch = [&](int kb0) {
        const int feature_block = at.m_tile * kPair + (int)rank;
        const bool some = feature_block < g.n_blocks;  // a pair's second CTA may have no features
        const float* const ws = g.weight_scales +
            ((long long)at.expert * g.n_blocks + (some ? feature_block : 0)) * g.k_blocks;
        const float* const rs =
            g.row_scales + ((long long)s.table.row_base[at.expert] + at.row0) * g.row_stride;
#pragma unroll
        for (int h = 0; h < kAhead; h++) {
          const bool real = kb0 + h < g.k_blocks;
          w[h] = some && real ? __ldg(ws + kb0 + h) : 0.f;
#pragma unroll
          for (int i = 0; i < kPer; i++) {
            const int c = half * (kBN / 2) + i * 32 + lane;
            r[h][i] = real && c < at.rows
                          ? __ldg(rs + c * g.row_stride + (kb0 + h) * g.block_stride) : 0.f;
          }
        }
      };
      int t = group, kb0 = 0;
      if (t < total_tiles) {
        at = tile_at(s.table, g.experts, g.m_tiles, t);
        fetch(0);
      }
      while (t < total_tiles && !failed) {
        float scale[kAhead][kPer];
#pragma unroll
        for (int h = 0; h < kAhead; h++)
#pragma unroll
          for (int i = 0; i < kPer; i++) scale[h][i] = r[h][i] * w[h];
        const int blocks = min(kAhead, g.k_blocks - kb0);
        kb0 += kAhead;
        if (kb0 >= g.k_blocks) {
          kb0 = 0;
          t += groups;
          if (t < total_tiles) at = tile_at(s.table, g.experts, g.m_tiles, t);
        }
        if (t < total_tiles) fetch(kb0);
#pragma unroll
        for (int h = 0; h < kAhead; h++) {
          if (h >= blocks) break;
          if (!mbar_wait(&s.scale_empty[slot], phase ^ 1)) { failed = true; break; }
#pragma unroll
          for (int i = 0; i < kPer; i++)
            s.scale[slot][scale_at(half * (kBN / 2) + i * 32 + lane)] = scale[h][i];
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.scale_full[slot]);
          if (++slot == kScaleSlots) { slot = 0; phase ^= 1; }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
    const int quarter = warp & 3;  // the 32 lanes of tensor memory that this warp may read
    const int half = (warp - kFirstAccWarp) / 4;
    unsigned char* const turn = s.turn[warp - kFirstAccWarp];
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    int slot = 0, buf = 0;
    uint32_t phase = 0, buf_phase = 0;
    for (int t = group; t < total_tiles && !failed; t += groups) {
      const TileAt at = tile_at(s.table, g.experts, g.m_tiles, t);
      const int cols = at.width / 2;  // of this warp: a multiple of 16
      const int col0 = half * cols;
      // [32 columns][16 lanes][8 columns][8 lanes]: two columns each
      uint64_t acc[4][2][4][2];
#pragma unroll
      for (int c = 0; c < 4; c++)
#pragma unroll
        for (int l = 0; l < 2; l++)
#pragma unroll
          for (int u = 0; u < 4; u++) acc[c][l][u][0] = acc[c][l][u][1] = 0;
      for (int kb = 0; kb < g.k_blocks; kb++) {
        if (!mbar_wait(&s.scale_full[slot], phase) || !mbar_wait(&s.acc_full[buf], buf_phase)) {
          failed = true;
          break;
        }
        tcgen05_after_sync();
        const float* const scales = s.scale[slot] + col0 + (lane & 3) * 4;
        const uint32_t at_buf = lanes + (uint32_t)(buf * kBN + col0);
#pragma unroll
        for (int c = 0; c < 4; c++) {
          if (c * 32 >= cols) continue;
          uint32_t v[2][16];
          tmem_load_16x32(at_buf + c * 32, v[0]);
          tmem_load_16x32(at_buf + c * 32 + (16u << 16), v[1]);
          const ulonglong2 s0 = *reinterpret_cast<const ulonglong2*>(scales + c * 32);
          const ulonglong2 s1 = *reinterpret_cast<const ulonglong2*>(scales + c * 32 + 16);
          tmem_load_wait();
#pragma unroll
          for (int l = 0; l < 2; l++)
#pragma unroll
            for (int u = 0; u < 4; u++) {
              const uint64_t scale = u == 0 ? s0.x : u == 1 ? s0.y : u == 2 ? s1.x : s1.y;
              scaled_add(acc[c][l][u][0], v[l][4 * u], v[l][4 * u + 1], scale);
              scaled_add(acc[c][l][u][1], v[l][4 * u + 2], v[l][4 * u + 3], scale);
            }
        }
        tcgen05_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (rank == 0) mbar_arrive(&s.acc_empty[buf]);
          else mbar_arrive_cluster_relaxed(map_to_cta(&s.acc_empty[buf], 0));
          mbar_arrive(&s.scale_empty[slot]);
        }
        if (++slot == kScaleSlots) { slot = 0; phase ^= 1; }
        buf ^= 1;
        if (buf == 0) buf_phase ^= 1;
      }
      if (failed) break;
      const int feature = (at.m_tile * kPair + (int)rank) * kBM + quarter * 32 + (lane & 3) * 8;
      __nv_bfloat16* const out =
          g.out + ((long long)s.table.row_base[at.expert] + at.row0 + col0) * g.N + feature;
      const int rows = min(cols, at.rows - col0);
#pragma unroll
      for (int c = 0; c < 4; c++) {
        if (c * 32 >= rows) continue;
#pragma unroll
        for (int u = 0; u < 4; u++) {
          uint32_t packed[4];
#pragma unroll
          for (int m = 0; m < 4; m++) {
            const uint64_t pair = acc[c][m >> 1][u][m & 1];
            float lo = __uint_as_float((uint32_t)pair);
            float hi = __uint_as_float((uint32_t)(pair >> 32));
            if (g.relu) { lo = fmaxf(lo, 0.f); hi = fmaxf(hi, 0.f); }
            const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
            memcpy(&packed[m], &p, 4);
          }
          // 64 bytes per row, its four pieces exchanged by the row's number: no bank conflicts
          const int r = u * 8 + (lane & 7);
          store_turned(smem_u32(turn + r * 64 + (((lane >> 3) ^ (r >> 1)) & 3) * 16), packed);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int r = i * 8 + (lane >> 2);
          if (c * 32 + r < rows && feature < g.N)
            *reinterpret_cast<uint4*>(out + (long long)(c * 32 + r) * g.N) =
                *reinterpret_cast<const uint4*>(turn + r * 64 + ((lane ^ (r >> 1)) & 3) * 16);
        }
        __syncwarp();
      }
    }
    if (g.zero_unused)
      zero_unused_rows(s.table, g, blockIdx.x * kAccWarps + warp - kFirstAccWarp,
                       gridDim.x * kAccWarps);
  }
  if (failed) atomicExch(g.error, BRT_ERR_TIMEOUT);
  __syncwarp();  // the single-lane roles rejoin their warps before the barrier

  tcgen05_before_sync();
  group_sync<kPair>();  // nobody leaves while the peer may still signal its barriers
  tcgen05_after_sync();
  if (warp == 1) tmem_free<kPair>(tmem);
}

// ---- many rows per expert: the rows are the M operand -------------------------------------
//
// A CTA pair computes 256 rows x 256 features, 128 rows (the lanes of tensor memory) in each CTA.
// A thread then holds 128 features of ONE row, a scale block, and needs one scale per block of K,
// which it multiplies itself from two global values fetched blocks ahead: no scale ring and no
// shared-memory reads beside the MMA's.  The last tile of an expert is computed in full, so
// this pays from some hundred rows per expert on.

constexpr int kRowsStages = 6;
constexpr int kRowsFew = 40, kRowsMany = 232;
static_assert(128 * kRowsFew + 32 * kAccWarps * kRowsMany == kThreads * 168, "registers");
constexpr int kRowsAsM = 512;  // rows per expert on average

struct alignas(1024) Fp8RowsSmem {
  unsigned char a[kRowsStages][kTileBytes];  // 128 rows
  unsigned char b[kRowsStages][kTileBytes];  // 128 features: half of the pair's
  unsigned char turn[kAccWarps][32 * 64];
  uint64_t full[kRowsStages];
  uint64_t empty[kRowsStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint32_t tmem_base;
  ExpertTable table;
};

static_assert(sizeof(Fp8RowsSmem) + 1024 <= 232448 && sizeof(Fp8Smem<1>) + 1024 <= 232448 &&
              sizeof(Fp8Smem<2>) + 1024 <= 232448, "shared memory of an SM");

struct RowsTile {
  int expert, n_tile;
  int row0, rows;  // within the expert
};
__device__ __forceinline__ RowsTile rows_tile(const ExpertTable& table, int experts, int n_tiles,
                                              int t) {
  RowsTile at;
  at.expert = expert_of_tile(table, experts, t);
  const int local = t - table.first_tile[at.expert];
  const int part = local / n_tiles;
  at.n_tile = local - part * n_tiles;
  at.row0 = part * 2 * kBM;
  at.rows = min(2 * kBM, table.load[at.expert] - at.row0);
  return at;
}

__global__ void __launch_bounds__(kThreads, 1)
expert_gemm_fp8_rows_kernel(const __grid_constant__ CUtensorMap map_w,
                            const __grid_constant__ CUtensorMap map_r, const Fp8Args g) {
  extern __shared__ __align__(1024) unsigned char s_raw[];
  Fp8RowsSmem& s = *reinterpret_cast<Fp8RowsSmem*>(
      (reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int group = blockIdx.x / 2;
  const int groups = gridDim.x / 2;
  const int n_tiles = g.m_tiles;

  if (warp == 0) {
    fill_expert_table(s.table, g.loads, g.experts, g.max_path_load, g.total_rows,
                      [n_tiles](int load) { return (load + 2 * kBM - 1) / (2 * kBM) * n_tiles; });
    if (lane == 0) {
      for (int i = 0; i < kRowsStages; i++) {
        mbar_init(&s.full[i], 1);
        mbar_init(&s.empty[i], 1);
      }
      for (int i = 0; i < 2; i++) {
        mbar_init(&s.acc_full[i], 1);
        mbar_init(&s.acc_empty[i], kAccWarps * 2);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  if (warp == 1) tmem_alloc<2>(&s.tmem_base);
  tcgen05_before_sync();
  __syncthreads();
  group_sync<2>();
  tcgen05_after_sync();
  const uint32_t tmem = s.tmem_base;
  const int total_tiles = s.table.first_tile[g.experts];
  bool failed = false;

  if (warp < kFirstAccWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRowsFew));
    if (warp == 0) {
      int slot = 0;
      uint32_t phase = 0;
      for (int t = group; t < total_tiles && !failed; t += groups) {
        const RowsTile at = rows_tile(s.table, g.experts, n_tiles, t);
        const int row0 = s.table.row_base[at.expert] + at.row0 + (int)rank * kBM;
        const int feature0 = (at.n_tile * 2 + (int)rank) * kBM;
        for (int kb = 0; kb < g.k_blocks; kb++) {
          if (!mbar_wait(&s.empty[slot], phase ^ 1)) { failed = true; break; }
          if (elect_one()) {
            if (rank == 0) mbar_expect_tx(&s.full[slot], 4 * kTileBytes);
            const uint32_t bar = map_to_cta(&s.full[slot], 0);
            tma_load_2d<2>(s.a[slot], &map_r, bar, kb * kBK, row0);
            tma_load_3d<2>(s.b[slot], &map_w, bar, kb * kBK, feature0, at.expert);
          }
          __syncwarp();
          if (++slot == kRowsStages) { slot = 0; phase ^= 1; }
        }
      }
      // copies still in flight land before the CTA's shared memory is given back
      if (failed)
        for (int i = 0; i < 1024; i++) __nanosleep(1000);
    } else if (warp == 1 && rank == 0) {
      int slot = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      const uint32_t idesc = fp8_idesc<2>(2 * kBM);
      for (int t = group; t < total_tiles && !failed; t += groups) {
        for (int kb = 0; kb < g.k_blocks; kb++) {
          if (!mbar_wait(&s.acc_empty[buf], buf_phase ^ 1) || !mbar_wait(&s.full[slot], phase)) {
            failed = true;
            break;
          }
          tcgen05_after_sync();
          if (elect_one()) {
            const uint64_t da = umma_desc(s.a[slot]);
            const uint64_t db = umma_desc(s.b[slot]);
            const uint32_t d = tmem + (uint32_t)buf * kBN;
#pragma unroll
            for (int k = 0; k < kBK / kMmaK; k++)
              mma_fp8<2>(d, da + 2 * k, db + 2 * k, idesc, k != 0);
            umma_commit<2>(&s.empty[slot]);
            umma_commit<2>(&s.acc_full[buf]);
          }
          __syncwarp();
          if (++slot == kRowsStages) { slot = 0; phase ^= 1; }
          buf ^= 1;
          if (buf == 0) buf_phase ^= 1;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowsMany));
    const int quarter = warp & 3;
    const int half = (warp - kFirstAccWarp) / 4;  // of the tile's features: one scale block
    unsigned char* const turn = s.turn[warp - kFirstAccWarp];
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * kBM);
    int buf = 0;
    uint32_t buf_phase = 0;
    constexpr int kAhead = 4;  // blocks whose scales are on their way
    for (int t = group; t < total_tiles && !failed; t += groups) {
      const RowsTile at = rows_tile(s.table, g.experts, n_tiles, t);
      const int row0 = (int)rank * kBM + quarter * 32;  // of the tile
      const long long first = (long long)s.table.row_base[at.expert] + at.row0 + row0;
      const int feature_block = at.n_tile * 2 + half;
      const bool some = feature_block < g.n_blocks && row0 + lane < at.rows;
      const float* const rs = g.row_scales + (some ? (first + lane) * g.row_stride : 0);
      const float* const ws = g.weight_scales +
          (some ? ((long long)at.expert * g.n_blocks + feature_block) * g.k_blocks : 0);
      float r[kAhead], w[kAhead];
#pragma unroll
      for (int h = 0; h < kAhead; h++) {
        r[h] = some && h < g.k_blocks ? __ldg(rs + h * g.block_stride) : 0.f;
        w[h] = some && h < g.k_blocks ? __ldg(ws + h) : 0.f;
      }
      float acc[kBM];
#pragma unroll
      for (int i = 0; i < kBM; i++) acc[i] = 0.f;
      for (int kb0 = 0; kb0 < g.k_blocks && !failed; kb0 += kAhead) {
#pragma unroll
        for (int h = 0; h < kAhead; h++) {
          const int kb = kb0 + h;
          if (kb >= g.k_blocks) break;
          const float scale = r[h] * w[h];
          if (some && kb + kAhead < g.k_blocks) {
            r[h] = __ldg(rs + (kb + kAhead) * g.block_stride);
            w[h] = __ldg(ws + kb + kAhead);
          }
          if (!mbar_wait(&s.acc_full[buf], buf_phase)) { failed = true; break; }
          tcgen05_after_sync();
          const uint32_t from = lanes + (uint32_t)(buf * kBN);
          uint32_t v[2][32];
          tmem_load_32(from, v[0]);
#pragma unroll
          for (int c = 0; c < 4; c++) {
            tmem_load_wait();
            if (c < 3) tmem_load_32(from + (c + 1) * 32, v[(c + 1) & 1]);
            if (c == 3) {  // everything is in registers: the next block may be multiplied into it
              tcgen05_before_sync();
              __syncwarp();
              if (lane == 0) {
                if (rank == 0) mbar_arrive(&s.acc_empty[buf]);
                else mbar_arrive_cluster_relaxed(map_to_cta(&s.acc_empty[buf], 0));
              }
            }
#pragma unroll
            for (int i = 0; i < 32; i++)
              acc[c * 32 + i] = fmaf(__uint_as_float(v[c & 1][i]), scale, acc[c * 32 + i]);
          }
          buf ^= 1;
          if (buf == 0) buf_phase ^= 1;
        }
      }
      if (failed) break;
      const int rows = at.rows - row0;
      const int feature = feature_block * kBM + (lane & 3) * 8;
      __nv_bfloat16* const out = g.out + first * g.N + feature;
#pragma unroll
      for (int c = 0; c < 4; c++) {
        uint32_t packed[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
          float lo = acc[c * 32 + 2 * i], hi = acc[c * 32 + 2 * i + 1];
          if (g.relu) { lo = fmaxf(lo, 0.f); hi = fmaxf(hi, 0.f); }
          const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
          memcpy(&packed[i], &p, 4);
        }
        // 64 bytes per row, its four pieces exchanged by the row's number: no bank conflicts
#pragma unroll
        for (int i = 0; i < 4; i++)
          *reinterpret_cast<uint4*>(turn + lane * 64 + ((i ^ (lane >> 1)) & 3) * 16) =
              make_uint4(packed[4 * i], packed[4 * i + 1], packed[4 * i + 2], packed[4 * i + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int row = i * 8 + (lane >> 2);
          if (row < rows && feature + c * 32 < g.N)
            *reinterpret_cast<uint4*>(out + (long long)row * g.N + c * 32) =
                *reinterpret_cast<const uint4*>(turn + row * 64 + ((lane ^ (row >> 1)) & 3) * 16);
        }
        __syncwarp();
      }
    }
    if (g.zero_unused)
      zero_unused_rows(s.table, g, blockIdx.x * kAccWarps + warp - kFirstAccWarp,
                       gridDim.x * kAccWarps);
  }
  if (failed) atomicExch(g.error, BRT_ERR_TIMEOUT);
  __syncwarp();

  tcgen05_before_sync();
  group_sync<2>();
  tcgen05_after_sync();
  if (warp == 1) tmem_free<2>(tmem);
}

template <typename Kernel, typename MapR>
int launch_fp8(Kernel kernel, int pair, size_t smem, const CUtensorMap& map_w, const MapR& map_r,
               const Fp8Args& g, cudaStream_t st) {
  BRT_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)smem));
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = pair;
  cluster.val.clusterDim.y = 1;
  cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(sm_count() / pair * pair));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = smem;
  config.stream = st;
  config.attrs = &cluster;
  config.numAttrs = 1;
  const KernelTimer timer("expert_gemm_fp8_kernel", st);
  BRT_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, map_w, map_r, g));
  note_launch();
  return BRT_OK;
}

}  // namespace
}  // namespace brt_b200

using namespace brt_b200;

extern "C" {

BRT_API int brt_grouped_expert_gemm_fp8(const void* rows, const float* row_scales,
                                        int64_t scale_row_stride, int64_t scale_block_stride,
                                        const void* weights, const float* weight_scales,
                                        void* out, const int32_t* loads, int path_num,
                                        int64_t total_rows, int32_t max_path_load,
                                        int64_t in_features, int64_t out_features, int relu,
                                        int zero_unused, void* error_word, void* stream) {
  clear_error();
  BRT_REQUIRE(path_num > 0 && path_num <= kMaxExperts, "path_num %d outside [1, %d]", path_num,
              kMaxExperts);
  BRT_REQUIRE(total_rows >= 0 && max_path_load >= 0, "negative size");
  BRT_REQUIRE(loads != nullptr && error_word != nullptr, "loads or error_word is null");
  if (in_features <= 0 || out_features <= 0 || in_features % 16 != 0 || out_features % 16 != 0)
    return set_error(BRT_ERR_UNSUPPORTED,
                     "the 8-bit expert GEMM needs in_features %% 16 == 0 and out_features %% 16 "
                     "== 0 (got %lld, %lld)",
                     (long long)in_features, (long long)out_features);
  if (total_rows == 0) return BRT_OK;
  BRT_REQUIRE(rows != nullptr && weights != nullptr && out != nullptr && row_scales != nullptr &&
                  weight_scales != nullptr, "null pointer argument");
  BRT_REQUIRE(aligned_to(rows, 16) && aligned_to(weights, 16) && aligned_to(out, 16),
              "rows, weights and out must be 16-byte aligned");
  BRT_REQUIRE(total_rows < (1LL << 31) - 1024, "too many rows");
  BRT_REQUIRE(in_features < (1LL << 31) - 256 && out_features < (1LL << 31) - 512,
              "too many features");
  const int n_blocks = (int)((out_features + kBM - 1) / kBM);
  // a pair of CTAs computes two blocks of 128 features; single CTAs where an odd number would
  // leave half a pair idle for a large share of the work
  const int pair = n_blocks % 2 == 0 || n_blocks > 6 ? 2 : 1;
  const int64_t mean_rows = max_path_load != 0 ? max_path_load : total_rows / path_num;
  const bool rows_as_m = pair == 2 && mean_rows >= kRowsAsM;
  const int m_tiles = (n_blocks + pair - 1) / pair;
  BRT_REQUIRE((total_rows / kBN + path_num) * (int64_t)m_tiles < (1LL << 31) - 1024,
              "more tiles than 32 bits count");
  EncodeTiledFn encode = encode_tiled();
  if (encode == nullptr)
    return set_error(BRT_ERR_CUDA, "the driver does not offer cuTensorMapEncodeTiled");

  alignas(64) CUtensorMap map_w;
  alignas(64) RowMaps map_r;
  const cuuint32_t elem[3] = {1, 1, 1};
  for (int i = 0; i < kBoxSizes; i++) {
    const cuuint64_t dims[2] = {(cuuint64_t)in_features, (cuuint64_t)total_rows};
    const cuuint64_t strides[1] = {(cuuint64_t)in_features};
    const cuuint32_t box[2] = {kBK, (cuuint32_t)((i + 1) * kBoxStep)};
    const CUresult r = encode(&map_r.box[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 2,
                              const_cast<void*>(rows), dims, strides, box, elem,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
      return set_error(BRT_ERR_CUDA, "cuTensorMapEncodeTiled(rows) failed with %d", (int)r);
  }
  {
    const cuuint64_t dims[3] = {(cuuint64_t)in_features, (cuuint64_t)out_features,
                                (cuuint64_t)path_num};
    const cuuint64_t strides[2] = {(cuuint64_t)in_features,
                                   (cuuint64_t)in_features * out_features};
    const cuuint32_t box[3] = {kBK, kBM, 1};
    const CUresult r = encode(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3,
                              const_cast<void*>(weights), dims, strides, box, elem,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
      return set_error(BRT_ERR_CUDA, "cuTensorMapEncodeTiled(weights) failed with %d", (int)r);
  }
  Fp8Args g;
  g.loads = loads;
  g.row_scales = row_scales;
  g.weight_scales = weight_scales;
  g.out = static_cast<__nv_bfloat16*>(out);
  g.error = static_cast<int*>(error_word);
  g.row_stride = scale_row_stride;
  g.block_stride = scale_block_stride;
  g.total_rows = total_rows;
  g.N = out_features;
  g.experts = path_num;
  g.max_path_load = max_path_load;
  g.m_tiles = m_tiles;
  g.n_blocks = n_blocks;
  g.k_blocks = (int)((in_features + kBK - 1) / kBK);
  g.relu = relu != 0;
  g.zero_unused = zero_unused != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows_as_m)
    return launch_fp8(expert_gemm_fp8_rows_kernel, 2, sizeof(Fp8RowsSmem) + 1024, map_w,
                      map_r.box[kBoxSizes - 1], g, st);
  if (pair == 2)
    return launch_fp8(expert_gemm_fp8_kernel<2>, 2, sizeof(Fp8Smem<2>) + 1024, map_w, map_r, g, st);
  return launch_fp8(expert_gemm_fp8_kernel<1>, 1, sizeof(Fp8Smem<1>) + 1024, map_w, map_r, g, st);
}

}  // extern "C"
