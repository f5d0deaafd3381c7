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
// K is one fresh accumulation in tensor memory (4 MMAs of K = 32), which the accumulating warps
// multiply by rs * ws and add to fp32 registers while the next block is being multiplied into
// the other half of tensor memory.  The rows are the M operand, 128 (the lanes of tensor memory)
// per CTA, and 256 features the N operand: a thread holds 128 features of ONE row, a scale block,
// and needs one scale per block of K.  (With the weights as M, as in the bf16 kernel, no row is
// computed for padding, but a thread needs the scales of 128 rows; the shared-memory reads for
// them made every size slower: 1024 rows per expert, 4096 -> 4096, 551 us against 322; 64 rows per
// expert, 102 against 82.)
// Two forms: CTA pairs (cta_group::2, 256 rows x 256 features, half of the features fetched by
// each) for many rows, single CTAs (128 x 256) for few: there the work on a block of K takes as
// long as ever for however few rows, and a CTA gets twice the weights through in that time.
//
// What bounds it: with many rows the accumulating warps (65536 rows in 32 even experts, 4096 -> 4096,
// three calls in a row: 1077 us, 2043 TFLOP/s; 790 us without them) and under a sustained load the
// 1000 W limit (uneven experts, for seconds: 1290 to 1330 us, 1650 to 1700 TFLOP/s); with few the
// reading of the weights (a row in each of 64 experts, 2048 -> 4096, calls in a row: 100 us, 5.4 TB/s).
// Roles inside a CTA (384 threads):
//   warp 0     TMA loads into a shared-memory ring, 128 bytes of K per slot and row (128-byte
//              swizzle): its 128 features, and of its 128 rows those that exist, in one box of
//              32, 64, 96 or 128 (what is left in the slot behind them are rows of the M
//              operand that nobody reads);
//   warp 1     allocates tensor memory; issues the MMAs of the pair (first CTA);
//   warps 2-3  copy the scales of 128 rows and of the weights into a ring, one warp for each of
//              the tile's two scale blocks, without waiting for the copies;
//   warps 4-11 scale and accumulate, four warps for each scale block; at the end ReLU, bf16, and
//              through shared memory out: whole groups of 32 rows by TMA stores, which go on under
//              the next tile (with pairs; 32768 rows, 1024 -> 4096: 189 -> 175 us), an expert's
//              last rows 64 bytes at a time.
// Every wait is bounded: after the limit the role records an error and leaves its loop, the
// copies in flight are given time to land, the CTAs meet, free tensor memory and return.
#include <cuda_fp8.h>

#include "expert_tiles.cuh"
#include "tensor_core.cuh"

namespace brt_b200 {
namespace {

constexpr int kBM = 128;      // rows per CTA, and features per scale block
constexpr int kBK = 128;      // codes of K per ring slot: one scale block, one swizzle row
constexpr int kBN = 256;      // features per tile
constexpr int kBoxStep = 32;  // the rows come in one box of 32, 64, 96 or 128
constexpr int kBoxSizes = 4;
constexpr int kMmaK = 32;
// ring slots: 32 KB each with a pair, 48 KB without
template <int kPair>
constexpr int kStages = kPair == 2 ? 5 : 4;
// Buffers of 32 rows x 32 features in which an accumulating warp turns its rows on their way out.
template <int kPair>
constexpr int kOutBuffers = kPair == 2 ? 2 : 1;
constexpr int kOutBytes = 32 * 64;
constexpr int kScaleSlots = 4;
constexpr int kAccWarps = 8;
constexpr int kFirstScaleWarp = 2;
constexpr int kFirstAccWarp = 4;  // warps are given registers by fours
constexpr int kThreads = 32 * (kFirstAccWarp + kAccWarps);
// The block starts with 168 registers a thread; the accumulators alone are 128 of an accumulating
// thread's, and the other four warps hand over some of theirs (more than 184 made the compiler
// hold more columns at once, and was up to 15 % slower).  At 168, ptxas -v counts 16 bytes of spill
// stores and 64 of spill loads per thread, in both forms.
constexpr int kFewRegisters = 136, kManyRegisters = 184;
static_assert(128 * kFewRegisters + 32 * kAccWarps * kManyRegisters == kThreads * 168, "registers");
// Rows per expert on average up to which single CTAs are taken.  16 experts, 4096 -> 4096, 16 calls
// in a row: 32 rows 58 us against 81 with pairs, 128 rows 64 against 87, 194 rows 102 against 93,
// 256 rows 105 against 95, 1024 rows 328 against 289; a row in each of 64 experts, 2048 -> 4096: 100
// against 146.
// The loads are on the device, so rows that dropped picks leave empty count here, and padded slots
// count as full: slots of more than 192 rows with few of them used take the slower form.
constexpr int kSingleRows = 192;
constexpr uint32_t kRowBytes = kBK;
constexpr uint32_t kTileBytes = kBM * kRowBytes;

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
  int n_tiles;         // of 256 features
  unsigned n_inverse;  // 2^32 / n_tiles, rounded up
  int n_blocks;        // of 128 features
  int k_blocks;
  int relu;
  int zero_unused;
};

// kind::f8f6f4: fp32 accumulators, e4m3 x e4m3, both operands K-major, N = 256.
template <int kPair>
__device__ __forceinline__ void mma_fp8(uint32_t tmem_d, uint64_t a, uint64_t b,
                                        uint32_t accumulate) {
  constexpr uint32_t kInstruction =
      (1u << 4) | ((uint32_t)(kBN >> 3) << 17) | ((uint32_t)(kPair * kBM >> 4) << 24);
  if constexpr (kPair == 2)
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(kInstruction), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(kInstruction), "r"(accumulate)
        : "memory");
}
// acc += v * scale for 32 columns, two at a time.  The empty statements keep the additions in
// front of the loads that follow: the compiler would move them behind, and then hold more columns
// in registers than there are.
__device__ __forceinline__ void add_scaled(float2* acc, const uint32_t (&v)[32], float scale) {
#pragma unroll
  for (int i = 0; i < 16; i++)
    acc[i] = __ffma2_rn(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])),
                        make_float2(scale, scale), acc[i]);
#pragma unroll
  for (int i = 0; i < 16; i += 4)
    asm volatile("" : "+f"(acc[i].x), "+f"(acc[i].y), "+f"(acc[i + 1].x), "+f"(acc[i + 1].y),
                      "+f"(acc[i + 2].x), "+f"(acc[i + 2].y), "+f"(acc[i + 3].x),
                      "+f"(acc[i + 3].y));
}

// Eight accumulators as bf16, ReLU applied.
__device__ __forceinline__ void pack_pairs(const float2* acc, int relu, uint32_t (&packed)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(acc[i].x, acc[i].y);
    const __nv_bfloat162 q = relu ? relu_pair(p) : p;
    memcpy(&packed[i], &q, 4);
  }
}

template <int kPair>
struct alignas(1024) Fp8Smem {
  unsigned char a[kStages<kPair>][kTileBytes];               // 128 rows
  unsigned char b[kStages<kPair>][kBN / kPair * kRowBytes];  // half of a pair's features, or all
  unsigned char out[kAccWarps][kOutBuffers<kPair>][kOutBytes];
  uint64_t full[kStages<kPair>];
  uint64_t empty[kStages<kPair>];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t scale_full[kScaleSlots][2];  // [slot][scale block of the tile]
  uint64_t scale_empty[kScaleSlots][2];
  float row_scale[kScaleSlots][2][kBM];
  float weight_scale[kScaleSlots][2];
  uint32_t tmem_base;
  ExpertTable table;
};
static_assert(sizeof(Fp8Smem<1>) + 1024 <= 232448 && sizeof(Fp8Smem<2>) + 1024 <= 232448,
              "shared memory of an SM");

struct TileAt {
  int expert, n_tile;
  int row0, rows;  // within the expert
};
// Walks over the tiles of a CTA or pair, every `step`-th of all; experts are followed from the last
// one, since a search of the whole table takes as long as two blocks of K.
template <int kPair>
struct TileWalk {
  const ExpertTable& table;
  const Fp8Args& g;
  int expert, local;  // number of the tile within its expert

  __device__ __forceinline__ TileWalk(const ExpertTable& table_, const Fp8Args& g_, int t)
      : table(table_), g(g_), expert(expert_of_tile(table_, g_.experts, t)),
        local(t - table_.first_tile[expert]) {}
  // `t`: the tile's number among all
  __device__ __forceinline__ void to(int t, int step) {
    local += step;
#pragma unroll 1
    for (int i = 0; i < 4; i++) {
      const int tiles = table.first_tile[expert + 1] - table.first_tile[expert];
      if (local < tiles) return;
      local -= tiles;
      expert++;
    }
    expert = expert_of_tile(table, g.experts, t);
    local = t - table.first_tile[expert];
  }
  __device__ __forceinline__ TileAt at() const {
    // local / n_tiles by its reciprocal, at most one too large
    int part = g.n_tiles == 1 ? local : (int)__umulhi((unsigned)local, g.n_inverse);
    if (part * g.n_tiles > local) part--;
    TileAt at;
    at.expert = expert;
    at.n_tile = local - part * g.n_tiles;
    at.row0 = part * kPair * kBM;
    at.rows = min(kPair * kBM, table.load[expert] - at.row0);
    return at;
  }
};
// Boxes of 32 rows that CTA `rank` fetches for a tile.
__device__ __forceinline__ int boxes_of(int rows, int rank) {
  const int mine = min(kBM, rows - rank * kBM);
  return mine > 0 ? (mine + kBoxStep - 1) / kBoxStep : 0;
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
                       const __grid_constant__ RowMaps map_r,
                       const __grid_constant__ CUtensorMap map_out, const Fp8Args g) {
  extern __shared__ __align__(1024) unsigned char s_raw[];
  Fp8Smem<kPair>& s = *reinterpret_cast<Fp8Smem<kPair>*>(
      (reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = kPair == 2 ? (int)cluster_rank() : 0;
  const int group = blockIdx.x / kPair;
  const int groups = gridDim.x / kPair;

  if (warp == 0) {
    const int n_tiles = g.n_tiles;
    fill_expert_table(s.table, g.loads, g.experts, g.max_path_load, g.total_rows,
                      [n_tiles](int load) {
                        return (load + kPair * kBM - 1) / (kPair * kBM) * n_tiles;
                      });
    if (lane == 0) {
      for (int i = 0; i < kStages<kPair>; i++) {
        mbar_init(&s.full[i], 1);
        mbar_init(&s.empty[i], 1);
      }
      for (int i = 0; i < 2; i++) {
        mbar_init(&s.acc_full[i], 1);
        mbar_init(&s.acc_empty[i], kAccWarps * kPair);
      }
      for (int i = 0; i < 2 * kScaleSlots; i++) {
        mbar_init(&s.scale_full[i >> 1][i & 1], 32);
        mbar_init(&s.scale_empty[i >> 1][i & 1], kAccWarps / 2);
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
  const int first = min(group, max(total_tiles - 1, 0));
  bool failed = false;

  if (warp < kFirstAccWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
    if (warp == 0) {
      int slot = 0;
      uint32_t phase = 0;
      TileWalk<kPair> walk(s.table, g, first);
      for (int t = group; t < total_tiles && !failed; t += groups) {
        if (t != group) walk.to(t, groups);
        const TileAt at = walk.at();
        const int boxes = boxes_of(at.rows, rank);
        const CUtensorMap* const map_box = &map_r.box[boxes > 0 ? boxes - 1 : 0];
        const int row0 = s.table.row_base[at.expert] + at.row0 + rank * kBM;
        const int feature0 = at.n_tile * kBN + rank * kBM;
        const int blocks = min(2, g.n_blocks - at.n_tile * 2);  // the last tile may have but one
        const uint32_t bytes =
            (uint32_t)(boxes_of(at.rows, 0) + (kPair == 2 ? boxes_of(at.rows, 1) : 0)) * kBoxStep *
                kRowBytes +
            (uint32_t)blocks * kTileBytes;
        for (int kb = 0; kb < g.k_blocks; kb++) {
          if (!mbar_wait_warp(&s.empty[slot], phase ^ 1)) { failed = true; break; }
          if (elect_one()) {
            if (rank == 0) mbar_expect_tx(&s.full[slot], bytes);  // of both CTAs
            const uint32_t bar =
                kPair == 2 ? map_to_cta(&s.full[slot], 0) : smem_u32(&s.full[slot]);
            if (rank < blocks)
              tma_load_3d<kPair>(s.b[slot], &map_w, bar, kb * kBK, feature0, at.expert);
            if (kPair == 1 && blocks == 2)
              tma_load_3d<kPair>(s.b[slot] + kTileBytes, &map_w, bar, kb * kBK, feature0 + kBM,
                                 at.expert);
            if (boxes > 0) tma_load_2d<kPair>(s.a[slot], map_box, bar, kb * kBK, row0);
          }
          __syncwarp();
          if (++slot == kStages<kPair>) { slot = 0; phase ^= 1; }
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
          for (int kb = 0; kb < g.k_blocks; kb++) {
            if (!mbar_wait_warp(&s.acc_empty[buf], buf_phase ^ 1) ||
                !mbar_wait_warp(&s.full[slot], phase)) {
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
                mma_fp8<kPair>(d, da + 2 * k, db + 2 * k, k != 0);
              umma_commit<kPair>(&s.empty[slot]);
              umma_commit<kPair>(&s.acc_full[buf]);
            }
            __syncwarp();
            if (++slot == kStages<kPair>) { slot = 0; phase ^= 1; }
            buf ^= 1;
            if (buf == 0) buf_phase ^= 1;
          }
        }
      }
    } else {
      const int half = warp - kFirstScaleWarp;
      int slot = 0;
      uint32_t phase = 0;
      TileWalk<kPair> walk(s.table, g, first);
      for (int t = group; t < total_tiles && !failed; t += groups) {
        if (t != group) walk.to(t, groups);
        const TileAt at = walk.at();
        const int feature_block = min(at.n_tile * 2 + half, g.n_blocks - 1);
        const float* const ws =
            g.weight_scales + ((long long)at.expert * g.n_blocks + feature_block) * g.k_blocks;
        const int row0 = rank * kBM + lane;
        const float* rs = g.row_scales +
            ((long long)s.table.row_base[at.expert] + at.row0 + row0) * g.row_stride;
#pragma unroll 1
        for (int kb = 0; kb < g.k_blocks; kb++) {
          if (!mbar_wait_warp(&s.scale_empty[slot][half], phase ^ 1)) { failed = true; break; }
#pragma unroll
          for (int i = 0; i < kBM / 32; i++)
            if (row0 + i * 32 < at.rows)
              cp_async_4(&s.row_scale[slot][half][i * 32 + lane], rs + i * 32 * g.row_stride);
          if (lane == 0) cp_async_4(&s.weight_scale[slot][half], ws + kb);
          mbar_arrive_copied(&s.scale_full[slot][half]);
          rs += g.block_stride;
          if (++slot == kScaleSlots) { slot = 0; phase ^= 1; }
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
    const int quarter = warp & 3;  // the 32 lanes of tensor memory that this warp may read
    const int half = (warp - kFirstAccWarp) / 4;  // of the tile's features: one scale block
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * kBM);
    const uint32_t handed_back =
        kPair == 2 ? map_to_cta(&s.acc_empty[0], 0) : smem_u32(&s.acc_empty[0]);
    const float* const row_scale = &s.row_scale[0][half][quarter * 32 + lane];
    const int row0 = rank * kBM + quarter * 32;  // of the tile
    int buf = 0, slot = 0, out_buffer = 0;
    uint32_t buf_phase = 0, phase = 0;
    TileWalk<kPair> walk(s.table, g, first);
    for (int t = group; t < total_tiles && !failed; t += groups) {
      if (t != group) walk.to(t, groups);
      const TileAt at = walk.at();
      const int feature0 = at.n_tile * kBN + half * kBM;
      const int rows = feature0 < g.N ? at.rows - row0 : 0;  // of this warp
      float2 acc[kBM / 2];
#pragma unroll
      for (int i = 0; i < kBM / 2; i++) acc[i] = make_float2(0.f, 0.f);
#pragma unroll 1
      for (int kb = 0; kb < g.k_blocks; kb++) {
        if (!mbar_wait_warp(&s.scale_full[slot][half], phase)) { failed = true; break; }
        const float scale = row_scale[slot * 2 * kBM] * s.weight_scale[slot][half];
        if (!mbar_wait_warp(&s.acc_full[buf], buf_phase)) { failed = true; break; }
        tcgen05_after_sync();
        const uint32_t from = lanes + (uint32_t)(buf * kBN);
        uint32_t v[2][32];
        tmem_load_32(from, v[0]);
#pragma unroll
        for (int c = 0; c < 4; c++) {
          tmem_load_wait();
          if (c < 3) {
            tmem_load_32(from + (c + 1) * 32, v[(c + 1) & 1]);
          } else {  // everything is in registers: the next block may be multiplied into it
            hand_back(handed_back + buf * (uint32_t)sizeof(uint64_t));
            if (lane == 0) mbar_arrive(&s.scale_empty[slot][half]);
          }
          add_scaled(acc + c * 16, v[c & 1], scale);
        }
        if (++slot == kScaleSlots) { slot = 0; phase ^= 1; }
        buf ^= 1;
        if (buf == 0) buf_phase ^= 1;
      }
      if (failed) break;
      const int row = s.table.row_base[at.expert] + at.row0 + row0;
#pragma unroll
      for (int c = 0; c < kBM / 32; c++) {
        const int feature = feature0 + c * 32;
        if (rows <= 0 || feature >= g.N) break;
        unsigned char* const staged = s.out[warp - kFirstAccWarp][out_buffer];
        if (++out_buffer == kOutBuffers<kPair>) out_buffer = 0;  // used in turn, tile after tile
        // the last store out of this buffer has read it (one lane issues them all)
        if (lane == 0)
          asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kOutBuffers<kPair> - 1)
                       : "memory");
        __syncwarp();
        // 64 bytes per row, its four pieces exchanged by the row's number (the 64-byte swizzle)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          uint32_t packed[4];
          pack_pairs(acc + c * 16 + i * 4, g.relu, packed);
          *reinterpret_cast<uint4*>(staged + lane * 64 + ((i ^ (lane >> 1)) & 3) * 16) =
              make_uint4(packed[0], packed[1], packed[2], packed[3]);
        }
        if (kPair == 2 && rows >= 32) {  // the TMA stores them while the warp goes on
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            asm volatile(
                "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                    &map_out),
                "r"(smem_u32(staged)), "r"(feature), "r"(row)
                : "memory");
          }
        } else {  // an expert's last rows: only those that exist
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int r = i * 8 + (lane >> 2);
            if (r < rows && feature + (lane & 3) * 8 < g.N)
              *reinterpret_cast<uint4*>(g.out + (long long)(row + r) * g.N + feature +
                                        (lane & 3) * 8) =
                  *reinterpret_cast<const uint4*>(staged + r * 64 + ((lane ^ (r >> 1)) & 3) * 16);
          }
          __syncwarp();
        }
        if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    if (g.zero_unused)
      zero_unused_rows(s.table, g, blockIdx.x * kAccWarps + warp - kFirstAccWarp,
                       gridDim.x * kAccWarps);
  }
  if (failed) atomicExch(g.error, BRT_ERR_TIMEOUT);
  __syncwarp();

  tcgen05_before_sync();
  group_sync<kPair>();  // nobody leaves while the peer may still signal its barriers
  tcgen05_after_sync();
  if (warp == 1) tmem_free<kPair>(tmem);
}

template <int kPair>
int launch_fp8(const CUtensorMap& map_w, const RowMaps& map_r, const CUtensorMap& map_out,
               const Fp8Args& g, cudaStream_t st) {
  const size_t smem = sizeof(Fp8Smem<kPair>) + 1024;
  static thread_local int configured_device = -1;
  int dev = 0;
  BRT_CUDA_TRY(cudaGetDevice(&dev));
  if (configured_device != dev) {
    BRT_CUDA_TRY(cudaFuncSetAttribute(expert_gemm_fp8_kernel<kPair>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured_device = dev;
  }
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = kPair;
  cluster.val.clusterDim.y = 1;
  cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(sm_count() / kPair * kPair));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = smem;
  config.stream = st;
  config.attrs = &cluster;
  config.numAttrs = 1;
  const KernelTimer timer("expert_gemm_fp8_kernel", st);
  BRT_CUDA_TRY(cudaLaunchKernelEx(&config, expert_gemm_fp8_kernel<kPair>, map_w, map_r, map_out, g));
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
  const int n_tiles = (n_blocks + 1) / 2;
  const int64_t mean_rows = max_path_load != 0 ? max_path_load : total_rows / path_num;
  const bool pair = mean_rows > kSingleRows;
  BRT_REQUIRE((total_rows / kBM + path_num) * (int64_t)n_tiles < (1LL << 31) - 1024,
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
  alignas(64) CUtensorMap map_out;
  {
    const cuuint64_t dims[2] = {(cuuint64_t)out_features, (cuuint64_t)total_rows};
    const cuuint64_t strides[1] = {(cuuint64_t)out_features * 2};
    const cuuint32_t box[2] = {32, 32};
    const CUresult r = encode(&map_out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, out, dims, strides, box,
                              elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                              CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
      return set_error(BRT_ERR_CUDA, "cuTensorMapEncodeTiled(out) failed with %d", (int)r);
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
  g.n_tiles = n_tiles;
  g.n_inverse = n_tiles == 1 ? 0u : (unsigned)((1ULL << 32) / (unsigned)n_tiles + 1);
  g.n_blocks = n_blocks;
  g.k_blocks = (int)((in_features + kBK - 1) / kBK);
  g.relu = relu != 0;
  g.zero_unused = zero_unused != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return pair ? launch_fp8<2>(map_w, map_r, map_out, g, st)
              : launch_fp8<1>(map_w, map_r, map_out, g, st);
}

}  // extern "C"
