// Gradient of the experts' weights on the dispatched layout, for sm_100a tensor cores.
//
//   out[e, n, k] = sum over the rows r of expert e of grads[r, n] * rows[r, k]
//
// grads [L, N] bf16: the gradient of an expert layer's output, packed or in slots as its rows
// rows  [L, K] bf16: the rows that went into the layer
// out   [E, N, K] bf16 or fp32; zeros for an expert without rows
// loads [E] int32 on the device
//
// The sum runs over rows, so both operands have their features contiguous and the summed axis
// strided ("MN-major"): a ring slot holds 64 rows of both, in boxes of 64 features (128 bytes, one
// swizzle row) x 64 rows.  N features are the M operand (128 per CTA), up to 256 of K the N
// operand (half of them in each CTA of a pair).  Where an expert's rows end inside a slot, the
// rows behind them are another expert's or none at all: of the last slot only ceil(rows / 16) MMA
// steps run, and warp 2 first writes zeros over what the last step would read beyond the end in
// both operands (zeros in one would not do: the other may hold NaN or infinities).
// Additions in tensor memory need not round to nearest, so their errors add up instead of
// cancelling: after 1024 rows an accumulator is added to fp32 registers and begun anew (9001 rows in
// 30 uneven experts to fp32, off from 64 bits by 1.5e-6 of the norm without, 6.6e-7 with; a plain fp32
// product is off by 2.8e-7).
// Roles inside a CTA (384 threads): warp 0 TMA loads, warp 1 tensor memory and MMAs, warp 2 the
// ends of experts, warps 4-11 sums and output, four warps for each half of the tile's columns,
// under the MMAs that follow thanks to two accumulators.  A thread holds up to 128 values of
// one row of the output and stores whole sectors.  Every wait is bounded as in the other expert
// kernels.
//
// What bounds it: the tensor pipe and shared memory together (65536 rows in 32 even experts, 1024 x
// 4096, a launch at a time: 336 to 344 us, 1600 TFLOP/s) and under a sustained load the 1000 W limit
// (uneven experts: 480 to 510 us, 1080 to 1150 TFLOP/s); with few rows per expert writing the
// gradients.
#include "expert_tiles.cuh"
#include "tensor_core.cuh"

namespace brt_b200 {
namespace {

constexpr int kBM = 128;       // features of N per CTA
constexpr int kBN = 256;       // features of K per tile, at most
constexpr int kBR = 64;        // rows per ring slot
constexpr int kBoxFeatures = 64;
constexpr uint32_t kBoxBytes = kBoxFeatures * kBR * 2;  // 8 KB
constexpr int kABoxes = kBM / kBoxFeatures;
constexpr int kMmaK = 16;
constexpr int kFirstSumWarp = 4;  // warps are given registers by fours
constexpr int kSumWarps = 8;
constexpr int kThreads = 32 * (kFirstSumWarp + kSumWarps);
constexpr int kFewRegisters = 88, kManyRegisters = 208;
static_assert(128 * kFewRegisters + 32 * kSumWarps * kManyRegisters == kThreads * 168, "registers");
constexpr int kMaxSorted = 256;
constexpr int kChunk = 16;     // ring slots (1024 rows) per accumulator
template <int kPair>
constexpr int kStages = kPair == 2 ? 6 : 4;
template <int kPair>
constexpr int kBBoxes = kBN / kPair / kBoxFeatures;

struct WgradArgs {
  const int* loads;
  void* out;
  int* error;
  long long total_rows;
  int experts;
  int max_path_load;
  int N, K;
  int m_tiles;  // of 128 * kPair features of N
  int n_tiles;  // of `width` features of K
  int width;    // a multiple of 32
};

// kind::f16: fp32 accumulators, bf16 x bf16, both operands MN-major.
template <int kPair>
__device__ __forceinline__ uint32_t wgrad_idesc(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kPair * kBM >> 4) << 24);
}
// MN-major tile with the 128-byte swizzle: atoms of 64 features x 8 rows (1024 bytes); the next 8
// rows are 1024 bytes on (stride byte offset), the next 64 features a box (leading byte offset).
__device__ __forceinline__ uint64_t wgrad_desc(const void* tile) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_u32(tile) & 0x3ffff) >> 4);
  d |= (uint64_t)(kBoxBytes >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

template <int kPair>
struct alignas(1024) WgradSmem {
  unsigned char a[kStages<kPair>][kABoxes * kBoxBytes];
  unsigned char b[kStages<kPair>][kBBoxes<kPair> * kBoxBytes];
  uint64_t full[kStages<kPair>];
  uint64_t empty[kStages<kPair>];
  uint64_t tail[kStages<kPair>];  // this CTA's bytes of a slot where an expert ends
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint32_t tmem_base;
  ExpertTable table;
  int order[kMaxExperts];  // experts by descending load
};

struct WgradTile {
  int expert, n0, k0;
  int row0, load;
  int blocks;  // ring slots
};
// The tiles of the largest experts come first, and are dealt out to and fro.
__device__ __forceinline__ int wgrad_turn(int round, int group, int groups) {
  return round * groups + (round & 1 ? groups - 1 - group : group);
}
template <int kPair>
__device__ __forceinline__ WgradTile wgrad_tile(const WgradSmem<kPair>& s, const WgradArgs& g,
                                                int t) {
  WgradTile at;
  const ExpertTable& table = s.table;
  const int per = g.m_tiles * g.n_tiles;
  const int which = t / per;
  at.expert = s.order[which];
  const int local = t - which * per;
  const int part = local / g.m_tiles;
  at.n0 = (local - part * g.m_tiles) * kBM * kPair;
  at.k0 = part * g.width;
  at.row0 = table.row_base[at.expert];
  at.load = table.load[at.expert];
  at.blocks = (at.load + kBR - 1) / kBR;
  return at;
}

// 32 bytes by one thread: a whole sector.
__device__ __forceinline__ void store_sector(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// The empty statements keep the additions in front of the loads that follow (the compiler would
// hold more columns in registers than there are).
__device__ __forceinline__ void add_columns(float* sum, const uint32_t (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i++) sum[i] += __uint_as_float(v[i]);
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile("" : "+f"(sum[i]), "+f"(sum[i + 1]), "+f"(sum[i + 2]), "+f"(sum[i + 3]),
                      "+f"(sum[i + 4]), "+f"(sum[i + 5]), "+f"(sum[i + 6]), "+f"(sum[i + 7]));
}

template <int kPair, bool kFloatOut>
__global__ void __launch_bounds__(kThreads, 1)
expert_wgrad_kernel(const __grid_constant__ CUtensorMap map_g,
                    const __grid_constant__ CUtensorMap map_r, const WgradArgs g) {
  constexpr int kRing = kStages<kPair>;
  extern __shared__ __align__(1024) unsigned char s_raw[];
  WgradSmem<kPair>& s = *reinterpret_cast<WgradSmem<kPair>*>(
      (reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = kPair == 2 ? cluster_rank() : 0;
  const int group = blockIdx.x / kPair;
  const int groups = gridDim.x / kPair;
  const int total_tiles = g.experts * g.m_tiles * g.n_tiles;
  const int half = g.width / kPair;  // features of K that this CTA stages

  if (warp == 0) {
    fill_expert_table(s.table, g.loads, g.experts, g.max_path_load, g.total_rows,
                      [](int) { return 0; });
    if (lane == 0) {
      for (int i = 0; i < kRing; i++) {
        mbar_init(&s.full[i], kPair);
        mbar_init(&s.empty[i], 1);
        mbar_init(&s.tail[i], 1);
      }
      for (int i = 0; i < 2; i++) {
        mbar_init(&s.acc_full[i], 1);
        mbar_init(&s.acc_empty[i], kSumWarps * kPair);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  if (warp == 1) tmem_alloc<kPair>(&s.tmem_base);
  __syncthreads();
  // A tile takes as long as its expert has rows, so uneven experts are dealt out by load.  All
  // pairs are compared; beyond kMaxSorted experts that would take longer than it gains.
  for (int e = threadIdx.x; e < g.experts; e += kThreads) {
    int rank = e;
    if (g.experts <= kMaxSorted) {
      rank = 0;
      const int mine = s.table.load[e];
      for (int j = 0; j < g.experts; j++) {
        const int other = s.table.load[j];
        rank += other > mine || (other == mine && j < e);
      }
    }
    s.order[rank] = e;
  }
  tcgen05_before_sync();
  __syncthreads();
  group_sync<kPair>();
  tcgen05_after_sync();
  const uint32_t tmem = s.tmem_base;
  bool failed = false;

  if (warp < kFirstSumWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
    if (warp == 0) {
      int slot = 0;
      uint32_t phase = 0;
      const int b_boxes = (half + kBoxFeatures - 1) / kBoxFeatures;
      const uint32_t bytes = (uint32_t)(kABoxes + b_boxes) * kBoxBytes;
      for (int round = 0, t = group; t < total_tiles && !failed;
         t = wgrad_turn(++round, group, groups)) {
        const WgradTile at = wgrad_tile<kPair>(s, g, t);
        const int n0 = at.n0 + (int)rank * kBM;
        const int k0 = at.k0 + (int)rank * half;
        for (int i = 0; i < at.blocks; i++) {
          if (!mbar_wait_warp(&s.empty[slot], phase ^ 1)) { failed = true; break; }
          if (elect_one()) {
            uint32_t bar;
            if (at.load - i * kBR < kBR) {  // the expert ends here: warp 2 passes the slot on
              mbar_expect_tx(&s.tail[slot], bytes);
              bar = kPair == 2 ? map_to_cta(&s.tail[slot], rank) : smem_u32(&s.tail[slot]);
            } else {
              bar = kPair == 2 ? map_to_cta(&s.full[slot], 0) : smem_u32(&s.full[slot]);
              if (rank == 0) mbar_expect_tx(&s.full[slot], kPair * bytes);
              else mbar_arrive_cluster_relaxed(bar);
            }
            const int row = at.row0 + i * kBR;
#pragma unroll
            for (int b = 0; b < kABoxes; b++)
              tma_load_2d<kPair>(s.a[slot] + b * kBoxBytes, &map_g, bar, n0 + b * kBoxFeatures, row);
#pragma unroll
            for (int b = 0; b < kBBoxes<kPair>; b++)
              if (b < b_boxes)
                tma_load_2d<kPair>(s.b[slot] + b * kBoxBytes, &map_r, bar, k0 + b * kBoxFeatures,
                                   row);
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
        int slot = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        const uint32_t idesc = wgrad_idesc<kPair>(g.width);
        for (int round = 0, t = group; t < total_tiles && !failed;
         t = wgrad_turn(++round, group, groups)) {
          const WgradTile at = wgrad_tile<kPair>(s, g, t);
          for (int i = 0; i < at.blocks; i++) {
            if ((i % kChunk == 0 && !mbar_wait_warp(&s.acc_empty[acc], acc_phase ^ 1)) ||
                !mbar_wait_warp(&s.full[slot], phase)) {
              failed = true;
              break;
            }
            tcgen05_after_sync();
            const int rows = at.load - i * kBR;
            const bool last = i % kChunk == kChunk - 1 || i + 1 == at.blocks;
            const uint32_t d = tmem + (uint32_t)acc * kBN;
            if (elect_one()) {
              const uint64_t da = wgrad_desc(s.a[slot]);
              const uint64_t db = wgrad_desc(s.b[slot]);
#pragma unroll
              for (int k = 0; k < kBR / kMmaK; k++)  // 16 rows of 128 bytes further each
                if (k * kMmaK < rows)
                  umma_bf16<kPair>(d, da + 128 * k, db + 128 * k, idesc, (i % kChunk | k) != 0);
              umma_commit<kPair>(&s.empty[slot]);
              if (last) umma_commit<kPair>(&s.acc_full[acc]);
            }
            __syncwarp();
            if (++slot == kRing) { slot = 0; phase ^= 1; }
            if (last && ++acc == 2) { acc = 0; acc_phase ^= 1; }
          }
        }
      }
    } else if (warp == 2) {
      int slot = 0;            // of the next tile's first block
      uint32_t phases = 0;     // one bit per tail barrier
      const int b_boxes = (half + kBoxFeatures - 1) / kBoxFeatures;
      for (int round = 0, t = group; t < total_tiles && !failed;
         t = wgrad_turn(++round, group, groups)) {
        const WgradTile at = wgrad_tile<kPair>(s, g, t);
        const int rows = at.load % kBR;
        if (rows != 0) {
          const int last = (slot + at.blocks - 1) % kRing;
          if (!mbar_wait_warp(&s.tail[last], (phases >> last) & 1)) { failed = true; break; }
          phases ^= 1u << last;
          const int until = (rows + kMmaK - 1) / kMmaK * kMmaK;
          const int pieces = (until - rows) * 8;  // of 16 bytes, in one box
          for (int b = 0; b < kABoxes + b_boxes; b++) {
            unsigned char* const box = (b < kABoxes ? s.a[last] + b * kBoxBytes
                                                    : s.b[last] + (b - kABoxes) * kBoxBytes) +
                                       rows * kBoxFeatures * 2;
            for (int i = lane; i < pieces; i += 32)
              *reinterpret_cast<uint4*>(box + i * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            if (rank == 0) mbar_arrive(&s.full[last]);
            else mbar_arrive_cluster(map_to_cta(&s.full[last], 0));
          }
        }
        slot = (slot + at.blocks) % kRing;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
    const int quarter = warp & 3;  // the 32 lanes of tensor memory that this warp may read
    const int cols = g.width / 2;  // of this warp: a multiple of 16
    const int col0 = (warp - kFirstSumWarp) / 4 * cols;
    const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)col0;
    constexpr int kSize = kFloatOut ? 4 : 2;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int round = 0, t = group; t < total_tiles && !failed;
         t = wgrad_turn(++round, group, groups)) {
      const WgradTile at = wgrad_tile<kPair>(s, g, t);
      float sum[kBN / 2];
#pragma unroll
      for (int i = 0; i < kBN / 2; i++) sum[i] = 0.f;
#pragma unroll 1
      for (int i = 0; i < at.blocks; i += kChunk) {
        if (!mbar_wait_warp(&s.acc_full[acc], acc_phase)) { failed = true; break; }
        tcgen05_after_sync();
#pragma unroll
        for (int c = 0; c < 4; c++) {
          if (c * 32 >= cols) continue;
          uint32_t v[32];
          tmem_load_32(from + (uint32_t)(acc * kBN + c * 32), v);
          tmem_load_wait();
          add_columns(sum + c * 32, v);
        }
        hand_back(kPair == 2 ? map_to_cta(&s.acc_empty[acc], 0) : smem_u32(&s.acc_empty[acc]));
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
      if (failed) break;
      const int n = at.n0 + (int)rank * kBM + quarter * 32 + lane;
      const int columns = n < g.N ? min(cols, g.K - at.k0 - col0) : 0;
      unsigned char* const out = static_cast<unsigned char*>(g.out) +
          (((long long)at.expert * g.N + n) * g.K + at.k0 + col0) * kSize;
#pragma unroll
      for (int c = 0; c < kBN / 2; c += 32 / kSize) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          if constexpr (kFloatOut) {
            w[e] = __float_as_uint(sum[c + e]);
          } else {
            const __nv_bfloat162 p = __floats2bfloat162_rn(sum[c + 2 * e], sum[c + 2 * e + 1]);
            memcpy(&w[e], &p, 4);
          }
        }
        if (c < columns) store_sector(out + c * kSize, w);
      }
    }
  }
  if (failed) atomicExch(g.error, BRT_ERR_TIMEOUT);
  __syncwarp();

  tcgen05_before_sync();
  group_sync<kPair>();
  tcgen05_after_sync();
  if (warp == 1) tmem_free<kPair>(tmem);
}

template <int kPair, bool kFloatOut>
int launch_wgrad(const CUtensorMap& map_g, const CUtensorMap& map_r, const WgradArgs& g,
                 cudaStream_t st) {
  const size_t smem = sizeof(WgradSmem<kPair>) + 1024;
  static_assert(sizeof(WgradSmem<kPair>) + 1024 <= 232448, "shared memory of an SM");
  static thread_local int configured_device = -1;
  int dev = 0;
  BRT_CUDA_TRY(cudaGetDevice(&dev));
  if (configured_device != dev) {
    BRT_CUDA_TRY(cudaFuncSetAttribute(expert_wgrad_kernel<kPair, kFloatOut>,
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
  const KernelTimer timer("expert_wgrad_kernel", st);
  BRT_CUDA_TRY(cudaLaunchKernelEx(&config, expert_wgrad_kernel<kPair, kFloatOut>, map_g, map_r, g));
  note_launch();
  return BRT_OK;
}

int encode_features(EncodeTiledFn encode, CUtensorMap* map, const void* base, int64_t features,
                    int64_t rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)features, (cuuint64_t)(rows > 0 ? rows : 1)};
  const cuuint64_t strides[1] = {(cuuint64_t)features * 2};
  const cuuint32_t box[2] = {kBoxFeatures, kBR};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims,
                            strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(BRT_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
  return BRT_OK;
}

}  // namespace
}  // namespace brt_b200

using namespace brt_b200;

extern "C" {

BRT_API int brt_grouped_expert_weight_grad(const void* grads, const void* rows, void* out,
                                           const int32_t* loads, int path_num, int64_t total_rows,
                                           int32_t max_path_load, int64_t in_features,
                                           int64_t out_features, int out_dtype, void* error_word,
                                           void* stream) {
  clear_error();
  BRT_REQUIRE(path_num > 0 && path_num <= kMaxExperts, "path_num %d outside [1, %d]", path_num,
              kMaxExperts);
  BRT_REQUIRE(total_rows >= 0 && max_path_load >= 0, "negative size");
  BRT_REQUIRE(loads != nullptr && error_word != nullptr, "loads or error_word is null");
  BRT_REQUIRE(out_dtype == BRT_F32 || out_dtype == BRT_BF16, "out_dtype %d is neither fp32 nor bf16",
              out_dtype);
  if (in_features <= 0 || out_features <= 0 || in_features % 16 != 0 || out_features % 16 != 0)
    return set_error(BRT_ERR_UNSUPPORTED,
                     "the weight gradient needs in_features %% 16 == 0 and out_features %% 16 == 0 "
                     "(got %lld, %lld)",
                     (long long)in_features, (long long)out_features);
  BRT_REQUIRE(out != nullptr && aligned_to(out, 32), "out must be 32-byte aligned");
  BRT_REQUIRE(in_features < (1LL << 31) - 512 && out_features < (1LL << 31) - 512,
              "too many features");
  BRT_REQUIRE(total_rows < (1LL << 31) - 1024, "too many rows");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (total_rows == 0) {
    BRT_CUDA_TRY(cudaMemsetAsync(out, 0, (size_t)path_num * in_features * out_features *
                                             dtype_size(out_dtype), st));
    return BRT_OK;
  }
  BRT_REQUIRE(rows != nullptr && grads != nullptr, "null pointer argument");
  BRT_REQUIRE(aligned_to(rows, 16) && aligned_to(grads, 16),
              "rows and grads must be 16-byte aligned");
  const int n_blocks = (int)((out_features + kBM - 1) / kBM);
  // A pair takes 256 features; of an odd number of blocks its last tile is half empty.  16384 rows in
  // 16 experts, K = 2048, us for single CTAs and pairs: 1 block 18.6 and 25.2, 2 blocks 24.8 and 22.7,
  // 3 blocks 32.8 and 32.9, 5 blocks 46.8 and 44.7, 7 blocks 64.7 and 53.8; 4096 rows in 64 experts,
  // K = 1024: 1 block 14.9 and 22.7, 3 blocks 28.8 and 33.0, 5 blocks 30.9 and 35.9, 7 blocks 37.4 and
  // 41.0, 9 blocks 45.2 and 49.3.
  const int pair = n_blocks % 2 == 0 || n_blocks > 6 ? 2 : 1;
  WgradArgs g;
  g.loads = loads;
  g.out = out;
  g.error = static_cast<int*>(error_word);
  g.total_rows = total_rows;
  g.experts = path_num;
  g.max_path_load = max_path_load;
  g.N = (int)out_features;
  g.K = (int)in_features;
  g.m_tiles = (n_blocks + pair - 1) / pair;
  g.n_tiles = (int)((in_features + kBN - 1) / kBN);
  g.width = (int)round_up((size_t)((in_features + g.n_tiles - 1) / g.n_tiles), 32);
  BRT_REQUIRE((int64_t)path_num * g.m_tiles * g.n_tiles < (1LL << 31) - 1024,
              "more tiles than 32 bits count");
  EncodeTiledFn encode = encode_tiled();
  if (encode == nullptr)
    return set_error(BRT_ERR_CUDA, "the driver does not offer cuTensorMapEncodeTiled");
  alignas(64) CUtensorMap map_g;
  alignas(64) CUtensorMap map_r;
  int rc = encode_features(encode, &map_g, grads, out_features, total_rows);
  if (rc == BRT_OK) rc = encode_features(encode, &map_r, rows, in_features, total_rows);
  if (rc != BRT_OK) return rc;
  if (out_dtype == BRT_F32)
    return pair == 2 ? launch_wgrad<2, true>(map_g, map_r, g, st)
                     : launch_wgrad<1, true>(map_g, map_r, g, st);
  return pair == 2 ? launch_wgrad<2, false>(map_g, map_r, g, st)
                   : launch_wgrad<1, false>(map_g, map_r, g, st);
}

}  // extern "C"
