// Order of the rows of a mixture-of-experts layer from compact picks (the indices of a top-k).
//
//   loads[e]     = number of picks that are e
//   places[t, j] = loads[0] + .. + loads[e-1] + number of earlier picks that are e
//                  (earlier: a smaller t * k + j), for e = picks[t, j]
//
// A stable counting sort.  Picks outside [0, paths) go nowhere: they count as one more path
// behind the last, and -2 - row stands in their place, the row at the end that stays empty for
// them.  Integer sums in a fixed order: the result does not depend on timing.
//
// A CTA owns a tile of consecutive picks and each of its warps a run of them.  Counting: a
// histogram per warp in shared memory; the lanes of a step that share a path are found with one
// match instruction and their first lane adds for all.  The exclusive sums over paths, tiles and
// warps turn the histograms into next places, and a second walk over the picks hands them out.
// Up to kOneCta picks one CTA does all of it in one launch; more take two launches, tile
// counts in between (the second launch is set up under the first).
#include "common.cuh"

namespace brt_b200 {
namespace {

constexpr int kMaxPaths = 1024;
constexpr int kWarps = 32;      // of a CTA with a large tile,
constexpr int kFewWarps = 16;   // and with few picks: fewer histograms to add up
constexpr int kBatch = 4;       // steps of 32 picks fetched together
// 2048 to 8192 picks took one CTA 6.4 to 20 us; two launches over tiles of 512 take 6 to 8.
constexpr int kOneCta = 1024;
constexpr int kSmallTile = 32 * kFewWarps;

struct OrderArgs {
  const void* picks;
  int* places;
  int* loads;
  int* counts;  // [tiles, paths + 1], two-launch form
  int n;
  int paths;
  int tile;  // picks per CTA, a multiple of 32 * warps
  int tiles;
};

template <typename P>
__device__ __forceinline__ int bucket_of(const P* picks, int i, int paths) {
  const P v = picks[i];
  return v >= 0 && v < (P)paths ? (int)v : paths;
}

// s_hist[warp][bucket] of this CTA's tile.
template <typename P>
__device__ __forceinline__ void count_tile(const OrderArgs& a, int* s_hist, int lo, int hi) {
  const int buckets = a.paths + 1;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < warps * buckets; i += blockDim.x) s_hist[i] = 0;
  __syncthreads();
  const P* picks = static_cast<const P*>(a.picks);
  const int run = a.tile / warps;
  const int end = min(lo + (warp + 1) * run, hi);
  int* const mine = s_hist + warp * buckets;
  for (int i0 = lo + warp * run; i0 < end; i0 += 32 * kBatch) {
    int b[kBatch];
#pragma unroll
    for (int s = 0; s < kBatch; s++) {
      const int i = i0 + s * 32 + lane;
      b[s] = i < end ? bucket_of(picks, i, a.paths) : buckets;
    }
#pragma unroll
    for (int s = 0; s < kBatch; s++) {
      const unsigned same = __match_any_sync(0xffffffffu, b[s]);
      if (b[s] < buckets && lane == __ffs(same) - 1) mine[b[s]] += __popc(same);
      __syncwarp();
    }
  }
  __syncthreads();
}

// s_hist[warp][bucket], behind s_base[bucket], is the next place of every warp and bucket: hands
// them out.
template <typename P>
__device__ __forceinline__ void place_tile(const OrderArgs& a, int* s_hist, const int* s_base,
                                           int lo, int hi) {
  const int buckets = a.paths + 1;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const P* picks = static_cast<const P*>(a.picks);
  const int run = a.tile / warps;
  const int end = min(lo + (warp + 1) * run, hi);
  int* const mine = s_hist + warp * buckets;
  for (int i0 = lo + warp * run; i0 < end; i0 += 32 * kBatch) {
    int b[kBatch];
#pragma unroll
    for (int s = 0; s < kBatch; s++) {
      const int i = i0 + s * 32 + lane;
      b[s] = i < end ? bucket_of(picks, i, a.paths) : buckets;
    }
#pragma unroll
    for (int s = 0; s < kBatch; s++) {
      const unsigned same = __match_any_sync(0xffffffffu, b[s]);
      int row = 0;
      if (b[s] < buckets) row = s_base[b[s]] + mine[b[s]] + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (b[s] < buckets && lane == __ffs(same) - 1) mine[b[s]] += __popc(same);
      __syncwarp();
      if (b[s] < buckets) a.places[i0 + s * 32 + lane] = b[s] < a.paths ? row : -2 - row;
    }
  }
}

// s_base[bucket] <- exclusive sums of s_total over the buckets (one warp, each lane a run of
// neighbouring buckets).
__device__ __forceinline__ void scan_buckets(const int* s_total, int* s_base, int buckets) {
  const int lane = threadIdx.x & 31;
  const int per = (buckets + 31) / 32;
  const int first = lane * per, last = min(first + per, buckets);
  int mine = 0;
  for (int b = first; b < last; b++) mine += s_total[b];
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  int next = incl - mine;
  for (int b = first; b < last; b++) {
    s_base[b] = next;
    next += s_total[b];
  }
}

template <typename P>
__global__ void __launch_bounds__(kWarps * 32) pick_order_kernel(const OrderArgs a) {
  extern __shared__ int s_mem[];
  const int buckets = a.paths + 1, warps = blockDim.x >> 5;
  int* const s_hist = s_mem;
  int* const s_total = s_hist + warps * buckets;
  int* const s_base = s_total + buckets;
  count_tile<P>(a, s_hist, 0, a.n);
  for (int b = threadIdx.x; b < buckets; b += blockDim.x) {
    int sum = 0;
#pragma unroll 8
    for (int w = 0; w < warps; w++) {
      const int c = s_hist[w * buckets + b];
      s_hist[w * buckets + b] = sum;
      sum += c;
    }
    s_total[b] = sum;
    if (b < a.paths) a.loads[b] = sum;
  }
  __syncthreads();
  if (threadIdx.x < 32) scan_buckets(s_total, s_base, buckets);
  __syncthreads();
  place_tile<P>(a, s_hist, s_base, 0, a.n);
}

template <typename P>
__global__ void __launch_bounds__(kWarps * 32) pick_count_kernel(const OrderArgs a) {
  extern __shared__ int s_mem[];
  const int buckets = a.paths + 1, warps = blockDim.x >> 5;
  const int lo = blockIdx.x * a.tile, hi = min(lo + a.tile, a.n);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  count_tile<P>(a, s_mem, lo, hi);
  for (int b = threadIdx.x; b < buckets; b += blockDim.x) {
    int sum = 0;
    for (int w = 0; w < warps; w++) sum += s_mem[w * buckets + b];
    a.counts[blockIdx.x * buckets + b] = sum;
  }
}

template <typename P>
__global__ void __launch_bounds__(kWarps * 32) pick_place_kernel(const OrderArgs a) {
  extern __shared__ int s_mem[];
  const int buckets = a.paths + 1, warps = blockDim.x >> 5;
  int* const s_hist = s_mem;
  int* const s_total = s_hist + warps * buckets;
  int* const s_base = s_total + buckets;
  int* const s_before = s_base + buckets;  // picks of the bucket in earlier tiles
  const int lo = blockIdx.x * a.tile, hi = min(lo + a.tile, a.n);
  for (int b = threadIdx.x; b < buckets; b += blockDim.x) s_total[b] = s_before[b] = 0;
  count_tile<P>(a, s_hist, lo, hi);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the tile counts are complete
  // neighbouring threads take neighbouring buckets; the tiles are dealt out to groups of threads
  const int groups = max(1, (int)blockDim.x / buckets);
  for (int at = threadIdx.x; at < groups * buckets; at += blockDim.x) {
    const int b = at % buckets;
    int total = 0, before = 0;
#pragma unroll 8
    for (int t = at / buckets; t < a.tiles; t += groups) {
      const int c = a.counts[t * buckets + b];
      total += c;
      if (t < (int)blockIdx.x) before += c;
    }
    atomicAdd(&s_total[b], total);  // integer sums: any order gives the same
    atomicAdd(&s_before[b], before);
  }
  __syncthreads();
  if (threadIdx.x < 32) scan_buckets(s_total, s_base, buckets);
  __syncthreads();
  for (int b = threadIdx.x; b < buckets; b += blockDim.x) {
    int next = s_before[b];
    for (int w = 0; w < warps; w++) {
      const int c = s_hist[w * buckets + b];
      s_hist[w * buckets + b] = next;
      next += c;
    }
    if (blockIdx.x == 0 && b < a.paths) a.loads[b] = s_total[b];
  }
  __syncthreads();
  place_tile<P>(a, s_hist, s_base, lo, hi);
}

int tile_for(int64_t n) {
  const int64_t tile = (n + sm_count() - 1) / sm_count();
  return tile <= kSmallTile ? kSmallTile : (int)round_up((size_t)tile, kWarps * 32);
}

// A tile ends at most 1024 picks per SM behind the last pick, which is within 32 bits; pick_total +
// tile is not.
int tiles_for(int64_t n) {
  const int64_t tile = tile_for(n);
  return (int)((n + tile - 1) / tile);
}

template <typename P>
int launch_order(OrderArgs a, cudaStream_t st) {
  const int buckets = a.paths + 1;
  static thread_local int configured_device = -1;
  int dev = 0;
  BRT_CUDA_TRY(cudaGetDevice(&dev));
  if (configured_device != dev) {
    const int most = (kWarps + 3) * (kMaxPaths + 1) * (int)sizeof(int);
    BRT_CUDA_TRY(cudaFuncSetAttribute(pick_order_kernel<P>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    BRT_CUDA_TRY(cudaFuncSetAttribute(pick_count_kernel<P>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    BRT_CUDA_TRY(cudaFuncSetAttribute(pick_place_kernel<P>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    configured_device = dev;
  }
  const KernelTimer timer("pick_order", st);
  if (a.n <= kOneCta) {
    int warps = (a.n + 31) / 32;
    if (warps > kFewWarps) warps = kFewWarps;
    a.tile = (int)round_up((size_t)a.n, (size_t)warps * 32);
    const size_t smem = (size_t)(warps + 2) * buckets * sizeof(int);
    pick_order_kernel<P><<<1, warps * 32, smem, st>>>(a);
    note_launch();
    BRT_LAUNCH_CHECK("pick_order_kernel");
    return BRT_OK;
  }
  const int warps = a.tile <= kSmallTile ? kFewWarps : kWarps;
  pick_count_kernel<P><<<a.tiles, warps * 32, (size_t)warps * buckets * sizeof(int), st>>>(a);
  note_launch();
  BRT_LAUNCH_CHECK("pick_count_kernel");
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)a.tiles);
  config.blockDim = dim3((unsigned)warps * 32);
  config.dynamicSmemBytes = (size_t)(warps + 3) * buckets * sizeof(int);
  config.stream = st;
  config.attrs = &early;
  config.numAttrs = 1;
  BRT_CUDA_TRY(cudaLaunchKernelEx(&config, pick_place_kernel<P>, a));
  note_launch();
  BRT_LAUNCH_CHECK("pick_place_kernel");
  return BRT_OK;
}

}  // namespace
}  // namespace brt_b200

using namespace brt_b200;

extern "C" {

BRT_API size_t brt_pick_order_scratch_bytes(int64_t pick_total, int path_num) {
  if (pick_total <= kOneCta || path_num <= 0) return 0;
  return (size_t)tiles_for(pick_total) * (size_t)(path_num + 1) * sizeof(int);
}

BRT_API int brt_order_picks(const void* picks, int picks_are_64bit, int64_t pick_total,
                            int path_num, int32_t* places, int32_t* loads, void* scratch,
                            size_t scratch_bytes, void* stream) {
  clear_error();
  BRT_REQUIRE(path_num > 0 && path_num <= kMaxPaths, "path_num %d outside [1, %d]", path_num,
              kMaxPaths);
  BRT_REQUIRE(pick_total >= 0 && pick_total < (1LL << 31) - (1 << 20),
              "%lld picks: the rows are counted in 32 bits", (long long)pick_total);
  BRT_REQUIRE(loads != nullptr, "loads is null");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (pick_total == 0) {
    BRT_CUDA_TRY(cudaMemsetAsync(loads, 0, (size_t)path_num * sizeof(int), st));
    return BRT_OK;
  }
  BRT_REQUIRE(picks != nullptr && places != nullptr, "null pointer argument");
  const size_t need = brt_pick_order_scratch_bytes(pick_total, path_num);
  if (need > 0 && (scratch == nullptr || scratch_bytes < need))
    return set_error(BRT_ERR_SCRATCH_TOO_SMALL, "scratch holds %zu bytes, %zu are needed",
                     scratch == nullptr ? (size_t)0 : scratch_bytes, need);
  OrderArgs a;
  a.picks = picks;
  a.places = places;
  a.loads = loads;
  a.counts = static_cast<int*>(scratch);
  a.n = (int)pick_total;
  a.paths = path_num;
  a.tile = tile_for(pick_total);
  a.tiles = tiles_for(pick_total);
  return picks_are_64bit ? launch_order<long long>(a, st) : launch_order<int>(a, st);
}

}  // extern "C"
