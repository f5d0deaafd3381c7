// Cells to rows sorted by path and back, over the places of brt_order_picks.
//
//   sort      rows[places[t, j]] = cells[t]
//   sort fp8  the same row as 8-bit codes with a scale for each block of 128 (block_codes.cuh)
//   unsort    cells[t] = sum over j of gates[t, j] * rows[places[t, j]]
//   backward of unsort
//             row_grads[places[t, j]] = gates[t, j] * cell_grads[t]
//             gate_grads[t, j]        = <cell_grads[t], rows[places[t, j]]>
//   (the backward of sort is unsort without gates)
//
// A place p >= 0 is a row; p <= -2 says that the pick goes nowhere and that row -2 - p at the
// end stays empty: sort and the row gradients write zeros there, so that every row of their
// output is written exactly once whatever was dropped.  Other numbers (-1, or outside the buffer)
// are skipped: places may be edited after brt_order_picks, and the rows that nothing names any more
// are found and set to zero as well.  Sums run in fp32 in the order of j and are rounded once; a gate
// of a pick that goes nowhere is not looked at.
//
// All are bound by HBM (a few operations per byte).  sort and unsort give a warp 2 KB of a cell:
// a cell is read once for its k copies, and written once; with few cells a warp gets one pick or
// one access per lane.  The backward of unsort
// gives a warp one route, so that its dot product stays in the warp and is summed in one fixed
// order; the k warps of a cell read its gradient from L1 or L2.
//
// Rows that no place names: a bitmap of the rows of a window, made from all places, says which of
// them to set to zero.  Few rows are one window, and a CTA in front of the others sees to them.  For
// more a launch of its own does, beside which the rows are moved (none of them is a row that it
// writes): one cluster reads the places once to see whether each row is named, and only where that is
// not so searches the windows.  It goes by the number of rows named and by a sum of 64-bit mixtures of
// them (the finisher of splitmix64), which other rows than 0, 1, .. share by an accident of 2^-64.
// What that costs, bf16, places as brt_order_picks made them: 512 rows of 4 KB nothing, 8192 of 256
// bytes 8 us as before, 27003 of 128 bytes 8 -> 11 us, 65536 of 2 KB nothing (37 us), 524288 of 64
// bytes 45 -> 52 us, 8.4 million of 128 bytes 627 -> 670 us; to set all rows to zero first took those
// 65536 from 37 to 60 us.
#include <cooperative_groups.h>

#include "block_codes.cuh"

namespace brt_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kCtaWarps = kThreads / 32;

// VB-byte accesses per lane and item: 2 KB (1 KB of 2-byte accesses) per warp where there are
// items enough for the GPU, else one access.
template <int VB>
constexpr int kUnroll = VB == 16 ? 4 : 16;
constexpr int kManyItems = 16;  // per SM
constexpr int kManyCells = 4;   // per SM, where long items also save reads

// The search for rows that no place names.
constexpr int kFewRows = 8192;          // searched by one CTA of the kernel that moves them
constexpr int kSearchThreads = 512;
constexpr int kSearchCtas = 8;          // a cluster
constexpr int kMostWindow = 40 * 8192;  // rows of a window: 40 KB of bits
struct Unnamed {
  int front = 0;   // CTAs in front that search
  int beside = 0;  // a launch of its own searches, and has to end before this one does
};

struct SortArgs {
  const unsigned char* cells;
  unsigned char* rows;
  float* scales;  // [blocks, rows], sort fp8
  const int* places;
  long long row_bytes;  // of a cell
  long long width;
  long long items;
  long long total_rows;
  int pieces;
  int picks;
  int group;   // picks of an item
  int groups;  // items of a piece of a cell
  Unnamed unnamed;
};

__device__ __forceinline__ float empty_scale() { return __fdiv_rn(kAmaxFloor, kCodeMax); }

// Sets those of the rows [from, from + n) to zero that no place names, with `scales` to the codes and
// scales of rows of zeros.  By a whole CTA; `named` has a bit for each of the rows.  Not inlined: the
// loops of the kernels that move rows compile as they do without it (inlined, the backward pass of
// unsort went from 215 to 185 us over 131072 rows of 4 KB and from 178 to 239 over 120000 of 2002 bytes).
template <int VB>
__device__ __noinline__ void clear_unnamed(unsigned* named, unsigned from, unsigned n,
                                           const int* places, long long total,
                                           unsigned char* rows, long long row_bytes,
                                           float* scales) {
  using V = typename Chunk<VB>::type;
  const int tid = threadIdx.x, threads = blockDim.x;
  const int words = (int)((n + 31) / 32);
  for (int i = tid; i < words; i += threads) named[i] = 0u;
  __syncthreads();
  constexpr int kAtOnce = 16;
  for (long long i0 = tid; i0 < total; i0 += (long long)threads * kAtOnce) {
    int p[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; u++)
      p[u] = i0 + (long long)u * threads < total ? __ldg(places + i0 + (long long)u * threads) : -1;
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) {
      const unsigned at = (unsigned)(p[u] >= 0 ? p[u] : -2 - p[u]) - from;  // -1: behind any window
      if (at < n) atomicOr(&named[at >> 5], 1u << (at & 31));
    }
  }
  __syncthreads();
  const int lane = tid & 31;
  for (int word = tid >> 5; word < words; word += threads >> 5) {
    unsigned left = ~named[word];
    if (n - word * 32u < 32u) left &= (1u << (n - word * 32u)) - 1;
    for (; left != 0; left &= left - 1) {
      const long long row = (long long)from + word * 32 + (__ffs(left) - 1);
      for (long long at = lane * VB; at < row_bytes; at += 32 * VB)
        *reinterpret_cast<V*>(rows + row * row_bytes + at) = zero_chunk<V>();
      if (scales != nullptr)
        for (long long b = lane; b * kCodeBlock < row_bytes; b += 32)
          scales[b * total + row] = empty_scale();
    }
  }
}

// In the kernels that move rows: the CTA in front does nothing else, the last one waits for the
// search beside (all of whose predecessors have ended, or it would not have begun).
template <int VB>
__device__ __forceinline__ bool searches(const Unnamed& u, const int* places, long long total,
                                         unsigned char* rows, long long row_bytes, float* scales) {
  __shared__ unsigned s_named[kFewRows / 32];
  if (u.beside && blockIdx.x + 1 == gridDim.x)
    asm volatile("griddepcontrol.wait;" ::: "memory");
  if ((int)blockIdx.x >= u.front) return false;
  clear_unnamed<VB>(s_named, 0u, (unsigned)total, places, total, rows, row_bytes, scales);
  return true;
}

struct SearchArgs {
  const int* places;
  unsigned char* rows;
  float* scales;  // or null
  long long total, row_bytes;
  unsigned window;
};
__device__ __forceinline__ unsigned long long mixed(unsigned row) {
  unsigned long long x = (row + 1ull) * 0x9e3779b97f4a7c15ull;
  x = (x ^ (x >> 30)) * 0xbf58476d1ce4e5b9ull;
  x = (x ^ (x >> 27)) * 0x94d049bb133111ebull;
  return x ^ (x >> 31);
}
template <int VB>
__global__ void __cluster_dims__(kSearchCtas) __launch_bounds__(kSearchThreads)
unnamed_rows_kernel(const SearchArgs a) {
  extern __shared__ unsigned s_bits[];
  __shared__ unsigned long long s_sums[2];  // rows named; mixtures of them less those of all rows
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const auto cluster = cooperative_groups::this_cluster();
  const unsigned rank = cluster.block_rank();
  if (threadIdx.x < 2) s_sums[threadIdx.x] = 0;
  __syncthreads();
  constexpr int kAtOnce = 16, kStep = kSearchCtas * kSearchThreads;
  unsigned long long mine[2] = {0, 0};
  for (long long i0 = rank * kSearchThreads + threadIdx.x; i0 < a.total; i0 += kStep * kAtOnce) {
    int p[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; u++)
      p[u] = i0 + u * kStep < a.total ? __ldg(a.places + i0 + u * kStep) : -1;
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) {
      const unsigned row = (unsigned)(p[u] >= 0 ? p[u] : -2 - p[u]);
      if (i0 + u * kStep < a.total) mine[1] -= mixed((unsigned)(i0 + u * kStep));
      if (row >= a.total) continue;  // -1, or outside
      mine[0]++;
      mine[1] += mixed(row);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; i++) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mine[i] += __shfl_xor_sync(0xffffffffu, mine[i], d);
    if ((threadIdx.x & 31) == 0) atomicAdd(&s_sums[i], mine[i]);
  }
  cluster.sync();
  unsigned long long all[2] = {0, 0};
  for (unsigned r = 0; r < kSearchCtas; r++)
    for (int i = 0; i < 2; i++) all[i] += cluster.map_shared_rank(s_sums, r)[i];
  cluster.sync();  // nobody leaves while others read its sums
  if (all[0] == (unsigned long long)a.total && all[1] == 0) return;
  for (long long from = (long long)rank * a.window; from < a.total;
       from += (long long)kSearchCtas * a.window) {
    clear_unnamed<VB>(s_bits, (unsigned)from, (unsigned)min((long long)a.window, a.total - from),
                      a.places, a.total, a.rows, a.row_bytes, a.scales);
    __syncthreads();
  }
}

// The item of this warp: a piece of a cell for some of its picks.
struct SortItem {
  long long cell;
  int piece, first, last;
};
__device__ __forceinline__ SortItem sort_item(const SortArgs& a, long long item) {
  SortItem it;
  const long long at = item / a.groups;
  const int part = (int)(item - at * a.groups);
  it.cell = at / a.pieces;
  it.piece = (int)(at - it.cell * a.pieces);
  it.first = part * a.group;
  it.last = min(a.picks, it.first + a.group);
  return it;
}

template <int VB, int U>
__global__ void __launch_bounds__(kThreads) sort_cells_kernel(const SortArgs a) {
  using V = typename Chunk<VB>::type;
  if (searches<VB>(a.unnamed, a.places, a.total_rows, a.rows, a.row_bytes, nullptr)) return;
  const int lane = threadIdx.x & 31;
  const long long item =
      (long long)(blockIdx.x - a.unnamed.front) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (item >= a.items) return;
  const SortItem it = sort_item(a, item);
  const long long at = (long long)it.piece * (32 * VB * U) + lane * VB;
  const unsigned char* const src = a.cells + it.cell * a.row_bytes + at;
  V v[U];
#pragma unroll
  for (int u = 0; u < U; u++)
    v[u] = at + u * (32 * VB) < a.row_bytes
               ? load_stream(reinterpret_cast<const V*>(src + u * (32 * VB)))
               : zero_chunk<V>();
  const int* const places = a.places + it.cell * a.picks;
  for (int j = it.first; j < it.last; j++) {
    const int p = __ldg(places + j);
    const long long row = p >= 0 ? p : -2LL - p;
    if (row < 0 || row >= a.total_rows) continue;
    unsigned char* const dst = a.rows + row * a.row_bytes + at;
#pragma unroll
    for (int u = 0; u < U; u++)
      if (at + u * (32 * VB) < a.row_bytes)
        *reinterpret_cast<V*>(dst + u * (32 * VB)) = p >= 0 ? v[u] : zero_chunk<V>();
  }
}

constexpr int kCodeUnroll = 4;  // x 256 values per warp and item

// kPlaced = false: one row per cell, in the order they come (a plain quantisation).
template <int DT, int U, bool kPlaced>
__global__ void __launch_bounds__(kThreads) sort_codes_kernel(const SortArgs a) {
  using T = typename Elem<DT>::type;
  if constexpr (kPlaced)
    if (searches<16>(a.unnamed, a.places, a.total_rows, a.rows, a.width, a.scales)) return;
  const int lane = threadIdx.x & 31;
  const long long item =
      (long long)(blockIdx.x - (kPlaced ? a.unnamed.front : 0)) * (blockDim.x >> 5) +
      (threadIdx.x >> 5);
  if (item >= a.items) return;
  const SortItem it = sort_item(a, item);
  const long long at = (long long)it.piece * (256 * U) + lane * 8;
  const T* const src = reinterpret_cast<const T*>(a.cells) + it.cell * a.width + at;
  Eight<DT> v[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    if (at + u * 256 < a.width) v[u].load(src + u * 256);
    else v[u].clear();
  }
  // 16 lanes hold a block.  Its two quotients are taken by one lane in U of them and handed round:
  // each is a dozen instructions, and taken by all lanes they cost more than the conversion.
  float mine = kAmaxFloor;
#pragma unroll
  for (int u = 0; u < U; u++) {
    float amax = v[u].max_abs();
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    if ((lane & 15) % U == u) mine = fmaxf(amax, kAmaxFloor);
  }
  const float my_scale = __fdiv_rn(mine, kCodeMax);
  const float my_inverse = __fdiv_rn(kCodeMax, mine);
  uint2 code[U];
  float scale[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    scale[u] = __shfl_sync(0xffffffffu, my_scale, (lane & 16) + u);
    code[u] = v[u].encode(scale[u], __shfl_sync(0xffffffffu, my_inverse, (lane & 16) + u));
  }
  for (int j = it.first; j < it.last; j++) {
    const int p = kPlaced ? __ldg(a.places + it.cell * a.picks + j) : 0;
    const long long row = !kPlaced ? it.cell : p >= 0 ? p : -2LL - p;
    if (row < 0 || row >= a.total_rows) continue;
    unsigned char* const dst = a.rows + row * a.width + at;
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (at + u * 256 >= a.width) continue;
      *reinterpret_cast<uint2*>(dst + u * 256) = p >= 0 ? code[u] : make_uint2(0u, 0u);
      if ((lane & 15) == 0)
        a.scales[((at + u * 256) / kCodeBlock) * a.total_rows + row] =
            p >= 0 ? scale[u] : empty_scale();
    }
  }
}

struct UnsortArgs {
  const unsigned char* rows;
  unsigned char* cells;
  const int* places;
  const void* gates;  // or null
  long long row_bytes;
  long long items;
  long long total_rows;
  int pieces;
  int picks;
};

template <int DT, int VB>
struct Pack {  // a VB-byte access as values
  static constexpr int kValues = VB / (int)sizeof(typename Elem<DT>::type);
  static __device__ __forceinline__ void values(const typename Chunk<VB>::type& raw,
                                                float (&v)[kValues]) {
    typename Elem<DT>::type part[kValues];
    memcpy(part, &raw, VB);
#pragma unroll
    for (int i = 0; i < kValues; i++) v[i] = Elem<DT>::to_f32(part[i]);
  }
  static __device__ __forceinline__ typename Chunk<VB>::type chunk(const float (&v)[kValues]) {
    typename Elem<DT>::type part[kValues];
#pragma unroll
    for (int i = 0; i < kValues; i++) part[i] = Elem<DT>::from_f32(v[i]);
    typename Chunk<VB>::type raw;
    memcpy(&raw, part, VB);
    return raw;
  }
};

// kGates: 0 none, 1 fp32, 2 of the data's type
template <int DT, int kGates>
__device__ __forceinline__ float gate_at(const void* gates, long long i) {
  if constexpr (kGates == 0) return 1.f;
  else if constexpr (kGates == 1) return __ldg(static_cast<const float*>(gates) + i);
  else return Elem<DT>::to_f32(static_cast<const typename Elem<DT>::type*>(gates)[i]);
}

template <int DT, int VB, int U, int kGates>
__global__ void __launch_bounds__(kThreads) unsort_cells_kernel(const UnsortArgs a) {
  using V = typename Chunk<VB>::type;
  using P = Pack<DT, VB>;
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (item >= a.items) return;
  const long long cell = item / a.pieces;
  const long long at = (item - cell * a.pieces) * (32 * VB * U) + lane * VB;
  float sum[U][P::kValues];
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int e = 0; e < P::kValues; e++) sum[u][e] = 0.f;
  // rows on their way at a time: as many as registers allow without losing warps
  constexpr int kAtOnce = VB < 16 && U > 1 ? 1 : U > 1 ? 2 : 8;
  for (int j0 = 0; j0 < a.picks; j0 += 32) {
    // a lane for each pick: its place and gate come with one access each
    int my_place = -1;
    float my_gate = 0.f;
    if (j0 + lane < a.picks) {
      const long long route = cell * a.picks + j0 + lane;
      my_place = __ldg(a.places + route);
      my_gate = gate_at<DT, kGates>(a.gates, route);
    }
    const int until = min(32, a.picks - j0);
    for (int j = 0; j < until; j += kAtOnce) {
      V raw[kAtOnce][U];
      int place[kAtOnce];
#pragma unroll
      for (int h = 0; h < kAtOnce; h++) {
        place[h] = __shfl_sync(0xffffffffu, my_place, (j + h) & 31);
        if (j + h >= until || place[h] >= a.total_rows) place[h] = -1;
        const unsigned char* const src = a.rows + (long long)place[h] * a.row_bytes + at;
#pragma unroll
        for (int u = 0; u < U; u++)
          raw[h][u] = place[h] >= 0 && at + u * (32 * VB) < a.row_bytes
                          ? load_stream(reinterpret_cast<const V*>(src + u * (32 * VB)))
                          : zero_chunk<V>();
      }
#pragma unroll
      for (int h = 0; h < kAtOnce; h++) {
        const float gate = __shfl_sync(0xffffffffu, my_gate, (j + h) & 31);
        if (place[h] < 0) continue;  // the whole warp: its gate may be anything
#pragma unroll
        for (int u = 0; u < U; u++) {
          float v[P::kValues];
          P::values(raw[h][u], v);
#pragma unroll
          for (int e = 0; e < P::kValues; e++)
            sum[u][e] = kGates == 0 ? sum[u][e] + v[e] : fmaf(gate, v[e], sum[u][e]);
        }
      }
    }
  }
  unsigned char* const dst = a.cells + cell * a.row_bytes + at;
#pragma unroll
  for (int u = 0; u < U; u++)
    if (at + u * (32 * VB) < a.row_bytes)
      store_stream(reinterpret_cast<V*>(dst + u * (32 * VB)), P::chunk(sum[u]));
}

struct BackArgs {
  const unsigned char* cell_grads;
  const unsigned char* rows;  // or null: no gate gradients
  unsigned char* row_grads;   // or null
  void* gate_grads;           // or null
  const int* places;
  const void* gates;
  long long row_bytes;
  long long routes;
  long long total_rows;
  int picks;
  Unnamed unnamed;
};

template <int DT, int VB, int kGates>
__global__ void __launch_bounds__(kThreads) unsort_backward_kernel(const BackArgs a) {
  using V = typename Chunk<VB>::type;
  using P = Pack<DT, VB>;
  if (searches<VB>(a.unnamed, a.places, a.total_rows, a.row_grads, a.row_bytes, nullptr)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long route = (long long)(blockIdx.x - a.unnamed.front) * kCtaWarps + warp;
  if (route >= a.routes) return;
  const int p = __ldg(a.places + route);
  const long long row = p >= 0 ? p : -2LL - p;
  const bool inside = row >= 0 && row < a.total_rows;
  const bool live = inside && p >= 0;
  float dot = 0.f;
  if (inside) {
    const float gate = live ? gate_at<DT, kGates>(a.gates, route) : 0.f;
    const unsigned char* const grad = a.cell_grads + route / a.picks * a.row_bytes;
    const bool dots = live && a.gate_grads != nullptr;
    constexpr int U = VB == 16 ? 4 : 8;
    for (long long at = lane * VB; at < a.row_bytes; at += 32 * VB * U) {
      V g[U], r[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const long long o = at + u * (32 * VB);
        const bool real = live && o < a.row_bytes;
        g[u] = real ? __ldg(reinterpret_cast<const V*>(grad + o)) : zero_chunk<V>();
        r[u] = real && dots
                   ? load_stream(reinterpret_cast<const V*>(a.rows + row * a.row_bytes + o))
                   : zero_chunk<V>();
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const long long o = at + u * (32 * VB);
        float gv[P::kValues], rv[P::kValues];
        P::values(g[u], gv);
        P::values(r[u], rv);
        if (dots && o < a.row_bytes) {
#pragma unroll
          for (int e = 0; e < P::kValues; e++) dot = fmaf(gv[e], rv[e], dot);
        }
        if (a.row_grads != nullptr && o < a.row_bytes) {
#pragma unroll
          for (int e = 0; e < P::kValues; e++) gv[e] = live ? gate * gv[e] : 0.f;
          store_stream(reinterpret_cast<V*>(a.row_grads + row * a.row_bytes + o), P::chunk(gv));
        }
      }
    }
  }
  if (a.gate_grads == nullptr) return;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
  if (lane == 0) {
    if constexpr (kGates == 2)
      static_cast<typename Elem<DT>::type*>(a.gate_grads)[route] = Elem<DT>::from_f32(dot);
    else
      static_cast<float*>(a.gate_grads)[route] = dot;
  }
}

// The widest access that rows of `row_bytes` at these addresses allow: 16, 4 or the element.
int access_bytes(long long row_bytes, int element, const void* a, const void* b, const void* c) {
  for (int vb = 16; vb > element; vb /= 4)
    if (row_bytes % vb == 0 && aligned_to(a, vb) && aligned_to(b, vb) && aligned_to(c, vb))
      return vb;
  return element;
}
// The search for rows that no place names: in front of the kernel that is launched next, or beside it.
template <int VB>
int search_unnamed(Unnamed* u, const int* places, long long total, unsigned char* rows,
                   long long row_bytes, float* scales, cudaStream_t st) {
  *u = Unnamed();
  if (total <= kFewRows) {
    u->front = 1;
    return BRT_OK;
  }
  u->beside = 1;
  SearchArgs a;
  a.places = places;
  a.rows = rows;
  a.scales = scales;
  a.total = total;
  a.row_bytes = row_bytes;
  a.window = (unsigned)round_up((size_t)((total + kSearchCtas - 1) / kSearchCtas), 32);
  if (a.window > kMostWindow) a.window = kMostWindow;
  unnamed_rows_kernel<VB><<<kSearchCtas, kSearchThreads, a.window / 8, st>>>(a);
  note_launch();
  BRT_LAUNCH_CHECK("unnamed_rows_kernel");
  return BRT_OK;
}
// Launches a kernel that moves rows.
template <typename Args>
int launch_rows(void (*kernel)(Args), const char* name, unsigned grid, unsigned threads,
                const Args& a, cudaStream_t st) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(threads);
  config.stream = st;
  config.attrs = &early;
  config.numAttrs = a.unnamed.beside;  // beside the search, else after everything before
  BRT_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, a));
  note_launch();
  BRT_LAUNCH_CHECK(name);
  return BRT_OK;
}
// Few items: one warp per CTA spreads them over the SMs.
struct Shape {
  unsigned grid = 0, threads = 0;
  explicit Shape(long long items, int more = 0) {
    const long long most = (long long)sm_count() * kManyItems;
    threads = items >= most ? kThreads : items * 4 >= most ? 128 : 32;
    const long long ctas = (items + threads / 32 - 1) / (threads / 32) + more;
    grid = ctas <= 0x7fffffffLL ? (unsigned)ctas : 0;
  }
};
template <int VB, int U>
long long pieces_of(long long row_bytes) {
  return (row_bytes + 32 * VB * U - 1) / (32 * VB * U);
}
bool many(long long items, int per_sm) { return items >= (long long)sm_count() * per_sm; }
// Accesses per lane and item: 3 where that leaves fewer lanes without work at a row's end.
template <int VB>
bool by_threes(long long row_bytes) {
  const long long accesses = (row_bytes + 32 * VB - 1) / (32 * VB);
  return VB == 16 && (accesses + 2) / 3 * 3 < (accesses + 3) / 4 * 4;
}

template <int DT, int VB, int U>
int launch_unsort(UnsortArgs a, long long cells, int gates, cudaStream_t st) {
  a.pieces = (int)pieces_of<VB, U>(a.row_bytes);
  a.items = cells * a.pieces;
  const Shape s(a.items);
  BRT_REQUIRE(s.grid > 0, "too many cells for one launch");
  const KernelTimer timer("unsort_cells_kernel", st);
  if (gates == 0) unsort_cells_kernel<DT, VB, U, 0><<<s.grid, s.threads, 0, st>>>(a);
  else if (gates == 1) unsort_cells_kernel<DT, VB, U, 1><<<s.grid, s.threads, 0, st>>>(a);
  else unsort_cells_kernel<DT, VB, U, 2><<<s.grid, s.threads, 0, st>>>(a);
  note_launch();
  BRT_LAUNCH_CHECK("unsort_cells_kernel");
  return BRT_OK;
}
template <int DT, int VB>
int launch_unsort(const UnsortArgs& a, long long cells, int gates, cudaStream_t st) {
  if (many(cells * pieces_of<VB, kUnroll<VB>>(a.row_bytes), kManyItems)) {
    if (by_threes<VB>(a.row_bytes))
      return launch_unsort<DT, VB, VB == 16 ? 3 : 1>(a, cells, gates, st);
    return launch_unsort<DT, VB, kUnroll<VB>>(a, cells, gates, st);
  }
  return launch_unsort<DT, VB, 1>(a, cells, gates, st);
}
template <int DT>
int launch_unsort(const UnsortArgs& a, long long cells, int vb, int gates, cudaStream_t st) {
  if (vb == 16) return launch_unsort<DT, 16>(a, cells, gates, st);
  if constexpr (DT != BRT_F32)
    if (vb == 2) return launch_unsort<DT, 2>(a, cells, gates, st);
  return launch_unsort<DT, 4>(a, cells, gates, st);
}

// Items of whole cells read each cell once; where they are too few to fill the GPU an item is
// one pick of a short piece.
template <int VB>
int launch_sort(SortArgs a, long long cells, cudaStream_t st) {
  constexpr int kLong = kUnroll<VB>;
  const bool whole = many(cells * pieces_of<VB, kLong>(a.row_bytes), kManyCells);
  a.pieces = (int)(whole ? pieces_of<VB, kLong>(a.row_bytes) : pieces_of<VB, 1>(a.row_bytes));
  a.group = whole ? a.picks : 1;
  a.groups = whole ? 1 : a.picks;
  a.items = cells * a.pieces * a.groups;
  const KernelTimer timer("sort_cells_kernel", st);
  BRT_REQUIRE(Shape(a.items, 1).grid > 0, "too many cells for one launch");
  const int rc = search_unnamed<VB>(&a.unnamed, a.places, a.total_rows, a.rows, a.row_bytes,
                                    nullptr, st);
  if (rc != BRT_OK) return rc;
  const Shape s(a.items, a.unnamed.front);
  return launch_rows(whole ? sort_cells_kernel<VB, kLong> : sort_cells_kernel<VB, 1>,
                     "sort_cells_kernel", s.grid, s.threads, a, st);
}

template <int DT, int VB>
int launch_back(BackArgs a, int gates, cudaStream_t st) {
  const KernelTimer timer("unsort_backward_kernel", st);
  const long long grid = (a.routes + kCtaWarps - 1) / kCtaWarps + 1;
  BRT_REQUIRE(grid <= 0x7fffffffLL, "too many cells for one launch");
  if (a.row_grads != nullptr) {
    const int rc = search_unnamed<VB>(&a.unnamed, a.places, a.total_rows, a.row_grads,
                                      a.row_bytes, nullptr, st);
    if (rc != BRT_OK) return rc;
  }
  return launch_rows(gates == 1 ? unsort_backward_kernel<DT, VB, 1>
                                : unsort_backward_kernel<DT, VB, 2>,
                     "unsort_backward_kernel", (unsigned)grid - 1 + a.unnamed.front, kThreads, a,
                     st);
}
template <int DT>
int launch_back(const BackArgs& a, int vb, int gates, cudaStream_t st) {
  if (vb == 16) return launch_back<DT, 16>(a, gates, st);
  if constexpr (DT != BRT_F32)
    if (vb == 2) return launch_back<DT, 2>(a, gates, st);
  return launch_back<DT, 4>(a, gates, st);
}

template <int DT, bool kPlaced>
int launch_codes(SortArgs a, long long cells, cudaStream_t st) {
  const bool threes = by_threes<16>(a.width * 2);  // 256 values per access, whatever their type
  const long long length = 256 * (threes ? 3 : kCodeUnroll);
  const bool whole = many(cells * ((a.width + length - 1) / length), kManyCells);
  a.pieces = (int)(whole ? (a.width + length - 1) / length : (a.width + 255) / 256);
  a.group = whole ? a.picks : 1;
  a.groups = whole ? 1 : a.picks;
  a.items = cells * a.pieces * a.groups;
  const KernelTimer timer("sort_codes_kernel", st);
  BRT_REQUIRE(Shape(a.items, 1).grid > 0, "too many rows for one launch");
  if (kPlaced) {
    const int rc = search_unnamed<16>(&a.unnamed, a.places, a.total_rows, a.rows, a.width,
                                      a.scales, st);
    if (rc != BRT_OK) return rc;
  }
  const Shape s(a.items, a.unnamed.front);
  return launch_rows(whole && threes ? sort_codes_kernel<DT, 3, kPlaced>
                     : whole         ? sort_codes_kernel<DT, kCodeUnroll, kPlaced>
                                     : sort_codes_kernel<DT, 1, kPlaced>,
                     "sort_codes_kernel", s.grid, s.threads, a, st);
}
template <bool kPlaced>
int launch_codes(const SortArgs& a, long long cells, int dtype, cudaStream_t st) {
  if (dtype == BRT_F32) return launch_codes<BRT_F32, kPlaced>(a, cells, st);
  if (dtype == BRT_F16) return launch_codes<BRT_F16, kPlaced>(a, cells, st);
  return launch_codes<BRT_BF16, kPlaced>(a, cells, st);
}

bool known_dtype(int dtype) { return dtype == BRT_F32 || dtype == BRT_F16 || dtype == BRT_BF16; }

int check_shape(int64_t cell_num, int pick_num, int64_t cell_size, int dtype) {
  BRT_REQUIRE(known_dtype(dtype), "unknown dtype %d", dtype);
  BRT_REQUIRE(cell_num >= 0 && pick_num >= 1 && cell_size >= 1, "bad shape: %lld cells, %d picks, "
              "%lld elements per cell", (long long)cell_num, pick_num, (long long)cell_size);
  BRT_REQUIRE(cell_num <= 0x7fffffffLL / pick_num, "the rows are counted in 32 bits");
  BRT_REQUIRE(cell_size <= (1LL << 34), "cell_size %lld", (long long)cell_size);
  return BRT_OK;
}

}  // namespace
}  // namespace brt_b200

using namespace brt_b200;

extern "C" {

BRT_API int brt_sort_cells(const void* cells, const int32_t* places, void* rows, int64_t cell_num,
                           int pick_num, int64_t cell_size, int dtype, void* stream) {
  clear_error();
  const int rc = check_shape(cell_num, pick_num, cell_size, dtype);
  if (rc != BRT_OK) return rc;
  if (cell_num == 0) return BRT_OK;
  BRT_REQUIRE(cells != nullptr && places != nullptr && rows != nullptr, "null pointer argument");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SortArgs a = {};
  a.cells = static_cast<const unsigned char*>(cells);
  a.rows = static_cast<unsigned char*>(rows);
  a.places = places;
  a.row_bytes = cell_size * dtype_size(dtype);
  a.total_rows = cell_num * pick_num;
  a.picks = pick_num;
  const int vb = access_bytes(a.row_bytes, dtype_size(dtype), cells, rows, nullptr);
  if (vb == 16) return launch_sort<16>(a, cell_num, st);
  if (vb == 4) return launch_sort<4>(a, cell_num, st);
  return launch_sort<2>(a, cell_num, st);
}

BRT_API int brt_sort_cells_fp8(const void* cells, const int32_t* places, void* codes,
                               float* scales, int64_t cell_num, int pick_num, int64_t cell_size,
                               int dtype, void* stream) {
  clear_error();
  const int rc = check_shape(cell_num, pick_num, cell_size, dtype);
  if (rc != BRT_OK) return rc;
  BRT_REQUIRE(cell_size % 16 == 0, "cell_size %lld is no multiple of 16", (long long)cell_size);
  if (cell_num == 0) return BRT_OK;
  BRT_REQUIRE(cells != nullptr && codes != nullptr && scales != nullptr && places != nullptr,
              "null pointer argument");
  BRT_REQUIRE(aligned_to(cells, 16) && aligned_to(codes, 16), "cells and codes must be 16-byte "
              "aligned");
  SortArgs a = {};
  a.cells = static_cast<const unsigned char*>(cells);
  a.rows = static_cast<unsigned char*>(codes);
  a.scales = scales;
  a.places = places;
  a.width = cell_size;
  a.total_rows = cell_num * pick_num;
  a.picks = pick_num;
  return launch_codes<true>(a, cell_num, dtype, static_cast<cudaStream_t>(stream));
}

BRT_API int brt_quantize_rows(const void* rows, void* codes, float* scales, int64_t row_num,
                              int64_t width, int dtype, void* stream) {
  clear_error();
  const int rc = check_shape(row_num, 1, width, dtype);
  if (rc != BRT_OK) return rc;
  BRT_REQUIRE(width % 16 == 0, "width %lld is no multiple of 16", (long long)width);
  if (row_num == 0) return BRT_OK;
  BRT_REQUIRE(rows != nullptr && codes != nullptr && scales != nullptr, "null pointer argument");
  BRT_REQUIRE(aligned_to(rows, 16) && aligned_to(codes, 16), "rows and codes must be 16-byte "
              "aligned");
  SortArgs a = {};
  a.cells = static_cast<const unsigned char*>(rows);
  a.rows = static_cast<unsigned char*>(codes);
  a.scales = scales;
  a.width = width;
  a.total_rows = row_num;
  a.picks = 1;
  return launch_codes<false>(a, row_num, dtype, static_cast<cudaStream_t>(stream));
}

BRT_API int brt_unsort_cells(const void* rows, const int32_t* places, const void* gates,
                             void* cells, int64_t cell_num, int pick_num, int64_t cell_size,
                             int dtype, int gates_dtype, void* stream) {
  clear_error();
  const int rc = check_shape(cell_num, pick_num, cell_size, dtype);
  if (rc != BRT_OK) return rc;
  BRT_REQUIRE(gates == nullptr || gates_dtype == BRT_F32 || gates_dtype == dtype,
              "gates are fp32 or of the data's type");
  if (cell_num == 0) return BRT_OK;
  BRT_REQUIRE(cells != nullptr && places != nullptr && rows != nullptr, "null pointer argument");
  UnsortArgs a = {};
  a.rows = static_cast<const unsigned char*>(rows);
  a.cells = static_cast<unsigned char*>(cells);
  a.places = places;
  a.gates = gates;
  a.row_bytes = cell_size * dtype_size(dtype);
  a.total_rows = cell_num * pick_num;
  a.picks = pick_num;
  const int vb = access_bytes(a.row_bytes, dtype_size(dtype), cells, rows, nullptr);
  const int kind = gates == nullptr ? 0 : gates_dtype == BRT_F32 ? 1 : 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == BRT_F32) return launch_unsort<BRT_F32>(a, cell_num, vb, kind, st);
  if (dtype == BRT_F16) return launch_unsort<BRT_F16>(a, cell_num, vb, kind, st);
  return launch_unsort<BRT_BF16>(a, cell_num, vb, kind, st);
}

BRT_API int brt_unsort_cells_backward(const void* cell_grads, const void* rows,
                                      const int32_t* places, const void* gates, void* row_grads,
                                      void* gate_grads, int64_t cell_num, int pick_num,
                                      int64_t cell_size, int dtype, int gates_dtype,
                                      void* stream) {
  clear_error();
  const int rc = check_shape(cell_num, pick_num, cell_size, dtype);
  if (rc != BRT_OK) return rc;
  BRT_REQUIRE(gates_dtype == BRT_F32 || gates_dtype == dtype,
              "gates are fp32 or of the data's type");
  if (cell_num == 0 || (row_grads == nullptr && gate_grads == nullptr)) return BRT_OK;
  BRT_REQUIRE(cell_grads != nullptr && places != nullptr && gates != nullptr &&
                  (rows != nullptr || gate_grads == nullptr), "null pointer argument");
  BackArgs a = {};
  a.cell_grads = static_cast<const unsigned char*>(cell_grads);
  a.rows = static_cast<const unsigned char*>(rows);
  a.row_grads = static_cast<unsigned char*>(row_grads);
  a.gate_grads = gate_grads;
  a.places = places;
  a.gates = gates;
  a.row_bytes = cell_size * dtype_size(dtype);
  a.routes = cell_num * pick_num;
  a.total_rows = a.routes;
  a.picks = pick_num;
  const int vb = access_bytes(a.row_bytes, dtype_size(dtype), cell_grads, rows, row_grads);
  const int kind = gates_dtype == BRT_F32 ? 1 : 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == BRT_F32) return launch_back<BRT_F32>(a, vb, kind, st);
  if (dtype == BRT_F16) return launch_back<BRT_F16>(a, vb, kind, st);
  return launch_back<BRT_BF16>(a, vb, kind, st);
}

}  // extern "C"
