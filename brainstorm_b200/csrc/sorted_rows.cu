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
// output is written exactly once whatever was dropped.  -1, and places outside the buffer, are
// skipped.  Sums run in fp32 in the order of j and are rounded once; a gate of a pick that goes
// nowhere is not looked at.
//
// All are bound by HBM (a few operations per byte).  sort and unsort give a warp 2 KB of a cell:
// a cell is read once for its k copies, and written once.  The backward of unsort
// gives a warp one route, so that its dot product stays in the warp and is summed in one fixed
// order; the k warps of a cell read its gradient from L1 or L2.
#include "block_codes.cuh"

namespace brt_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kCtaWarps = kThreads / 32;
constexpr int kItemsPerWarp = 2;

// VB-byte accesses per lane and item: 2 KB (1 KB of 2-byte accesses) per warp
template <int VB>
constexpr int kUnroll = VB == 16 ? 4 : 16;

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
};

template <int VB>
__global__ void __launch_bounds__(kThreads) sort_cells_kernel(const SortArgs a) {
  using V = typename Chunk<VB>::type;
  constexpr int U = kUnroll<VB>;
  constexpr int kPiece = 32 * VB * U;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long first = (long long)blockIdx.x * (kCtaWarps * kItemsPerWarp) + warp;
#pragma unroll 1
  for (int i = 0; i < kItemsPerWarp; i++) {
    const long long item = first + (long long)i * kCtaWarps;
    if (item >= a.items) return;
    const long long cell = item / a.pieces;
    const long long at = (item - cell * a.pieces) * kPiece + lane * VB;
    const unsigned char* const src = a.cells + cell * a.row_bytes + at;
    V v[U];
#pragma unroll
    for (int u = 0; u < U; u++)
      v[u] = at + u * (32 * VB) < a.row_bytes
                 ? load_stream(reinterpret_cast<const V*>(src + u * (32 * VB)))
                 : zero_chunk<V>();
    const int* const places = a.places + cell * a.picks;
    for (int j = 0; j < a.picks; j++) {
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
}

constexpr int kCodeUnroll = 4;  // 4 x 256 values per warp and item

// kPlaced = false: one row per cell, in the order they come (a plain quantisation).
template <int DT, bool kPlaced>
__global__ void __launch_bounds__(kThreads) sort_codes_kernel(const SortArgs a) {
  using T = typename Elem<DT>::type;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long first = (long long)blockIdx.x * (kCtaWarps * kItemsPerWarp) + warp;
#pragma unroll 1
  for (int i = 0; i < kItemsPerWarp; i++) {
    const long long item = first + (long long)i * kCtaWarps;
    if (item >= a.items) return;
    const long long cell = item / a.pieces;
    const long long at = (item - cell * a.pieces) * (256 * kCodeUnroll) + lane * 8;
    const T* const src = reinterpret_cast<const T*>(a.cells) + cell * a.width + at;
    uint2 code[kCodeUnroll];
    float scale[kCodeUnroll];
#pragma unroll
    for (int u = 0; u < kCodeUnroll; u++) {
      float v[8];
      if (at + u * 256 < a.width) {
        load_eight<DT>(src + u * 256, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = 0.f;
      }
      float amax = max_abs(v);  // of the block: 16 lanes hold its 128 values
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
      amax = fmaxf(amax, kAmaxFloor);
      scale[u] = __fdiv_rn(amax, kCodeMax);
      code[u] = encode_eight(v, __fdiv_rn(kCodeMax, amax));
    }
    const int copies = kPlaced ? a.picks : 1;
    for (int j = 0; j < copies; j++) {
      const int p = kPlaced ? __ldg(a.places + cell * a.picks + j) : 0;
      const long long row = !kPlaced ? cell : p >= 0 ? p : -2LL - p;
      if (row < 0 || row >= a.total_rows) continue;
      unsigned char* const dst = a.rows + row * a.width + at;
#pragma unroll
      for (int u = 0; u < kCodeUnroll; u++) {
        if (at + u * 256 >= a.width) continue;
        *reinterpret_cast<uint2*>(dst + u * 256) = p >= 0 ? code[u] : make_uint2(0u, 0u);
        if ((lane & 15) == 0)
          a.scales[((at + u * 256) / kCodeBlock) * a.total_rows + row] =
              p >= 0 ? scale[u] : __fdiv_rn(kAmaxFloor, kCodeMax);
      }
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

template <int DT, int VB, int kGates>
__global__ void __launch_bounds__(kThreads) unsort_cells_kernel(const UnsortArgs a) {
  using V = typename Chunk<VB>::type;
  using P = Pack<DT, VB>;
  constexpr int U = kUnroll<VB>;
  constexpr int kPiece = 32 * VB * U;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * kCtaWarps + warp;
  if (item >= a.items) return;
  const long long cell = item / a.pieces;
  const long long at = (item - cell * a.pieces) * kPiece + lane * VB;
  const int* const places = a.places + cell * a.picks;
  float sum[U][P::kValues];
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int e = 0; e < P::kValues; e++) sum[u][e] = 0.f;
#pragma unroll 2
  for (int j = 0; j < a.picks; j++) {
    const int p = __ldg(places + j);
    if (p < 0 || p >= a.total_rows) continue;
    const float gate = gate_at<DT, kGates>(a.gates, cell * a.picks + j);
    const unsigned char* const src = a.rows + (long long)p * a.row_bytes + at;
    V raw[U];
#pragma unroll
    for (int u = 0; u < U; u++)
      raw[u] = at + u * (32 * VB) < a.row_bytes
                   ? load_stream(reinterpret_cast<const V*>(src + u * (32 * VB)))
                   : zero_chunk<V>();
#pragma unroll
    for (int u = 0; u < U; u++) {
      float v[P::kValues];
      P::values(raw[u], v);
#pragma unroll
      for (int e = 0; e < P::kValues; e++)
        sum[u][e] = kGates == 0 ? sum[u][e] + v[e] : fmaf(gate, v[e], sum[u][e]);
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
};

template <int DT, int VB, int kGates>
__global__ void __launch_bounds__(kThreads) unsort_backward_kernel(const BackArgs a) {
  using V = typename Chunk<VB>::type;
  using P = Pack<DT, VB>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long route = (long long)blockIdx.x * kCtaWarps + warp;
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
#pragma unroll 4
    for (long long at = lane * VB; at < a.row_bytes; at += 32 * VB) {
      float g[P::kValues], out[P::kValues];
      if (live) {
        P::values(__ldg(reinterpret_cast<const V*>(grad + at)), g);
        if (dots) {
          float r[P::kValues];
          P::values(load_stream(reinterpret_cast<const V*>(a.rows + row * a.row_bytes + at)), r);
#pragma unroll
          for (int e = 0; e < P::kValues; e++) dot = fmaf(g[e], r[e], dot);
        }
      }
      if (a.row_grads != nullptr) {
#pragma unroll
        for (int e = 0; e < P::kValues; e++) out[e] = live ? gate * g[e] : 0.f;
        store_stream(reinterpret_cast<V*>(a.row_grads + row * a.row_bytes + at), P::chunk(out));
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
template <int VB>
int pieces_of(long long row_bytes) {
  return (int)((row_bytes + 32 * VB * kUnroll<VB> - 1) / (32 * VB * kUnroll<VB>));
}
int pieces_of(long long row_bytes, int vb) {
  return vb == 16 ? pieces_of<16>(row_bytes) : vb == 4 ? pieces_of<4>(row_bytes)
                                                       : pieces_of<2>(row_bytes);
}

template <int DT, int VB>
int launch_unsort(const UnsortArgs& a, int gates, cudaStream_t st) {
  const long long grid = (a.items + kCtaWarps - 1) / kCtaWarps;
  BRT_REQUIRE(grid <= 0x7fffffffLL, "too many cells for one launch");
  const KernelTimer timer("unsort_cells_kernel", st);
  if (gates == 0) unsort_cells_kernel<DT, VB, 0><<<(unsigned)grid, kThreads, 0, st>>>(a);
  else if (gates == 1) unsort_cells_kernel<DT, VB, 1><<<(unsigned)grid, kThreads, 0, st>>>(a);
  else unsort_cells_kernel<DT, VB, 2><<<(unsigned)grid, kThreads, 0, st>>>(a);
  note_launch();
  BRT_LAUNCH_CHECK("unsort_cells_kernel");
  return BRT_OK;
}
template <int DT>
int launch_unsort(const UnsortArgs& a, int vb, int gates, cudaStream_t st) {
  if (vb == 16) return launch_unsort<DT, 16>(a, gates, st);
  if constexpr (DT != BRT_F32)
    if (vb == 2) return launch_unsort<DT, 2>(a, gates, st);
  return launch_unsort<DT, 4>(a, gates, st);
}

template <int DT, int VB>
int launch_back(const BackArgs& a, int gates, cudaStream_t st) {
  const long long grid = (a.routes + kCtaWarps - 1) / kCtaWarps;
  BRT_REQUIRE(grid <= 0x7fffffffLL, "too many cells for one launch");
  const KernelTimer timer("unsort_backward_kernel", st);
  if (gates == 1) unsort_backward_kernel<DT, VB, 1><<<(unsigned)grid, kThreads, 0, st>>>(a);
  else unsort_backward_kernel<DT, VB, 2><<<(unsigned)grid, kThreads, 0, st>>>(a);
  note_launch();
  BRT_LAUNCH_CHECK("unsort_backward_kernel");
  return BRT_OK;
}
template <int DT>
int launch_back(const BackArgs& a, int vb, int gates, cudaStream_t st) {
  if (vb == 16) return launch_back<DT, 16>(a, gates, st);
  if constexpr (DT != BRT_F32)
    if (vb == 2) return launch_back<DT, 2>(a, gates, st);
  return launch_back<DT, 4>(a, gates, st);
}

template <bool kPlaced>
int launch_codes(SortArgs a, long long cells, int dtype, cudaStream_t st) {
  a.pieces = (int)((a.width + 256 * kCodeUnroll - 1) / (256 * kCodeUnroll));
  a.items = cells * a.pieces;
  const long long per = kCtaWarps * kItemsPerWarp;
  const long long grid = (a.items + per - 1) / per;
  BRT_REQUIRE(grid <= 0x7fffffffLL, "too many rows for one launch");
  const KernelTimer timer("sort_codes_kernel", st);
  const unsigned g = (unsigned)grid;
  if (dtype == BRT_F32) sort_codes_kernel<BRT_F32, kPlaced><<<g, kThreads, 0, st>>>(a);
  else if (dtype == BRT_F16) sort_codes_kernel<BRT_F16, kPlaced><<<g, kThreads, 0, st>>>(a);
  else sort_codes_kernel<BRT_BF16, kPlaced><<<g, kThreads, 0, st>>>(a);
  note_launch();
  BRT_LAUNCH_CHECK("sort_codes_kernel");
  return BRT_OK;
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
  a.pieces = pieces_of(a.row_bytes, vb);
  a.items = cell_num * a.pieces;
  const long long per = kCtaWarps * kItemsPerWarp;
  const long long grid = (a.items + per - 1) / per;
  BRT_REQUIRE(grid <= 0x7fffffffLL, "too many cells for one launch");
  const KernelTimer timer("sort_cells_kernel", st);
  if (vb == 16) sort_cells_kernel<16><<<(unsigned)grid, kThreads, 0, st>>>(a);
  else if (vb == 4) sort_cells_kernel<4><<<(unsigned)grid, kThreads, 0, st>>>(a);
  else sort_cells_kernel<2><<<(unsigned)grid, kThreads, 0, st>>>(a);
  note_launch();
  BRT_LAUNCH_CHECK("sort_cells_kernel");
  return BRT_OK;
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
  a.pieces = pieces_of(a.row_bytes, vb);
  a.items = cell_num * a.pieces;
  const int kind = gates == nullptr ? 0 : gates_dtype == BRT_F32 ? 1 : 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == BRT_F32) return launch_unsort<BRT_F32>(a, vb, kind, st);
  if (dtype == BRT_F16) return launch_unsort<BRT_F16>(a, vb, kind, st);
  return launch_unsort<BRT_BF16>(a, vb, kind, st);
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
