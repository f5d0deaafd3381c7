// Expert weights as 8-bit codes with a scale for each block of 128 x 128 (block_codes.cuh).
//
//   weights [E, N, K] -> codes [E, N, K] and scales [E, ceil(N / 128), ceil(K / 128)], or, for the
//   product that takes the gradient of the output back to the rows, transposed: codes [E, K, N]
//   and scales [E, ceil(K / 128), ceil(N / 128)].
//
// Bound by HBM: every weight is read once and its code written once.  A CTA holds one block in
// registers (8 x 8 neighbouring values per thread), so the maximum needs no second read; codes
// are turned in 16 KB of shared memory for the transposed form.
#include "block_codes.cuh"

namespace brt_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kParts = kCodeBlock * kCodeBlock / 8 / kThreads;  // groups of 8 values per thread
constexpr int kPitch = kCodeBlock / 4 + 1;                       // words of a turned row

template <int DT, bool kTransposed>
__global__ void __launch_bounds__(kThreads)
weight_codes_kernel(const typename Elem<DT>::type* __restrict__ weights,
                    unsigned char* __restrict__ codes, float* __restrict__ scales, int N, int K) {
  __shared__ float s_max[kThreads / 32];
  __shared__ uint32_t s_turn[kTransposed ? kCodeBlock * kPitch : 1];
  const int tid = threadIdx.x;
  const int k0 = blockIdx.x * kCodeBlock, n0 = blockIdx.y * kCodeBlock;
  const long long expert = blockIdx.z;
  const auto* const w = weights + expert * N * (long long)K;
  const int my_k = (tid & 15) * 8;       // 16 threads hold a row of the block,
  const int my_n = (tid >> 4) * kParts;  // each of them in kParts rows
  Eight<DT> v[kParts];
#pragma unroll
  for (int i = 0; i < kParts; i++) {
    const int n = n0 + my_n + i;
    if (n < N && k0 + my_k < K) v[i].load(w + (long long)n * K + k0 + my_k);
    else v[i].clear();
  }
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < kParts; i++) amax = fmaxf(amax, v[i].max_abs());
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
  if ((tid & 31) == 0) s_max[tid >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; i++) amax = fmaxf(amax, s_max[i]);
  amax = fmaxf(amax, kAmaxFloor);
  const float scale = __fdiv_rn(amax, kCodeMax);
  const float inverse = __fdiv_rn(kCodeMax, amax);
  if (tid == 0) {
    const long long block = kTransposed
        ? (expert * gridDim.x + blockIdx.x) * gridDim.y + blockIdx.y
        : (expert * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
    scales[block] = scale;
  }
  unsigned char* const out = codes + expert * N * (long long)K;
  if constexpr (!kTransposed) {
#pragma unroll
    for (int i = 0; i < kParts; i++) {
      const int n = n0 + my_n + i;
      if (n < N && k0 + my_k < K)
        *reinterpret_cast<uint2*>(out + (long long)n * K + k0 + my_k) = v[i].encode(scale, inverse);
    }
  } else {
    // Row k of s_turn: the codes of 128 neighbouring n, four to a word.  A thread makes words of
    // four of its rows; their place in a row is exchanged by k / 32, so that the threads of a
    // warp meet in a bank by twos.
#pragma unroll
    for (int q = 0; q < kParts / 4; q++) {
      uint2 c[4];
#pragma unroll
      for (int i = 0; i < 4; i++) c[i] = v[q * 4 + i].encode(scale, inverse);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const uint32_t pick = (uint32_t)(e & 3) | (uint32_t)(4 + (e & 3)) << 4;
        const uint32_t lo = __byte_perm(e < 4 ? c[0].x : c[0].y, e < 4 ? c[1].x : c[1].y, pick);
        const uint32_t hi = __byte_perm(e < 4 ? c[2].x : c[2].y, e < 4 ? c[3].x : c[3].y, pick);
        const int k = my_k + e;
        s_turn[k * kPitch + ((my_n / 4 + q) ^ (k >> 5))] = __byte_perm(lo, hi, 0x5410);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = tid; i < kCodeBlock * kCodeBlock / 16; i += kThreads) {
      const int k = i >> 3, n = (i & 7) * 16;
      if (k0 + k < K && n0 + n < N) {
        const uint32_t* const from = s_turn + k * kPitch;
        const int at = n / 4, x = k >> 5;
        *reinterpret_cast<uint4*>(out + (long long)(k0 + k) * N + n0 + n) =
            make_uint4(from[at ^ x], from[(at + 1) ^ x], from[(at + 2) ^ x], from[(at + 3) ^ x]);
      }
    }
  }
}

template <int DT>
void launch(const void* weights, void* codes, float* scales, int paths, int N, int K,
            bool transposed, cudaStream_t st) {
  const dim3 grid((K + kCodeBlock - 1) / kCodeBlock, (N + kCodeBlock - 1) / kCodeBlock, paths);
  const auto* w = static_cast<const typename Elem<DT>::type*>(weights);
  auto* c = static_cast<unsigned char*>(codes);
  if (transposed) weight_codes_kernel<DT, true><<<grid, kThreads, 0, st>>>(w, c, scales, N, K);
  else weight_codes_kernel<DT, false><<<grid, kThreads, 0, st>>>(w, c, scales, N, K);
}

}  // namespace
}  // namespace brt_b200

using namespace brt_b200;

extern "C" {

BRT_API int brt_quantize_expert_weights(const void* weights, void* codes, float* scales,
                                        int path_num, int64_t in_features, int64_t out_features,
                                        int transposed, int dtype, void* stream) {
  clear_error();
  BRT_REQUIRE(dtype == BRT_F32 || dtype == BRT_F16 || dtype == BRT_BF16, "unknown dtype %d", dtype);
  BRT_REQUIRE(path_num >= 0 && path_num <= 65535, "path_num %d outside [0, 65535]", path_num);
  BRT_REQUIRE(in_features > 0 && out_features > 0 && in_features % 16 == 0 &&
                  out_features % 16 == 0 && in_features < (1LL << 31) - 128 &&
                  out_features <= 65535LL * 128,
              "in_features and out_features must be positive multiples of 16 (got %lld, %lld)",
              (long long)in_features, (long long)out_features);
  if (path_num == 0) return BRT_OK;
  BRT_REQUIRE(weights != nullptr && codes != nullptr && scales != nullptr,
              "null pointer argument");
  BRT_REQUIRE(aligned_to(weights, 16) && aligned_to(codes, 16), "weights and codes must be "
              "16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int N = (int)out_features, K = (int)in_features;
  const KernelTimer timer("weight_codes_kernel", st);
  if (dtype == BRT_F32) launch<BRT_F32>(weights, codes, scales, path_num, N, K, transposed, st);
  else if (dtype == BRT_F16) launch<BRT_F16>(weights, codes, scales, path_num, N, K, transposed, st);
  else launch<BRT_BF16>(weights, codes, scales, path_num, N, K, transposed, st);
  note_launch();
  BRT_LAUNCH_CHECK("weight_codes_kernel");
  return BRT_OK;
}

}  // extern "C"
