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

template <int DT, bool kTransposed>
__global__ void __launch_bounds__(kThreads)
weight_codes_kernel(const typename Elem<DT>::type* __restrict__ weights,
                    unsigned char* __restrict__ codes, float* __restrict__ scales, int N, int K) {
  __shared__ float s_max[kThreads / 32];
  __shared__ uint32_t s_turn[kTransposed ? kCodeBlock * (kCodeBlock / 4 + 1) : 1];
  const int tid = threadIdx.x;
  const int k0 = blockIdx.x * kCodeBlock, n0 = blockIdx.y * kCodeBlock;
  const long long expert = blockIdx.z;
  const auto* const w = weights + expert * N * (long long)K;
  const int my_k = (tid & 15) * 8;  // 16 threads hold a row of the block
  const int my_n = tid >> 4;
  float v[kParts][8];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < kParts; i++) {
    const int n = n0 + my_n + i * (kThreads / 16);
    if (n < N && k0 + my_k < K) {
      load_eight<DT>(w + (long long)n * K + k0 + my_k, v[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = 0.f;
    }
    amax = fmaxf(amax, max_abs(v[i]));
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
  if ((tid & 31) == 0) s_max[tid >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; i++) amax = fmaxf(amax, s_max[i]);
  amax = fmaxf(amax, kAmaxFloor);
  const float inverse = __fdiv_rn(kCodeMax, amax);
  if (tid == 0) {
    const long long block = kTransposed
        ? (expert * gridDim.x + blockIdx.x) * gridDim.y + blockIdx.y
        : (expert * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
    scales[block] = __fdiv_rn(amax, kCodeMax);
  }
  unsigned char* const out = codes + expert * N * (long long)K;
  if constexpr (!kTransposed) {
#pragma unroll
    for (int i = 0; i < kParts; i++) {
      const int n = n0 + my_n + i * (kThreads / 16);
      if (n < N && k0 + my_k < K)
        *reinterpret_cast<uint2*>(out + (long long)n * K + k0 + my_k) =
            encode_eight(v[i], inverse);
    }
  } else {
    // row k of s_turn: the codes of 128 neighbouring n, four to a word, one word of padding
    unsigned char* const turn = reinterpret_cast<unsigned char*>(s_turn);
    constexpr int kPitch = kCodeBlock + 4;
#pragma unroll
    for (int i = 0; i < kParts; i++) {
      const uint2 c = encode_eight(v[i], inverse);
      const int n = my_n + i * (kThreads / 16);
#pragma unroll
      for (int e = 0; e < 8; e++)
        turn[(my_k + e) * kPitch + n] = (unsigned char)((e < 4 ? c.x : c.y) >> (8 * (e & 3)));
    }
    __syncthreads();
    for (int i = tid; i < kCodeBlock * kCodeBlock / 16; i += kThreads) {
      const int k = i >> 3, n = (i & 7) * 16;
      if (k0 + k < K && n0 + n < N) {
        const uint32_t* const from = s_turn + k * (kPitch / 4) + n / 4;
        *reinterpret_cast<uint4*>(out + (long long)(k0 + k) * N + n0 + n) =
            make_uint4(from[0], from[1], from[2], from[3]);
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
