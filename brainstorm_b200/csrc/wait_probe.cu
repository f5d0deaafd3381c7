// The bounded wait of the tensor-core kernels by itself, for tests: whether a warp whose lanes have
// different limits, and of whom some see the barrier complete, still goes on as one.
#include "tensor_core.cuh"

namespace brt_b200 {
namespace {

constexpr unsigned long long kMostNs = 100000000ull;

__global__ void __launch_bounds__(64)
wait_probe_kernel(int* results, unsigned long long first_limit, unsigned long long limit,
                  unsigned long long arrive_after) {
  __shared__ uint64_t s_bar;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) mbar_init(&s_bar, 1);
  __syncthreads();
  if (threadIdx.x >= 32) {
    if (lane == 0) {
      const unsigned long long begin = now_ns();
      while (now_ns() - begin < arrive_after) __nanosleep(1000);
      mbar_arrive(&s_bar);
    }
  } else {
    results[lane] = mbar_wait_warp(&s_bar, 0, lane == 0 ? first_limit : limit);
  }
  __syncthreads();
}

}  // namespace
}  // namespace brt_b200

using namespace brt_b200;

extern "C" {

BRT_API int brt_expert_wait_probe(int32_t* results, uint64_t first_limit_ns, uint64_t limit_ns,
                                  uint64_t arrive_after_ns, void* stream) {
  clear_error();
  BRT_REQUIRE(results != nullptr, "results is null");
  BRT_REQUIRE(first_limit_ns <= kMostNs && limit_ns <= kMostNs && arrive_after_ns <= kMostNs,
              "a limit of more than %llu ns", kMostNs);
  wait_probe_kernel<<<1, 64, 0, static_cast<cudaStream_t>(stream)>>>(results, first_limit_ns,
                                                                    limit_ns, arrive_after_ns);
  note_launch();
  BRT_LAUNCH_CHECK("wait_probe_kernel");
  return BRT_OK;
}

}  // extern "C"
