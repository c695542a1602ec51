// The bounded waits of the attention kernels by themselves: warps that wait for a barrier which a thread completes after
// a while, or which nobody completes. Built and driven by test_bounded_waits.py.
#include <cuda_runtime.h>

#include "mup_attn_common.cuh"

namespace {

struct Probe {
  uint32_t* outcome;   // [128]: what each lane of warps 0 to 3 got
  uint64_t* elapsed;   // [2]: of the waits, of a drain
  uint32_t* status;
  uint64_t limit_ns, others_limit_ns;  // of warp 0, of warps 1 to 3
  uint64_t delay_ns;   // until the barrier is completed
  int completes;       // or never
  int drains;          // then drains the barrier
};

__global__ void __launch_bounds__(160) probe_kernel(Probe p) {
  __shared__ __align__(8) uint64_t barrier;
  __shared__ uint32_t abort_word;
  const uint32_t bar = mup::smem_u32(&barrier);
  const int warp = threadIdx.x / 32;
  if (threadIdx.x == 0) {
    abort_word = 0u;
    mup::mbar_init(bar, 1);
    mup::fence_mbar_init();
  }
  __syncthreads();
  const uint64_t start = mup::globaltimer_ns();
  if (warp < 4) {
    const mup::WaitControl ctl{&abort_word, p.status, warp == 0 ? p.limit_ns : p.others_limit_ns};
    p.outcome[threadIdx.x] = ctl.wait(bar, 0, MUP_ST_MMA_FULL_TIMEOUT);
  } else if (threadIdx.x == 128 && p.completes) {
    while (mup::globaltimer_ns() - start < p.delay_ns) {
    }
    mup::mbar_arrive(bar);
  }
  __syncthreads();
  if (threadIdx.x == 0) p.elapsed[0] = mup::globaltimer_ns() - start;
  if (p.drains && warp == 0) {
    mup::drain_barrier(bar, 0);
    if (threadIdx.x == 0) p.elapsed[1] = mup::globaltimer_ns() - start - p.elapsed[0];
  }
}

// Products without anybody who waits for them, then the drain: their sums have to be there behind it.
__global__ void __launch_bounds__(128) products_kernel(float* sums, int repeats) {
  extern __shared__ __align__(1024) uint8_t tiles[];  // two tiles of 128 rows of 64, all ones: any order of them is the same
  __shared__ __align__(8) uint64_t barrier;
  __shared__ uint32_t tmem_slot;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t bar = mup::smem_u32(&barrier);
  for (int i = threadIdx.x; i < 2 * mup::kPanelBytes / 4; i += 128) reinterpret_cast<uint32_t*>(tiles)[i] = 0x3f803f80u;
  mup::fence_proxy_async_smem();
  if (threadIdx.x == 0) {
    mup::mbar_init(bar, 1);
    mup::fence_mbar_init();
  }
  if (warp == 1) {
    mup::tmem_alloc<1>(mup::smem_u32(&tmem_slot), 128);
    mup::tmem_relinquish<1>();
  }
  mup::tc_fence_before_sync();
  __syncthreads();
  mup::tc_fence_after_sync();
  const uint32_t tmem = tmem_slot, base = mup::smem_u32(tiles);
  if (warp == 0) {
    const bool leader = mup::elect_one_sync();
    for (int i = 0; i < repeats; ++i)
      if (leader) mup::umma_rows_by_rows<64>(tmem, base, base + mup::kPanelBytes);
    __syncwarp();
    mup::drain_products(bar);
  }
  mup::tc_fence_before_sync();
  __syncthreads();
  mup::tc_fence_after_sync();
  for (int b = 0; b < 4; ++b) {
    uint32_t v[32];
    mup::tmem_ld_32x32(tmem + (static_cast<uint32_t>(warp * 32) << 16) + b * 32, v);
    mup::tmem_ld_wait();
    for (int x = 0; x < 32; ++x) sums[(warp * 32 + lane) * 128 + b * 32 + x] = __uint_as_float(v[x]);
  }
  mup::tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    mup::tc_fence_after_sync();
    mup::tmem_dealloc<1>(tmem, 128);
  }
}

}  // namespace

// `sums`: [128, 128].
extern "C" int products_probe(float* sums, int repeats) {
  if (repeats < 1 || repeats > 1000) return -1;
  products_kernel<<<1, 128, 2 * mup::kPanelBytes>>>(sums, repeats);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  return static_cast<int>(e);
}

extern "C" int bounded_wait_probe(uint32_t* outcome, uint64_t* elapsed, uint32_t* status, uint64_t limit_ns,
                                  uint64_t others_limit_ns, uint64_t delay_ns, int completes, int drains) {
  if (limit_ns > 2000000000ull || delay_ns > 2000000000ull) return -1;
  probe_kernel<<<1, 160>>>({outcome, elapsed, status, limit_ns, others_limit_ns, delay_ns, completes, drains});
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  return static_cast<int>(e);
}
