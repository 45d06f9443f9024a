// Device code of every load into LDS, each with a descriptor whose words come out of vector registers right before it
// (tests/test_lds_dma.py reads the assembly; nothing runs).
#include "tree_attention.cuh"

namespace tv {

__global__ void lds_dma_check(const uint32_t* words, const unsigned char* rows, uint32_t* out) {
  __shared__ __attribute__((aligned(16))) unsigned char smem[4096];
  const uint32_t base = sgpr((uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem);
  const uint32_t* w = words + threadIdx.x;
  const u32x4 a = u32x4{sgpr(w[0]), sgpr(w[64]), sgpr(w[128]), sgpr(w[192])};
  load_lds16(a, base, threadIdx.x * 16);
  const u32x4 b = u32x4{sgpr(w[256]), sgpr(w[320]), sgpr(w[384]), sgpr(w[448])};
  load_lds16_nt(b, sgpr(base + 1024), threadIdx.x * 16);
  load_lds16_at(rows + threadIdx.x * 16, sgpr(base + 2048));
  wait_vmcnt<0>();
  __syncthreads();
  out[threadIdx.x] = reinterpret_cast<const uint32_t*>(smem)[threadIdx.x];
}

}  // namespace tv
