// Linear attention with waits that give up at once, without a look at their barrier, in chosen warps: what others have under way then lands all the same.
#include <cuda_runtime.h>

#include <cstdint>

__device__ uint32_t gives_up_warps, gives_up_parity;  // a bit a warp; of waits for a phase of this parity
extern "C" int set_gives_up(uint32_t warps, uint32_t parity) {
    const cudaError_t e = cudaMemcpyToSymbol(gives_up_warps, &warps, sizeof(warps));
    return e != cudaSuccess ? e : cudaMemcpyToSymbol(gives_up_parity, &parity, sizeof(parity));
}
#define KVB_CHUNK_PROBES ((gives_up_warps >> (threadIdx.x >> 5) & 1u) != 0u && gives_up_parity == parity ? 0u : kSpinLimit)

#include "kvb_linear.cu"
#include "kvb_linear_chunk.cu"
