// The start of a kernel that allocates tensor memory and lets the next kernel of the stream start early.
#pragma once
#include "ptx.cuh"

namespace dlfb200 {
namespace ptx {

// By one converged warp: the allocation, then - in the same warp, with the tensor memory in hand, as ptx.cuh asks for - the
// leave for the dependents. One call, so that no kernel can have them the other way round.
__device__ __forceinline__ void tmem_alloc_then_dependents(uint32_t smem_dst, uint32_t ncols) {
    tmem_alloc(smem_dst, ncols);
    tmem_relinquish();
    launch_dependents();
}
__device__ __forceinline__ void tmem_alloc_pair_then_dependents(uint32_t smem_dst, uint32_t ncols) {
    tmem_alloc_pair(smem_dst, ncols);
    tmem_relinquish_pair();
    launch_dependents();
}

}  // namespace ptx
}  // namespace dlfb200
