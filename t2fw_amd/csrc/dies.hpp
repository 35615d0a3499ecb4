// Which of a grid's pieces of work a workgroup has.  The hardware deals workgroups out to the eight dies in turn, each with a cache of its own:
// runs of neighbouring pieces go to one die, so that the lines that neighbours share are fetched and written once.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace t2fw {

template <uint32_t NEAR> __device__ __forceinline__ uint32_t piece_of_work() {
    constexpr uint32_t DIES = 8, ROUND = DIES * NEAR;
    const uint32_t n = blockIdx.x;
    if (n >= gridDim.x / ROUND * ROUND) return n;        // (the last ones as they come)
    const uint32_t in = n % ROUND;
    return n - in + in % DIES * NEAR + in / DIES;
}

}  // namespace t2fw
