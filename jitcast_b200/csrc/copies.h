// Which barrier phases the copies of a ring of stages still complete (host and device).
#pragma once

#ifdef __CUDACC__
#define JC_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define JC_HOST_DEVICE inline
#endif

namespace jc {

// Copy i of `issued` went to stage i % stages and completes phase i / stages of that stage's barrier. A stage is filled again
// only after its last copy was consumed, so what may be in flight is the last copy of each stage, and waiting for its phase's
// parity is exact: wait(stage, parity). Stages that no copy went to are not waited for.
template <typename Wait>
JC_HOST_DEVICE void for_last_copies(int issued, int stages, Wait wait) {
  for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
    wait(i % stages, static_cast<unsigned>(i / stages) & 1u);
}

}  // namespace jc
