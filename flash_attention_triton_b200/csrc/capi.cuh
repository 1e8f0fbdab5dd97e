// What the files with C entry points share.
#pragma once
#include <cstdint>

#include "common.cuh"

namespace fa2 {

// Status word, work counter and SM count of the current device, which must be of compute capability 10.x; binds its
// primary context to the calling thread.  Returns a code of fa2_b200.h or a cudaError_t.
int launch_context(LaunchCtx* ctx);

inline bool aligned_to(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace fa2
