// Which half of a finishing warp's 4 KB a result leaves through while earlier ones are still being copied out.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define TB_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define TB_HOST_DEVICE inline
#endif

namespace tb {

// A warp's shared memory is two pieces (bits 1 and 2); a copy out of it reads one of them or both, and a block may
// pass from a product whose results take both to one whose results take one.  So what the newest copy reads is
// kept, and a piece that is about to be written is compared with it.
struct OutPieces {
  uint32_t read; // by the newest copy; 0: no copy is under way

  // A piece that the newest copy leaves alone, where there is one.
  TB_HOST_DEVICE uint32_t other() const { return read & 1 ? 2 : 1; }
  // `pieces` are about to be written and then copied out: how many of the newest copies may still be under way
  // meanwhile.  (The one before the newest has been waited for here, in the call before this one.)
  TB_HOST_DEVICE uint32_t claim(uint32_t pieces) {
    const uint32_t may = (read & pieces) == 0;
    read = pieces;
    return may;
  }
};

} // namespace tb
