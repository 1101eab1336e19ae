// Where the prompt kernel's search for an item's sequence stands.  Host and device, no CUDA types.
#pragma once
#ifdef __CUDACC__
#define QMTP_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define QMTP_HOST_DEVICE inline
#endif

namespace qmtp {

// Sequences [0, seq) hold `before` row tiles.  The search goes on from here for a later tile and starts over for one that
// lies before: a block takes its own item and then those of blocks that have not started, in whichever order it is given
// them (as a rule rising, so that few searches start over).
struct ItemCursor {
  int seq = 0;
  long long before = 0;
  QMTP_HOST_DEVICE void seek(long long tile) {
    if (tile < before) {
      seq = 0;
      before = 0;
    }
  }
  // Past the next `n` sequences, which hold `tiles` row tiles.
  QMTP_HOST_DEVICE void pass(int n, long long tiles) {
    seq += n;
    before += tiles;
  }
};

}  // namespace qmtp
