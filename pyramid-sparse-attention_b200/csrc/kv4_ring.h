// A ring of barriers that copies are armed on, one after another.  Whoever copies advances it with each barrier that it arms and with no
// other, or counts them, so that it knows at any time which copies may still be in flight.
#pragma once
#ifdef __CUDACC__
#define PSA_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define PSA_HOST_DEVICE inline
#endif

namespace psa {

template <int N>
struct Ring {
  int at;           // the barrier to be armed next, and the parity of the phase that arming it begins
  unsigned phase;
  PSA_HOST_DEVICE void advance() {
    if (++at == N) at = 0, phase ^= 1;
  }
  static PSA_HOST_DEVICE Ring after(int armed) { return {armed % N, (unsigned)(armed / N) & 1u}; }
  // Parity to wait for barrier i with, until all that was armed on it has landed: its last phase - or, where it was never armed, the one
  // before its first, which counts as over.
  PSA_HOST_DEVICE unsigned last(int i) const { return i < at ? phase : phase ^ 1; }
};

}  // namespace psa
