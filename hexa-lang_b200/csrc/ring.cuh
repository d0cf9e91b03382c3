// ring.cuh — a ring of copies in flight, counted: copy n fills slot
// n % kSlots, and its wait has parity (n / kSlots) & 1.
#pragma once
#ifdef __CUDACC__
#define RING_FN __host__ __device__ __forceinline__
#else
#define RING_FN inline
#endif

// After a wait has run out: waits once more for every copy that is not known
// to have landed, the one whose wait ran out (n_out) first. wait(slot, parity)
// is bounded, so this is what can be done before a CTA exits, not a guarantee.
template <int kSlots, typename Wait>
RING_FN void ring_drain(int n_out, int n_in, Wait wait) {
    for (int n = n_out; n < n_in; ++n) wait(n % kSlots, (n / kSlots) & 1);
}
