// Sequences that go on from a kept state: packed rows, state slots, and the scan's step sizes, as the launchers for prompts and single
// tokens take them (include/mp_kernels.h, "sequences that go on from a kept state").
#pragma once

#include "mp_async.cuh"

// Sequence i has the rows starts[i] .. starts[i + 1] of the packed buffers and row slots[i] of the state buffer; it goes on from that state
// where resume[i] is not zero.  The three arrays lie on the device: nothing about them is known when a launch is made, so every use is clamped
// to the buffers that the launch names.
struct Sequences {
  const int* starts;
  const int* slots;    // NULL: slot i
  const int* resume;   // NULL: none does
  int nseq;
  long long rows, nslots;
};

__device__ __forceinline__ long long seq_first(const Sequences& q, int i) {
  const long long v = q.starts[i];
  return v < 0 ? 0 : v > q.rows ? q.rows : v;
}
// The slot of sequence (or token row) i, -1 where it has none: such a sequence is left alone.
__device__ __forceinline__ long long seq_slot(const int* slots, long long nslots, long long i) {
  const long long v = slots == nullptr ? i : slots[i];
  return v >= 0 && v < nslots ? v : -1;
}
__device__ __forceinline__ bool seq_resumes(const Sequences& q, int i) { return q.resume != nullptr && q.resume[i] != 0; }

// The last i in [0, n] with key(i) <= v, -1 where there is none; key does not fall.  By a whole warp, 32 places at a time: a batch of up to a
// thousand sequences takes two rounds of loads instead of ten.
template <typename Key>
__device__ __forceinline__ int warp_last_not_above(int n, long long v, Key key) {
  const int lane = threadIdx.x & 31;
  int lo = 0, count = n + 1;      // the answer is below lo + count
  while (true) {
    const int step = (count + 31) / 32;
    const int at = lo + lane * step;
    const unsigned m = __ballot_sync(0xffffffffu, lane * step < count && key(at) <= v);
    if (m == 0) return lo - 1;    // only in the first round: later ones begin at a place that is not above
    const int k = 31 - __clz(m);
    if (step == 1) return lo + k;
    lo += k * step;
    count = min(step, count - k * step);
  }
}

template <typename A> __device__ __forceinline__ A seq_exp(A v);
template <> __device__ __forceinline__ float seq_exp<float>(float v) { return expf(v); }
template <> __device__ __forceinline__ double seq_exp<double>(double v) { return exp(v); }
// softplus; where it is the identity to the last bit, it is taken for it
__device__ __forceinline__ float seq_softplus(float v) { return v > 20.f ? v : log1pf(expf(v)); }
__device__ __forceinline__ double seq_softplus(double v) { return v > 37.0 ? v : log1p(exp(v)); }
