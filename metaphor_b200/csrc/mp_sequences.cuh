// Sequences that go on from a kept state: packed rows, state slots, and the scan's step sizes, as the launchers for prompts and single
// tokens take them (include/mp_kernels.h, "sequences that go on from a kept state").
#pragma once

#include "mp_async.cuh"

// Sizes are counted in 31 bits, and so are products of two (each asked first: the product of larger ones may wrap round).
inline bool fits(len_t v) { return v <= 0x7fffffffull; }
inline bool fits(len_t a, len_t b) { return fits(a) && fits(b) && fits(a * b); }
// A head's rows p: the kernels round them up to whole tiles.
constexpr len_t SEQ_HEADDIM = 1ull << 30;

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

// V neighbouring values.
template <typename T, int V>
struct alignas(sizeof(T) * V) StVec { T v[V]; };

template <typename T, int V>
__device__ __forceinline__ void ld_vec(const T* p, typename Acc<T>::type* out) {
  const StVec<T, V> x = *reinterpret_cast<const StVec<T, V>*>(p);
#pragma unroll
  for (int e = 0; e < V; ++e) out[e] = mp_up(x.v[e]);
}
template <typename T, int V>
__device__ __forceinline__ void st_vec(T* p, const typename Acc<T>::type* in) {
  StVec<T, V> x;
#pragma unroll
  for (int e = 0; e < V; ++e) x.v[e] = mp_down<T>(in[e]);
  *reinterpret_cast<StVec<T, V>*>(p) = x;
}

// out = a b + c, value by value; fp32 values two at a time.
template <int V>
__device__ __forceinline__ void fma_vec(float (&out)[V], const float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int e = 0; e < V; e += 2)
      asm("{\n.reg .b64 a, b, c;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\nfma.rn.f32x2 c, a, b, c;\nmov.b64 {%0, %1}, c;\n}"
          : "=f"(out[e]), "=f"(out[e + 1])
          : "f"(a[e]), "f"(a[e + 1]), "f"(b[e]), "f"(b[e + 1]), "f"(c[e]), "f"(c[e + 1]));
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = a[e] * b[e] + c[e];
  }
}
template <int V>
__device__ __forceinline__ void fma_vec(double (&out)[V], const double (&a)[V], const double (&b)[V], const double (&c)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) out[e] = a[e] * b[e] + c[e];
}
template <int V>
__device__ __forceinline__ void mul_vec(float (&out)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int e = 0; e < V; e += 2)
      asm("{\n.reg .b64 c, a, b;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 c, a, b;\nmov.b64 {%0, %1}, c;\n}"
          : "=f"(out[e]), "=f"(out[e + 1])
          : "f"(a[e]), "f"(a[e + 1]), "f"(b[e]), "f"(b[e + 1]));
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = a[e] * b[e];
  }
}
template <int V>
__device__ __forceinline__ void mul_vec(double (&out)[V], const double (&a)[V], const double (&b)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) out[e] = a[e] * b[e];
}
template <typename T, int V>
__device__ __forceinline__ void widen(const StVec<T, V>& x, typename Acc<T>::type (&out)[V]) {
  if constexpr (std::is_same<T, __half>::value && V % 2 == 0) {
    const __half2* h = reinterpret_cast<const __half2*>(x.v);
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 f = __half22float2(h[e / 2]);
      out[e] = f.x;
      out[e + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = mp_up(x.v[e]);
  }
}

// The sum over the L lanes of a group of s[u], U of them: a lane is left with that of u = its number in the group / (L / U), where
// L < U with those of u = number * (U / L) + k in s[k].
template <int L, int U, typename A>
__device__ __forceinline__ void sum_rows(A (&s)[U], int lane) {
  int have = U;
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    if (have > 1) {
      have >>= 1;
      const bool up = (lane & o) != 0;
#pragma unroll
      for (int k = 0; k < (U + 1) / 2; ++k)
        if (k < have) {
          const A send = up ? s[k] : s[k + have], keep = up ? s[k + have] : s[k];
          s[k] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    } else {
      s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
    }
  }
}
