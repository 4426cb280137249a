// Selection of a beam search: the `picks` best continuations over the beams and the vocabulary (launch_beam_select_*).
//
// With lse_i = log sum_v exp(logits_iv) the score of token v behind beam i is scores_i + logits_iv - lse_i.  Inside a beam the order is that of
// the logits, so the first kernel reads them once and leaves, per piece of a row, the maximum, the sum of exponentials below it (online) and the
// 32 best logits; the second adds the pieces up, forms the scores in r64 and merges the beams.
//
// The best of a piece.  While it streams by, a thread keeps its own maximum only.  Sorted inside a warp, the maxima give a bound that at least
// `picks` values reach: the least of the warps' values at place ceil(picks / warps).  Threads whose maximum reaches it (some tens of 128) look
// again at the one or two packs that they remember for it, or at all of theirs where a third one reaches it too, which the L2 still has, and put
// what reaches it on a list in shared memory; the warps sort it, 32 at a time, by bitonic stages and merge what they have.  So what is done for
// every value is one exponential, its sum and a comparison.  Where the list would overflow (rows of few different values), every value is offered
// to a warp's list of 32 in turn instead.
// Measured (r16, 50280 logits a row): 64 searches of 8 beams and 16 picks 27.4 us (rows 19, beams 7; the bytes take 7.9), one of 4 beams and 4
// picks 10.7 us.  Rows come at 4 TB/s, one exponential a value keeps the special-function unit busy for 4.9 us; beside them stand about 8 us of
// latency in a row's own steps (maxima, bound, second look, list) and the merge's sorts, shuffle behind shuffle.  Inserting every candidate into a
// warp's list instead took 70.7 and 18.8 us.
#include "mp_common.cuh"

namespace {

constexpr int BM_THREADS = 128, BM_WARPS = BM_THREADS / 32;
constexpr int BM_LIST = 32;
constexpr int BM_HELD = 512;             // values on a CTA's list
constexpr int BM_NONE = 0x7fffffff;      // token of an empty place
constexpr int BM_MAX_BEAMS = 64;

// A value and its token (or beam and place) as whole numbers in the order of better-first: comparisons of floating point values in r64 take ten
// times as long.  A value of 32 bits and its token make one number.  (-0 is taken for 0.)
template <typename V> struct Entry;
template <> struct Entry<float> { unsigned long long k; };
template <> struct Entry<double> { long long v; int i; };
__device__ __forceinline__ Entry<float> entry(float v, int i) {
  const int bits = __float_as_int(v + 0.f);
  const unsigned up = bits < 0 ? ~static_cast<unsigned>(bits) : static_cast<unsigned>(bits) | 0x80000000u;
  return {static_cast<unsigned long long>(up) << 32 | static_cast<unsigned>(BM_NONE - i)};
}
__device__ __forceinline__ Entry<double> entry(double v, int i) {
  const long long bits = __double_as_longlong(v + 0.0);
  return {bits < 0 ? bits ^ 0x7fffffffffffffffll : bits, i};
}
__device__ __forceinline__ float value_of(const Entry<float>& e) {
  const unsigned up = static_cast<unsigned>(e.k >> 32);
  return __int_as_float(static_cast<int>(up & 0x80000000u ? up & 0x7fffffffu : ~up));
}
__device__ __forceinline__ double value_of(const Entry<double>& e) { return __longlong_as_double(e.v < 0 ? e.v ^ 0x7fffffffffffffffll : e.v); }
__device__ __forceinline__ int index_of(const Entry<float>& e) { return BM_NONE - static_cast<int>(static_cast<unsigned>(e.k)); }
__device__ __forceinline__ int index_of(const Entry<double>& e) { return e.i; }
__device__ __forceinline__ bool better(const Entry<float>& a, const Entry<float>& b) { return a.k > b.k; }
__device__ __forceinline__ bool better(const Entry<double>& a, const Entry<double>& b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }
__device__ __forceinline__ Entry<float> entry_xor(const Entry<float>& e, int o) { return {__shfl_xor_sync(0xffffffffu, e.k, o)}; }
__device__ __forceinline__ Entry<double> entry_xor(const Entry<double>& e, int o) { return {__shfl_xor_sync(0xffffffffu, e.v, o), __shfl_xor_sync(0xffffffffu, e.i, o)}; }
__device__ __forceinline__ Entry<float> entry_at(const Entry<float>& e, int lane) { return {__shfl_sync(0xffffffffu, e.k, lane)}; }
__device__ __forceinline__ Entry<double> entry_at(const Entry<double>& e, int lane) { return {__shfl_sync(0xffffffffu, e.v, lane), __shfl_sync(0xffffffffu, e.i, lane)}; }
__device__ __forceinline__ float lowest(float) { return -INFINITY; }
__device__ __forceinline__ double lowest(double) { return -INFINITY; }

// The 32 best of two lists, best first.
template <typename V>
__device__ __forceinline__ void merge_lists(Entry<V>& a, const Entry<V>& b, int lane) {
  const Entry<V> r = entry_at(b, 31 - lane);
  if (better(r, a)) a = r;               // now bitonic
#pragma unroll 1
  for (int o = 16; o > 0; o >>= 1) {
    const Entry<V> other = entry_xor(a, o);
    const bool upper = (lane & o) != 0;  // keeps the worse one
    if (better(other, a) != upper) a = other;
  }
}
// A warp's entries, best first.
template <typename V>
__device__ __forceinline__ void sort_list(Entry<V>& a, int lane) {
#pragma unroll 1
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll 1
    for (int o = size >> 1; o > 0; o >>= 1) {
      const Entry<V> other = entry_xor(a, o);
      const bool worse = ((lane & o) != 0) != ((lane & size) != 0);      // this lane keeps the worse one
      if (better(other, a) != worse) a = other;
    }
}
// The warp's value at place `place` (0: the largest), counting equal ones.
__device__ __forceinline__ float nth_largest(float v, int place) {
  const int bits = __float_as_int(v);
  int key = bits < 0 ? bits ^ 0x7fffffff : bits, most = key;      // whole numbers in the same order
  for (int i = 0; i <= place; ++i) {
    most = __reduce_max_sync(0xffffffffu, key);
    const unsigned who = __ballot_sync(0xffffffffu, key == most);
    if ((threadIdx.x & 31) == __ffs(who) - 1) key = 0x80000000;
  }
  return __int_as_float(most < 0 ? most ^ 0x7fffffff : most);
}
__device__ __forceinline__ double nth_largest(double v, int place) {
  double most = v;
  for (int i = 0; i <= place; ++i) {
    most = warp_reduce<MaxOp>(v);
    const unsigned who = __ballot_sync(0xffffffffu, v == most);
    if ((threadIdx.x & 31) == __ffs(who) - 1) v = -INFINITY;
  }
  return most;
}
// `e` takes its place in the list.
template <typename V>
__device__ __forceinline__ void insert(Entry<V>& list, const Entry<V>& e, int lane) {
  const int at = __popc(__ballot_sync(0xffffffffu, better(list, e)));
  const Entry<V> before = entry_at(list, lane > 0 ? lane - 1 : 0);
  if (lane == at) list = e;
  else if (lane > at) list = before;
}
// Every lane's value that belongs among the first `picks`; `last`: the entry at that place.
template <typename V>
__device__ __forceinline__ void offer(Entry<V>& list, Entry<V>& last, const Entry<V>& e, int picks, int lane) {
  unsigned m = __ballot_sync(0xffffffffu, better(e, last));
  while (m != 0) {
    insert(list, entry_at(e, __ffs(m) - 1), lane);
    last = entry_at(list, picks - 1);
    m &= m - 1;
    m &= __ballot_sync(0xffffffffu, better(e, last));
  }
}

// exp(v) for v <= 0: the sum of them needs no more than 22 bits of each value
__device__ __forceinline__ float below_exp(float v) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * 1.4426950408889634f));
  return e;
}
__device__ __forceinline__ double below_exp(double v) { return exp(v); }
template <typename A> __device__ __forceinline__ A most_negative();
template <> __device__ __forceinline__ float most_negative<float>() { return -3.402823466e+38f; }
template <> __device__ __forceinline__ double most_negative<double>() { return -1.7976931348623157e+308; }

// The largest of a pack's values (a NaN is passed over: it shows in the sum).
template <typename T>
__device__ __forceinline__ typename Acc<T>::type pack_most(const Pack<T>& p) {
  typename Acc<T>::type m = mp_up(p.v[0]);
#pragma unroll
  for (int e = 1; e < Pack<T>::N; ++e) {
    const auto v = mp_up(p.v[e]);
    m = v > m || m != m ? v : m;
  }
  return m;
}
template <>
__device__ __forceinline__ float pack_most<__half>(const Pack<__half>& p) {
  const __half2* h = reinterpret_cast<const __half2*>(p.v);
  const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return __half2float(__hmax(__low2half(m), __high2half(m)));
}
// sum += exp(v - top) for two values (r16 and r32: the arithmetic of both in one instruction each)
__device__ __forceinline__ void add_exp2(float (&sum)[2], float top, float v0, float v1) {
  float d0, d1;
  asm("{\n.reg .b64 v, t, l;\nmov.b64 v, {%2, %3};\nmov.b64 t, {%4, %4};\nmov.b64 l, {%5, %5};\nadd.rn.f32x2 v, v, t;\nmul.rn.f32x2 v, v, l;\nmov.b64 {%0, %1}, v;\n}"
      : "=f"(d0), "=f"(d1)
      : "f"(v0), "f"(v1), "f"(-top), "f"(1.4426950408889634f));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(d0));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(d1));
  asm("{\n.reg .b64 s, d;\nmov.b64 s, {%0, %1};\nmov.b64 d, {%2, %3};\nadd.rn.f32x2 s, s, d;\nmov.b64 {%0, %1}, s;\n}" : "+f"(sum[0]), "+f"(sum[1]) : "f"(d0), "f"(d1));
}
__device__ __forceinline__ void add_exp2(double (&sum)[2], double top, double v0, double v1) {
  sum[0] += below_exp(v0 - top);
  sum[1] += below_exp(v1 - top);
}

template <typename A>
struct BeamScratch {     // per row and piece
  A* top;                // maximum
  double* sum;           // sum of exp(logit - maximum)
  Entry<A>* best;        // [32] best logits
};
template <typename A>
__host__ __device__ inline BeamScratch<A> beam_carve(void* scratch, size_t pieces) {
  BeamScratch<A> b;
  unsigned char* p = static_cast<unsigned char*>(scratch);
  b.sum = reinterpret_cast<double*>(p); p += pieces * sizeof(double);
  b.top = reinterpret_cast<A*>(p); p += pieces * sizeof(double);
  b.best = reinterpret_cast<Entry<A>*>(p);
  return b;
}
template <typename A> inline size_t beam_bytes(size_t pieces) { return pieces * (2 * sizeof(double) + BM_LIST * sizeof(Entry<A>)); }

// Pieces of a row: two packs for each thread of a CTA at least, eight CTAs for every SM where the rows are too few.  (148 SMs: the scratch function,
// which goes by the same numbers, knows no device.)
constexpr size_t BM_CTAS = 8 * 148;
inline size_t beam_most_pieces(size_t vocab, size_t size) { return (vocab * size + 2 * 16 * BM_THREADS - 1) / (2 * 16 * BM_THREADS); }
inline int beam_pieces(size_t rows, size_t vocab, size_t size) {
  const size_t most = beam_most_pieces(vocab, size);
  size_t want = BM_CTAS / rows;
  if (want > most) want = most;
  return static_cast<int>(want < 1 ? 1 : want);
}

// Pack k (of `packs`) of a row that begins off the 16-byte boundary: two aligned words, moved together.  Its first and last pack, whose words reach
// over the row's ends, are read value by value.
template <typename T>
__device__ __forceinline__ Pack<T> fetch_shifted(const T* src, int k, int packs) {
  union { uint32_t w[8]; uint4 u[2]; Pack<T> p; } x;
  const unsigned off = reinterpret_cast<uintptr_t>(src) & 15u;
  if (k == 0 || k == packs - 1) {
#pragma unroll
    for (int e = 0; e < Pack<T>::N; ++e) x.p.v[e] = src[static_cast<size_t>(k) * Pack<T>::N + e];
    return x.p;
  }
  const uint4* at = reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned char*>(src) - off) + k;
  x.u[0] = at[0];
  x.u[1] = off != 0 ? at[1] : x.u[0];
#pragma unroll
  for (int e = 0; e < 6; ++e) x.w[e] = off & 8 ? x.w[e + 2] : x.w[e];
#pragma unroll
  for (int e = 0; e < 5; ++e) x.w[e] = off & 4 ? x.w[e + 1] : x.w[e];
  if constexpr (sizeof(T) == 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) x.w[e] = __funnelshift_r(x.w[e], x.w[e + 1], off & 2 ? 16 : 0);
  return x.p;
}

// A beam from which nothing goes on, or nothing but the end: its logits are not read.
template <typename A> __device__ __forceinline__ bool beam_dead(A score) { return !(score > lowest(score)); }

template <typename T, bool WHOLE>
__global__ void __launch_bounds__(BM_THREADS, sizeof(T) == 8 ? 6 : 8) beam_rows_kernel(const T* __restrict__ logits, size_t pitch, const typename Acc<T>::type* __restrict__ scores,
                                                               const int* __restrict__ finished, BeamScratch<typename Acc<T>::type> out, int vocab, int picks,
                                                               int pieces) {
  mp_grid_dependency();
  using A = typename Acc<T>::type;
  constexpr int V = Pack<T>::N, U = WHOLE ? 8 : 4;
  __shared__ A s_top[BM_WARPS];
  __shared__ double s_sum[BM_WARPS];
  __shared__ int s_count;
  __shared__ A s_bound[BM_WARPS];
  __shared__ Entry<A> s_held[BM_HELD], s_best[BM_WARPS][BM_LIST];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long row = blockIdx.x / pieces;
  const int piece = blockIdx.x % pieces;
  if (beam_dead(scores[row]) || (finished != nullptr && finished[row] != 0)) return;
  const T* src = logits + row * pitch;
  // Which thread adds up which value goes by the token alone, not by the address: equal rows get equal sums, and their beams tie.
  const int packs = vocab / V, tail = vocab - packs * V;
  const int each = (packs + pieces - 1) / pieces;
  const int first = min(piece * each, packs), end = min(first + each, packs);

  A top = most_negative<A>(), sums[2] = {A(0), A(0)};
  auto fetch = [&](int k) {
    if constexpr (WHOLE) return ld_pack(src, k);
    return fetch_shifted(src, k, packs);
  };
  // this thread's packs, U at a time: what(pack, its number)
  auto stream = [&](auto what) {
    for (int k0 = first + tid; k0 < end; k0 += BM_THREADS * U) {
      Pack<T> in[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k0 + u * BM_THREADS < end) in[u] = fetch(k0 + u * BM_THREADS);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k0 + u * BM_THREADS < end) what(in[u], k0 + u * BM_THREADS);
    }
  };
  // The sum is kept relative to a value that was the maximum once: it moves on only when the maximum is more than 4 above it (the exponents'
  // rounding grows with the distance: 4 half steps at 4), which a stream does a few times.
  A base = most_negative<A>();
  auto raise = [&](A most) {
    top = most > top ? most : top;
    if (most > base + A(4)) {
      const A f = below_exp(base - most);
      sums[0] *= f;
      sums[1] *= f;
      base = most;
    }
  };
  // the two packs with the largest maxima, and the largest maximum of the others
  A most1 = lowest(A(0)), most2 = most1, most3 = most1;
  int pack1 = 0, pack2 = 0;
  stream([&](const Pack<T>& in, int k) {
    const A m = pack_most(in);
    if (m > most2) {
      most3 = most2;
      const bool first_now = m > most1;
      most2 = first_now ? most1 : m;
      pack2 = first_now ? pack1 : k;
      most1 = first_now ? m : most1;
      pack1 = first_now ? k : pack1;
    } else {
      most3 = m > most3 ? m : most3;
    }
    raise(m);
    A v[V];
    unpack(in, v);
#pragma unroll
    for (int e = 0; e < V; e += 2) add_exp2(sums, base, v[e], v[e + 1]);
  });
  const int at_tail = packs * V + tid;      // fewer than a pack
  const bool has_tail = piece == 0 && tid < tail;
  if (has_tail) {
    const A v = mp_up(src[at_tail]);
    raise(v);
    sums[0] += below_exp(v - base);
  }
  const A sum = sums[0] + sums[1];
  if (tid == 0) s_count = 0;
  {
    const A at = nth_largest(top, (picks + BM_WARPS - 1) / BM_WARPS - 1);
    if (lane == 0) s_bound[warp] = at;
  }
  __syncthreads();
  A bound = s_bound[0];
#pragma unroll
  for (int w = 1; w < BM_WARPS; ++w) bound = s_bound[w] < bound ? s_bound[w] : bound;
  if (bound == most_negative<A>()) bound = lowest(A(0));      // threads without a value above minus infinity have it too
  auto take = [&](A v, int i) {
    if (v >= bound) {
      const int at = atomicAdd(&s_count, 1);
      if (at < BM_HELD) s_held[at] = entry(v, i);
    }
  };
  if (!(top < bound)) {
    auto look = [&](const Pack<T>& in, int k) {
      A v[V];
      unpack(in, v);
#pragma unroll
      for (int e = 0; e < V; ++e) take(v[e], k * V + e);
    };
    if (most3 < bound) {
      if (most1 >= bound) look(fetch(pack1), pack1);
      if (most2 >= bound) look(fetch(pack2), pack2);
    } else {
      stream([&](const Pack<T>& in, int k) { if (!(pack_most(in) < bound)) look(in, k); });
    }
    if (has_tail) take(mp_up(src[at_tail]), at_tail);
  }
  __syncthreads();
  const int count = s_count;
  const Entry<A> none = entry(lowest(A(0)), BM_NONE);
  Entry<A> list = none;
  if (count <= BM_HELD) {
    // warp w has places 32 w ..; mostly there is work for the first ones only
    for (int k = warp * 32; k < count; k += BM_THREADS) {
      Entry<A> e = none;
      if (k + lane < count) e = s_held[k + lane];
      sort_list(e, lane);
      merge_lists(list, e, lane);
    }
  } else {
    Entry<A> last = list;
    for (int k0 = first + warp * 32; k0 < end; k0 += BM_THREADS) {
      const int k = k0 + lane;
#pragma unroll 1
      for (int e = 0; e < V; ++e) {
        Entry<A> mine = none;
        if (k < end) mine = entry(mp_up(src[static_cast<size_t>(k) * V + e]), k * V + e);
        offer(list, last, mine, picks, lane);
      }
    }
    Entry<A> mine = none;
    if (has_tail) mine = entry(mp_up(src[at_tail]), at_tail);
    offer(list, last, mine, picks, lane);
  }
  // the warp's sum, then the CTA's
  const A wtop = warp_reduce<MaxOp>(top);
  const double wsum = warp_reduce<SumOp>(static_cast<double>(sum) * static_cast<double>(below_exp(base - wtop)));
  s_best[warp][lane] = list;
  if (lane == 0) { s_top[warp] = wtop; s_sum[warp] = wsum; }
  __syncthreads();
  const int busy = count <= BM_HELD ? (count + 31) / 32 : BM_WARPS;      // warps that have something on their lists
  for (int half = BM_WARPS / 2; half > 0; half >>= 1) {
    if (half >= busy) continue;
    if (warp < half) {
      merge_lists(list, s_best[warp + half][lane], lane);
      s_best[warp][lane] = list;
    }
    __syncthreads();
  }
  if (warp == 0) {
    const size_t at = static_cast<size_t>(row) * pieces + piece;
    out.best[at * BM_LIST + lane] = list;
    const A t = s_top[lane % BM_WARPS], ct = warp_reduce<MaxOp>(t);
    const double cs = warp_reduce_width<SumOp, BM_WARPS>(s_sum[lane % BM_WARPS] * static_cast<double>(below_exp(t - ct)));
    if (lane == 0) { out.top[at] = ct; out.sum[at] = cs; }
  }
}

// One CTA per search.  `share` warps have a beam's pieces, so that few beams keep all warps busy; a warp's share of the pieces is `seats` lists
// at a time, the first 32 / seats places of each (at least `picks`), sorted together.
constexpr int BM_MERGE_WARPS = 16;
template <typename A>
__global__ void __launch_bounds__(BM_MERGE_WARPS * 32) beam_merge_kernel(BeamScratch<A> in, const A* scores, const int* finished, int eos, A* next_scores,
                                                                         int* parents, int* tokens, int* next_finished, int beams, int vocab, int picks,
                                                                         int pieces, int share, int seats) {
  __shared__ Entry<A> s_best[BM_MERGE_WARPS][BM_LIST];
  __shared__ Entry<double> s_score[BM_MERGE_WARPS][BM_LIST];
  __shared__ int s_token[BM_MAX_BEAMS][BM_LIST], s_done[BM_MAX_BEAMS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t search = blockIdx.x;
  const int places = BM_LIST / seats, seat = lane / places, place = lane % places;
  const int beams_at_once = BM_MERGE_WARPS / share;
  const Entry<A> none = entry(lowest(A(0)), BM_NONE);
  Entry<double> best = entry(lowest(0.0), BM_NONE);
  mp_grid_dependency();
  for (int b0 = 0; b0 < beams; b0 += beams_at_once) {
    const int beam = b0 + warp / share, part = warp % share;
    const bool live = beam < beams;
    const size_t row = search * beams + (live ? beam : 0);
    // (what a beam that is not looked at has in its place is anything: it is not used)
    Entry<A> list = none;
    A top = most_negative<A>();
    double sum = 0;
    const A had = scores[row];
    const bool done = finished != nullptr && finished[row] != 0, dead = beam_dead(had);
    if (part == 0) {      // the pieces' sums under one maximum
      for (int k = lane; k < pieces; k += 32) {
        const A t = in.top[row * pieces + k];
        const double more = in.sum[row * pieces + k];
        const A both = t > top ? t : top;
        sum = sum * static_cast<double>(below_exp(top - both)) + more * static_cast<double>(below_exp(t - both));
        top = both;
      }
    }
    for (int k0 = part * seats; k0 < pieces; k0 += share * seats) {
      const int k = k0 + seat;
      Entry<A> e = none;
      if (live && k < pieces) e = in.best[(row * pieces + k) * BM_LIST + place];
      if (seats > 1) sort_list(e, lane);
      merge_lists(list, e, lane);
    }
    if (part == 0) {
      const A all = warp_reduce<MaxOp>(top);
      sum = warp_reduce<SumOp>(sum * static_cast<double>(below_exp(top - all)));
      top = all;
    }
    if (share > 1) {
      if (b0 != 0) __syncthreads();      // the lists of the beams before have been read
      s_best[warp][lane] = list;
      __syncthreads();
      for (int half = share / 2; half > 0; half >>= 1) {
        if (part < half) {
          merge_lists(list, s_best[warp + half][lane], lane);
          s_best[warp][lane] = list;
        }
        if (half > 1) __syncthreads();
      }
    }
    if (live && part == 0) {
      double score = lowest(0.0);
      int token = lane;
      if (dead) {
        // its tokens rank in their order
      } else if (done) {
        token = lane == 0 ? eos : lane - 1 < eos ? lane - 1 : lane;
        if (lane == 0) score = static_cast<double>(had);
      } else if (sum > 0 && sum < 1.0 / 0.0) {
        // (the maximum goes first: beside one of 1e38, a mask's, the sum's logarithm would be lost)
        score = static_cast<double>(had) + ((static_cast<double>(value_of(list)) - static_cast<double>(top)) - log(sum));
        if (score != score) score = lowest(0.0);      // an infinite score behind a token that is ruled out
        token = index_of(list);
      }      // else a NaN or an infinity among the logits, or nothing above minus infinity: no probabilities
      s_token[beam][lane] = token;
      if (lane == 0) s_done[beam] = done;
      const bool wanted = lane < picks;
      const Entry<double> e = entry(wanted ? score : lowest(0.0), wanted ? beam * BM_LIST + lane : BM_NONE);
      if (b0 == 0) best = e;
      else merge_lists(best, e, lane);
    }
  }
  // the warps with beams: every `share`-th
  s_score[warp][lane] = best;
  __syncthreads();
  for (int half = BM_MERGE_WARPS / 2; half >= share; half >>= 1) {
    if (half >= beams * share) continue;
    if (warp < half) {
      merge_lists(best, s_score[warp + half][lane], lane);
      s_score[warp][lane] = best;
    }
    __syncthreads();
  }
  if (warp == 0 && lane < picks) {
    const size_t at = search * picks + lane;
    const int key = index_of(best), beam = key / BM_LIST, token = s_token[beam][key % BM_LIST];
    next_scores[at] = static_cast<A>(value_of(best));
    parents[at] = beam;
    tokens[at] = token;
    if (next_finished != nullptr) next_finished[at] = s_done[beam] != 0 || token == eos;
  }
}

template <typename T>
void beam_select_impl(const void* logits, len_t logits_pitch, const void* scores, const void* finished, len_t eos, void* next_scores, void* parents,
                      void* tokens, void* next_finished, void* scratch, len_t batch, len_t beams, len_t vocab, len_t picks, StreamContext ctx) {
  using A = typename Acc<T>::type;
  if (beams == 0 || beams > BM_MAX_BEAMS) MP_FATAL("beam_select: %lu beams (1 to %d)", beams, BM_MAX_BEAMS);
  if (picks == 0 || picks > BM_LIST || picks > vocab) MP_FATAL("beam_select: %lu picks (1 to %d, and no more than the vocabulary of %lu)", picks, BM_LIST, vocab);
  if (vocab > 0x7ffffff0ull || logits_pitch < vocab) MP_FATAL("beam_select: vocabulary of %lu, row pitch %lu", vocab, logits_pitch);
  if (batch == 0) return;
  if (scratch == nullptr) MP_FATAL("beam_select: scratch must not be NULL (mpBeamSelectScratchBytes)");
  if (reinterpret_cast<uintptr_t>(scratch) % 8 != 0) MP_FATAL("beam_select: scratch must be 8-byte aligned");
  if (batch > 0x7fffffffull) MP_FATAL("beam_select: %lu searches are too many for one launch", batch);
  const size_t rows = static_cast<size_t>(batch) * beams;
  const int pieces = beam_pieces(rows, vocab, sizeof(T));
  if (rows * pieces > 0x7fffffffull) MP_FATAL("beam_select: %lu searches are too many for one launch", batch);
  if (eos >= vocab) { finished = nullptr; next_finished = nullptr; }      // no end token
  const BeamScratch<A> sc = beam_carve<A>(scratch, rows * pieces);
  const bool whole = mp_aligned16(logits) && logits_pitch % Pack<T>::N == 0;
  MpLaunch(static_cast<unsigned>(rows * pieces), BM_THREADS, 0, mp_stream(ctx))(
      whole ? beam_rows_kernel<T, true> : beam_rows_kernel<T, false>, static_cast<const T*>(logits), logits_pitch, static_cast<const A*>(scores),
      static_cast<const int*>(finished), sc, static_cast<int>(vocab), static_cast<int>(picks), pieces);
  MP_LAUNCH_CHECK();
  int share = 1, seats = 1;
  while (share < BM_MERGE_WARPS && 2 * share * static_cast<int>(beams) <= BM_MERGE_WARPS && share < pieces) share <<= 1;
  while (2 * seats * static_cast<int>(picks) <= BM_LIST && seats < pieces) seats <<= 1;
  MpLaunch(static_cast<unsigned>(batch), BM_MERGE_WARPS * 32, 0, mp_stream(ctx))(
      beam_merge_kernel<A>, sc, static_cast<const A*>(scores), static_cast<const int*>(finished), eos < vocab ? static_cast<int>(eos) : -1,
      static_cast<A*>(next_scores), static_cast<int*>(parents), static_cast<int*>(tokens), static_cast<int*>(next_finished), static_cast<int>(beams),
      static_cast<int>(vocab), static_cast<int>(picks), pieces, share, seats);
  MP_LAUNCH_CHECK();
}

}  // namespace

extern "C" len_t mpBeamSelectScratchBytes(uint32_t dtype_key, len_t batch, len_t beams, len_t vocab, len_t picks) {
  (void)picks;
  const size_t rows = static_cast<size_t>(batch) * beams;
  if (rows == 0) return 256;
  // No call of as many rows and tokens or fewer has more pieces in all: one a row, or not above BM_CTAS and not above the most that its rows have.
  const size_t size = dtype_key == MP_R16 ? 2 : dtype_key == MP_R32 ? 4 : 8, most = beam_most_pieces(vocab, size);
  const size_t cut = most != 0 && rows > BM_CTAS / most ? BM_CTAS : rows * most, pieces = cut > rows ? cut : rows;
  return static_cast<len_t>((dtype_key == MP_R64 ? beam_bytes<double>(pieces) : beam_bytes<float>(pieces)) + 256);
}

MP_STAMP3(beam_select,
          (const void* logits, len_t logits_pitch, const void* scores, const void* finished, len_t eos, void* next_scores, void* parents, void* tokens,
           void* next_finished, void* scratch, len_t batch, len_t beams, len_t vocab, len_t picks, StreamContext ctx),
          (logits, logits_pitch, scores, finished, eos, next_scores, parents, tokens, next_finished, scratch, batch, beams, vocab, picks, ctx))
