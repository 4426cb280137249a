// Selection of a beam search: the `picks` best continuations over the beams and the vocabulary (launch_beam_select_*).
//
// With lse_i = log sum_v exp(logits_iv) the score of token v behind beam i is scores_i + logits_iv - lse_i.  Inside a beam the order is that of
// the logits, so the first kernel reads them once and leaves, per piece of a row, the maximum, the sum of exponentials below it (online) and the
// 32 best logits; the second adds the pieces up, forms the scores in r64 and merges the beams.
//
// A list of 32 lies in a warp's lanes, best first.  While a row streams by, a value has to beat the list's last wanted place to be looked at
// again (for random rows `picks` x ln(values / picks) of them do).  Two lists are merged by one bitonic stage and a bitonic sort of 32.
#include "mp_common.cuh"

namespace {

constexpr int BM_THREADS = 256, BM_WARPS = BM_THREADS / 32;
constexpr int BM_LIST = 32;
constexpr int BM_NONE = 0x7fffffff;      // token of an empty place
constexpr int BM_MAX_BEAMS = 64;

template <typename V> struct Entry { V v; int i; };
template <typename V> __device__ __forceinline__ bool better(const Entry<V>& a, const Entry<V>& b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }
template <typename V> __device__ __forceinline__ Entry<V> entry_xor(const Entry<V>& e, int o) {
  return {__shfl_xor_sync(0xffffffffu, e.v, o), __shfl_xor_sync(0xffffffffu, e.i, o)};
}
template <typename V> __device__ __forceinline__ Entry<V> entry_at(const Entry<V>& e, int lane) {
  return {__shfl_sync(0xffffffffu, e.v, lane), __shfl_sync(0xffffffffu, e.i, lane)};
}
__device__ __forceinline__ float lowest(float) { return -INFINITY; }
__device__ __forceinline__ double lowest(double) { return -INFINITY; }

// The 32 best of two lists, best first.
template <typename V>
__device__ __forceinline__ void merge_lists(Entry<V>& a, const Entry<V>& b, int lane) {
  const Entry<V> r = entry_at(b, 31 - lane);
  if (better(r, a)) a = r;               // now bitonic
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Entry<V> other = entry_xor(a, o);
    const bool upper = (lane & o) != 0;  // keeps the worse one
    if (better(other, a) != upper) a = other;
  }
}
// `e` takes its place in the list.
template <typename V>
__device__ __forceinline__ void insert(Entry<V>& list, const Entry<V>& e, int lane) {
  const int at = __popc(__ballot_sync(0xffffffffu, better(list, e)));
  const Entry<V> before = {__shfl_up_sync(0xffffffffu, list.v, 1), __shfl_up_sync(0xffffffffu, list.i, 1)};
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

template <typename A>
struct BeamScratch {     // per row and piece
  A* top;                // maximum
  double* sum;           // sum of exp(logit - maximum)
  A* value;              // [32] best logits
  int* token;            // [32] their tokens
};
template <typename A>
__host__ __device__ inline BeamScratch<A> beam_carve(void* scratch, size_t pieces) {
  BeamScratch<A> b;
  unsigned char* p = static_cast<unsigned char*>(scratch);
  b.sum = reinterpret_cast<double*>(p); p += pieces * sizeof(double);
  b.top = reinterpret_cast<A*>(p); p += pieces * sizeof(double);
  b.value = reinterpret_cast<A*>(p); p += pieces * BM_LIST * sizeof(A);
  b.token = reinterpret_cast<int*>(p);
  return b;
}
inline size_t beam_bytes(size_t pieces, size_t acc) { return pieces * (2 * sizeof(double) + BM_LIST * (acc + sizeof(int))); }

// Pieces of a row: two packs for each thread of a CTA at least, four CTAs for every SM where the rows are too few.
inline int beam_pieces(size_t rows, size_t vocab, size_t size) {
  const size_t most = (vocab * size + 2 * 16 * BM_THREADS - 1) / (2 * 16 * BM_THREADS);
  size_t want = (4 * 148 + rows - 1) / rows;
  if (want > most) want = most;
  return static_cast<int>(want < 1 ? 1 : want);
}

// A beam from which nothing goes on, or nothing but the end: its logits are not read.
template <typename A> __device__ __forceinline__ bool beam_dead(A score) { return !(score > lowest(score)); }

template <typename T>
__global__ void __launch_bounds__(BM_THREADS) beam_rows_kernel(const T* __restrict__ logits, size_t pitch, const typename Acc<T>::type* __restrict__ scores,
                                                               const int* __restrict__ finished, BeamScratch<typename Acc<T>::type> out, int vocab, int picks,
                                                               int pieces) {
  mp_grid_dependency();
  using A = typename Acc<T>::type;
  constexpr int V = Pack<T>::N, U = 2;
  __shared__ A s_value[BM_WARPS][BM_LIST], s_top[BM_WARPS];
  __shared__ double s_sum[BM_WARPS];
  __shared__ int s_token[BM_WARPS][BM_LIST];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long row = blockIdx.x / pieces;
  const int piece = blockIdx.x % pieces;
  if (beam_dead(scores[row]) || (finished != nullptr && finished[row] != 0)) return;
  const T* src = logits + row * pitch;
  // Which thread adds up which value goes by the token alone, not by the address: equal rows get equal sums, and their beams tie.  A row off the
  // 16-byte boundary is read value by value.
  const bool whole = (reinterpret_cast<uintptr_t>(src) & 15u) == 0;
  const int packs = vocab / V, tail = vocab - packs * V;
  const int each = (packs + pieces - 1) / pieces;
  const int first = min(piece * each, packs), end = min(first + each, packs);

  Entry<A> list = {lowest(A(0)), BM_NONE}, last = list;
  A top = most_negative<A>(), sum = A(0);
  auto add = [&](A v) {
    if (v > top) { sum *= below_exp(top - v); top = v; }
    sum += below_exp(v - top);
  };
  for (int k0 = first; k0 < end; k0 += BM_THREADS * U) {
    Pack<T> in[U];
    bool have[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * BM_THREADS + tid;
      have[u] = k < end;
      if (have[u]) {
        if (whole) {
          in[u] = ld_pack_stream(src, k);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) in[u].v[e] = src[static_cast<size_t>(k) * V + e];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      A v[V], most = lowest(A(0));
      if (have[u]) {
        unpack(in[u], v);
#pragma unroll
        for (int e = 0; e < V; ++e) most = v[e] > most ? v[e] : most;
        if (most > top) { sum *= below_exp(top - most); top = most; }
#pragma unroll
        for (int e = 0; e < V; ++e) sum += below_exp(v[e] - top);
      }
      const int i = (k0 + u * BM_THREADS + tid) * V;
      if (__any_sync(0xffffffffu, have[u] && (most >= last.v))) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const Entry<A> mine = have[u] ? Entry<A>{v[e], i + e} : Entry<A>{lowest(A(0)), BM_NONE};
          offer(list, last, mine, picks, lane);
        }
      }
    }
  }
  if (piece == 0 && warp == 0) {
    const int i = packs * V + lane;
    Entry<A> e = {lowest(A(0)), BM_NONE};
    if (lane < tail) {
      e = {mp_up(src[i]), i};
      add(e.v);
    }
    offer(list, last, e, picks, lane);
  }
  // the warp's sum, then the CTA's
  const A wtop = warp_reduce<MaxOp>(top);
  const double wsum = warp_reduce<SumOp>(static_cast<double>(sum) * static_cast<double>(below_exp(top - wtop)));
  s_value[warp][lane] = list.v;
  s_token[warp][lane] = list.i;
  if (lane == 0) { s_top[warp] = wtop; s_sum[warp] = wsum; }
  __syncthreads();
  for (int half = BM_WARPS / 2; half > 0; half >>= 1) {
    if (warp < half) {
      merge_lists(list, Entry<A>{s_value[warp + half][lane], s_token[warp + half][lane]}, lane);
      s_value[warp][lane] = list.v;
      s_token[warp][lane] = list.i;
    }
    __syncthreads();
  }
  if (warp == 0) {
    const size_t at = static_cast<size_t>(row) * pieces + piece;
    out.value[at * BM_LIST + lane] = list.v;
    out.token[at * BM_LIST + lane] = list.i;
    const A t = s_top[lane % BM_WARPS], ct = warp_reduce<MaxOp>(t);
    const double cs = warp_reduce_width<SumOp, BM_WARPS>(s_sum[lane % BM_WARPS] * static_cast<double>(below_exp(t - ct)));
    if (lane == 0) { out.top[at] = ct; out.sum[at] = cs; }
  }
}

// One CTA per search.
template <typename A>
__global__ void __launch_bounds__(BM_THREADS) beam_merge_kernel(BeamScratch<A> in, const A* scores, const int* finished, int eos, A* next_scores,
                                                                int* parents, int* tokens, int* next_finished, int beams, int vocab, int picks, int pieces) {
  mp_grid_dependency();
  __shared__ A s_value[BM_WARPS][BM_LIST];
  __shared__ int s_from[BM_WARPS][BM_LIST], s_key[BM_WARPS][BM_LIST];
  __shared__ double s_score[BM_WARPS][BM_LIST];
  __shared__ int s_token[BM_MAX_BEAMS][BM_LIST], s_done[BM_MAX_BEAMS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t search = blockIdx.x;
  // `share` warps have a beam's pieces, so that few beams keep all warps busy
  int share = BM_WARPS;
  while (share > 1 && share * beams > BM_WARPS) share >>= 1;
  Entry<double> best = {lowest(0.0), BM_NONE};
  for (int b0 = 0; b0 < beams; b0 += BM_WARPS / share) {
    const int beam = b0 + warp / share, part = warp % share;
    const bool live = beam < beams;
    const size_t row = search * beams + (live ? beam : 0);
    const A had = scores[row];
    const bool dead = beam_dead(had), done = finished != nullptr && finished[row] != 0;
    Entry<A> list = {lowest(A(0)), BM_NONE};
    if (live && !dead && !done) {
      for (int k = part; k < pieces; k += share) {
        const size_t at = (row * pieces + k) * BM_LIST + lane;
        merge_lists(list, Entry<A>{in.value[at], in.token[at]}, lane);
      }
    }
    __syncthreads();      // the lists of the beams before have been read
    s_value[warp][lane] = list.v;
    s_from[warp][lane] = list.i;
    __syncthreads();
    if (live && part == 0) {
      double score = lowest(0.0);
      if (dead) {
        list.i = lane;
      } else if (done) {
        list.i = lane == 0 ? eos : lane - 1 < eos ? lane - 1 : lane;
        if (lane == 0) score = static_cast<double>(had);
      } else {
        for (int k = 1; k < share; ++k) merge_lists(list, Entry<A>{s_value[warp + k][lane], s_from[warp + k][lane]}, lane);
        A top = most_negative<A>();
        for (int k = lane; k < pieces; k += 32) { const A t = in.top[row * pieces + k]; top = t > top ? t : top; }
        top = warp_reduce<MaxOp>(top);
        double sum = 0;
        for (int k = lane; k < pieces; k += 32) sum += in.sum[row * pieces + k] * static_cast<double>(below_exp(in.top[row * pieces + k] - top));
        sum = warp_reduce<SumOp>(sum);
        // a NaN or an infinity among the logits, or nothing above minus infinity: no probabilities
        if (sum > 0 && sum < 1.0 / 0.0) score = static_cast<double>(had) + (static_cast<double>(list.v) - (static_cast<double>(top) + log(sum)));
        else list.i = lane;
      }
      s_token[beam][lane] = list.i;
      if (lane == 0) s_done[beam] = done;
      const bool wanted = lane < picks;
      merge_lists(best, Entry<double>{wanted ? score : lowest(0.0), wanted ? beam * BM_LIST + lane : BM_NONE}, lane);
    }
  }
  s_score[warp][lane] = best.v;
  s_key[warp][lane] = best.i;
  __syncthreads();
  for (int half = BM_WARPS / 2; half > 0; half >>= 1) {
    if (warp < half) {
      merge_lists(best, Entry<double>{s_score[warp + half][lane], s_key[warp + half][lane]}, lane);
      s_score[warp][lane] = best.v;
      s_key[warp][lane] = best.i;
    }
    __syncthreads();
  }
  if (warp == 0 && lane < picks) {
    const size_t at = search * picks + lane;
    const int beam = best.i / BM_LIST, token = s_token[beam][best.i % BM_LIST];
    next_scores[at] = static_cast<A>(best.v);
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
  const size_t rows = static_cast<size_t>(batch) * beams;
  const int pieces = beam_pieces(rows, vocab, sizeof(T));
  if (rows * pieces > 0x7fffffffull) MP_FATAL("beam_select: %lu searches are too many for one launch", batch);
  if (eos >= vocab) { finished = nullptr; next_finished = nullptr; }      // no end token
  const BeamScratch<A> sc = beam_carve<A>(scratch, rows * pieces);
  MpLaunch(static_cast<unsigned>(rows * pieces), BM_THREADS, 0, mp_stream(ctx))(
      beam_rows_kernel<T>, static_cast<const T*>(logits), logits_pitch, static_cast<const A*>(scores), static_cast<const int*>(finished), sc,
      static_cast<int>(vocab), static_cast<int>(picks), pieces);
  MP_LAUNCH_CHECK();
  MpLaunch(static_cast<unsigned>(batch), BM_THREADS, 0, mp_stream(ctx))(
      beam_merge_kernel<A>, sc, static_cast<const A*>(scores), static_cast<const int*>(finished), eos < vocab ? static_cast<int>(eos) : -1,
      static_cast<A*>(next_scores), static_cast<int*>(parents), static_cast<int*>(tokens), static_cast<int*>(next_finished), static_cast<int>(beams),
      static_cast<int>(vocab), static_cast<int>(picks), pieces);
  MP_LAUNCH_CHECK();
}

}  // namespace

extern "C" len_t mpBeamSelectScratchBytes(uint32_t dtype_key, len_t batch, len_t beams, len_t vocab, len_t picks) {
  (void)picks;
  const size_t rows = static_cast<size_t>(batch) * beams;
  if (rows == 0) return 256;
  const size_t size = dtype_key == MP_R16 ? 2 : dtype_key == MP_R32 ? 4 : 8;
  return static_cast<len_t>(beam_bytes(rows * beam_pieces(rows, vocab, size), dtype_key == MP_R64 ? 8 : 4) + 256);
}

MP_STAMP3(beam_select,
          (const void* logits, len_t logits_pitch, const void* scores, const void* finished, len_t eos, void* next_scores, void* parents, void* tokens,
           void* next_finished, void* scratch, len_t batch, len_t beams, len_t vocab, len_t picks, StreamContext ctx),
          (logits, logits_pitch, scores, finished, eos, next_scores, parents, tokens, next_finished, scratch, batch, beams, vocab, picks, ctx))
