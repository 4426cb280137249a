// Operators of a Mamba-2 block that go on from a kept state: the causal convolution + SiLU over packed prompts and over one token per
// sequence, the scan over one token per sequence, and the kept states that follow the beams of a search.  All of them are bound by memory:
// every input is read once, every output and state written once, in 16-byte accesses where the addresses allow it.
#include "mp_sequences.cuh"

namespace {

// The taps of V neighbouring channels lie in a row: as many whole vectors as there are taps.
template <typename T, int V, int W>
__device__ __forceinline__ void load_taps(const T* __restrict__ w, int c, typename Acc<T>::type (&tap)[W][V]) {
  typename Acc<T>::type flat[W * V];
#pragma unroll
  for (int k = 0; k < W; ++k) ld_vec<T, V>(w + static_cast<size_t>(c) * W + k * V, flat + k * V);
#pragma unroll
  for (int k = 0; k < W; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) tap[k][e] = flat[e * W + k];
}

// pre * sigmoid(pre).  r16 results have 11 bits: the special-function unit's exponential and reciprocal (22 bits) lose nothing there.
template <typename T, int V>
__device__ __forceinline__ StVec<T, V> silu_vec(const typename Acc<T>::type (&v)[V]) {
  StVec<T, V> x;
  if constexpr (std::is_same<T, __half>::value) {
    float r[V], by[V], one[V];
#pragma unroll
    for (int e = 0; e < V; ++e) { by[e] = -1.4426950408889634f; one[e] = 1.f; }
    mul_vec(r, v, by);
#pragma unroll
    for (int e = 0; e < V; ++e) asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(r[e]));
    fma_vec(r, r, one, one);
#pragma unroll
    for (int e = 0; e < V; ++e) asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r[e]));
    mul_vec(r, v, r);
    if constexpr (V % 2 == 0) {
      __half2* h = reinterpret_cast<__half2*>(x.v);
#pragma unroll
      for (int e = 0; e < V; e += 2) h[e / 2] = __floats2half2_rn(r[e], r[e + 1]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) x.v[e] = __float2half_rn(r[e]);
    }
  } else {
    using A = typename Acc<T>::type;
#pragma unroll
    for (int e = 0; e < V; ++e) x.v[e] = mp_down<T>(v[e] / (A(1) + seq_exp(-v[e])));
  }
  return x;
}

// ---------------------------------------------------------------------------
// Convolution over packed prompts.  A thread has V channels and a run of `run` rows, which it walks with the last W - 1 inputs in registers.
// Rows that reach into the kept state (the first W - 1 of a sequence) belong to the thread that has the sequence's first row, even behind its
// run's end, and that thread writes the new state too, from inputs that it fetches again: so nobody else reads what it overwrites.
// Measured (r16, 16 prompts of 7375 rows in all, 1792 channels): 17.5 us, 3.0 TB/s.  The special-function unit, which gives 16 of a value's two
// results a clock, is busy for 6.6 us of it; the rest is the way to the first inputs (sequence, state, taps) and too few warps to hide it.
// ---------------------------------------------------------------------------
constexpr int CS_TX = 32, CS_TY = 4, CS_U = 8;

template <typename T, int V, int W>
__global__ void __launch_bounds__(CS_TX * CS_TY, sizeof(T) == 2 ? 7 : 5) conv_prompt_kernel(const T* __restrict__ x, size_t xp, const T* __restrict__ w, const T* __restrict__ bias,
                                                                    T* __restrict__ states, T* __restrict__ y, size_t yp, const Sequences q, int channels,
                                                                    int run) {
  mp_grid_dependency();
  using A = typename Acc<T>::type;
  const int c = (blockIdx.x * CS_TX + threadIdx.x) * V;
  const bool live = c < channels;
  const int piece = blockIdx.y * CS_TY + threadIdx.y, pieces = gridDim.y * CS_TY;
  const long long r0 = static_cast<long long>(piece) * run, r1 = min(r0 + run, q.rows);
  A tap[W][V], b[V];
  if (live) {
    if (bias != nullptr) ld_vec<T, V>(bias + c, b);
    else
#pragma unroll
      for (int e = 0; e < V; ++e) b[e] = A(0);
    load_taps<T, V, W>(w, c, tap);
  }
  // a sequence without rows keeps nothing but zeros where it does not go on; they are dealt out over the pieces
  for (int s = piece; s < q.nseq; s += pieces) {
    const long long slot = seq_slot(q.slots, q.nslots, s);
    if (live && slot >= 0 && seq_first(q, s) >= seq_first(q, s + 1) && !seq_resumes(q, s)) {
      A zero[V] = {};
#pragma unroll
      for (int k = 0; k < W - 1; ++k) st_vec<T, V>(states + (slot * (W - 1) + k) * channels + c, zero);
    }
  }
  if (r0 >= r1) return;
  int s = warp_last_not_above(q.nseq, r0, [&](int i) { return seq_first(q, i); });
  long long at = r0;
  if (s < 0) { s = 0; at = seq_first(q, 0); }
  for (; s < q.nseq && at < r1; ++s) {
    const long long lo = seq_first(q, s), hi = seq_first(q, s + 1), slot = seq_slot(q.slots, q.nslots, s);
    if (hi <= at || slot < 0) { at = max(at, hi); continue; }
    StVec<T, V> before[W - 1] = {};
    long long end;
    if (lo >= at) {      // its first row is here
      at = lo;
      if (at >= r1) break;
      T* kept = states + slot * (W - 1) * channels + c;
      if (live) {
        if (seq_resumes(q, s))
#pragma unroll
          for (int k = 0; k < W - 1; ++k) before[k] = *reinterpret_cast<const StVec<T, V>*>(kept + static_cast<size_t>(k) * channels);
        StVec<T, V> last[W - 1] = {};
        const long long len = hi - lo;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
          const long long p = len - (W - 1) + k;      // in the sequence; before it lies what was kept
          if (p >= 0) {
            last[k] = *reinterpret_cast<const StVec<T, V>*>(x + (lo + p) * xp + c);
          } else {
            if (k + 1 < W - 1 && len == 1) last[k] = before[k + 1 < W - 1 ? k + 1 : 0];
            if (k + 2 < W - 1 && len == 2) last[k] = before[k + 2 < W - 1 ? k + 2 : 0];
          }
        }
#pragma unroll
        for (int k = 0; k < W - 1; ++k) *reinterpret_cast<StVec<T, V>*>(kept + static_cast<size_t>(k) * channels) = last[k];
      }
      end = min(hi, max(r1, lo + W - 1));
    } else {
      at = max(at, lo + W - 1);
      end = min(hi, r1);
      if (at < end && live) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) before[k] = *reinterpret_cast<const StVec<T, V>*>(x + (at - (W - 1) + k) * xp + c);
      }
    }
    if (live) {
      constexpr int U = CS_U;
      A h[W - 1][V];
#pragma unroll
      for (int k = 0; k < W - 1; ++k) widen(before[k], h[k]);
      const T* from = x + at * xp + c;
      T* to = y + at * yp + c;
      for (int left = static_cast<int>(end - at); left > 0; left -= U) {
        StVec<T, V> in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u < left) in[u] = *reinterpret_cast<const StVec<T, V>*>(from);
          from += xp;
        }
        // (rows behind the last are worked out too, from whatever is there: without a branch around each the taps' inputs move on by name)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          A now[V], pre[V];
          widen(in[u], now);
          fma_vec(pre, tap[0], h[0], b);
#pragma unroll
          for (int k = 1; k < W - 1; ++k) fma_vec(pre, tap[k], h[k], pre);
          fma_vec(pre, tap[W - 1], now, pre);
          const StVec<T, V> out = silu_vec<T, V>(pre);
          if (u < left) *reinterpret_cast<StVec<T, V>*>(to) = out;
          to += yp;
#pragma unroll
          for (int e = 0; e < V; ++e) {
#pragma unroll
            for (int k = 0; k + 1 < W - 1; ++k) h[k][e] = h[k + 1][e];
            h[W - 2][e] = now[e];
          }
        }
      }
    }
    at = max(end, r0);
    if (end < hi) break;
  }
}

// One token per sequence: V channels of a row per thread.  y may be x.
template <typename T, int V, int W>
__global__ void __launch_bounds__(128) conv_token_kernel(const T* x, size_t xp, const T* __restrict__ w, const T* __restrict__ bias, T* __restrict__ states,
                                                         const int* __restrict__ slots, T* y, size_t yp, long long rows, long long nslots, int channels) {
  mp_grid_dependency();
  using A = typename Acc<T>::type;
  const int per_row = (channels + V - 1) / V;
  const long long i = blockIdx.x * 128ll + threadIdx.x;
  const long long r = i / per_row;
  if (r >= rows) return;
  const int c = static_cast<int>(i - r * per_row) * V;
  const long long slot = seq_slot(slots, nslots, r);
  if (slot < 0) return;
  T* kept = states + slot * (W - 1) * channels + c;
  A in[W][V], tap[W][V], b[V] = {};
#pragma unroll
  for (int k = 0; k < W - 1; ++k) ld_vec<T, V>(kept + static_cast<size_t>(k) * channels, in[k]);
  ld_vec<T, V>(x + r * xp + c, in[W - 1]);
  load_taps<T, V, W>(w, c, tap);
  if (bias != nullptr) ld_vec<T, V>(bias + c, b);
#pragma unroll
  for (int k = 0; k < W; ++k) fma_vec(b, tap[k], in[k], b);
#pragma unroll
  for (int k = 0; k < W - 1; ++k) st_vec<T, V>(kept + static_cast<size_t>(k) * channels, in[k + 1]);
  *reinterpret_cast<StVec<T, V>*>(y + r * yp + c) = silu_vec<T, V>(b);
}

// ---------------------------------------------------------------------------
// Scan of one token per sequence:  S = exp(dt A) S + dt x (x) B,  y = S C.  The state ([P][N], accumulator type) is read and written once and
// is nearly all of the traffic.  L lanes have a row p of it, V values at a time; a warp takes ST_U rows per lane group at a time, `batches` times,
// so that what a row costs beside its own values (step size, B and C, addresses) is shared.  Measured (r16, 24 heads of 64 x 128): 300 tokens 82 us,
// 5.8 TB/s of the 6.5 that a copy has; one token 4.4 us, the way to the state and a launch.  The ST_U sums of a lane group are added up across
// its lanes by halves: in each of three rounds a lane hands on half of its sums and keeps the others.
// ---------------------------------------------------------------------------
constexpr int ST_U = 8;

template <typename T, int V, int L>
__global__ void __launch_bounds__(128, sizeof(T) == 8 ? 3 : 6) scan_token_kernel(const T* __restrict__ x, size_t xp, const T* __restrict__ raw, size_t rp,
                                                         const typename Acc<T>::type* __restrict__ dt_bias, const typename Acc<T>::type* __restrict__ A_log,
                                                         const T* __restrict__ Bm, const T* __restrict__ Cm, size_t bcp,
                                                         typename Acc<T>::type* __restrict__ states, const int* __restrict__ slots, T* __restrict__ y,
                                                         size_t yp, long long nslots, int H, int P, int N, int G, int batches, int splits) {
  mp_grid_dependency();
  using A = typename Acc<T>::type;
  constexpr int GROUPS = 32 / L, ROWS = ST_U * GROUPS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const unsigned split = blockIdx.x % splits, rh = blockIdx.x / splits, r = rh / H, h = rh % H;
  const int sub = lane / L, n0 = (lane % L) * V;
  const int first = (split * warps + warp) * batches * ROWS;      // rows first + u GROUPS + sub
  if (first >= P) return;
  const A step = mp_up(raw[r * rp + h]) + dt_bias[h], rate = A_log[h];
  const T* b = Bm + r * bcp + static_cast<size_t>(h / (H / G)) * N;
  const T* cc = Cm + r * bcp + static_cast<size_t>(h / (H / G)) * N;
  const T* xr = x + r * xp + static_cast<size_t>(h) * P;
  T* yr = y + r * yp + static_cast<size_t>(h) * P;
  StVec<T, V> braw, craw;
  auto fetch_bc = [&](int n) {
#pragma unroll
    for (int e = 0; e < V; ++e) { braw.v[e] = n < N ? b[n + e] : T(0.f); craw.v[e] = n < N ? cc[n + e] : T(0.f); }
  };
  fetch_bc(n0);
  const long long slot = seq_slot(slots, nslots, r);
  if (slot < 0) return;
  A* state = states + (slot * H + h) * static_cast<long long>(P) * N;
  A dt, decay[V];
  bool begun = false;
  for (int p0 = first; p0 < min(P, first + batches * ROWS); p0 += ROWS) {
    A sum[ST_U], xd[ST_U];
#pragma unroll
    for (int u = 0; u < ST_U; ++u) {
      sum[u] = A(0);
      const int p = p0 + u * GROUPS + sub;
      xd[u] = p < P ? mp_up(xr[p]) : A(0);
    }
    for (int n = n0; n - n0 < N; n += L * V) {
      StVec<A, V> s[ST_U];
      A* at = state + static_cast<size_t>(p0 + sub) * N + n;
#pragma unroll
      for (int u = 0; u < ST_U; ++u)
        if (p0 + u * GROUPS + sub < P && n < N) s[u] = *reinterpret_cast<const StVec<A, V>*>(at + static_cast<size_t>(u * GROUPS) * N);
      if (!begun) {      // while the first values are on their way
        dt = seq_softplus(step);
        const A d = seq_exp(dt * -seq_exp(rate));
#pragma unroll
        for (int e = 0; e < V; ++e) decay[e] = d;
        begun = true;
      }
      if (N > L * V) fetch_bc(n);
      A bv[V], cv[V];
      widen(braw, bv);
      widen(craw, cv);
#pragma unroll
      for (int u = 0; u < ST_U; ++u) {
        if (p0 + u * GROUPS + sub < P && n < N) {
          A xv[V], now[V], part[V];
          const A d = dt * xd[u];
#pragma unroll
          for (int e = 0; e < V; ++e) xv[e] = d;
          mul_vec(now, decay, s[u].v);
          fma_vec(now, xv, bv, now);
          mul_vec(part, now, cv);
#pragma unroll
          for (int e = 0; e < V; ++e) { s[u].v[e] = now[e]; sum[u] += part[e]; }
          *reinterpret_cast<StVec<A, V>*>(at + static_cast<size_t>(u * GROUPS) * N) = s[u];
        }
      }
    }
    sum_rows<L, ST_U>(sum, lane);
    constexpr int HELD = L >= ST_U ? 1 : ST_U / L, SHARED = L >= ST_U ? L / ST_U : 1;      // sums of a lane, lanes with the same one
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      const int u = (lane % L) / SHARED * HELD + k, p = p0 + u * GROUPS + sub;
      if (lane % SHARED == 0 && p < P) yr[p] = mp_down<T>(sum[k]);
    }
  }
}

// ---------------------------------------------------------------------------
// States that follow the beams, in place.  The CTA lists the beams that another one follows (each is read once) and the beams that change
// (each is written once); beams that keep their state cost nothing.  A thread has W bytes of every state of one search, RE_TURNS times: it
// fetches them into shared memory, the next turn's while this one's are written.  No other thread touches these bytes, so no barrier stands between.
// Measured (24 layers, 8 searches of 5 beams, rows of 768 KB): 152 us, 5.97 TB/s of the 6.5 that a copy has; with one word a thread and the lists
// made out by every thread, 185.
// ---------------------------------------------------------------------------
constexpr int RE_BEAMS = 64, RE_STAGES = 2;

template <int W> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = unsigned short; };

template <int W>
__device__ __forceinline__ void fetch_word(typename Word<W>::type* to, const typename Word<W>::type* from) {
  if constexpr (W == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mp_smem_u32(to)), "l"(from) : "memory");
  else if constexpr (W >= 4) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(mp_smem_u32(to)), "l"(from), "n"(W) : "memory");
  else *to = *from;
}

template <int W>
__global__ void reorder_kernel(unsigned char* __restrict__ states, const int* __restrict__ slots, const int* __restrict__ parents, int batch, int beams,
                               long long nslots, long long row_words, int turns) {
  mp_grid_dependency();
  using U = typename Word<W>::type;
  extern __shared__ __align__(16) unsigned char reorder_smem[];
  __shared__ long long s_source[RE_BEAMS], s_target[RE_BEAMS];      // places of the rows
  __shared__ int s_from[RE_BEAMS];                                  // which source a target takes
  __shared__ unsigned s_needed[2], s_moves[2];
  U* held = reinterpret_cast<U*>(reorder_smem) + threadIdx.x;
  const int b = blockIdx.y % batch, threads = blockDim.x;
  const long long layer = blockIdx.y / batch;
  if (threadIdx.x < 2) s_needed[threadIdx.x] = s_moves[threadIdx.x] = 0;
  __syncthreads();
  auto slot_of = [&](int j) { return seq_slot(slots, nslots, static_cast<long long>(b) * beams + j); };
  for (int j = threadIdx.x; j < beams; j += threads) {
    const int p = parents[static_cast<size_t>(b) * beams + j];
    if (p >= 0 && p < beams && p != j && slot_of(j) >= 0 && slot_of(p) >= 0) {
      atomicOr(&s_moves[j >> 5], 1u << (j & 31));
      atomicOr(&s_needed[p >> 5], 1u << (p & 31));
    }
  }
  __syncthreads();
  const unsigned m0 = s_moves[0], m1 = s_moves[1], n0 = s_needed[0], n1 = s_needed[1];
  const int targets = __popc(m0) + __popc(m1), sources = __popc(n0) + __popc(n1);
  if (targets == 0) return;
  auto rank = [](unsigned lo, unsigned hi, int j) { return j < 32 ? __popc(lo & ((1u << j) - 1)) : __popc(lo) + __popc(hi & ((1u << (j - 32)) - 1)); };
  for (int j = threadIdx.x; j < beams; j += threads) {
    if ((j < 32 ? n0 >> j : n1 >> (j - 32)) & 1) s_source[rank(n0, n1, j)] = slot_of(j) * row_words;
    if ((j < 32 ? m0 >> j : m1 >> (j - 32)) & 1) {
      const int k = rank(m0, m1, j);
      s_target[k] = slot_of(j) * row_words;
      s_from[k] = rank(n0, n1, parents[static_cast<size_t>(b) * beams + j]) * threads;
    }
  }
  __syncthreads();
  U* base = reinterpret_cast<U*>(states) + layer * nslots * row_words;
  const long long first = static_cast<long long>(blockIdx.x) * turns * threads + threadIdx.x;
  const int stage = beams * threads;
  auto fetch = [&](int t) {
    const long long word = first + static_cast<long long>(t) * threads;
    if (t < turns && word < row_words)
      for (int k = 0; k < sources; ++k) fetch_word<W>(held + (t % RE_STAGES) * stage + k * threads, base + s_source[k] + word);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int t = 0; t < RE_STAGES - 1; ++t) fetch(t);
  for (int t = 0; t < turns; ++t) {
    fetch(t + RE_STAGES - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(RE_STAGES - 1) : "memory");
    const long long word = first + static_cast<long long>(t) * threads;
    if (word >= row_words) break;
    const U* from = held + (t % RE_STAGES) * stage;
    for (int k = 0; k < targets; ++k) base[s_target[k] + word] = from[s_from[k]];
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ------------------------------- launch bodies ------------------------------
template <typename T, int V>
void conv_prompt_run(const T* x, size_t xp, const T* w, const T* bias, T* states, T* y, size_t yp, const Sequences& q, int channels, int width, StreamContext ctx) {
  const int cols = (channels + V * CS_TX - 1) / (V * CS_TX);
  // Rows of a run so that seven CTAs on each SM, as many as fit in r16, take all of them at once; a run reads W - 1 rows more than it writes.
  const long long per_sm = (q.rows * cols + 28ll * mp_sm_count(ctx) - 1) / (28ll * mp_sm_count(ctx));
  int run = static_cast<int>(per_sm < 4 ? 4 : per_sm > 64 ? 64 : per_sm);
  long long tiles = (q.rows + static_cast<long long>(run) * CS_TY - 1) / (static_cast<long long>(run) * CS_TY);
  while (tiles > 65535) { run *= 2; tiles = (q.rows + static_cast<long long>(run) * CS_TY - 1) / (static_cast<long long>(run) * CS_TY); }
  const dim3 grid(cols, static_cast<unsigned>(tiles < 1 ? 1 : tiles)), block(CS_TX, CS_TY);
  MpLaunch go(grid, block, 0, mp_stream(ctx));
  switch (width) {
    case 2: go(conv_prompt_kernel<T, V, 2>, x, xp, w, bias, states, y, yp, q, channels, run); break;
    case 3: go(conv_prompt_kernel<T, V, 3>, x, xp, w, bias, states, y, yp, q, channels, run); break;
    default: go(conv_prompt_kernel<T, V, 4>, x, xp, w, bias, states, y, yp, q, channels, run);
  }
  MP_LAUNCH_CHECK();
}

template <typename T>
void conv_check(const char* name, len_t rows, len_t nslots, len_t channels, len_t width, len_t x_pitch, len_t y_pitch) {
  if (width < 2 || width > 4) MP_FATAL("%s: width %lu is not 2, 3 or 4", name, width);
  if (x_pitch < channels || y_pitch < channels) MP_FATAL("%s: a row pitch is below the %lu channels", name, channels);
  if (!fits(rows) || !fits(nslots) || !fits(channels, width)) MP_FATAL("%s: rows, slots and channels are counted in 31 bits", name);
}

template <typename T>
void causal_conv1d_silu_prompt_impl(const void* x, len_t x_pitch, const void* w, const void* bias, void* states, const void* slots, const void* resume,
                                    const void* starts, void* y, len_t y_pitch, len_t nseq, len_t rows, len_t nslots, len_t channels, len_t width,
                                    StreamContext ctx) {
  conv_check<T>("causal_conv1d_silu_prompt", rows, nslots, channels, width, x_pitch, y_pitch);
  if (!fits(nseq)) MP_FATAL("causal_conv1d_silu_prompt: sequences are counted in 31 bits");
  if (nseq == 0 || channels == 0) return;
  const Sequences q{static_cast<const int*>(starts), static_cast<const int*>(slots), static_cast<const int*>(resume), static_cast<int>(nseq),
                    static_cast<long long>(rows), static_cast<long long>(nslots)};
  constexpr int PN = Pack<T>::N;
  const T *xt = static_cast<const T*>(x), *wt = static_cast<const T*>(w), *bt = static_cast<const T*>(bias);
  T *st = static_cast<T*>(states), *yt = static_cast<T*>(y);
  // (r16: 8 bytes at a time.  With 16 a thread holds twice the taps and inputs, and half as many warps fit: 19.1 us for 16 prompts of 1792
  // channels instead of 17.5.)
  constexpr int PV = PN > 4 ? 4 : PN;
  if (mp_aligned16(x) && mp_aligned16(w) && (bias == nullptr || mp_aligned16(bias)) && mp_aligned16(y) && mp_aligned16(states) && x_pitch % PV == 0 && y_pitch % PV == 0 && channels % PV == 0)
    conv_prompt_run<T, PV>(xt, x_pitch, wt, bt, st, yt, y_pitch, q, static_cast<int>(channels), static_cast<int>(width), ctx);
  else
    conv_prompt_run<T, 1>(xt, x_pitch, wt, bt, st, yt, y_pitch, q, static_cast<int>(channels), static_cast<int>(width), ctx);
}

template <typename T, int V>
void conv_token_run(const T* x, size_t xp, const T* w, const T* bias, T* states, const int* slots, T* y, size_t yp, long long rows, long long nslots,
                    int channels, int width, StreamContext ctx) {
  const long long threads = rows * ((channels + V - 1) / V);
  MpLaunch go(static_cast<unsigned>((threads + 127) / 128), 128, 0, mp_stream(ctx));
  switch (width) {
    case 2: go(conv_token_kernel<T, V, 2>, x, xp, w, bias, states, slots, y, yp, rows, nslots, channels); break;
    case 3: go(conv_token_kernel<T, V, 3>, x, xp, w, bias, states, slots, y, yp, rows, nslots, channels); break;
    default: go(conv_token_kernel<T, V, 4>, x, xp, w, bias, states, slots, y, yp, rows, nslots, channels);
  }
  MP_LAUNCH_CHECK();
}

template <typename T>
void causal_conv1d_silu_token_impl(const void* x, len_t x_pitch, const void* w, const void* bias, void* states, const void* slots, void* y, len_t y_pitch,
                                   len_t rows, len_t nslots, len_t channels, len_t width, StreamContext ctx) {
  conv_check<T>("causal_conv1d_silu_token", rows, nslots, channels, width, x_pitch, y_pitch);
  if (rows == 0 || channels == 0) return;
  constexpr int PN = Pack<T>::N;
  const T *xt = static_cast<const T*>(x), *wt = static_cast<const T*>(w), *bt = static_cast<const T*>(bias);
  T *st = static_cast<T*>(states), *yt = static_cast<T*>(y);
  const int* sl = static_cast<const int*>(slots);
  const long long r = static_cast<long long>(rows), n = static_cast<long long>(nslots);
  if (mp_aligned16(x) && mp_aligned16(w) && (bias == nullptr || mp_aligned16(bias)) && mp_aligned16(y) && mp_aligned16(states) && x_pitch % PN == 0 && y_pitch % PN == 0 && channels % PN == 0 &&
      r * (channels / PN) <= 0x7fffffffll * 128)
    conv_token_run<T, PN>(xt, x_pitch, wt, bt, st, sl, yt, y_pitch, r, n, static_cast<int>(channels), static_cast<int>(width), ctx);
  else
    conv_token_run<T, 1>(xt, x_pitch, wt, bt, st, sl, yt, y_pitch, r, n, static_cast<int>(channels), static_cast<int>(width), ctx);
}

template <typename T>
void ssd_scan_token_impl(const void* x, len_t x_pitch, const void* dt_raw, len_t dt_pitch, const void* dt_bias, const void* A_log, const void* Bm,
                         const void* Cm, len_t bc_pitch, void* states, const void* slots, void* y, len_t y_pitch, len_t rows, len_t nslots, len_t heads,
                         len_t headdim, len_t dstate, len_t ngroups, StreamContext ctx) {
  using A = typename Acc<T>::type;
  if (ngroups == 0 || heads % ngroups != 0) MP_FATAL("ssd_scan_token: heads %lu not divisible by groups %lu", heads, ngroups);
  if (!fits(rows) || !fits(nslots) || !fits(heads, headdim) || !fits(headdim, dstate) || !fits(ngroups, dstate) || headdim > SEQ_HEADDIM || dstate > 1ull << 30)
    MP_FATAL("ssd_scan_token: rows, slots and sizes are counted in 31 bits");
  if (x_pitch < heads * headdim || y_pitch < heads * headdim || bc_pitch < ngroups * dstate || dt_pitch < heads) MP_FATAL("ssd_scan_token: a row pitch is below its columns");
  if (rows == 0 || heads == 0 || headdim == 0) return;
  if (dstate == 0) MP_FATAL("ssd_scan_token: no state");
  const int P = static_cast<int>(headdim), N = static_cast<int>(dstate);
  const bool vec = mp_aligned16(states) && dstate % (16 / sizeof(A)) == 0;
  const int V = vec ? static_cast<int>(16 / sizeof(A)) : 1;
  int width = 1;
  while (width < 32 && width * V < N) width <<= 1;
  // A warp has ST_U rows p for each of its lane groups at a time, twice where that leaves four warps for every scheduler; a CTA of up to four warps.
  const int at_once = ST_U * (32 / width), turns = (P + at_once - 1) / at_once;
  const long long units = static_cast<long long>(rows) * static_cast<long long>(heads), plenty = 16ll * mp_sm_count(ctx);
  const int batches = turns > 1 && units * ((turns + 1) / 2) >= plenty ? 2 : 1;
  const int need = (turns + batches - 1) / batches;
  const int warps = units * need < 2ll * mp_sm_count(ctx) ? 1 : need >= 4 ? 4 : need >= 2 ? 2 : 1;
  const int splits = (need + warps - 1) / warps;
  if (units * splits > 0x7fffffffll) MP_FATAL("ssd_scan_token: %lu rows of %lu heads are too many for one launch", rows, heads);
  MpLaunch go(static_cast<unsigned>(units * splits), 32 * warps, 0, mp_stream(ctx));
  auto run = [&](auto kernel) {
    go(kernel, static_cast<const T*>(x), x_pitch, static_cast<const T*>(dt_raw), dt_pitch, static_cast<const A*>(dt_bias), static_cast<const A*>(A_log),
       static_cast<const T*>(Bm), static_cast<const T*>(Cm), bc_pitch, static_cast<A*>(states), static_cast<const int*>(slots), static_cast<T*>(y), y_pitch,
       static_cast<long long>(nslots), static_cast<int>(heads), P, N, static_cast<int>(ngroups), batches, splits);
  };
  auto by_width = [&](auto vec_size) {
    constexpr int VS = decltype(vec_size)::value;
    switch (width) {
      case 1: run(scan_token_kernel<T, VS, 1>); break;
      case 2: run(scan_token_kernel<T, VS, 2>); break;
      case 4: run(scan_token_kernel<T, VS, 4>); break;
      case 8: run(scan_token_kernel<T, VS, 8>); break;
      case 16: run(scan_token_kernel<T, VS, 16>); break;
      default: run(scan_token_kernel<T, VS, 32>);
    }
  };
  if (vec) by_width(std::integral_constant<int, static_cast<int>(16 / sizeof(A))>());
  else by_width(std::integral_constant<int, 1>());
  MP_LAUNCH_CHECK();
}

template <int W>
void reorder_run(void* states, const int* slots, const int* parents, long long layers, long long batch, int beams, long long nslots, long long row_bytes,
                 StreamContext ctx) {
  const long long words = row_bytes / W;
  // 48 KB of shared memory hold the words of a CTA's threads, a few KB of them its lists (64 beams: 16 threads)
  int threads = 128;
  while (threads > 16 && RE_STAGES * threads * beams * W > 46 * 1024) threads >>= 1;
  while (threads > 32 && threads / 2 >= words) threads >>= 1;
  // turns: twenty CTAs for every SM and more share the lists' making out over up to eight
  const long long per_sm = words * layers * batch / (static_cast<long long>(threads) * 20 * mp_sm_count(ctx));
  const int turns = static_cast<int>(per_sm < 1 ? 1 : per_sm > 8 ? 8 : per_sm);
  const long long blocks = (words + static_cast<long long>(threads) * turns - 1) / (static_cast<long long>(threads) * turns);
  // at most 65535 searches and layers in the grid's second dimension
  const long long step = batch <= 65535 ? 65535 / batch : 1;
  for (long long l = 0; l < layers; l += step) {
    const long long n = layers - l < step ? layers - l : step;
    MpLaunch(dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(n * batch)), threads, static_cast<size_t>(RE_STAGES) * threads * beams * W, mp_stream(ctx))(
        reorder_kernel<W>, static_cast<unsigned char*>(states) + l * nslots * row_bytes, slots, parents, static_cast<int>(batch), beams, nslots, words, turns);
    MP_LAUNCH_CHECK();
  }
}

template <typename T>
void reorder_states_impl(void* states, const void* slots, const void* parents, len_t layers, len_t batch, len_t beams, len_t nslots, len_t row,
                         StreamContext ctx) {
  if (beams > 64) MP_FATAL("reorder_states: %lu beams (64 at most)", beams);
  if (batch > 65535 || !fits(nslots) || !fits(layers)) MP_FATAL("reorder_states: searches are counted in 16 bits, slots and layers in 31");
  if (layers == 0 || batch == 0 || beams == 0 || row == 0) return;
  if (row > (0x7fffffffull * 32 + 31) / sizeof(T)) MP_FATAL("reorder_states: rows of %lu elements are too long", row);
  const size_t bytes = static_cast<size_t>(row) * sizeof(T);
  const int *sl = static_cast<const int*>(slots), *pa = static_cast<const int*>(parents);
  const size_t align = reinterpret_cast<uintptr_t>(states) | bytes;
  const long long L = static_cast<long long>(layers), b = static_cast<long long>(batch), n = static_cast<long long>(nslots), rb = static_cast<long long>(bytes);
  if (align % 16 == 0) reorder_run<16>(states, sl, pa, L, b, static_cast<int>(beams), n, rb, ctx);
  else if (align % 8 == 0) reorder_run<8>(states, sl, pa, L, b, static_cast<int>(beams), n, rb, ctx);
  else if (align % 4 == 0) reorder_run<4>(states, sl, pa, L, b, static_cast<int>(beams), n, rb, ctx);
  else reorder_run<2>(states, sl, pa, L, b, static_cast<int>(beams), n, rb, ctx);
}

}  // namespace

MP_STAMP3(causal_conv1d_silu_prompt,
          (const void* x, len_t x_pitch, const void* w, const void* bias, void* states, const void* slots, const void* resume, const void* starts, void* y,
           len_t y_pitch, len_t nseq, len_t rows, len_t nslots, len_t channels, len_t width, StreamContext ctx),
          (x, x_pitch, w, bias, states, slots, resume, starts, y, y_pitch, nseq, rows, nslots, channels, width, ctx))
MP_STAMP3(causal_conv1d_silu_token,
          (const void* x, len_t x_pitch, const void* w, const void* bias, void* states, const void* slots, void* y, len_t y_pitch, len_t rows, len_t nslots,
           len_t channels, len_t width, StreamContext ctx),
          (x, x_pitch, w, bias, states, slots, y, y_pitch, rows, nslots, channels, width, ctx))
MP_STAMP3(ssd_scan_token,
          (const void* x, len_t x_pitch, const void* dt_raw, len_t dt_pitch, const void* dt_bias, const void* A_log, const void* Bm, const void* Cm,
           len_t bc_pitch, void* states, const void* slots, void* y, len_t y_pitch, len_t rows, len_t nslots, len_t heads, len_t headdim, len_t dstate,
           len_t ngroups, StreamContext ctx),
          (x, x_pitch, dt_raw, dt_pitch, dt_bias, A_log, Bm, Cm, bc_pitch, states, slots, y, y_pitch, rows, nslots, heads, headdim, dstate, ngroups, ctx))
MP_STAMP3(reorder_states,
          (void* states, const void* slots, const void* parents, len_t layers, len_t batch, len_t beams, len_t nslots, len_t row, StreamContext ctx),
          (states, slots, parents, layers, batch, beams, nslots, row, ctx))
