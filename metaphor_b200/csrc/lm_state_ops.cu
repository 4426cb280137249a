// Operators of a Mamba-2 block that go on from a kept state: the causal convolution + SiLU over packed prompts and over one token per
// sequence, the scan over one token per sequence, and the kept states that follow the beams of a search.  All of them are bound by memory:
// every input is read once, every output and state written once, in 16-byte accesses where the addresses allow it.
#include "mp_sequences.cuh"

namespace {

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

// pre * sigmoid(pre).  r16 results have 11 bits: the special-function unit's exponential and reciprocal (22 bits) lose nothing there.
template <typename T> __device__ __forceinline__ typename Acc<T>::type silu_of(typename Acc<T>::type v) { return v / (typename Acc<T>::type(1) + seq_exp(-v)); }
template <> __device__ __forceinline__ float silu_of<__half>(float v) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return v * r;
}

// ---------------------------------------------------------------------------
// Convolution over packed prompts.  A thread has V channels and a run of `run` rows, which it walks with the last W - 1 inputs in registers.
// Rows that reach into the kept state (the first W - 1 of a sequence) belong to the thread that has the sequence's first row, even behind its
// run's end, and that thread writes the new state too, from inputs that it fetches again: so nobody else reads what it overwrites.
// ---------------------------------------------------------------------------
constexpr int CS_TX = 32, CS_TY = 4;

template <typename T, int V, int W>
__global__ void __launch_bounds__(CS_TX * CS_TY) conv_prompt_kernel(const T* __restrict__ x, size_t xp, const T* __restrict__ w, const T* __restrict__ bias,
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
#pragma unroll
    for (int e = 0; e < V; ++e) {
      b[e] = bias != nullptr ? mp_up(bias[c + e]) : A(0);
#pragma unroll
      for (int k = 0; k < W; ++k) tap[k][e] = mp_up(w[static_cast<size_t>(c + e) * W + k]);
    }
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
    A h[W - 1][V];
    long long end;
    if (lo >= at) {      // its first row is here
      at = lo;
      if (at >= r1) break;
      T* kept = states + slot * (W - 1) * channels + c;
      if (live) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
          if (seq_resumes(q, s)) ld_vec<T, V>(kept + static_cast<size_t>(k) * channels, h[k]);
          else
#pragma unroll
            for (int e = 0; e < V; ++e) h[k][e] = A(0);
        }
        A last[W - 1][V];
        const long long len = hi - lo;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
          const long long p = len - (W - 1) + k;      // in the sequence; before it lies what was kept
          if (p >= 0) {
            ld_vec<T, V>(x + (lo + p) * xp + c, last[k]);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) last[k][e] = A(0);
#pragma unroll
            for (int j = 1; j < W - 1; ++j)           // p + W - 1 = len + k < W - 1
              if (j == len + k)
#pragma unroll
                for (int e = 0; e < V; ++e) last[k][e] = h[j][e];
          }
        }
#pragma unroll
        for (int k = 0; k < W - 1; ++k) st_vec<T, V>(kept + static_cast<size_t>(k) * channels, last[k]);
      }
      end = min(hi, max(r1, lo + W - 1));
    } else {
      at = max(at, lo + W - 1);
      end = min(hi, r1);
      if (at < end && live) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) ld_vec<T, V>(x + (at - (W - 1) + k) * xp + c, h[k]);
      }
    }
    if (live) {
      constexpr int U = 4;
      for (; at < end; at += U) {
        A in[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (at + u < end) ld_vec<T, V>(x + (at + u) * xp + c, in[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (at + u < end) {
            A out[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
              A pre = b[e];
#pragma unroll
              for (int k = 0; k < W - 1; ++k) {
                const int j = u - (W - 1) + k;      // input of tap k: in this group, or before it
                pre += tap[k][e] * (j >= 0 ? in[j >= 0 ? j : 0][e] : h[j < 0 ? j + W - 1 : 0][e]);
              }
              pre += tap[W - 1][e] * in[u][e];
              out[e] = silu_of<T>(pre);
            }
            st_vec<T, V>(y + (at + u) * yp + c, out);
          }
        }
        if (at + U < end) {
#pragma unroll
          for (int k = 0; k < W - 1; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) h[k][e] = in[U - (W - 1) + k][e];
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
  A in[W][V], out[V];
#pragma unroll
  for (int k = 0; k < W - 1; ++k) ld_vec<T, V>(kept + static_cast<size_t>(k) * channels, in[k]);
  ld_vec<T, V>(x + r * xp + c, in[W - 1]);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    A pre = bias != nullptr ? mp_up(bias[c + e]) : A(0);
#pragma unroll
    for (int k = 0; k < W; ++k) pre += mp_up(w[static_cast<size_t>(c + e) * W + k]) * in[k][e];
    out[e] = silu_of<T>(pre);
  }
#pragma unroll
  for (int k = 0; k < W - 1; ++k) st_vec<T, V>(kept + static_cast<size_t>(k) * channels, in[k + 1]);
  st_vec<T, V>(y + r * yp + c, out);
}

// ---------------------------------------------------------------------------
// Scan of one token per sequence:  S = exp(dt A) S + dt x (x) B,  y = S C.  The state ([P][N], accumulator type) is read and written once and
// is nearly all of the traffic.  `width` lanes have a row p of it, V values at a time; a warp has U rows per lane group in flight.
// ---------------------------------------------------------------------------
constexpr int ST_U = 8;

template <typename T, int V>
__global__ void __launch_bounds__(128) scan_token_kernel(const T* __restrict__ x, size_t xp, const T* __restrict__ raw, size_t rp,
                                                         const typename Acc<T>::type* __restrict__ dt_bias, const typename Acc<T>::type* __restrict__ A_log,
                                                         const T* __restrict__ Bm, const T* __restrict__ Cm, size_t bcp,
                                                         typename Acc<T>::type* __restrict__ states, const int* __restrict__ slots, T* __restrict__ y,
                                                         size_t yp, long long nslots, int H, int P, int N, int G, int width, int splits) {
  mp_grid_dependency();
  using A = typename Acc<T>::type;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int split = blockIdx.x % splits;
  const long long rh = blockIdx.x / splits, r = rh / H;
  const int h = static_cast<int>(rh % H);
  const long long slot = seq_slot(slots, nslots, r);
  if (slot < 0) return;
  const int groups = 32 / width, sub = lane / width, n0 = (lane % width) * V;
  const int p0 = (split * warps + warp) * ST_U * groups + sub;      // rows p0, p0 + groups, ...
  if (p0 - sub >= P) return;
  A* state = states + (slot * H + h) * static_cast<long long>(P) * N;
  const A dt = seq_softplus(mp_up(raw[r * rp + h]) + dt_bias[h]);
  const A decay = seq_exp(dt * -seq_exp(A_log[h]));
  const T* b = Bm + r * bcp + static_cast<size_t>(h / (H / G)) * N;
  const T* cc = Cm + r * bcp + static_cast<size_t>(h / (H / G)) * N;
  A xd[ST_U], sum[ST_U];
#pragma unroll
  for (int u = 0; u < ST_U; ++u) {
    const int p = p0 + u * groups;
    xd[u] = p < P ? dt * mp_up(x[r * xp + static_cast<size_t>(h) * P + p]) : A(0);
    sum[u] = A(0);
  }
  for (int n = n0; n - n0 < N; n += width * V) {
    StVec<A, V> s[ST_U];
#pragma unroll
    for (int u = 0; u < ST_U; ++u) {
      const int p = p0 + u * groups;
      if (p < P && n < N) s[u] = *reinterpret_cast<const StVec<A, V>*>(state + static_cast<size_t>(p) * N + n);
    }
    A bv[V], cv[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      bv[e] = n < N ? mp_up(b[n + e]) : A(0);
      cv[e] = n < N ? mp_up(cc[n + e]) : A(0);
    }
#pragma unroll
    for (int u = 0; u < ST_U; ++u) {
      const int p = p0 + u * groups;
      if (p < P && n < N) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          s[u].v[e] = decay * s[u].v[e] + xd[u] * bv[e];
          sum[u] += s[u].v[e] * cv[e];
        }
        *reinterpret_cast<StVec<A, V>*>(state + static_cast<size_t>(p) * N + n) = s[u];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < ST_U; ++u) {
    for (int o = width >> 1; o > 0; o >>= 1) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], o);
    const int p = p0 + u * groups;
    if (p < P && lane % width == 0) y[r * yp + static_cast<size_t>(h) * P + p] = mp_down<T>(sum[u]);
  }
}

// ---------------------------------------------------------------------------
// States that follow the beams, in place.  A thread has W bytes of a row in every state of one search: it fetches those that a beam takes from
// another one into shared memory, which serves as its array with a variable index, then writes the beams that change.  No other thread
// touches these bytes, so no barrier stands between; beams that keep their state cost nothing, and a state that several take is read once.
// ---------------------------------------------------------------------------
template <int W> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = unsigned short; };

template <int W>
__global__ void reorder_kernel(unsigned char* __restrict__ states, const int* __restrict__ slots, const int* __restrict__ parents, int batch, int beams,
                               long long nslots, long long row_words) {
  mp_grid_dependency();
  using U = typename Word<W>::type;
  extern __shared__ __align__(16) unsigned char reorder_smem[];
  U* held = reinterpret_cast<U*>(reorder_smem) + threadIdx.x;
  const int b = blockIdx.y % batch;
  const long long layer = blockIdx.y / batch;
  const long long word = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
  const int* par = parents + static_cast<size_t>(b) * beams;
  unsigned long long moves = 0, needed = 0;
  for (int j = 0; j < beams; ++j) {
    const int p = par[j];
    if (p < 0 || p >= beams || p == j) continue;
    if (seq_slot(slots, nslots, static_cast<long long>(b) * beams + j) < 0 || seq_slot(slots, nslots, static_cast<long long>(b) * beams + p) < 0) continue;
    moves |= 1ull << j;
    needed |= 1ull << p;
  }
  if (moves == 0 || word >= row_words) return;
  U* base = reinterpret_cast<U*>(states) + layer * nslots * row_words + word;
  for (int p = 0; p < beams; ++p)
    if (needed >> p & 1) held[p * blockDim.x] = base[seq_slot(slots, nslots, static_cast<long long>(b) * beams + p) * row_words];
  for (int j = 0; j < beams; ++j)
    if (moves >> j & 1) base[seq_slot(slots, nslots, static_cast<long long>(b) * beams + j) * row_words] = held[par[j] * blockDim.x];
}

// ------------------------------- launch bodies ------------------------------
bool fits(len_t v) { return v <= 0x7fffffffull; }

template <typename T, int V>
void conv_prompt_run(const T* x, size_t xp, const T* w, const T* bias, T* states, T* y, size_t yp, const Sequences& q, int channels, int width, StreamContext ctx) {
  const int cols = (channels + V * CS_TX - 1) / (V * CS_TX);
  // runs of 16 rows read 19; shorter ones where there are too few threads for every SM
  int run = 16;
  const long long enough = static_cast<long long>(mp_sm_count(ctx)) * 8;
  while (run > 4 && static_cast<long long>(cols) * ((q.rows + run * CS_TY - 1) / (run * CS_TY)) < enough) run >>= 1;
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
  if (!fits(rows) || !fits(nslots) || !fits(channels * width)) MP_FATAL("%s: rows, slots and channels are counted in 31 bits", name);
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
  if (mp_aligned16(x) && mp_aligned16(y) && mp_aligned16(states) && x_pitch % PN == 0 && y_pitch % PN == 0 && channels % PN == 0)
    conv_prompt_run<T, PN>(xt, x_pitch, wt, bt, st, yt, y_pitch, q, static_cast<int>(channels), static_cast<int>(width), ctx);
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
  if (mp_aligned16(x) && mp_aligned16(y) && mp_aligned16(states) && x_pitch % PN == 0 && y_pitch % PN == 0 && channels % PN == 0 &&
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
  if (x_pitch < heads * headdim || y_pitch < heads * headdim || bc_pitch < ngroups * dstate || dt_pitch < heads) MP_FATAL("ssd_scan_token: a row pitch is below its columns");
  if (!fits(rows) || !fits(nslots) || !fits(heads * headdim) || !fits(headdim * dstate)) MP_FATAL("ssd_scan_token: rows, slots and sizes are counted in 31 bits");
  if (rows == 0 || heads == 0 || headdim == 0) return;
  if (dstate == 0) MP_FATAL("ssd_scan_token: no state");
  const int P = static_cast<int>(headdim), N = static_cast<int>(dstate);
  const bool vec = mp_aligned16(states) && dstate % (16 / sizeof(A)) == 0;
  const int V = vec ? static_cast<int>(16 / sizeof(A)) : 1;
  int width = 1;
  while (width < 32 && width * V < N) width <<= 1;
  // a warp has ST_U rows p for each of its lane groups; a CTA of up to four warps
  const int rows_per_warp = ST_U * (32 / width), need = (P + rows_per_warp - 1) / rows_per_warp;
  const long long units = static_cast<long long>(rows) * static_cast<long long>(heads);
  const int warps = units >= 2ll * mp_sm_count(ctx) && need >= 4 ? 4 : need >= 2 && units >= mp_sm_count(ctx) ? 2 : 1;
  const int splits = (need + warps - 1) / warps;
  if (units * splits > 0x7fffffffll) MP_FATAL("ssd_scan_token: %lu rows of %lu heads are too many for one launch", rows, heads);
  MpLaunch go(static_cast<unsigned>(units * splits), 32 * warps, 0, mp_stream(ctx));
  auto run = [&](auto kernel) {
    go(kernel, static_cast<const T*>(x), x_pitch, static_cast<const T*>(dt_raw), dt_pitch, static_cast<const A*>(dt_bias), static_cast<const A*>(A_log),
       static_cast<const T*>(Bm), static_cast<const T*>(Cm), bc_pitch, static_cast<A*>(states), static_cast<const int*>(slots), static_cast<T*>(y), y_pitch,
       static_cast<long long>(nslots), static_cast<int>(heads), P, N, static_cast<int>(ngroups), width, splits);
  };
  if (vec) run(scan_token_kernel<T, static_cast<int>(16 / sizeof(A))>);
  else run(scan_token_kernel<T, 1>);
  MP_LAUNCH_CHECK();
}

template <int W>
void reorder_run(void* states, const int* slots, const int* parents, long long layers, long long batch, int beams, long long nslots, long long row_bytes,
                 StreamContext ctx) {
  const long long words = row_bytes / W;
  // 48 KB of shared memory hold the beams' words of a CTA's threads
  int threads = 256;
  while (threads > 32 && threads * beams * W > 48 * 1024) threads >>= 1;
  while (threads > 32 && threads / 2 >= words) threads >>= 1;
  const long long blocks = (words + threads - 1) / threads;
  // at most 65535 searches and layers in the grid's second dimension
  const long long step = batch <= 65535 ? 65535 / batch : 1;
  for (long long l = 0; l < layers; l += step) {
    const long long n = layers - l < step ? layers - l : step;
    MpLaunch(dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(n * batch)), threads, static_cast<size_t>(threads) * beams * W, mp_stream(ctx))(
        reorder_kernel<W>, static_cast<unsigned char*>(states) + l * nslots * row_bytes, slots, parents, static_cast<int>(batch), beams, nslots, words);
    MP_LAUNCH_CHECK();
  }
}

template <typename T>
void reorder_states_impl(void* states, const void* slots, const void* parents, len_t layers, len_t batch, len_t beams, len_t nslots, len_t row,
                         StreamContext ctx) {
  if (beams > 64) MP_FATAL("reorder_states: %lu beams (64 at most)", beams);
  if (batch > 65535 || !fits(nslots) || !fits(layers)) MP_FATAL("reorder_states: searches are counted in 16 bits, slots and layers in 31");
  if (layers == 0 || batch == 0 || beams == 0 || row == 0) return;
  const size_t bytes = static_cast<size_t>(row) * sizeof(T);
  if (bytes / 2 / 32 > 0x7fffffffull) MP_FATAL("reorder_states: rows of %lu elements are too long", row);
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
