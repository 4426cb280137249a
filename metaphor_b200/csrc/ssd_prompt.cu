// The SSD scan over packed prompts that go on from a kept state (launch_ssd_scan_prompt_*):
//   dt = softplus(raw + dt_bias[h]),  a_t = exp(-dt_t exp(A_log[h])),  S_t = a_t S_{t-1} + dt_t x_t (x) B_t,  y_t = S_t C_t
// per sequence and head, S_{-1} the sequence's kept state or zero, the last S kept again.
#include "ssd_prompt.cuh"

namespace {

// ---------------------------------------------------------------------------
// The recurrence, step by step, for every type and shape.  LN lanes have PV rows p of a state, each lane NV of their columns in registers, so
// that nothing but B, C and x moves: they come through shared memory RT steps at a time, for the four warps of a CTA at once, the next steps'
// while these are worked on.  A step is three operations for every value of the state (decay, product, sum over the columns), two values to an
// instruction in fp32: bound by the fp32 pipe.  A lane leaves its share of y_t in shared memory; the LN shares of a value are added up behind
// the RT steps, so that no step waits for shuffles.  More lanes to a row make more and smaller CTAs; fewer rows to a lane would too, but then
// B and C, of which a lane reads as many values as it has columns, would come from shared memory no faster than now for a quarter of the products.
// Measured (r32, 64 rows and 128 columns a head): one prompt of 4095 steps and 24 heads 203 us, 12 of up to 1200 369 us (half of the fp32 pipe's
// rate), one of 37 steps 8 us (0.1 us a step: one warp on each scheduler, and a step's reads of shared memory and sums in a row); r64, 4 heads,
// three of up to 900 steps 51 us (61 with the step sizes made by one of the four warps: the others wait for it).
// Where the sequences and heads are too few for the GPU, long sequences are cut into ranges: first the states that all but the last ranges add
// (`STATES`: from zero, without y), then carried from range to range, then the ranges side by side from the states that they receive.
// ---------------------------------------------------------------------------
template <typename T, int NP_, int LN>
struct RecurrenceSizes {
  using A = typename Acc<T>::type;
  static constexpr int NP = NP_, NV = NP / LN, PV = sizeof(A) == 8 ? 2 : 4;   // columns (padded) of a state and of a lane, rows of a lane
  static constexpr int WARPS = 4, THREADS = 32 * WARPS;
  static constexpr int ROWS = PV * (32 / LN), PS = ROWS * WARPS;               // rows p of a warp, of the CTA
  static constexpr int RT = sizeof(A) == 8 ? 8 : 16;                           // steps at a time
  static constexpr int TILE = 2 * RT * NP + RT * PS + 2 * RT;                  // B, C, x, decays, step sizes
  static constexpr size_t BYTES = sizeof(A) * (2 * TILE + RT * THREADS * PV);  // two tiles, the lanes' shares of y
};

struct Ranges {
  void* local;      // acc [id][head][P][N]: states that a range adds, later those that it receives
  void* decay;      // acc [id][head]: what is left of a state behind it
  int steps;        // of a range, 0: whole sequences
  bool packs;       // rows of x, B and C are whole 16-byte packs
};

// RT rows of NP values, 16 bytes at a time or one by one; zeros behind row `steps` and column `cols`.  Values that need no conversion are copied
// asynchronously.
template <typename T, int NP, int RT, int THREADS>
__device__ __forceinline__ void fetch_rows(typename Acc<T>::type* dst, const T* src, size_t pitch, int steps, int cols, bool packs) {
  using A = typename Acc<T>::type;
  constexpr int V = Pack<T>::N;
  if (packs && NP % V == 0) {
#pragma unroll
    for (int k = 0; k < (RT * NP / V + THREADS - 1) / THREADS; ++k) {
      const int i = threadIdx.x + k * THREADS, t = i / (NP / V), n = i % (NP / V) * V;
      if (RT * NP / V % THREADS != 0 && i >= RT * NP / V) break;
      const bool in = t < steps && n < cols;
      const T* from = src + (in ? t * pitch + n : 0);
      if constexpr (std::is_same<T, A>::value) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(mp_smem_u32(dst + t * NP + n)), "l"(from), "r"(in ? 16 : 0) : "memory");
      } else {
        A v[V] = {};
        if (in) unpack(ld_pack(from, 0), v);
#pragma unroll
        for (int e = 0; e < V; e += 16 / sizeof(A)) *reinterpret_cast<StVec<A, 16 / sizeof(A)>*>(dst + t * NP + n + e) = *reinterpret_cast<StVec<A, 16 / sizeof(A)>*>(v + e);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < (RT * NP + THREADS - 1) / THREADS; ++k) {
      const int i = threadIdx.x + k * THREADS, t = i / NP, n = i % NP;
      if (RT * NP % THREADS == 0 || i < RT * NP) dst[i] = t < steps && n < cols ? mp_up(src[t * pitch + n]) : A(0);
    }
  }
}

template <typename T, int NP, int LN, bool STATES>
__global__ void __launch_bounds__(160, 3) recurrence_kernel(const PromptArgs g, const Ranges ranges, int splits) {
  mp_grid_dependency();
  using Z = RecurrenceSizes<T, NP, LN>;
  using A = typename Z::A;
  constexpr int NV = Z::NV, PV = Z::PV, RT = Z::RT, PS = Z::PS, THREADS = Z::THREADS, CV = 16 / sizeof(A);      // columns side by side
  extern __shared__ __align__(16) unsigned char rc_smem[];
  // a tile: B [RT][NP], columns past N zero; C the same; x [RT][PS]; decays [RT]; step sizes [RT]
  A* shares = reinterpret_cast<A*>(rc_smem) + 2 * Z::TILE;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // a fifth warp makes the step sizes and decays of the next tile: exponential and logarithm are as long as several steps
  const bool helper = warp == Z::WARPS;
  const int split = blockIdx.x % splits, idh = blockIdx.x / splits, h = idh % g.H, grp = h / (g.H / g.G);
  const Span sp = span_of(g.q, ranges.steps, idh / g.H);
  if (!sp.any || (STATES && sp.hi >= sp.seq_hi)) return;      // (nothing lies behind it)
  const T* x = static_cast<const T*>(g.x) + static_cast<size_t>(h) * g.P + split * PS;
  const T* raw = static_cast<const T*>(g.raw) + h;
  const T* Bm = static_cast<const T*>(g.Bm) + static_cast<size_t>(grp) * g.N;
  const T* Cm = static_cast<const T*>(g.Cm) + static_cast<size_t>(grp) * g.N;
  T* y = static_cast<T*>(g.y) + static_cast<size_t>(h) * g.P;
  const A bias = static_cast<const A*>(g.dt_bias)[h], rate = -seq_exp(static_cast<const A*>(g.A_log)[h]);
  const int pg = lane / LN, nl = lane % LN;
  const int pl = warp * Z::ROWS + pg * PV, p0 = split * PS + pl;     // this lane's first row, in the CTA and in the head
  A* state = static_cast<A*>(g.states) + (sp.slot * g.H + h) * static_cast<long long>(g.P) * g.N;
  A* local = static_cast<A*>(ranges.local) + static_cast<size_t>(idh) * g.P * g.N;
  // a lane's columns are neighbours CV at a time: 16-byte reads of B and C, the lanes of a row next to each other
  A S[PV][NV / CV][CV];
  auto column = [&](int i, int e) { return (i * LN + nl) * CV + e; };
  // (the first of several ranges too has what it receives in `local`: the last one may be writing the sequence's state by now)
  const bool received = !STATES && ranges.steps != 0 && sp.seq_hi - sp.seq_lo > ranges.steps, any = !helper && (received || (!STATES && seq_resumes(g.q, sp.s)));
  const A* from = received ? local : state;
  const bool vectors = g.N % CV == 0 && mp_aligned16(g.states);
#pragma unroll
  for (int p = 0; p < PV; ++p)
#pragma unroll
    for (int i = 0; i < NV / CV; ++i) {
      const A* at = from + static_cast<size_t>(p0 + p) * g.N + column(i, 0);
      StVec<A, CV> v = {};
      if (any && p0 + p < g.P) {
        if (vectors) {
          if (column(i, 0) < g.N) v = *reinterpret_cast<const StVec<A, CV>*>(at);
        } else {
#pragma unroll
          for (int e = 0; e < CV; ++e)
            if (column(i, e) < g.N) v.v[e] = at[e];
        }
      }
#pragma unroll
      for (int e = 0; e < CV; ++e) S[p][i][e] = v.v[e];
    }

  // (raw step sizes are asked for a tile earlier)
  auto raw_at = [&](long long t0) { return helper && lane < RT && t0 + lane < sp.hi ? mp_up(raw[(t0 + lane) * g.rp]) : A(0); };
  A raw_here = raw_at(sp.lo);
  auto fetch = [&](long long t0) {
    A* tile = reinterpret_cast<A*>(rc_smem) + ((t0 - sp.lo) / RT & 1) * Z::TILE;
    const int steps = sp.hi - t0 < RT ? static_cast<int>(sp.hi - t0) : RT;
    if (!helper) {
      fetch_rows<T, NP, RT, THREADS>(tile, Bm + t0 * g.bcp, g.bcp, steps, g.N, ranges.packs);
      if (!STATES) fetch_rows<T, NP, RT, THREADS>(tile + RT * NP, Cm + t0 * g.bcp, g.bcp, steps, g.N, ranges.packs);
      fetch_rows<T, PS, RT, THREADS>(tile + 2 * RT * NP, x + t0 * g.xp, g.xp, steps, g.P - split * PS, ranges.packs);
    } else if (lane < RT) {
      const A dt = lane < steps ? seq_softplus(raw_here + bias) : A(0);
      raw_here = raw_at(t0 + RT);
      tile[2 * RT * NP + RT * PS + lane] = lane < steps ? seq_exp(dt * rate) : A(1);
      tile[2 * RT * NP + RT * PS + RT + lane] = dt;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  A left = A(1);
  if (sp.lo < sp.hi) fetch(sp.lo);
  for (long long t0 = sp.lo; t0 < sp.hi; t0 += RT) {
    const int steps = sp.hi - t0 < RT ? static_cast<int>(sp.hi - t0) : RT;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    if (t0 + RT < sp.hi) fetch(t0 + RT);
    if (helper) continue;
    const A* sB = reinterpret_cast<const A*>(rc_smem) + ((t0 - sp.lo) / RT & 1) * Z::TILE;
    const A *sC = sB + RT * NP, *sx = sC + RT * NP, *sa = sx + RT * PS, *sdt = sa + RT;
    // UN steps at a time, so that one's operands are read and its sums finished beside another one's products; steps behind the last have a size
    // of zero and change nothing.  (The shares are stored behind all of them: no read of a tile may pass a store.)
    constexpr int UN = NV <= 4 ? 4 : 2;
    auto work = [&](auto padded) {
      for (int tu = 0; tu < steps; tu += UN) {
        StVec<A, PV> total[UN];
#pragma unroll
        for (int q = 0; q < UN; ++q) {
          const int t = tu + q;
          A a[CV], xd[PV][CV], sum[PV][CV];
          const A dt = sdt[t], a1 = sa[t];
          if (STATES) left *= a1;
#pragma unroll
          for (int e = 0; e < CV; ++e) a[e] = a1;
#pragma unroll
          for (int p = 0; p < PV; ++p) {
            const A v = dt * sx[t * PS + pl + p];
#pragma unroll
            for (int e = 0; e < CV; ++e) { xd[p][e] = v; sum[p][e] = A(0); }
          }
#pragma unroll
          for (int i = 0; i < NV / CV; ++i) {
            const StVec<A, CV> b = *reinterpret_cast<const StVec<A, CV>*>(sB + t * NP + column(i, 0));
            StVec<A, CV> c;
            if (!STATES) c = *reinterpret_cast<const StVec<A, CV>*>(sC + t * NP + column(i, 0));
#pragma unroll
            for (int p = 0; p < PV; ++p) {
              mul_vec(S[p][i], a, S[p][i]);
              fma_vec(S[p][i], xd[p], b.v, S[p][i]);
              if constexpr (decltype(padded)::value) {      // columns behind the last stay zero: an infinity times nothing would reach y
#pragma unroll
                for (int e = 0; e < CV; ++e) S[p][i][e] = column(i, e) < g.N ? S[p][i][e] : A(0);
              }
              if (!STATES) fma_vec(sum[p], c.v, S[p][i], sum[p]);
            }
          }
#pragma unroll
          for (int p = 0; p < PV; ++p) {
            total[q].v[p] = sum[p][0];
#pragma unroll
            for (int e = 1; e < CV; ++e) total[q].v[p] += sum[p][e];
          }
        }
        if (!STATES) {
#pragma unroll
          for (int q = 0; q < UN; ++q) *reinterpret_cast<StVec<A, PV>*>(shares + ((tu + q) * THREADS + tid) * PV) = total[q];
        }
      }
    };
    if (g.N < NP) work(std::true_type()); else work(std::false_type());
    if (!STATES) {
      __syncwarp();
      // a lane has one of the warp's ROWS values of every (32 / ROWS)-th step; it begins with another one of the shares than its
      // neighbours, which would all wait for the same bank
      const int row = lane % Z::ROWS, first = lane / PV;
      const A* at = shares + (warp * 32 + row / PV * LN) * PV + row % PV;
      const int p = split * PS + warp * Z::ROWS + row;
      for (int t = lane / Z::ROWS; t < steps; t += 32 / Z::ROWS) {
        A v = A(0);
#pragma unroll
        for (int k = 0; k < LN; ++k) v += at[(t * THREADS + (first + k) % LN) * PV];
        if (p < g.P) y[(t0 + t) * g.yp + p] = mp_down<T>(v);
      }
      __syncwarp();
    }
  }
  A* to = STATES ? local : state;
  if (helper || (!STATES && sp.hi < sp.seq_hi)) return;
#pragma unroll
  for (int p = 0; p < PV; ++p)
#pragma unroll
    for (int i = 0; i < NV / CV; ++i) {
      A* at = to + static_cast<size_t>(p0 + p) * g.N + column(i, 0);
      StVec<A, CV> v;
#pragma unroll
      for (int e = 0; e < CV; ++e) v.v[e] = S[p][i][e];
      if (p0 + p < g.P) {
        if (vectors) {
          if (column(i, 0) < g.N) *reinterpret_cast<StVec<A, CV>*>(at) = v;
        } else {
#pragma unroll
          for (int e = 0; e < CV; ++e)
            if (column(i, e) < g.N) at[e] = v.v[e];
        }
      }
    }
  if (STATES && split == 0 && tid == 0) static_cast<A*>(ranges.decay)[idh] = left;
}

// From range to range: what each adds is replaced by what it receives, the first one by the kept state.  A thread has one value of a state, four
// ranges' on their way.
template <typename A>
__global__ void __launch_bounds__(256) recurrence_carry_kernel(const PromptArgs g, const Ranges ranges, int parts) {
  mp_grid_dependency();
  const int part = blockIdx.x % parts, sh = blockIdx.x / parts, s = sh / g.H, h = sh % g.H;
  const long long lo = seq_first(g.q, s), hi = seq_first(g.q, s + 1), slot = seq_slot(g.q.slots, g.q.nslots, s);
  const long long n = (hi - lo + ranges.steps - 1) / ranges.steps, size = static_cast<long long>(g.P) * g.N, e = part * 256ll + threadIdx.x;
  if (slot < 0 || n < 2 || e >= size) return;
  // a state that is infinite stays so however many steps are behind it, as it does step by step
  const A least = sizeof(A) == 8 ? A(4.9406564584124654e-324) : A(1.401298464324817e-45f);
  A v = seq_resumes(g.q, s) ? static_cast<const A*>(g.states)[(slot * g.H + h) * size + e] : A(0);
  const size_t first = (static_cast<size_t>(lo / ranges.steps + s)) * g.H + h;
  A* at = static_cast<A*>(ranges.local) + first * size + e;
  const A* decay = static_cast<const A*>(ranges.decay) + first;
  const size_t next = static_cast<size_t>(g.H) * size;
  constexpr int U = 4;
  A ahead = at[0];      // (place j + 1 is read before it is written: what its range adds goes to the one behind)
  at[0] = v;
  for (long long j = 0; j + 1 < n; j += U) {
    A add[U + 1], left[U];
    add[0] = ahead;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j + u + 1 < n) left[u] = decay[u * g.H];
      if (j + u + 2 < n) add[u + 1] = at[(u + 1) * next];
    }
    ahead = add[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j + u + 1 < n) {
        v = (left[u] < least ? least : left[u]) * v + add[u];
        at[(u + 1) * next] = v;
      }
    at += U * next;
    decay += U * g.H;
  }
}

// How a call is cut up.  The host knows how many sequences and rows there are, not how long each is.
struct Cut { int lanes, splits, steps; size_t ids; };      // lanes of a row; CTAs of a head; steps of a range (0: whole sequences); ranges or sequences
// `least`, `most`: lanes of a row; `held`: rows p of a lane.  Ranges of 32 steps or more where a sequence may be longer than 320 steps and there
// are not eight CTAs for each of 148 SMs all the same (three fit at a time, two of 256 columns in fp32): a range's state is made twice.  Measured,
// r32, whole and in ranges: one sequence of 256 steps and 24 heads 28 and 46 us, of 512 steps 52 and 44, with 4 heads 51 and 22 (25 with ranges of
// 64 steps at least); five of up to 333 steps and 8 heads 39 and 41, which the guess at the longest cannot tell from one long among short ones.
// Rows get more lanes where a head is small, or where there are fewer than two CTAs for an SM (12 sequences of up to 300 steps: 95 us, with one CTA
// for an SM 143, with four 105).  (148 SMs: the scratch function, which goes by the same numbers, knows no device.)
constexpr size_t RC_SMS = 148, RC_CTAS = 8 * RC_SMS, RC_LONG = 320, RC_RANGE = 32;
Cut recurrence_cut(size_t nseq, size_t rows, size_t heads, size_t headdim, int held, int least, int most) {
  Cut c{least, 0, 0, nseq};
  auto rows_of = [&] { return static_cast<size_t>(held) * (128 / c.lanes); };
  auto splits = [&] { return (headdim + rows_of() - 1) / rows_of(); };
  while (c.lanes < most && 2 * headdim <= rows_of()) c.lanes <<= 1;
  const size_t units = heads * splits(), longest = 2 * rows / nseq < rows ? 2 * rows / nseq : rows;      // (a guess)
  if (nseq * units < RC_CTAS && longest > RC_LONG) {
    const size_t want = RC_CTAS / units + 1;
    size_t range = ((rows + want - 1) / want + 15) / 16 * 16;
    if (range < RC_RANGE) range = RC_RANGE;
    if (range < rows) { c.steps = static_cast<int>(range); c.ids = rows / range + nseq; }
  }
  while (c.lanes < most && c.ids * heads * splits() < 2 * RC_SMS) c.lanes <<= 1;
  c.splits = static_cast<int>(splits());
  return c;
}

template <typename T, int NP, int LN>
void recurrence_run(const PromptArgs& g, const Ranges& r, const Cut& c, StreamContext ctx) {
  using Z = RecurrenceSizes<T, NP, LN>;
  using A = typename Z::A;
  const size_t ctas = c.ids * g.H * c.splits;
  if (ctas > 0x7fffffffull) MP_FATAL("ssd_scan_prompt: too many sequences and heads for one launch");
  auto go = [&](auto kernel) {
    if (Z::BYTES > 48 * 1024) MP_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Z::BYTES)));
    MpLaunch(static_cast<unsigned>(ctas), Z::THREADS + 32, Z::BYTES, mp_stream(ctx))(kernel, g, r, c.splits);
    MP_LAUNCH_CHECK();
  };
  if (r.steps != 0) {
    go(recurrence_kernel<T, NP, LN, true>);
    const size_t parts = (static_cast<size_t>(g.P) * g.N + 255) / 256, carries = static_cast<size_t>(g.q.nseq) * g.H * parts;
    if (carries > 0x7fffffffull) MP_FATAL("ssd_scan_prompt: too many sequences and heads for one launch");
    MpLaunch(static_cast<unsigned>(carries), 256, 0, mp_stream(ctx))(recurrence_carry_kernel<A>, g, r, static_cast<int>(parts));
    MP_LAUNCH_CHECK();
  }
  go(recurrence_kernel<T, NP, LN, false>);
}

// what(padded columns, least and most lanes of a row): a lane has 4 to 16 columns
template <typename F>
auto by_columns(size_t dstate, F what) {
  using std::integral_constant;
  if (dstate <= 32) return what(integral_constant<int, 32>(), integral_constant<int, 8>(), integral_constant<int, 8>());
  if (dstate <= 64) return what(integral_constant<int, 64>(), integral_constant<int, 8>(), integral_constant<int, 16>());
  if (dstate <= 128) return what(integral_constant<int, 128>(), integral_constant<int, 8>(), integral_constant<int, 32>());
  return what(integral_constant<int, 256>(), integral_constant<int, 16>(), integral_constant<int, 32>());
}
template <typename T> constexpr int recurrence_held = RecurrenceSizes<T, 32, 8>::PV;

// Enough for every call of as many sequences and rows or fewer: those that are cut have fewer than RC_CTAS units in all (a head's CTAs do not depend on
// either), ranges of RC_RANGE steps or more, no more of them than `recurrence_cut` wants, and a sequence above RC_LONG by its guess.
template <typename T>
size_t recurrence_scratch(size_t nseq, size_t rows, size_t heads, size_t headdim, size_t dstate) {
  if (nseq == 0 || heads == 0 || headdim == 0 || dstate == 0 || dstate > 256) return 256;
  const size_t units = by_columns(dstate, [&](auto, auto least, auto most) {
    return heads * static_cast<size_t>(recurrence_cut(RC_CTAS, 0, heads, headdim, recurrence_held<T>, least.value, most.value).splits);
  });
  size_t sequences = (RC_CTAS - 1) / units, ranges = RC_CTAS / units + 1;
  if (sequences > nseq) sequences = nseq;
  if (sequences > 2 && sequences > 2 * rows / RC_LONG) sequences = 2 * rows / RC_LONG;
  if (ranges > rows / RC_RANGE) ranges = rows / RC_RANGE;
  if (sequences == 0 || rows <= RC_LONG) return 256;
  return (ranges + sequences) * heads * (headdim * dstate + 1) * sizeof(typename Acc<T>::type) + 256;
}

template <typename T>
void recurrence(const PromptArgs& g, void* scratch, StreamContext ctx) {
  using A = typename Acc<T>::type;
  constexpr size_t V = Pack<T>::N;
  Ranges r{nullptr, nullptr, 0, g.P % V == 0 && g.N % V == 0 && g.xp % V == 0 && g.bcp % V == 0 && mp_aligned16(g.x) && mp_aligned16(g.Bm) && mp_aligned16(g.Cm)};
  by_columns(g.N, [&](auto np, auto least, auto most) {
    constexpr int NP = decltype(np)::value, LEAST = decltype(least)::value, MOST = decltype(most)::value;
    const size_t nseq = g.q.nseq, heads = g.H;
    // (without scratch: whole sequences, as if there were no rows to cut)
    const Cut c = recurrence_cut(nseq, scratch != nullptr ? g.q.rows : 0, heads, g.P, recurrence_held<T>, LEAST, MOST);
    if (c.steps != 0) {
      r.steps = c.steps;
      r.local = scratch;
      r.decay = static_cast<A*>(scratch) + c.ids * heads * static_cast<size_t>(g.P) * g.N;
    }
    if constexpr (LEAST <= 8)
      if (c.lanes == 8) return recurrence_run<T, NP, 8>(g, r, c, ctx);
    if constexpr (MOST >= 16)
      if (c.lanes == 16) return recurrence_run<T, NP, 16>(g, r, c, ctx);
    if constexpr (MOST >= 32) recurrence_run<T, NP, 32>(g, r, c, ctx);
  });
}

template <typename T>
void ssd_scan_prompt_impl(const void* x, len_t x_pitch, const void* dt_raw, len_t dt_pitch, const void* dt_bias, const void* A_log, const void* Bm,
                          const void* Cm, len_t bc_pitch, void* states, const void* slots, const void* resume, const void* starts, void* y, len_t y_pitch,
                          void* scratch, len_t nseq, len_t rows, len_t nslots, len_t heads, len_t headdim, len_t dstate, len_t ngroups, StreamContext ctx) {
  if (ngroups == 0 || heads % ngroups != 0) MP_FATAL("ssd_scan_prompt: heads %lu not divisible by groups %lu", heads, ngroups);
  if (dstate == 0 || dstate > 256) MP_FATAL("ssd_scan_prompt: state size %lu (1 to 256)", dstate);
  if (!fits(nseq) || !fits(rows) || !fits(nslots) || !fits(heads, headdim) || !fits(ngroups, dstate) || headdim > SEQ_HEADDIM)
    MP_FATAL("ssd_scan_prompt: sequences, rows, slots and columns are counted in 31 bits");
  if (x_pitch < heads * headdim || y_pitch < heads * headdim || bc_pitch < ngroups * dstate || dt_pitch < heads) MP_FATAL("ssd_scan_prompt: a row pitch is below its columns");
  if (nseq == 0 || heads == 0 || headdim == 0) return;
  PromptArgs g{x, dt_raw, dt_bias, A_log, Bm, Cm, states, y, x_pitch, dt_pitch, bc_pitch, y_pitch,
               Sequences{static_cast<const int*>(starts), static_cast<const int*>(slots), static_cast<const int*>(resume), static_cast<int>(nseq),
                         static_cast<long long>(rows), static_cast<long long>(nslots)},
               static_cast<int>(heads), static_cast<int>(headdim), static_cast<int>(dstate), static_cast<int>(ngroups)};
  if (scratch != nullptr && !mp_aligned16(scratch)) MP_FATAL("ssd_scan_prompt: scratch must be 16-byte aligned");
  if constexpr (std::is_same<T, __half>::value) {
    if (mp_ssd_prompt_chunks_take(g)) {
      mp_ssd_prompt_chunks(g, scratch, ctx);
      return;
    }
  }
  recurrence<T>(g, scratch, ctx);
}

}  // namespace

extern "C" len_t mpSsdScanPromptScratchBytes(uint32_t dtype_key, len_t nseq, len_t rows, len_t heads, len_t headdim, len_t dstate, len_t ngroups) {
  (void)ngroups;
  if (dtype_key == MP_R64) return recurrence_scratch<double>(nseq, rows, heads, headdim, dstate);
  if (dtype_key != MP_R16) return recurrence_scratch<float>(nseq, rows, heads, headdim, dstate);
  // which form takes an r16 call is known when the addresses are
  const size_t chunks = mp_ssd_prompt_chunks_scratch(nseq, rows, heads, headdim, dstate), steps = recurrence_scratch<__half>(nseq, rows, heads, headdim, dstate);
  return chunks > steps ? chunks : steps;
}

MP_STAMP3(ssd_scan_prompt,
          (const void* x, len_t x_pitch, const void* dt_raw, len_t dt_pitch, const void* dt_bias, const void* A_log, const void* Bm, const void* Cm,
           len_t bc_pitch, void* states, const void* slots, const void* resume, const void* starts, void* y, len_t y_pitch, void* scratch, len_t nseq,
           len_t rows, len_t nslots, len_t heads, len_t headdim, len_t dstate, len_t ngroups, StreamContext ctx),
          (x, x_pitch, dt_raw, dt_pitch, dt_bias, A_log, Bm, Cm, bc_pitch, states, slots, resume, starts, y, y_pitch, scratch, nseq, rows, nslots, heads,
           headdim, dstate, ngroups, ctx))
