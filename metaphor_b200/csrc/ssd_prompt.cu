// The SSD scan over packed prompts that go on from a kept state (launch_ssd_scan_prompt_*):
//   dt = softplus(raw + dt_bias[h]),  a_t = exp(-dt_t exp(A_log[h])),  S_t = a_t S_{t-1} + dt_t x_t (x) B_t,  y_t = S_t C_t
// per sequence and head, S_{-1} the sequence's kept state or zero, the last S kept again.
#include "ssd_prompt.cuh"

namespace {

// ---------------------------------------------------------------------------
// The recurrence, step by step, for every type and shape.  Eight lanes have PV rows p of a state, each lane NV of their columns in registers, so
// that nothing but B, C and x moves: they come through shared memory RT steps at a time, for the four warps of a CTA at once.  A step is three
// operations for every value of the state (decay, product, sum over the columns), two values to an instruction in fp32: bound by the fp32 pipe.
// Where the sequences and heads are too few for the GPU, long sequences are cut into ranges: first the states that all but the last ranges add
// (`STATES`: from zero, without y), then carried from range to range, then the ranges side by side from the states that they receive.
// ---------------------------------------------------------------------------
constexpr int RC_LN = 8;

template <typename T, int NV, int WARPS>
struct RecurrenceSizes {
  using A = typename Acc<T>::type;
  static constexpr int PV = (sizeof(A) == 8 ? 2 : 4) / (NV > 16 ? 2 : 1);      // rows p of a lane: 64 registers of state
  static constexpr int ROWS = PV * (32 / RC_LN);
  static constexpr int NP = NV * RC_LN, THREADS = 32 * WARPS, PS = ROWS * WARPS;
  static constexpr int RT = sizeof(A) == 8 ? 8 : 16;                           // steps at a time
  static constexpr size_t BYTES = sizeof(A) * (2 * RT * NP + RT * PS + 2 * RT);
};

struct Ranges {
  void* local;      // acc [id][head][P][N]: states that a range adds, later those that it receives
  void* decay;      // acc [id][head]: what is left of a state behind it
  int steps;        // of a range, 0: whole sequences
  bool packs;       // rows of x, B and C are whole 16-byte packs
};

// `rows` rows of NP values, 16 bytes at a time or one by one; zeros behind row `steps` and column `cols`.
template <typename T, int NP, int RT, int THREADS>
__device__ __forceinline__ void fetch_rows(typename Acc<T>::type* dst, const T* src, size_t pitch, int steps, int cols, bool packs) {
  using A = typename Acc<T>::type;
  constexpr int V = Pack<T>::N;
  if (packs && NP % V == 0) {
#pragma unroll
    for (int i = threadIdx.x; i < RT * NP / V; i += THREADS) {
      const int t = i / (NP / V), n = i % (NP / V) * V;
      A v[V] = {};
      if (t < steps && n < cols) unpack(ld_pack(src + t * pitch + n, 0), v);
#pragma unroll
      for (int e = 0; e < V; e += 16 / sizeof(A)) *reinterpret_cast<StVec<A, 16 / sizeof(A)>*>(dst + t * NP + n + e) = *reinterpret_cast<StVec<A, 16 / sizeof(A)>*>(v + e);
    }
  } else {
#pragma unroll 8
    for (int i = threadIdx.x; i < RT * NP; i += THREADS) {
      const int t = i / NP, n = i % NP;
      dst[i] = t < steps && n < cols ? mp_up(src[t * pitch + n]) : A(0);
    }
  }
}

template <typename T, int NV, int WARPS, bool STATES>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS) recurrence_kernel(const PromptArgs g, const Ranges ranges, int splits) {
  mp_grid_dependency();
  using Z = RecurrenceSizes<T, NV, WARPS>;
  using A = typename Z::A;
  constexpr int NP = Z::NP, RT = Z::RT, PS = Z::PS, THREADS = Z::THREADS, PV = Z::PV, CV = 16 / sizeof(A);      // columns side by side
  extern __shared__ __align__(16) unsigned char rc_smem[];
  A* sB = reinterpret_cast<A*>(rc_smem);      // [RT][NP], columns past N zero
  A* sC = sB + RT * NP;
  A* sx = sC + RT * NP;                       // [RT][PS]
  A* sa = sx + RT * PS;                       // [RT]: decay
  A* sdt = sa + RT;                           // [RT]: step size
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x % splits, idh = blockIdx.x / splits, h = idh % g.H, grp = h / (g.H / g.G);
  const Span sp = span_of(g.q, ranges.steps, idh / g.H);
  if (!sp.any || (STATES && sp.hi >= sp.seq_hi)) return;      // (nothing lies behind it)
  const T* x = static_cast<const T*>(g.x) + static_cast<size_t>(h) * g.P + split * PS;
  const T* raw = static_cast<const T*>(g.raw) + h;
  const T* Bm = static_cast<const T*>(g.Bm) + static_cast<size_t>(grp) * g.N;
  const T* Cm = static_cast<const T*>(g.Cm) + static_cast<size_t>(grp) * g.N;
  T* y = static_cast<T*>(g.y) + static_cast<size_t>(h) * g.P;
  const A bias = static_cast<const A*>(g.dt_bias)[h], rate = -seq_exp(static_cast<const A*>(g.A_log)[h]);
  const int pg = lane / RC_LN, nl = lane % RC_LN;
  const int pl = warp * Z::ROWS + pg * PV, p0 = split * PS + pl;     // this lane's first row, in the CTA and in the head
  A* state = static_cast<A*>(g.states) + (sp.slot * g.H + h) * static_cast<long long>(g.P) * g.N;
  A* local = static_cast<A*>(ranges.local) + static_cast<size_t>(idh) * g.P * g.N;
  // a lane's columns are neighbours CV at a time: 16-byte reads of B and C, the eight lanes next to each other
  A S[PV][NV / CV][CV];
  auto column = [&](int i, int e) { return (i * RC_LN + nl) * CV + e; };
  const bool received = !STATES && ranges.steps != 0 && sp.lo > sp.seq_lo, any = received || (!STATES && seq_resumes(g.q, sp.s));
  const A* from = received ? local : state;
#pragma unroll
  for (int p = 0; p < PV; ++p)
#pragma unroll
    for (int i = 0; i < NV / CV; ++i)
#pragma unroll
      for (int e = 0; e < CV; ++e) S[p][i][e] = any && p0 + p < g.P && column(i, e) < g.N ? from[static_cast<size_t>(p0 + p) * g.N + column(i, e)] : A(0);

  A left = A(1);
  for (long long t0 = sp.lo; t0 < sp.hi; t0 += RT) {
    const int steps = sp.hi - t0 < RT ? static_cast<int>(sp.hi - t0) : RT;
    __syncthreads();
    fetch_rows<T, NP, RT, THREADS>(sB, Bm + t0 * g.bcp, g.bcp, steps, g.N, ranges.packs);
    if (!STATES) fetch_rows<T, NP, RT, THREADS>(sC, Cm + t0 * g.bcp, g.bcp, steps, g.N, ranges.packs);
    fetch_rows<T, PS, RT, THREADS>(sx, x + t0 * g.xp, g.xp, steps, g.P - split * PS, ranges.packs);
    if (tid < RT) {
      const A dt = tid < steps ? seq_softplus(mp_up(raw[(t0 + tid) * g.rp]) + bias) : A(0);
      sdt[tid] = dt;
      sa[tid] = seq_exp(dt * rate);
    }
    __syncthreads();
    T* out = y + t0 * g.yp + p0;
#pragma unroll 1
    for (int t = 0; t < steps; ++t) {
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
          if (!STATES) fma_vec(sum[p], c.v, S[p][i], sum[p]);
        }
      }
      if (!STATES) {
        A total[PV];
#pragma unroll
        for (int p = 0; p < PV; ++p) {
          total[p] = sum[p][0];
#pragma unroll
          for (int e = 1; e < CV; ++e) total[p] += sum[p][e];
        }
        sum_rows<RC_LN, PV>(total, nl);
        constexpr int SHARED = RC_LN / PV;      // lanes with the same sum
        if (nl % SHARED == 0 && p0 + nl / SHARED < g.P) out[nl / SHARED] = mp_down<T>(total[0]);
        out += g.yp;
      }
    }
  }
  A* to = STATES ? local : state;
  if (!STATES && sp.hi < sp.seq_hi) return;
#pragma unroll
  for (int p = 0; p < PV; ++p)
#pragma unroll
    for (int i = 0; i < NV / CV; ++i)
#pragma unroll
      for (int e = 0; e < CV; ++e)
        if (p0 + p < g.P && column(i, e) < g.N) to[static_cast<size_t>(p0 + p) * g.N + column(i, e)] = S[p][i][e];
  if (STATES && split == 0 && tid == 0) static_cast<A*>(ranges.decay)[idh] = left;
}

// From range to range: what each adds is replaced by what it receives.  A thread has one value of a state, four ranges' on their way.
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

// Steps of a range, 0 for whole sequences.  The host knows how many sequences and rows there are, not how long each is.  `units`: CTAs for one
// sequence.  Two CTAs on each of 148 SMs keep the fp32 pipe fed: from there on whole sequences, since a range's state is made twice.  Otherwise
// four CTAs for each SM, of 32 steps at least (one CTA takes them in about the time of the launches).
int recurrence_range(size_t nseq, size_t rows, size_t units) {
  if (nseq * units >= 2 * 148) return 0;
  const size_t want = 4 * 148 / units + 1;
  size_t range = ((rows + want - 1) / want + 15) / 16 * 16;
  if (range < 32) range = 32;
  return range >= rows ? 0 : static_cast<int>(range);
}
size_t recurrence_ids(size_t nseq, size_t rows, int range) { return range == 0 ? nseq : rows / range + nseq; }

template <typename T, int NV>
int recurrence_warps(size_t headdim) {
  constexpr size_t ROWS = RecurrenceSizes<T, NV, 1>::ROWS;
  return headdim > 2 * ROWS ? 4 : headdim > ROWS ? 2 : 1;
}
template <typename T, int NV>
size_t recurrence_splits(size_t headdim) {
  const size_t rows = static_cast<size_t>(RecurrenceSizes<T, NV, 1>::ROWS) * recurrence_warps<T, NV>(headdim);
  return (headdim + rows - 1) / rows;
}

template <typename T, int NV, int WARPS>
void recurrence_run(const PromptArgs& g, const Ranges& r, StreamContext ctx) {
  using Z = RecurrenceSizes<T, NV, WARPS>;
  using A = typename Z::A;
  const int splits = static_cast<int>(recurrence_splits<T, NV>(g.P));
  const size_t ctas = recurrence_ids(g.q.nseq, g.q.rows, r.steps) * g.H * splits;
  if (ctas > 0x7fffffffull) MP_FATAL("ssd_scan_prompt: too many sequences and heads for one launch");
  auto go = [&](auto kernel) {
    if (Z::BYTES > 48 * 1024) MP_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Z::BYTES)));
    MpLaunch(static_cast<unsigned>(ctas), Z::THREADS, Z::BYTES, mp_stream(ctx))(kernel, g, r, splits);
    MP_LAUNCH_CHECK();
  };
  if (r.steps != 0) {
    go(recurrence_kernel<T, NV, WARPS, true>);
    const size_t parts = (static_cast<size_t>(g.P) * g.N + 255) / 256, carries = static_cast<size_t>(g.q.nseq) * g.H * parts;
    if (carries > 0x7fffffffull) MP_FATAL("ssd_scan_prompt: too many sequences and heads for one launch");
    MpLaunch(static_cast<unsigned>(carries), 256, 0, mp_stream(ctx))(recurrence_carry_kernel<A>, g, r, static_cast<int>(parts));
    MP_LAUNCH_CHECK();
  }
  go(recurrence_kernel<T, NV, WARPS, false>);
}

// what(columns of a lane)
template <typename F>
auto by_columns(size_t dstate, F what) {
  if (dstate <= 32) return what(std::integral_constant<int, 4>());
  if (dstate <= 64) return what(std::integral_constant<int, 8>());
  if (dstate <= 128) return what(std::integral_constant<int, 16>());
  return what(std::integral_constant<int, 32>());
}

template <typename T>
int recurrence_steps(size_t nseq, size_t rows, size_t heads, size_t headdim, size_t dstate) {
  return by_columns(dstate, [&](auto nv) { return recurrence_range(nseq, rows, heads * recurrence_splits<T, decltype(nv)::value>(headdim)); });
}
template <typename T>
size_t recurrence_scratch(size_t nseq, size_t rows, size_t heads, size_t headdim, size_t dstate) {
  if (nseq == 0 || heads == 0 || headdim == 0 || dstate == 0 || dstate > 256) return 256;
  const int range = recurrence_steps<T>(nseq, rows, heads, headdim, dstate);
  return range == 0 ? 256 : recurrence_ids(nseq, rows, range) * heads * (headdim * dstate + 1) * sizeof(typename Acc<T>::type) + 256;
}

template <typename T>
void recurrence(const PromptArgs& g, void* scratch, StreamContext ctx) {
  using A = typename Acc<T>::type;
  constexpr size_t V = Pack<T>::N;
  Ranges r{nullptr, nullptr, 0, g.P % V == 0 && g.N % V == 0 && g.xp % V == 0 && g.bcp % V == 0 && mp_aligned16(g.x) && mp_aligned16(g.Bm) && mp_aligned16(g.Cm)};
  if (scratch != nullptr) {
    r.steps = recurrence_steps<T>(g.q.nseq, g.q.rows, g.H, g.P, g.N);
    r.local = scratch;
    r.decay = static_cast<A*>(scratch) + recurrence_ids(g.q.nseq, g.q.rows, r.steps) * g.H * static_cast<size_t>(g.P) * g.N;
  }
  by_columns(g.N, [&](auto nv) {
    constexpr int NV = decltype(nv)::value;
    const int warps = recurrence_warps<T, NV>(g.P);
    if (warps == 4) recurrence_run<T, NV, 4>(g, r, ctx);
    else if (warps == 2) recurrence_run<T, NV, 2>(g, r, ctx);
    else recurrence_run<T, NV, 1>(g, r, ctx);
  });
}

bool fits(len_t v) { return v <= 0x7fffffffull; }

template <typename T>
void ssd_scan_prompt_impl(const void* x, len_t x_pitch, const void* dt_raw, len_t dt_pitch, const void* dt_bias, const void* A_log, const void* Bm,
                          const void* Cm, len_t bc_pitch, void* states, const void* slots, const void* resume, const void* starts, void* y, len_t y_pitch,
                          void* scratch, len_t nseq, len_t rows, len_t nslots, len_t heads, len_t headdim, len_t dstate, len_t ngroups, StreamContext ctx) {
  if (ngroups == 0 || heads % ngroups != 0) MP_FATAL("ssd_scan_prompt: heads %lu not divisible by groups %lu", heads, ngroups);
  if (x_pitch < heads * headdim || y_pitch < heads * headdim || bc_pitch < ngroups * dstate || dt_pitch < heads) MP_FATAL("ssd_scan_prompt: a row pitch is below its columns");
  if (!fits(nseq) || !fits(rows) || !fits(nslots) || !fits(heads * headdim)) MP_FATAL("ssd_scan_prompt: sequences, rows, slots and columns are counted in 31 bits");
  if (dstate == 0 || dstate > 256) MP_FATAL("ssd_scan_prompt: state size %lu (1 to 256)", dstate);
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
