// The SSD scan over packed prompts that go on from a kept state (launch_ssd_scan_prompt_*):
//   dt = softplus(raw + dt_bias[h]),  a_t = exp(-dt_t exp(A_log[h])),  S_t = a_t S_{t-1} + dt_t x_t (x) B_t,  y_t = S_t C_t
// per sequence and head, S_{-1} the sequence's kept state or zero, the last S kept again.
#include "ssd_prompt.cuh"

namespace {

// ---------------------------------------------------------------------------
// The recurrence, step by step.  A warp has ROWS rows p of a state, PV to a lane group of eight, each lane NV of their columns in registers, so
// that nothing but B, C and x moves: they come through shared memory RT steps at a time, and the next steps' are fetched meanwhile.
// ---------------------------------------------------------------------------
constexpr int RC_LN = 8;

template <typename T, int NV, int WARPS>
struct RecurrenceSizes {
  using A = typename Acc<T>::type;
  static constexpr int PV = sizeof(A) == 8 ? 2 : 4;         // rows p of a lane: at most 128 registers of state
  static constexpr int ROWS = PV * (32 / RC_LN);
  static constexpr int NP = NV * RC_LN, THREADS = 32 * WARPS, PS = ROWS * WARPS;
  static constexpr int RT = sizeof(A) == 8 ? 8 : 16;        // steps at a time
  static constexpr size_t BYTES = sizeof(A) * (2 * RT * NP + RT * PS + RT);
};

template <typename T, int NV, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) recurrence_kernel(const PromptArgs g, int splits) {
  mp_grid_dependency();
  using Z = RecurrenceSizes<T, NV, WARPS>;
  using A = typename Z::A;
  constexpr int NP = Z::NP, RT = Z::RT, PS = Z::PS, THREADS = Z::THREADS, RC_PV = Z::PV;
  extern __shared__ __align__(16) unsigned char rc_smem[];
  A* sB = reinterpret_cast<A*>(rc_smem);      // [RT][NP], columns past N zero
  A* sC = sB + RT * NP;
  A* sx = sC + RT * NP;                       // [RT][PS]: dt x
  A* sa = sx + RT * PS;                       // [RT]: decay
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x % splits;
  const int sh = blockIdx.x / splits, s = sh / g.H, h = sh % g.H, grp = h / (g.H / g.G);
  const long long lo = seq_first(g.q, s), hi = seq_first(g.q, s + 1), slot = seq_slot(g.q.slots, g.q.nslots, s);
  if (slot < 0) return;
  const T* x = static_cast<const T*>(g.x) + static_cast<size_t>(h) * g.P;
  const T* raw = static_cast<const T*>(g.raw) + h;
  const T* Bm = static_cast<const T*>(g.Bm) + static_cast<size_t>(grp) * g.N;
  const T* Cm = static_cast<const T*>(g.Cm) + static_cast<size_t>(grp) * g.N;
  T* y = static_cast<T*>(g.y) + static_cast<size_t>(h) * g.P;
  const A bias = static_cast<const A*>(g.dt_bias)[h], rate = -seq_exp(static_cast<const A*>(g.A_log)[h]);
  const int pg = lane / RC_LN, nl = lane % RC_LN;
  const int pl = warp * Z::ROWS + pg * RC_PV, p0 = split * PS + pl;     // this lane's first row, in the CTA and in the head
  A* state = static_cast<A*>(g.states) + (slot * g.H + h) * static_cast<long long>(g.P) * g.N;
  // Columns nl, nl + 8, ... in pairs would conflict less, but a lane's columns are neighbours four at a time: 16-byte reads of B and C, the
  // eight lanes next to each other.
  A S[RC_PV][NV];
  const bool from_state = seq_resumes(g.q, s);
  auto column = [&](int i) { return (i / 4) * (4 * RC_LN) + nl * 4 + i % 4; };
#pragma unroll
  for (int p = 0; p < RC_PV; ++p)
#pragma unroll
    for (int i = 0; i < NV; ++i) S[p][i] = from_state && p0 + p < g.P && column(i) < g.N ? state[static_cast<size_t>(p0 + p) * g.N + column(i)] : A(0);

  for (long long t0 = lo; t0 < hi; t0 += RT) {
    const int steps = hi - t0 < RT ? static_cast<int>(hi - t0) : RT;
    __syncthreads();
    for (int i = tid; i < RT * NP; i += THREADS) {
      const int t = i / NP, n = i % NP;
      const bool in = t < steps && n < g.N;
      sB[i] = in ? mp_up(Bm[(t0 + t) * g.bcp + n]) : A(0);
      sC[i] = in ? mp_up(Cm[(t0 + t) * g.bcp + n]) : A(0);
    }
    for (int i = tid; i < RT * PS; i += THREADS) {
      const int t = i / PS, p = split * PS + i % PS;
      A v = A(0);
      if (t < steps && p < g.P) v = seq_softplus(mp_up(raw[(t0 + t) * g.rp]) + bias) * mp_up(x[(t0 + t) * g.xp + p]);
      sx[i] = v;
    }
    if (tid < RT) sa[tid] = tid < steps ? seq_exp(seq_softplus(mp_up(raw[(t0 + tid) * g.rp]) + bias) * rate) : A(1);
    __syncthreads();
    for (int t = 0; t < steps; ++t) {
      const A a = sa[t];
      A xd[RC_PV], out[RC_PV];
#pragma unroll
      for (int p = 0; p < RC_PV; ++p) { xd[p] = sx[t * PS + pl + p]; out[p] = A(0); }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const A b = sB[t * NP + column(i)], c = sC[t * NP + column(i)];
#pragma unroll
        for (int p = 0; p < RC_PV; ++p) {
          S[p][i] = a * S[p][i] + b * xd[p];
          out[p] += c * S[p][i];
        }
      }
#pragma unroll
      for (int p = 0; p < RC_PV; ++p) {
#pragma unroll
        for (int o = RC_LN / 2; o > 0; o >>= 1) out[p] += __shfl_xor_sync(0xffffffffu, out[p], o);
        if (nl == p && p0 + p < g.P) y[(t0 + t) * g.yp + p0 + p] = mp_down<T>(out[p]);
      }
    }
  }
#pragma unroll
  for (int p = 0; p < RC_PV; ++p)
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (p0 + p < g.P && column(i) < g.N) state[static_cast<size_t>(p0 + p) * g.N + column(i)] = S[p][i];
}

template <typename T, int NV, int WARPS>
void recurrence_run(const PromptArgs& g, StreamContext ctx) {
  using Z = RecurrenceSizes<T, NV, WARPS>;
  const int splits = (g.P + Z::PS - 1) / Z::PS;
  const long long ctas = static_cast<long long>(g.q.nseq) * g.H * splits;
  if (ctas > 0x7fffffffll) MP_FATAL("ssd_scan_prompt: too many sequences and heads for one launch");
  if (Z::BYTES > 48 * 1024)
    MP_CUDA_CHECK(cudaFuncSetAttribute(recurrence_kernel<T, NV, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Z::BYTES)));
  MpLaunch(static_cast<unsigned>(ctas), Z::THREADS, Z::BYTES, mp_stream(ctx))(recurrence_kernel<T, NV, WARPS>, g, splits);
  MP_LAUNCH_CHECK();
}

template <typename T, int NV>
void recurrence_warps(const PromptArgs& g, StreamContext ctx) {
  constexpr int ROWS = RecurrenceSizes<T, NV, 1>::ROWS;
  // CTAs of one warp fetch B and C once per ROWS rows of a head: only while there are not enough of them to fill the GPU
  const long long units = static_cast<long long>(g.q.nseq) * g.H * ((g.P + ROWS - 1) / ROWS);
  if (units >= 8ll * mp_sm_count(ctx) && g.P > 2 * ROWS) recurrence_run<T, NV, 4>(g, ctx);
  else if (units >= 4ll * mp_sm_count(ctx) && g.P > ROWS) recurrence_run<T, NV, 2>(g, ctx);
  else recurrence_run<T, NV, 1>(g, ctx);
}

template <typename T>
void recurrence(const PromptArgs& g, StreamContext ctx) {
  if (g.N <= 32) recurrence_warps<T, 4>(g, ctx);
  else if (g.N <= 64) recurrence_warps<T, 8>(g, ctx);
  else if (g.N <= 128) recurrence_warps<T, 16>(g, ctx);
  else recurrence_warps<T, 32>(g, ctx);
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
  if constexpr (std::is_same<T, __half>::value) {
    if (mp_ssd_prompt_chunks_take(g)) {
      if (scratch != nullptr && !mp_aligned16(scratch)) MP_FATAL("ssd_scan_prompt: scratch must be 16-byte aligned");
      mp_ssd_prompt_chunks(g, scratch, ctx);
      return;
    }
  }
  recurrence<T>(g, ctx);
}

}  // namespace

extern "C" len_t mpSsdScanPromptScratchBytes(uint32_t dtype_key, len_t nseq, len_t rows, len_t heads, len_t headdim, len_t dstate, len_t ngroups) {
  (void)ngroups;
  return dtype_key == MP_R16 ? static_cast<len_t>(mp_ssd_prompt_chunks_scratch(nseq, rows, heads, headdim, dstate)) : 256;
}

MP_STAMP3(ssd_scan_prompt,
          (const void* x, len_t x_pitch, const void* dt_raw, len_t dt_pitch, const void* dt_bias, const void* A_log, const void* Bm, const void* Cm,
           len_t bc_pitch, void* states, const void* slots, const void* resume, const void* starts, void* y, len_t y_pitch, void* scratch, len_t nseq,
           len_t rows, len_t nslots, len_t heads, len_t headdim, len_t dstate, len_t ngroups, StreamContext ctx),
          (x, x_pitch, dt_raw, dt_pitch, dt_bias, A_log, Bm, Cm, bc_pitch, states, slots, resume, starts, y, y_pitch, scratch, nseq, rows, nslots, heads,
           headdim, dstate, ngroups, ctx))
