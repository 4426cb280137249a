// The scan over packed prompts (see ssd_prompt.cu) for r16 tensors, in chunks of 128 steps on the tensor cores (tcgen05, accumulators in TMEM).
//
// With cum the inclusive sums of dt A inside a chunk, E their last one and S the state the chunk receives:
//   y_i = sum_{j <= i} (C_i . B_j) exp(cum_i - cum_j) dt_j x_j + exp(cum_i) S C_i          S' = exp(E) S + sum_j exp(E - cum_j) dt_j x_j (x) B_j
// Four products of 128 rows: G = C B^T, C S^T (128 x 64 x 128), W x with W the weighted scores, and B^T V with V the weighted x.  S stays in
// registers as fp32 values from chunk to chunk; where it, W or V is an operand, it is two r16 terms under one power of two (22 bits, down to
// 2^-38 of the largest value in the tile), so that y is an r16 rounding of fp32 sums and the kept state has fp32's accuracy to 2^-22 a term.
// x, B and C are r16 in memory and enter as they are.
//
// A CTA of eight warps walks one sequence of one head (64 of its rows p); two CTAs share an SM, so that one's products run beside the
// other's scaling.  Shared memory, 112 KB of tiles: C, B (two halves of 64 columns each), x, and one place for the terms of S, later those of V.
// TMEM, 256 columns: G, overwritten in place by W (the first operand of W x is read from there); C S^T, later B^T V; W x.
// Sequences too long and too few to fill the SMs are cut into ranges, whose own states are made first (states_kernel: B^T V alone), then carried
// from range to range (carry_kernel), then walked side by side.
//
// A chunk with an infinity or a NaN among its values does not go through the products, where a zero weight would spread it: it is taken step by
// step (chunk_plain).
#include "mp_tcgen05.cuh"
#include "ssd_prompt.cuh"

namespace {

constexpr int CQ = 128, CP = 64, CN = 128;      // steps, rows p and state columns of a tile
constexpr int CK_THREADS = 256;
constexpr int CK_HALF = CQ * 128;               // [128 rows][128 bytes], 128-byte swizzle
constexpr int CK_C = 0, CK_B = 2 * CK_HALF, CK_X = 4 * CK_HALF, CK_T = 5 * CK_HALF, CK_TAIL = 7 * CK_HALF;
struct ChunkTail {
  float colf[CQ];            // dt_j exp(l_end - l_j), l the sums inside a piece of eight steps
  float piece[CQ / 8];       // exp(sum over the piece)
  uint32_t most[4][8];       // per warp: largest |G|, |V|, |S|, dt as bits
  uint64_t bar[3];
  uint32_t tmem;
  int abort;
};
constexpr int CK_SMEM = CK_TAIL + 1024;
static_assert(sizeof(ChunkTail) <= 1024, "two CTAs on an SM have 113 KB each");
constexpr uint32_t TM_G = 0, TM_Y0 = 128, TM_Y1 = 192, TM_COLS = 256;

__device__ __forceinline__ uint32_t ck_at(int row, int piece16) { return row * 128 + ((piece16 ^ (row & 7)) << 4); }
__device__ __forceinline__ void ck_cp_async(uint32_t dst, const void* src, bool in) {      // 16 bytes, zeros where `in` is false
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ck_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void ck_cp_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ uint4 ck_ld(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void ck_st(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float2 ck_f2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
// Two values as r16 terms: the rounded values and the rounded rest.
__device__ __forceinline__ void ck_split(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
// The power of two that takes the largest value (its bits) to [2^13, 2^14), and its inverse.
struct Scale { float up, down; };
__device__ __forceinline__ Scale ck_scale(uint32_t most) {
  int k = most == 0 ? 0 : 13 - (static_cast<int>(most >> 23) - 127);
  k = k > 120 ? 120 : k < -120 ? -120 : k;
  return {__int_as_float((127 + k) << 23), __int_as_float((127 - k) << 23)};
}
__device__ __forceinline__ bool ck_infinite(uint32_t bits) { return bits >= 0x7f800000u; }

struct ChunkArgs {
  PromptArgs g;
  float* local;        // ranges: [id][unit][64 p][128 n] states that a range adds, later those that it receives
  float* decay;        // ranges: [id][unit] what is left of a state behind it
  int range;           // steps of a range, 0: whole sequences
  int slices;          // of 64 rows p in a head
  uint32_t* status;
};

// Which steps a CTA has.  Ranges are numbered without a table: sequence s has the numbers from starts[s] / range + s on, which is at least as
// many as it has ranges.
struct Span { int s; long long lo, hi, seq_lo, seq_hi, slot; bool any; };
__device__ __forceinline__ Span span_of(const ChunkArgs& a, int id) {
  Span r;
  if (a.range == 0) {
    r.s = id;
  } else {
    const long long range = a.range;
    r.s = warp_last_not_above(a.g.q.nseq - 1, id, [&](int i) { return seq_first(a.g.q, i) / range + i; });
    if (r.s < 0) { r.s = 0; r.any = false; return r; }
  }
  r.seq_lo = seq_first(a.g.q, r.s);
  r.seq_hi = seq_first(a.g.q, r.s + 1);
  r.slot = seq_slot(a.g.q.slots, a.g.q.nslots, r.s);
  if (a.range == 0) {
    r.lo = r.seq_lo;
    r.hi = r.seq_hi;
    r.any = r.slot >= 0;
  } else {
    const long long j = id - (r.seq_lo / a.range + r.s);
    r.lo = r.seq_lo + j * a.range;
    r.hi = min(r.lo + a.range, r.seq_hi);
    r.any = r.slot >= 0 && (r.lo < r.seq_hi || j == 0);
  }
  return r;
}

// What the two walks share: a thread's row (step, or state column n) and half of the 64 rows p; the fetch of a chunk; its step sizes.
struct Lane { int warp, lane, row, half; };
__device__ __forceinline__ Lane lane_of() {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  return {warp, lane, (warp & 3) * 32 + lane, warp >> 2};
}
// 128 rows of `cols` r16 values into halves of 64 columns; rows past `rows` and columns past `cols` become zeros.
template <int HALVES>
__device__ __forceinline__ void fetch_tile(uint32_t dst, const __half* src, size_t pitch, int rows, int cols) {
#pragma unroll
  for (int k = 0; k < CQ * 8 * HALVES / CK_THREADS; ++k) {
    const int i = k * CK_THREADS + threadIdx.x, r = i / (8 * HALVES), c = i % (8 * HALVES);
    const bool in = r < rows && c * 8 < cols;
    ck_cp_async(dst + (c >> 3) * CK_HALF + ck_at(r, c & 7), in ? src + r * pitch + c * 8 : src, in);
  }
}

// Step sizes of a chunk.  A thread has step `row`: dt, l = sum of dt A from its piece's first step on, and the piece's sum.  r64, because their
// differences count: behind steps of strong decay a sum has no digits left in r32 for one of weak decay.
struct StepSizes {
  float dt;
  double l, end;
  __device__ __forceinline__ float behind() const { return expf(static_cast<float>(end - l)); }      // decay from this step to the end of its piece
};
__device__ __forceinline__ StepSizes step_sizes(float raw, float bias, float rate, bool in, int lane) {
  StepSizes s;
  s.dt = in ? seq_softplus(raw + bias) : 0.f;
  s.l = static_cast<double>(s.dt) * static_cast<double>(rate);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, s.l, o, 8);
    if ((lane & 7) >= o) s.l += up;
  }
  s.end = __shfl_sync(0xffffffffu, s.l, 7, 8);
  return s;
}
__device__ __forceinline__ uint32_t warp_most(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint32_t cta_most(const uint32_t* most) {
  uint32_t m = most[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) m = max(m, most[w]);
  return m;
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// This thread's 32 values of row `row` of the x tile, and the largest of their magnitudes (NaN above all).
__device__ __forceinline__ float load_x(uint32_t tile, const Lane& t, uint4 (&x)[4]) {
  __half2 m = __float2half2_rn(0.f);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[k] = ck_ld(tile + ck_at(t.row, t.half * 4 + k));
    const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&w[e])));
  }
  const float2 f = __half22float2(m);
  return f.x != f.x || f.y != f.y ? __int_as_float(0x7fffffff) : fmaxf(f.x, f.y);
}
// V = x w in two terms, each a [128][64] tile.
__device__ __forceinline__ void store_v(uint32_t tile, const Lane& t, const uint4 (&x)[4], float w) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t in[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = ck_f2(in[e]);
      ck_split(f.x * w, f.y * w, hi[e], lo[e]);
    }
    const uint32_t at = tile + ck_at(t.row, t.half * 4 + k);
    ck_st(at, make_uint4(hi[0], hi[1], hi[2], hi[3]));
    ck_st(at + CK_HALF, make_uint4(lo[0], lo[1], lo[2], lo[3]));
  }
}
// S in two terms the same way: this thread's row is a state column n.
__device__ __forceinline__ void store_s(uint32_t tile, const Lane& t, const float (&S)[32], float up) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) ck_split(S[k * 8 + 2 * e] * up, S[k * 8 + 2 * e + 1] * up, hi[e], lo[e]);
    const uint32_t at = tile + ck_at(t.row, t.half * 4 + k);
    ck_st(at, make_uint4(hi[0], hi[1], hi[2], hi[3]));
    ck_st(at + CK_HALF, make_uint4(lo[0], lo[1], lo[2], lo[3]));
  }
}
__device__ __forceinline__ uint32_t most_of(const float (&S)[32]) {
  uint32_t m = 0;
#pragma unroll
  for (int p = 0; p < 32; ++p) m = max(m, abs_bits(S[p]));
  return m;
}

// A chunk step by step, for values that the products would spread.  The thread has S[n = row][p = 32 half ..]; y_p is summed over a warp's 32
// columns n lane against lane, then over the four warps through shared memory.  OUT: with y.
template <bool OUT>
__device__ __noinline__ void chunk_plain_steps(unsigned char* smem, uint32_t base, const Lane t, float* state, float dt, float rate, int steps, __half* y, size_t yp,
                                         int pcols) {
  float* sdt = reinterpret_cast<float*>(smem + CK_T);                   // the place of the terms, which no product reads now
  float* part = sdt + CQ;                                               // [4][64]
  float S[32];
#pragma unroll
  for (int p = 0; p < 32; ++p) S[p] = state[p];
  __syncthreads();
  if (t.half == 0) sdt[t.row] = dt;
  __syncthreads();
  for (int i = 0; i < steps; ++i) {
    const float d = sdt[i], a = expf(d * rate);
    const uint32_t col = (t.row >> 6) * CK_HALF + ck_at(i, (t.row & 63) >> 3) + (t.row & 7) * 2;
    const float b = __half2float(*reinterpret_cast<const __half*>(smem + CK_B + col));
    const float c = OUT ? __half2float(*reinterpret_cast<const __half*>(smem + CK_C + col)) : 0.f;
    float v[32];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint4 x = ck_ld(base + CK_X + ck_at(i, t.half * 4 + k));
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = ck_f2(w[e]);
        const int p = k * 8 + 2 * e;
        S[p] = a * S[p] + d * f.x * b;
        S[p + 1] = a * S[p + 1] + d * f.y * b;
        v[p] = c * S[p];
        v[p + 1] = c * S[p + 1];
      }
    }
    if (OUT) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int p = 0; p < o; ++p) {
          const bool up = (t.lane & o) != 0;
          const float send = up ? v[p] : v[p + o], keep = up ? v[p + o] : v[p];
          v[p] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      part[(t.warp & 3) * 64 + t.half * 32 + t.lane] = v[0];
      __syncthreads();
      if (threadIdx.x < CP && static_cast<int>(threadIdx.x) < pcols)
        y[i * yp + threadIdx.x] = __float2half_rn(part[threadIdx.x] + part[64 + threadIdx.x] + part[128 + threadIdx.x] + part[192 + threadIdx.x]);
      __syncthreads();
    }
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < 32; ++p) state[p] = S[p];
}
template <bool OUT>      // (a copy goes through memory, so that S itself stays in registers)
__device__ __forceinline__ void chunk_plain(unsigned char* smem, uint32_t base, const Lane& t, float (&S)[32], float dt, float rate, int steps, __half* y, size_t yp,
                                            int pcols) {
  float copy[32];
#pragma unroll
  for (int p = 0; p < 32; ++p) copy[p] = S[p];
  chunk_plain_steps<OUT>(smem, base, t, copy, dt, rate, steps, y, yp, pcols);
#pragma unroll
  for (int p = 0; p < 32; ++p) S[p] = copy[p];
}

// ---------------------------------------------------------------------------
// The walk.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(CK_THREADS, 2) chunk_walk_kernel(const ChunkArgs a) {
  extern __shared__ __align__(1024) unsigned char ck_smem[];
  ChunkTail* tail = reinterpret_cast<ChunkTail*>(ck_smem + CK_TAIL);
  const PromptArgs& g = a.g;
  const Lane t = lane_of();
  const uint32_t base = mp_smem_u32(ck_smem);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 3; ++i) mbar_init(tail->bar + i, 1);
    mbar_fence_init();
    tail->abort = 0;
  }
  mp_grid_wait();
  const int units = g.H * a.slices;
  const int id = blockIdx.x / units, unit = blockIdx.x % units, h = unit / a.slices, p0 = unit % a.slices * CP, grp = h / (g.H / g.G);
  const Span sp = span_of(a, id);
  if (!sp.any) { mp_launch_dependents(); return; }
  if (t.warp == 0) tmem_alloc(&tail->tmem, TM_COLS);
  const int pcols = min(CP, g.P - p0);
  const __half* x = static_cast<const __half*>(g.x) + static_cast<size_t>(h) * g.P + p0;
  const __half* raw = static_cast<const __half*>(g.raw) + h;
  const __half* Bm = static_cast<const __half*>(g.Bm) + static_cast<size_t>(grp) * g.N;
  const __half* Cm = static_cast<const __half*>(g.Cm) + static_cast<size_t>(grp) * g.N;
  __half* y = static_cast<__half*>(g.y) + static_cast<size_t>(h) * g.P + p0;
  float* state = static_cast<float*>(g.states) + ((sp.slot * g.H + h) * g.P + p0) * static_cast<long long>(g.N);
  const float bias = static_cast<const float*>(g.dt_bias)[h], rate = -expf(static_cast<const float*>(g.A_log)[h]);

  auto fetch = [&](long long t0, int steps) {
    fetch_tile<2>(base + CK_C, Cm + t0 * g.bcp, g.bcp, steps, g.N);
    fetch_tile<2>(base + CK_B, Bm + t0 * g.bcp, g.bcp, steps, g.N);
    fetch_tile<1>(base + CK_X, x + t0 * g.xp, g.xp, steps, pcols);
    ck_cp_commit();
  };
  auto steps_at = [&](long long t0) { return sp.hi - t0 < CQ ? static_cast<int>(sp.hi - t0) : CQ; };
  float raw_next = 0.f;
  auto fetch_raw = [&](long long t0) { raw_next = t0 + t.row < sp.hi ? __half2float(raw[(t0 + t.row) * g.rp]) : 0.f; };
  if (sp.lo < sp.hi) {
    fetch(sp.lo, steps_at(sp.lo));
    fetch_raw(sp.lo);
  }
  // the state that the span receives: this thread's column n = row, rows p = 32 half ..
  float S[32];
  {
    const float* from = nullptr;
    long long pitch = g.N;
    if (a.range != 0 && sp.lo > sp.seq_lo) {
      from = a.local + (static_cast<size_t>(id) * units + unit) * CP * CN;
      pitch = CN;
    } else if (seq_resumes(g.q, sp.s)) {
      from = state;
    }
#pragma unroll
    for (int p = 0; p < 32; ++p) S[p] = from != nullptr && t.row < g.N && t.half * 32 + p < pcols ? from[(t.half * 32 + p) * pitch + t.row] : 0.f;
  }
  auto publish = [&]() {      // S becomes an operand of the next chunk: its terms under one power of two
    const uint32_t m = warp_most(most_of(S));
    if (t.lane == 0) tail->most[2][t.warp] = m;
    __syncthreads();
    const uint32_t most = cta_most(tail->most[2]);
    if (!ck_infinite(most)) store_s(base + CK_T, t, S, ck_scale(most).up);
    return most;
  };
  uint32_t s_most = publish();

  const uint64_t d_c = umma_smem_desc(base + CK_C, 16, 1024), d_b = umma_smem_desc(base + CK_B, 16, 1024), d_bt = umma_smem_desc(base + CK_B, CK_HALF, 1024);
  const uint64_t d_x = umma_smem_desc(base + CK_X, CK_HALF, 1024), d_t = umma_smem_desc(base + CK_T, CK_HALF, 1024);
  constexpr uint32_t id_g = umma_instr_desc(UMMA_FMT_F16, 0, 0, 128, 128), id_y = umma_instr_desc(UMMA_FMT_F16, 0, 1, 128, CP), id_s = umma_instr_desc(UMMA_FMT_F16, 1, 1, 128, CP);
  constexpr uint32_t HALF_U = CK_HALF / 16, ROWS_U = 16 * 128 / 16;
  auto kslice = [](int ks) { return static_cast<uint32_t>((ks >> 2) * HALF_U + (ks & 3) * 2); };
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem = tail->tmem, tq = tmem + (static_cast<uint32_t>(t.warp & 3) << 21);      // this warp's 32 lanes
  uint32_t issued = 0, finished = 0;      // phases of the barriers: scores and C S^T, the other two products
  const bool odd = !(fabsf(rate) < INFINITY);
  for (long long t0 = sp.lo; t0 < sp.hi; t0 += CQ) {
    const int steps = steps_at(t0);
    const bool carried = s_most != 0, products = !odd && !ck_infinite(s_most);
    ck_cp_wait();
    fence_proxy_async_smem();
    tcgen05_fence_before_sync();
    __syncthreads();
    if (tail->abort != 0) break;      // a wait ran out
    tcgen05_fence_after_sync();
    if (t.warp == 0 && products && elect_one()) {
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) umma<false>(tmem + TM_G, d_c + kslice(ks), d_b + kslice(ks), id_g, ks != 0 ? 1u : 0u);
      umma_commit(tail->bar + 0);
      if (carried) {
#pragma unroll
        for (int ks = 0; ks < 16; ++ks)
          umma<false>(tmem + TM_Y0, d_c + kslice(ks & 7), d_t + (ks >> 3) * HALF_U + (ks & 7) * ROWS_U, id_y, ks != 0 ? 1u : 0u);
      }
      umma_commit(tail->bar + 1);
    }
    __syncwarp();
    const StepSizes z = step_sizes(raw_next, bias, rate, t.row < steps, t.lane);
    if (t.half == 0) {
      tail->colf[t.row] = z.dt * z.behind();
      if ((t.lane & 7) == 7) tail->piece[t.row >> 3] = expf(static_cast<float>(z.end));
    }
    uint4 xv[4];
    const float x_most = load_x(base + CK_X, t, xv);
    const uint32_t vm = warp_most(abs_bits(x_most * z.dt)), dm = warp_most(abs_bits(z.dt));
    if (t.lane == 0) { tail->most[1][t.warp] = vm; tail->most[3][t.warp] = dm; }
    if (products) {
      (void)mbar_wait_abortable(tail->bar + 0, issued, a.status, &tail->abort);
      tcgen05_fence_after_sync();
      uint32_t gm = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t v[16];
        tmem_ld_32x16(tq + TM_G + (2 * b + t.half) * 16, v);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) gm = max(gm, v[e] & 0x7fffffffu);
      }
      gm = warp_most(gm);
      if (t.lane == 0) tail->most[0][t.warp] = gm;
      (void)mbar_wait_abortable(tail->bar + 1, issued, a.status, &tail->abort);
      tcgen05_fence_after_sync();
      issued ^= 1;
    }
    __syncthreads();
    // bounds of V and W: the weights that are left out of them are at most one
    const uint32_t v_most = cta_most(tail->most[1]);
    const uint32_t w_most = products ? abs_bits(__uint_as_float(cta_most(tail->most[0])) * __uint_as_float(cta_most(tail->most[3]))) : 0u;
    float after = 1.f, total = 1.f, before = 1.f;      // decay behind this thread's piece, of the chunk, and up to this step
#pragma unroll
    for (int k = 0; k < CQ / 8; ++k) {
      const float d = tail->piece[k];
      total *= d;
      if (k > (t.row >> 3)) after *= d;
      if (k < (t.row >> 3)) before *= d;
    }
    before *= expf(static_cast<float>(z.l));
    if (!products || ck_infinite(v_most) || ck_infinite(w_most)) {
      chunk_plain<true>(ck_smem, base, t, S, z.dt, rate, steps, y + t0 * g.yp, g.yp, pcols);
    } else {
      const Scale sv = ck_scale(v_most), sw = ck_scale(w_most);
      store_v(base + CK_T, t, xv, z.dt * z.behind() * after * sv.up);
      float y0[32];
      if (carried) {
        tmem_ld_32x32(tq + TM_Y0 + t.half * 32, reinterpret_cast<uint32_t*>(y0));
        tmem_ld_wait();
        const float f = before * ck_scale(s_most).down;
#pragma unroll
        for (int p = 0; p < 32; ++p) y0[p] *= f;
      } else {
#pragma unroll
        for (int p = 0; p < 32; ++p) y0[p] = 0.f;
      }
      // W over G: sixteen columns of scores become eight of the upper terms and eight of the lower ones
      float diag[8];      // this row's weights inside its own piece
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double lj = __shfl_sync(0xffffffffu, z.l, e, 8);
        const float dj = __shfl_sync(0xffffffffu, z.dt, e, 8);
        diag[e] = e <= (t.lane & 7) ? dj * expf(static_cast<float>(z.l - lj)) * sw.up : 0.f;
      }
      const int mine = t.row >> 3;
      const float enter = expf(static_cast<float>(z.l)) * sw.up;      // towards the end of the piece before
      float far = 0.f;
#pragma unroll 1
      for (int blk = 7; blk >= 0; --blk) {
        const bool here = (blk & 1) == t.half, none = blk > 2 * (t.warp & 3) + 1;
        uint32_t v[16], w[16];
        if (here && !none) {
          tmem_ld_32x16(tq + TM_G + blk * 16, v);
          tmem_ld_wait();
        }
#pragma unroll
        for (int hp = 1; hp >= 0; --hp) {
          const int piece = 2 * blk + hp;
          if (mine == piece + 1) far = enter;
          if (here && !none) {
            const float4 c0 = *reinterpret_cast<const float4*>(tail->colf + piece * 8), c1 = *reinterpret_cast<const float4*>(tail->colf + piece * 8 + 4);
            const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w0 = mine == piece ? diag[2 * e] : far * c[2 * e], w1 = mine == piece ? diag[2 * e + 1] : far * c[2 * e + 1];
              ck_split(__uint_as_float(v[hp * 8 + 2 * e]) * w0, __uint_as_float(v[hp * 8 + 2 * e + 1]) * w1, w[hp * 4 + e], w[8 + hp * 4 + e]);
            }
          }
          far *= tail->piece[piece];
        }
        if (here) {
          if (none) {
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = 0;
          }
          tmem_st_32x16(tq + TM_G + blk * 16, w);
        }
      }
      tmem_st_wait();
      fence_proxy_async_smem();
      tcgen05_fence_before_sync();
      __syncthreads();
      tcgen05_fence_after_sync();
      if (t.warp == 0 && elect_one()) {
#pragma unroll
        for (int ks = 0; ks < 16; ++ks)
          umma_f16_ta(tmem + TM_Y1, tmem + TM_G + (ks & 7) * 16 + (ks >> 3) * 8, d_x + (ks & 7) * ROWS_U, id_y, ks != 0 ? 1u : 0u);
#pragma unroll
        for (int ks = 0; ks < 16; ++ks)
          umma<false>(tmem + TM_Y0, d_bt + (ks & 7) * ROWS_U, d_t + (ks >> 3) * HALF_U + (ks & 7) * ROWS_U, id_s, ks != 0 ? 1u : 0u);
        umma_commit(tail->bar + 2);
      }
      __syncwarp();
      (void)mbar_wait_abortable(tail->bar + 2, finished, a.status, &tail->abort);
      finished ^= 1;
      tcgen05_fence_after_sync();
      {
        float v[32];
        tmem_ld_32x32(tq + TM_Y1 + t.half * 32, reinterpret_cast<uint32_t*>(v));
        tmem_ld_wait();
        if (t.row < steps) {
          __half* out = y + (t0 + t.row) * g.yp + t.half * 32;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int p = k * 8 + 2 * e;
              const __half2 hv = __floats2half2_rn(y0[p] + v[p] * sw.down, y0[p + 1] + v[p + 1] * sw.down);
              o[e] = *reinterpret_cast<const uint32_t*>(&hv);
            }
            if (t.half * 32 + k * 8 < pcols) *reinterpret_cast<uint4*>(out + k * 8) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
        tmem_ld_32x32(tq + TM_Y0 + t.half * 32, reinterpret_cast<uint32_t*>(v));
        tmem_ld_wait();
#pragma unroll
        for (int p = 0; p < 32; ++p) S[p] = total * S[p] + v[p] * sv.down;
      }
    }
    if (t0 + CQ < sp.hi) {
      __syncthreads();      // plain: every thread has read the tiles
      fetch(t0 + CQ, steps_at(t0 + CQ));
      fetch_raw(t0 + CQ);
      s_most = publish();
    }
  }
  mp_launch_dependents();
  if (sp.hi == sp.seq_hi && t.row < g.N) {
#pragma unroll
    for (int p = 0; p < 32; ++p)
      if (t.half * 32 + p < pcols) state[(t.half * 32 + p) * static_cast<long long>(g.N) + t.row] = S[p];
  }
  ck_cp_wait();
  tcgen05_fence_before_sync();
  __syncthreads();
  if (t.warp == 0) tmem_dealloc(tmem, TM_COLS);
}

// ---------------------------------------------------------------------------
// Ranges of long sequences: the state that a range adds, from B^T V alone, and what its decay leaves of the one before.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(CK_THREADS, 2) chunk_states_kernel(const ChunkArgs a) {
  extern __shared__ __align__(1024) unsigned char ck_smem[];
  ChunkTail* tail = reinterpret_cast<ChunkTail*>(ck_smem + CK_TAIL);
  const PromptArgs& g = a.g;
  const Lane t = lane_of();
  const uint32_t base = mp_smem_u32(ck_smem);
  if (threadIdx.x == 0) {
    mbar_init(tail->bar + 2, 1);
    mbar_fence_init();
    tail->abort = 0;
  }
  mp_grid_wait();
  const int units = g.H * a.slices;
  const int id = blockIdx.x / units, unit = blockIdx.x % units, h = unit / a.slices, p0 = unit % a.slices * CP, grp = h / (g.H / g.G);
  const Span sp = span_of(a, id);
  if (!sp.any || sp.hi >= sp.seq_hi) { mp_launch_dependents(); return; }      // nothing lies behind it
  if (t.warp == 0) tmem_alloc(&tail->tmem, CP);
  const int pcols = min(CP, g.P - p0);
  const __half* x = static_cast<const __half*>(g.x) + static_cast<size_t>(h) * g.P + p0;
  const __half* raw = static_cast<const __half*>(g.raw) + h;
  const __half* Bm = static_cast<const __half*>(g.Bm) + static_cast<size_t>(grp) * g.N;
  const float bias = static_cast<const float*>(g.dt_bias)[h], rate = -expf(static_cast<const float*>(g.A_log)[h]);
  float raw_next = 0.f;
  auto fetch = [&](long long t0) {      // whole chunks: a range that others follow is a multiple of them
    fetch_tile<2>(base + CK_B, Bm + t0 * g.bcp, g.bcp, CQ, g.N);
    fetch_tile<1>(base + CK_X, x + t0 * g.xp, g.xp, CQ, pcols);
    ck_cp_commit();
    raw_next = __half2float(raw[(t0 + t.row) * g.rp]);
  };
  fetch(sp.lo);
  float S[32], left = 1.f;
#pragma unroll
  for (int p = 0; p < 32; ++p) S[p] = 0.f;
  const uint64_t d_bt = umma_smem_desc(base + CK_B, CK_HALF, 1024), d_t = umma_smem_desc(base + CK_T, CK_HALF, 1024);
  constexpr uint32_t id_s = umma_instr_desc(UMMA_FMT_F16, 1, 1, 128, CP), HALF_U = CK_HALF / 16, ROWS_U = 16 * 128 / 16;
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem = tail->tmem, tq = tmem + (static_cast<uint32_t>(t.warp & 3) << 21);
  uint32_t finished = 0;
  const bool odd = !(fabsf(rate) < INFINITY);
  for (long long t0 = sp.lo; t0 < sp.hi; t0 += CQ) {
    ck_cp_wait();
    fence_proxy_async_smem();
    __syncthreads();
    if (tail->abort != 0) break;
    const StepSizes z = step_sizes(raw_next, bias, rate, true, t.lane);
    if (t.half == 0 && (t.lane & 7) == 7) tail->piece[t.row >> 3] = expf(static_cast<float>(z.end));
    uint4 xv[4];
    const float x_most = load_x(base + CK_X, t, xv);
    uint32_t bm = 0;      // an infinity in B, against the two terms of V, would be a NaN
    {
      __half2 m = __float2half2_rn(0.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint4 b = ck_ld(base + CK_B + t.half * CK_HALF + ck_at(t.row, k));
        const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&w[e])));
      }
      const float2 f = __half22float2(m);
      if (!(f.x < INFINITY && f.y < INFINITY)) bm = 0x7fffffffu;
    }
    const uint32_t vm = warp_most(max(bm, abs_bits(x_most * z.dt)));
    if (t.lane == 0) tail->most[1][t.warp] = vm;
    __syncthreads();
    const uint32_t v_most = cta_most(tail->most[1]);
    float after = 1.f, total = 1.f;
#pragma unroll
    for (int k = 0; k < CQ / 8; ++k) {
      const float d = tail->piece[k];
      total *= d;
      if (k > (t.row >> 3)) after *= d;
    }
    left *= total;
    if (odd || ck_infinite(v_most)) {
      chunk_plain<false>(ck_smem, base, t, S, z.dt, rate, CQ, nullptr, 0, pcols);
    } else {
      const Scale sv = ck_scale(v_most);
      store_v(base + CK_T, t, xv, z.dt * z.behind() * after * sv.up);
      fence_proxy_async_smem();
      tcgen05_fence_before_sync();
      __syncthreads();
      tcgen05_fence_after_sync();
      if (t.warp == 0 && elect_one()) {
#pragma unroll
        for (int ks = 0; ks < 16; ++ks)
          umma<false>(tmem, d_bt + (ks & 7) * ROWS_U, d_t + (ks >> 3) * HALF_U + (ks & 7) * ROWS_U, id_s, ks != 0 ? 1u : 0u);
        umma_commit(tail->bar + 2);
      }
      __syncwarp();
      (void)mbar_wait_abortable(tail->bar + 2, finished, a.status, &tail->abort);
      finished ^= 1;
      tcgen05_fence_after_sync();
      float v[32];
      tmem_ld_32x32(tq + t.half * 32, reinterpret_cast<uint32_t*>(v));
      tmem_ld_wait();
#pragma unroll
      for (int p = 0; p < 32; ++p) S[p] = total * S[p] + v[p] * sv.down;
    }
    if (t0 + CQ < sp.hi) {
      __syncthreads();
      fetch(t0 + CQ);
    }
  }
  mp_launch_dependents();
  const size_t at = static_cast<size_t>(id) * units + unit;
#pragma unroll
  for (int p = 0; p < 32; ++p) a.local[at * CP * CN + (t.half * 32 + p) * CN + t.row] = S[p];
  // not zero, however many steps: an infinite state stays infinite then, as it does step by step
  if (threadIdx.x == 0) a.decay[at] = fmaxf(left, __int_as_float(1));
  ck_cp_wait();
  tcgen05_fence_before_sync();
  __syncthreads();
  if (t.warp == 0) tmem_dealloc(tmem, CP);
}

// From range to range: what each adds is replaced by what it receives.  A thread has four neighbouring values of a state.
constexpr int CR_PARTS = CP * CN / 4 / 256;
__global__ void __launch_bounds__(256) chunk_carry_kernel(const ChunkArgs a) {
  mp_grid_dependency();
  const PromptArgs& g = a.g;
  const int units = g.H * a.slices;
  const int part = blockIdx.x % CR_PARTS, su = blockIdx.x / CR_PARTS, s = su / units, unit = su % units, h = unit / a.slices, p0 = unit % a.slices * CP;
  const long long lo = seq_first(g.q, s), hi = seq_first(g.q, s + 1), slot = seq_slot(g.q.slots, g.q.nslots, s);
  const long long ranges = (hi - lo + a.range - 1) / a.range;
  if (slot < 0 || ranges < 2) return;
  const int e = (part * 256 + threadIdx.x) * 4, p = e / CN, n = e % CN;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (seq_resumes(g.q, s) && p0 + p < g.P) {
    const float* state = static_cast<const float*>(g.states) + ((slot * g.H + h) * g.P + p0 + p) * static_cast<long long>(g.N);
    if (n < g.N) v.x = state[n];
    if (n + 1 < g.N) v.y = state[n + 1];
    if (n + 2 < g.N) v.z = state[n + 2];
    if (n + 3 < g.N) v.w = state[n + 3];
  }
  const size_t first = (static_cast<size_t>(lo / a.range + s)) * units + unit;
  auto place = [&](long long j) { return reinterpret_cast<float4*>(a.local + (first + j * units) * CP * CN + e); };
  float4 add = *place(0);
  for (long long j = 0; j + 1 < ranges; ++j) {
    const float left = a.decay[first + j * units];
    const float4 now = add;
    if (j + 2 < ranges) add = *place(j + 1);
    v.x = left * v.x + now.x;
    v.y = left * v.y + now.y;
    v.z = left * v.z + now.z;
    v.w = left * v.w + now.w;
    *place(j + 1) = v;
  }
}

// Steps of a range, 0 for whole sequences.  The host knows how many sequences and rows there are, not how long each is.  Where the sequences'
// heads fill the SMs, whole ones: ranges make every state twice.  Otherwise two CTAs for each of 148 SMs, of two chunks at least.
int chunk_range(size_t nseq, size_t rows, size_t units) {
  if (nseq * units >= 148) return 0;
  const size_t want = 2 * 148 / units;
  size_t range = ((rows + want - 1) / want + CQ - 1) / CQ * CQ;
  if (range < 2 * CQ) range = 2 * CQ;
  return range >= rows ? 0 : static_cast<int>(range);
}
size_t chunk_ids(size_t nseq, size_t rows, int range) { return range == 0 ? nseq : rows / range + nseq; }

}  // namespace

bool mp_ssd_prompt_chunks_take(const PromptArgs& g) {
  return g.P % 8 == 0 && g.N % 8 == 0 && g.N <= CN && g.xp % 8 == 0 && g.bcp % 8 == 0 && g.yp % 8 == 0 && mp_aligned16(g.x) && mp_aligned16(g.Bm) &&
         mp_aligned16(g.Cm) && mp_aligned16(g.y);
}

size_t mp_ssd_prompt_chunks_scratch(size_t nseq, size_t rows, size_t heads, size_t headdim, size_t dstate) {
  const size_t units = heads * ((headdim + CP - 1) / CP);
  if (units == 0 || nseq == 0 || dstate > CN) return 256;
  const int range = chunk_range(nseq, rows, units);
  return range == 0 ? 256 : chunk_ids(nseq, rows, range) * units * (CP * CN + 1) * sizeof(float) + 256;
}

void mp_ssd_prompt_chunks(const PromptArgs& g, void* scratch, StreamContext ctx) {
  ChunkArgs a{g, nullptr, nullptr, 0, (g.P + CP - 1) / CP, mp_state(ctx)->status_dev};
  const size_t units = static_cast<size_t>(g.H) * a.slices;
  if (scratch != nullptr) a.range = chunk_range(g.q.nseq, g.q.rows, units);
  const size_t ids = chunk_ids(g.q.nseq, g.q.rows, a.range), ctas = ids * units;
  if (ctas > 0x7fffffffull) MP_FATAL("ssd_scan_prompt: too many sequences and heads for one launch");
  MP_CUDA_CHECK(cudaFuncSetAttribute(chunk_walk_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, CK_SMEM));
  if (a.range != 0) {
    a.local = static_cast<float*>(scratch);
    a.decay = a.local + ctas * CP * CN;
    MP_CUDA_CHECK(cudaFuncSetAttribute(chunk_states_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, CK_SMEM));
    MpLaunch(static_cast<unsigned>(ctas), CK_THREADS, CK_SMEM, mp_stream(ctx))(chunk_states_kernel, a);
    MP_LAUNCH_CHECK();
    MpLaunch(static_cast<unsigned>(g.q.nseq * units * CR_PARTS), 256, 0, mp_stream(ctx))(chunk_carry_kernel, a);
    MP_LAUNCH_CHECK();
  }
  MpLaunch(static_cast<unsigned>(ctas), CK_THREADS, CK_SMEM, mp_stream(ctx))(chunk_walk_kernel, a);
  MP_LAUNCH_CHECK();
}
