// The scan over packed prompts (see ssd_prompt.cu) for r16 tensors, in chunks of 128 steps on the tensor cores (tcgen05, accumulators in TMEM).
//
// With cum the inclusive sums of dt A inside a chunk, E their last one and S the state the chunk receives:
//   y_i = sum_{j <= i} (C_i . B_j) exp(cum_i - cum_j) dt_j x_j + exp(cum_i) S C_i          S' = exp(E) S + sum_j exp(E - cum_j) dt_j x_j (x) B_j
// Four products of 128 rows: G = C B^T, C S^T (128 x 64 x 128), W x with W the weighted scores, and B^T V with V the weighted x.  S stays in
// registers as fp32 values from chunk to chunk; where it, W or V is an operand, it is two r16 terms under a power of two: one for each row p of the
// head in S and V, one for each step in W, since these are columns or rows of the products by themselves (22 bits, down to 2^-38 of the largest
// value among the row's 128).  So y is an r16 rounding of fp32 sums and the kept state has fp32's accuracy to 2^-22 a term, whatever the other
// rows hold.  (One power of two for a whole tile took 72, 112 and 8.7 us below, and left a row p that is 2^28 times smaller than another
// one with 11 bits.)  x, B and C are r16 in memory and enter as they are.
//
// A CTA of eight warps walks one sequence of one head (64 of its rows p); two CTAs share an SM, so that one's products run beside the
// other's scaling.  Shared memory, 112 KB of tiles: C, B (two halves of 64 columns each), x, and one place for the terms of S, later those of V.
// TMEM, 256 columns: G, overwritten in place by W (the first operand of W x is read from there); C S^T, later B^T V; W x.
// Sequences too long and too few to fill the SMs are cut into ranges, whose own states are made first (states_kernel: B^T V alone), then carried
// from range to range (carry_kernel), then walked side by side.
//
// Measured (r16, 64 rows and 128 columns a head, one group): 16 prompts of up to 1023 steps and 24 heads 80 us, where the bytes would take 10.4 and
// 64 MMAs of 128 x 64 x 16 a chunk a fifth of the time.  A chunk takes a CTA about 9 us beside another one, eight of them in a row for the longest
// prompt: the scaling between the products (weights, two terms per value, sums) is what it waits for, a third of it the way through barriers.
// One prompt of 8191 steps and 32 heads 124 us, one of 37 steps and 24 heads 9.2 us.
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
  float piece[CQ / 8];       // decay over each piece of eight steps
  uint32_t most[4][8];       // per warp: largest |G| as bits, exponents of V and of S, dt as bits
  uint64_t bar[4];
  uint32_t tmem;
  int abort;
  // What a CTA needs now and then: kept here, not in registers, of which there are none to spare (a spilled value comes back from the L2, 500
  // cycles away: the L1 beside this much shared memory holds no thread's stack).
  const __half *x, *B, *C, *raw;      // at the span's first row
  __half* y;
  float* state;                       // where the last state goes, NULL for ranges that are not a sequence's last
  float bias, rate;
  alignas(16) uint16_t s_down[CP], v_down[CP];    // per row p: a power of two, the value of a unit in the terms of S and V (the upper half of the float)
  signed char y_up[CQ];               // per step: the exponent of the last chunk's scale of W and of its results in TMEM
  union {
    uint8_t column[4][CP];            // per 32 rows of S or V: the largest exponent of each column
    struct { float plain_dt, plain_y[CP]; };
  };
};
// Weights of a chunk.  They lie over C once its products are done.
struct ChunkWeights {
  float diag[CQ][8];         // row i: dt_j exp(cum_i - cum_j) over its own piece, zero behind i
  float far[CQ / 32][CQ];    // [q][j]: dt_j exp(cum - cum_j), cum up to step 32 q, for j < 32 q
  float enter[CQ];           // decay from the beginning of the row's piece
  float before[CQ];          // decay from the beginning of the chunk
  float v[CQ];               // dt_j exp(E - cum_j)
  float row[2][CQ];          // largest score of a row, among each half's columns
  float colf[CQ];            // dt_j times the decay towards the end of its piece
};
static_assert(sizeof(ChunkWeights) <= 2 * CK_HALF, "it lies over C");
constexpr int CK_SMEM = CK_TAIL + 1024;
static_assert(sizeof(ChunkTail) <= 1024, "two CTAs on an SM have 113 KB each");
constexpr uint32_t TM_G = 0, TM_Y0 = 128, TM_Y1 = 192, TM_COLS = 256;

__device__ __forceinline__ uint32_t ck_at(int row, int piece16) { return row * 128 + ((piece16 ^ (row & 7)) << 4); }
__device__ __forceinline__ void ck_cp_async(uint32_t dst, const void* src, bool in) {      // 16 bytes, zeros where `in` is false
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ck_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int GROUPS>
__device__ __forceinline__ void ck_cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(GROUPS) : "memory"); }
__device__ __forceinline__ uint4 ck_ld(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void ck_st(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// Two fp32 values at a time.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pk(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 upk(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 both(float a) { return pk(a, a); }
__device__ __forceinline__ float2 ck_f2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ f2 ck_wide(uint32_t v) {
  const float2 f = ck_f2(v);
  return pk(f.x, f.y);
}
__device__ __forceinline__ uint32_t ck_narrow(f2 v) {
  const float2 f = upk(v);
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Two values as r16 terms: the rounded values and the rounded rest.
__device__ __forceinline__ void ck_split(f2 v, uint32_t& hi, uint32_t& lo) {
  hi = ck_narrow(v);
  lo = ck_narrow(fma2(ck_wide(hi), both(-1.f), v));
}
// Largest magnitude, NaN above all.
__device__ __forceinline__ float most_abs(float m, float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
  return r;
}
// The exponent of the power of two that takes the largest value (its bits) to [2^13, 2^14).
__device__ __forceinline__ int ck_scale(uint32_t most, int largest) {
  const int k = most == 0 ? 0 : 13 - (static_cast<int>(most >> 23) - 127);
  return k > largest ? largest : k < -120 ? -120 : k;
}
__device__ __forceinline__ float ck_power(int k) { return __int_as_float((127 + k) << 23); }
__device__ __forceinline__ bool ck_infinite(uint32_t bits) { return bits >= 0x7f800000u; }
constexpr uint32_t CK_INFINITE = 255;      // the exponent of an infinity or NaN
// Two neighbouring powers of two from their upper halves, and their inverses.
__device__ __forceinline__ f2 ck_down(uint32_t w) { return pk(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ f2 ck_up(uint32_t w) { return ck_down(0x7f007f00u - w); }
// The largest exponents (biased) of 32 columns over a warp's rows; lane l is left with column l's.  Two columns to a word; in each round a lane hands
// on half of its words and keeps the others.
__device__ __forceinline__ uint32_t column_exponents(const f2 (&v)[16], int lane) {
  uint32_t w[16];
#pragma unroll
  for (int p = 0; p < 16; ++p) {
    const float2 f = upk(v[p]);
    w[p] = __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x7632) & 0x7f807f80u;
  }
#pragma unroll
  for (int o = 16; o > 1; o >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int k = 0; k < o / 2; ++k) {
      const uint32_t send = up ? w[k] : w[k + o / 2], keep = up ? w[k + o / 2] : w[k];
      w[k] = __vmaxu2(keep, __shfl_xor_sync(0xffffffffu, send, o));
    }
  }
  w[0] = __vmaxu2(w[0], __shfl_xor_sync(0xffffffffu, w[0], 1));
  return (lane & 1 ? w[0] >> 16 : w[0] & 0xffffu) >> 7;
}

// The products are a few hundred nanoseconds away: look for a while before the bounded wait, whose suspended warps wake up late.
__device__ __forceinline__ void ck_wait(uint64_t* bar, uint32_t parity, uint32_t* status, volatile int* abort) {
#pragma unroll 1
  for (int i = 0; i < 4096; ++i) {
    uint32_t done;
    asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done)
                 : "r"(mp_smem_u32(bar)), "r"(parity)
                 : "memory");
    if (done) return;
  }
  (void)mbar_wait_abortable(bar, parity, status, abort);
}

struct ChunkArgs {
  PromptArgs g;
  float* local;        // ranges: [id][unit][64 p][128 n] states that a range adds, later those that it receives
  float* decay;        // ranges: [id][unit] what is left of a state behind it
  int range;           // steps of a range, 0: whole sequences
  int slices;          // of 64 rows p in a head
  uint32_t* status;
};

// A value that the compiler takes for a new one, so that what is made of it is made here and not kept in registers across the loop.
__device__ __forceinline__ uint32_t fresh(uint32_t v) {
  asm volatile("" : "+r"(v));
  return v;
}
// What the two walks share: a thread's row (step, or state column n) and half of the 64 rows p; the fetch of a chunk; its step sizes.
struct Lane { int warp, lane, row, half; };
__device__ __forceinline__ Lane lane_of() {
  // (the shuffle tells the compiler that a warp takes one way: otherwise every shuffle behind a branch on it gathers the warp first)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  return {warp, lane, (warp & 3) * 32 + lane, warp >> 2};
}
// 128 rows of `cols` r16 values into halves of 64 columns; rows past `rows` and columns past `cols` become zeros.  A thread has one 16-byte
// column of every 32nd (one half) or 16th row, at the same place of the swizzle.
template <int HALVES>
__device__ __forceinline__ void fetch_tile(uint32_t dst, const __half* src, size_t pitch, int rows, int cols) {
  constexpr int STEP = CK_THREADS / (8 * HALVES);
  const int r = threadIdx.x / (8 * HALVES), c = threadIdx.x % (8 * HALVES);
  const __half* from = src + r * pitch + c * 8;
  const uint32_t to = dst + (c >> 3) * CK_HALF + ck_at(r, c & 7);
  const int left = c * 8 < cols ? rows - r : 0;
#pragma unroll
  for (int k = 0; k < CQ / STEP; ++k) {
    const bool in = k * STEP < left;
    ck_cp_async(to + k * STEP * 128, in ? from : src, in);
    from += STEP * pitch;
  }
}

// Step sizes of a chunk.  A thread has step `row`: dt, its decay, and the decays inside its piece of eight steps, as products of up to eight
// factors (sums of exponents would cancel behind steps of strong decay).
struct StepSizes { float dt, a, enter, leave, piece; };      // decay from the piece's beginning, towards its end, over all of it
__device__ __forceinline__ StepSizes step_sizes(float raw, float bias, float rate, bool in, int lane) {
  StepSizes s;
  s.dt = in ? seq_softplus(raw + bias) : 0.f;
  s.a = expf(s.dt * rate);
  s.enter = s.a;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const float up = __shfl_up_sync(0xffffffffu, s.enter, o, 8);
    if ((lane & 7) >= o) s.enter *= up;
  }
  s.leave = __shfl_down_sync(0xffffffffu, s.a, 1, 8);
  if ((lane & 7) == 7) s.leave = 1.f;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const float down = __shfl_down_sync(0xffffffffu, s.leave, o, 8);
    if ((lane & 7) + o < 8) s.leave *= down;
  }
  s.piece = __shfl_sync(0xffffffffu, s.enter, 7, 8);
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

// What this thread's warp knows of the columns of S or V goes to the others; behind a barrier, `column_scales` makes the powers of two of it.
__device__ __forceinline__ void column_publish(ChunkTail* tail, const Lane& t, const f2 (&v)[16], uint32_t* most, bool infinite = false) {
  const uint32_t e = column_exponents(v, t.lane), m = infinite ? CK_INFINITE : warp_most(e);
  tail->column[t.warp & 3][t.half * 32 + t.lane] = static_cast<uint8_t>(e);
  if (t.lane == 0) most[t.warp] = m;
}
// Every row p has a power of two of its own, which takes its largest value to [2^13, 2^14): a row of small values keeps its bits beside one of large
// ones.  (The four warps of a half write the same values.)
__device__ __forceinline__ void column_scales(ChunkTail* tail, const Lane& t, uint16_t* down) {
  const int c = t.half * 32 + t.lane;
  const int e = max(max(tail->column[0][c], tail->column[1][c]), max(tail->column[2][c], tail->column[3][c])) - 13;
  down[c] = static_cast<uint16_t>((e < 7 ? 7 : e > 247 ? 247 : e) << 7);
  __syncwarp();
}
// V = x w: 32 columns of a row.
__device__ __forceinline__ void weigh(f2 (&v)[16], uint32_t x_tile, int row, int half, float w) {
  const f2 w2 = both(w);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint4 x = ck_ld(x_tile + ck_at(row, half * 4 + k));
    const uint32_t in[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) v[4 * k + e] = mul2(ck_wide(in[e]), w2);
  }
}
// 32 columns of a row in two terms, each a [128][64] tile.
__device__ __forceinline__ void store_terms(uint32_t tile, int row, int half, const f2 (&v)[16], const uint16_t* down) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint4 d = *reinterpret_cast<const uint4*>(down + half * 32 + k * 8);
    const uint32_t scale[4] = {d.x, d.y, d.z, d.w};
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) ck_split(mul2(v[4 * k + e], ck_up(scale[e])), hi[e], lo[e]);
    const uint32_t at = tile + ck_at(row, half * 4 + k);
    ck_st(at, make_uint4(hi[0], hi[1], hi[2], hi[3]));
    ck_st(at + CK_HALF, make_uint4(lo[0], lo[1], lo[2], lo[3]));
  }
}
// S = total S + v, v from TMEM in the units of `down`
__device__ __forceinline__ void add_state(f2 (&S)[16], uint32_t tmem, float total, const uint16_t* down) {
  const f2 t2 = both(total);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    uint32_t v[16];
    tmem_ld_32x16(tmem + k * 16, v);
    const uint4 d0 = *reinterpret_cast<const uint4*>(down + k * 16), d1 = *reinterpret_cast<const uint4*>(down + k * 16 + 8);
    const uint32_t d[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
    tmem_ld_wait();
#pragma unroll
    for (int p = 0; p < 8; ++p) S[8 * k + p] = fma2(t2, S[8 * k + p], mul2(ck_down(d[p]), pk(__uint_as_float(v[2 * p]), __uint_as_float(v[2 * p + 1]))));
  }
}

// A chunk step by step, for values that the products would spread.  S lies where the operands' terms were, [64 p][128 n]; a thread has column
// n = row, 32 rows p.  y_p is summed over a warp's 32 columns lane against lane, then over the warps in turn.  OUT: with y.
template <bool OUT>
__device__ __forceinline__ void chunk_plain(unsigned char* smem, ChunkTail* tail, const Lane& t, f2 (&S)[16], float dt, int steps, __half* y, size_t yp, int pcols, int ncols) {
  float* held = reinterpret_cast<float*>(smem + CK_T) + t.half * 32 * CN + t.row;
#pragma unroll
  for (int p = 0; p < 16; ++p) {
    const float2 v = upk(S[p]);
    held[2 * p * CN] = v.x;
    held[(2 * p + 1) * CN] = v.y;
  }
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    __syncthreads();
    if (t.half == 0 && t.row == i) tail->plain_dt = dt;
    if (threadIdx.x < CP) tail->plain_y[threadIdx.x] = 0.f;
    __syncthreads();
    const float d = tail->plain_dt, a = expf(d * tail->rate);
    const uint32_t col = (t.row >> 6) * CK_HALF + ck_at(i, (t.row & 63) >> 3) + (t.row & 7) * 2;
    const float b = __half2float(*reinterpret_cast<const __half*>(smem + CK_B + col));
    const float c = OUT ? __half2float(*reinterpret_cast<const __half*>(smem + CK_C + col)) : 0.f;
    float v[32];
#pragma unroll
    for (int p = 0; p < 32; ++p) {
      const float x = __half2float(*reinterpret_cast<const __half*>(smem + CK_X + ck_at(i, t.half * 4 + (p >> 3)) + (p & 7) * 2));
      const float now = t.row < ncols ? a * held[p * CN] + d * x * b : 0.f;      // (columns behind the last: an infinity times nothing would reach y)
      held[p * CN] = now;
      v[p] = c * now;
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
#pragma unroll 1
      for (int w = 0; w < 4; ++w) {
        if ((t.warp & 3) == w) tail->plain_y[t.half * 32 + t.lane] += v[0];
        __syncthreads();
      }
      if (static_cast<int>(threadIdx.x) < pcols) y[i * yp + threadIdx.x] = __float2half_rn(tail->plain_y[threadIdx.x]);
    }
  }
#pragma unroll
  for (int p = 0; p < 16; ++p) S[p] = pk(held[2 * p * CN], held[(2 * p + 1) * CN]);
  __syncthreads();
}

// ---------------------------------------------------------------------------
// The walk.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(CK_THREADS, 2) chunk_walk_kernel(const ChunkArgs a) {
  extern __shared__ __align__(1024) unsigned char ck_smem[];
  ChunkTail* tail = reinterpret_cast<ChunkTail*>(ck_smem + CK_TAIL);
  ChunkWeights* wt = reinterpret_cast<ChunkWeights*>(ck_smem + CK_C);
  const PromptArgs& g = a.g;
  const Lane t = lane_of();
  const uint32_t base = mp_smem_u32(ck_smem);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(tail->bar + i, 1);
    mbar_fence_init();
    tail->abort = 0;
  }
  mp_grid_wait();
  const int units = g.H * a.slices;
  const int id = blockIdx.x / units, unit = blockIdx.x % units, h = unit / a.slices, p0 = unit % a.slices * CP, grp = h / (g.H / g.G);
  const Span sp = span_of(a.g.q, a.range, id);
  if (!sp.any) { mp_launch_dependents(); return; }
  if (t.warp == 0) tmem_alloc(&tail->tmem, TM_COLS);
  const int pcols = min(CP, g.P - p0), length = static_cast<int>(sp.hi - sp.lo);
  float* state = static_cast<float*>(g.states) + ((sp.slot * g.H + h) * g.P + p0) * static_cast<long long>(g.N);
  if (threadIdx.x == 0) {
    tail->x = static_cast<const __half*>(g.x) + sp.lo * g.xp + static_cast<size_t>(h) * g.P + p0;
    tail->B = static_cast<const __half*>(g.Bm) + sp.lo * g.bcp + static_cast<size_t>(grp) * g.N;
    tail->C = static_cast<const __half*>(g.Cm) + sp.lo * g.bcp + static_cast<size_t>(grp) * g.N;
    tail->raw = static_cast<const __half*>(g.raw) + sp.lo * g.rp + h;
    tail->y = static_cast<__half*>(g.y) + sp.lo * g.yp + static_cast<size_t>(h) * g.P + p0;
    tail->state = sp.hi == sp.seq_hi ? state : nullptr;
    tail->bias = static_cast<const float*>(g.dt_bias)[h];
    tail->rate = -expf(static_cast<const float*>(g.A_log)[h]);
  }
  __syncthreads();
  auto steps_at = [&](int t0) { return min(length - t0, CQ); };
  float raw_next = 0.f;      // of the warps that make the weights
  auto fetch_bc = [&](int t0) {
    const int steps = steps_at(t0);
    const uint32_t at = fresh(base);
    fetch_tile<2>(at + CK_C, tail->C + t0 * g.bcp, g.bcp, steps, g.N);
    fetch_tile<2>(at + CK_B, tail->B + t0 * g.bcp, g.bcp, steps, g.N);
    ck_cp_commit();
    if (t.half == 0) raw_next = t.row < steps ? __half2float(tail->raw[(t0 + t.row) * g.rp]) : 0.f;
  };
  auto fetch_x = [&](int t0) {
    fetch_tile<1>(fresh(base) + CK_X, tail->x + t0 * g.xp, g.xp, steps_at(t0), pcols);
    ck_cp_commit();
  };
  if (length > 0) {
    fetch_bc(0);
    fetch_x(0);
  }
  // the state that the span receives: this thread's column n = row, rows p = 32 half ..
  f2 S[16];
  {
    const float* from = state;
    long long pitch = g.N;
    bool any = true;
    if (a.range != 0 && sp.seq_hi - sp.seq_lo > a.range) {      // (the first range too: the last one may be writing the sequence's state by now)
      from = a.local + (static_cast<size_t>(id) * units + unit) * CP * CN;
      pitch = CN;
    } else {
      any = seq_resumes(g.q, sp.s);
    }
    const int live = any && t.row < g.N ? pcols - t.half * 32 : 0;
    from += t.half * 32 * pitch + t.row;
#pragma unroll
    for (int p = 0; p < 16; ++p) {
      float v0 = 0.f, v1 = 0.f;
      if (2 * p < live) v0 = *from;
      from += pitch;
      if (2 * p + 1 < live) v1 = *from;
      from += pitch;
      S[p] = pk(v0, v1);
    }
  }
  auto publish = [&]() {      // S becomes an operand of the next chunk: this thread's row of it is a state column n
    column_publish(tail, t, S, tail->most[2]);
    __syncthreads();
    const uint32_t most = cta_most(tail->most[2]);
    column_scales(tail, t, tail->s_down);
    if (most != CK_INFINITE) store_terms(fresh(base) + CK_T, t.row, t.half, S, tail->s_down);
    return most;
  };
  uint32_t s_most = publish();

  constexpr uint32_t id_g = umma_instr_desc(UMMA_FMT_F16, 0, 0, 128, 128), id_y = umma_instr_desc(UMMA_FMT_F16, 0, 1, 128, CP), id_s = umma_instr_desc(UMMA_FMT_F16, 1, 1, 128, CP);
  constexpr uint32_t HALF_U = CK_HALF / 16, ROWS_U = 16 * 128 / 16;
  auto kslice = [](int ks) { return static_cast<uint32_t>((ks >> 2) * HALF_U + (ks & 3) * 2); };
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  auto lanes = [&]() { return tail->tmem + (static_cast<uint32_t>(t.warp & 3) << 21); };      // this warp's 32 lanes of TMEM
  uint32_t issued = 0, finished = 0;      // phases of the barriers: scores and C S^T, the other two products
  // The results of a chunk leave TMEM while the next one's first products run.
  bool pending = false;
  auto store_y = [&](int t0, int steps) {
    const f2 down = both(ck_power(-tail->y_up[t.row]));
    __half* out = tail->y + (t0 + t.row) * g.yp + t.half * 32;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t v[16], o[8];
      tmem_ld_32x16(lanes() + TM_Y1 + t.half * 32 + k * 16, v);
      tmem_ld_wait();
#pragma unroll
      for (int p = 0; p < 8; ++p) o[p] = ck_narrow(mul2(pk(__uint_as_float(v[2 * p]), __uint_as_float(v[2 * p + 1])), down));
      if (t.row < steps && t.half * 32 + k * 16 < pcols) *reinterpret_cast<uint4*>(out + k * 16) = make_uint4(o[0], o[1], o[2], o[3]);
      if (t.row < steps && t.half * 32 + k * 16 + 8 < pcols) *reinterpret_cast<uint4*>(out + k * 16 + 8) = make_uint4(o[4], o[5], o[6], o[7]);
    }
  };
  for (int t0 = 0; t0 < length; t0 += CQ) {
    const int steps = steps_at(t0);
    const bool carried = s_most != 0, products = s_most != CK_INFINITE && fabsf(tail->rate) < INFINITY;
    ck_cp_wait<1>();      // C and B
    fence_proxy_async_smem();
    tcgen05_fence_before_sync();
    __syncthreads();
    if (tail->abort != 0) break;      // a wait ran out
    tcgen05_fence_after_sync();
    if (t.warp == 0 && products && elect_one()) {
      const uint32_t at = fresh(base), tmem = tail->tmem;
      const uint64_t d_c = umma_smem_desc(at + CK_C, 16, 1024), d_b = umma_smem_desc(at + CK_B, 16, 1024), d_t = umma_smem_desc(at + CK_T, CK_HALF, 1024);
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
    if (pending) store_y(t0 - CQ, CQ);
    pending = false;
    // half of the warps make the weights
    StepSizes z;
    float far[4], diag[8], before = 1.f;      // far: from this step's piece on to steps 32, 64, 96 and the end
    if (t.half == 0) {
      z = step_sizes(raw_next, tail->bias, tail->rate, t.row < steps, t.lane);
      if ((t.lane & 7) == 7) tail->piece[t.row >> 3] = z.piece;
      const uint32_t dm = warp_most(abs_bits(z.dt));
      if (t.lane == 0) tail->most[3][t.warp] = dm;
      named_bar_sync(1, CK_THREADS / 2);
      float f = z.dt * z.leave;
#pragma unroll
      for (int k = 0; k < CQ / 8; ++k) {
        const float d = tail->piece[k];
        if (k < (t.row >> 3)) before *= d;
        if (k > (t.row >> 3)) f *= d;
        if ((k & 3) == 3) far[k >> 2] = f;
      }
      float left = 1.f, au = z.a, du = z.dt;      // k steps back: the decays of the steps behind, dt
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        diag[k] = k <= (t.lane & 7) ? du * left : 0.f;
        left *= au;
        au = __shfl_up_sync(0xffffffffu, au, 1, 8);
        du = __shfl_up_sync(0xffffffffu, du, 1, 8);
      }
    }
    ck_cp_wait<0>();      // this thread's x
    const int q = t.warp & 3;      // this warp's rows begin at 32 q: blocks of 16 score columns up to 2 q + 1 are below or on the diagonal; it has
                                   // every other one
    if (products) {
      ck_wait(tail->bar + 0, issued, a.status, &tail->abort);
      tcgen05_fence_after_sync();
      float gm = 0.f;
      const uint32_t tg = lanes() + TM_G + t.half * 16;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if (b <= q) {
          uint32_t v[16];
          tmem_ld_32x16(tg + b * 32, v);
          tmem_ld_wait();
          if (b == q) {      // scores above the diagonal are not used
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (t.half * 16 + e > t.lane) v[e] = 0;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) gm = most_abs(gm, __uint_as_float(v[e]));
        }
      }
      const uint32_t gw = warp_most(abs_bits(gm));
      if (t.lane == 0) tail->most[0][t.warp] = gw;
      ck_wait(tail->bar + 1, issued, a.status, &tail->abort);
      tcgen05_fence_after_sync();
      issued ^= 1;
      wt->row[t.half][t.row] = gm;      // C is free
      if (t.half == 0) {
        wt->enter[t.row] = z.enter;
        wt->before[t.row] = before * z.enter;
        wt->colf[t.row] = z.dt * z.leave;
        wt->v[t.row] = far[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) wt->far[k + 1][t.row] = far[k];
#pragma unroll
        for (int k = 0; k < 8; ++k) wt->diag[t.row][(t.lane - k) & 7] = diag[k];
      }
    }
    __syncthreads();
    // the largest values of V, and a bound of W's: the decays that are left out of it are at most one
    float dt_most = 0.f;
    bool odd = !products;
    if (products) {
      f2 v[16];
      weigh(v, fresh(base) + CK_X, t.row, t.half, wt->v[t.row]);
      column_publish(tail, t, v, tail->most[1]);
      __syncthreads();
      dt_most = __uint_as_float(max(max(tail->most[3][0], tail->most[3][1]), max(tail->most[3][2], tail->most[3][3])));
      odd = cta_most(tail->most[1]) == CK_INFINITE || ck_infinite(abs_bits(__uint_as_float(cta_most(tail->most[0])) * dt_most));
    }
    if (odd) {
      if (products) {      // the weights lie over C
        __syncthreads();
        fetch_tile<2>(base + CK_C, tail->C + t0 * g.bcp, g.bcp, steps, g.N);
        ck_cp_commit();
        ck_cp_wait<0>();
      }
      chunk_plain<true>(ck_smem, tail, t, S, z.dt, steps, tail->y + t0 * g.yp, g.yp, pcols, g.N);
    } else {
      const uint32_t tiles = fresh(base);
      column_scales(tail, t, tail->v_down);
      // V goes to the warps with few blocks of W: two pieces of 32 rows to the first, one each to the next two
      for (int b = q == 0 ? 0 : q + 1, n = q == 0 ? 2 : q == 3 ? 0 : 1; n > 0; ++b, --n) {
        const int row = b * 32 + t.lane;
        f2 v[16];
        weigh(v, tiles + CK_X, row, t.half, wt->v[row]);
        store_terms(tiles + CK_T, row, t.half, v, tail->v_down);
      }
      // A row of W (a step) has a power of two of its own.  (2^60: scores below 2^-47 do not show in y, and the state's share, which takes the same
      // scale, stays finite where y does.)
      const int y_up = ck_scale(abs_bits(fmaxf(wt->row[0][t.row], wt->row[1][t.row]) * dt_most), 60);
      const float w_up = ck_power(y_up);
      tail->y_up[t.row] = static_cast<signed char>(y_up);      // (by two threads)
      {
        // W over G: sixteen columns of scores become eight of the upper terms and eight of the lower ones
        const float4 P = *reinterpret_cast<const float4*>(tail->piece + 4 * q);
        const int r = t.lane >> 3;      // this row's piece among the four of its warp
        const float enter = wt->enter[t.row] * w_up;
        const float p1 = r > 1 ? P.y : 1.f, p2 = r > 2 ? P.z : 1.f;
        const f2 lead = both(enter * (r > 0 ? P.x : 1.f) * p1 * p2), up = both(w_up);
        const uint32_t tg = lanes() + TM_G + t.half * 16;
        uint32_t v[16];
        tmem_ld_32x16(tg, v);
#pragma unroll 1
        for (int b = 0; b < 4; ++b) {
          uint32_t w[16];
          if (b <= q) {
            tmem_ld_wait();
            const float4* cf = reinterpret_cast<const float4*>((b < q ? wt->far[q] : wt->colf) + b * 32 + t.half * 16);
#pragma unroll
            for (int k = 0; k < 2; ++k) {      // a piece of eight columns
              // Below the warp's own 32 columns one factor for a row; there, two pieces for each half: those before the row's own, its own, zeros behind
              const int piece = 2 * t.half + k;
              const bool own = b == q && r == piece;
              const f2 row = b < q ? lead : own ? up : r > piece ? both(t.half == 0 ? (k == 0 ? enter * p1 * p2 : enter * p2) : enter) : both(0.f);
              const float4* from = own ? reinterpret_cast<const float4*>(wt->diag[t.row]) : cf + 2 * k;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float4 c = from[e];
                const int at = 8 * k + 4 * e;
                ck_split(mul2(pk(__uint_as_float(v[at]), __uint_as_float(v[at + 1])), mul2(row, pk(c.x, c.y))), w[4 * k + 2 * e], w[8 + 4 * k + 2 * e]);
                ck_split(mul2(pk(__uint_as_float(v[at + 2]), __uint_as_float(v[at + 3])), mul2(row, pk(c.z, c.w))), w[4 * k + 2 * e + 1], w[8 + 4 * k + 2 * e + 1]);
              }
            }
            if (b < q) tmem_ld_32x16(tg + (b + 1) * 32, v);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = 0;
          }
          tmem_st_32x16(tg + b * 32, w);
        }
      }
      if (carried) {      // the state's share of y, to the scale of W: W x is added to it
        const f2 f = both(wt->before[t.row] * w_up);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t v[16];
          tmem_ld_32x16(lanes() + TM_Y0 + t.half * 32 + k * 16, v);
          const uint4 d0 = *reinterpret_cast<const uint4*>(tail->s_down + t.half * 32 + k * 16), d1 = *reinterpret_cast<const uint4*>(tail->s_down + t.half * 32 + k * 16 + 8);
          const uint32_t d[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
          tmem_ld_wait();
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            const float2 r = upk(mul2(f, mul2(ck_down(d[p]), pk(__uint_as_float(v[2 * p]), __uint_as_float(v[2 * p + 1])))));
            v[2 * p] = __float_as_uint(r.x);
            v[2 * p + 1] = __float_as_uint(r.y);
          }
          tmem_st_32x16(lanes() + TM_Y1 + t.half * 32 + k * 16, v);
        }
      }
      tmem_st_wait();
      fence_proxy_async_smem();
      tcgen05_fence_before_sync();
      __syncthreads();
      tcgen05_fence_after_sync();
      if (t.warp == 0 && elect_one()) {
        const uint32_t at = fresh(base), tmem = tail->tmem;
        const uint64_t d_bt = umma_smem_desc(at + CK_B, CK_HALF, 1024), d_t = umma_smem_desc(at + CK_T, CK_HALF, 1024), d_x = umma_smem_desc(at + CK_X, CK_HALF, 1024);
#pragma unroll
        for (int ks = 0; ks < 16; ++ks)
          umma<false>(tmem + TM_Y0, d_bt + (ks & 7) * ROWS_U, d_t + (ks >> 3) * HALF_U + (ks & 7) * ROWS_U, id_s, ks != 0 ? 1u : 0u);
        umma_commit(tail->bar + 2);
#pragma unroll
        for (int ks = 0; ks < 16; ++ks)
          umma_f16_ta(tmem + TM_Y1, tmem + TM_G + (ks & 7) * 16 + (ks >> 3) * 8, d_x + (ks & 7) * ROWS_U, id_y, ks != 0 || carried ? 1u : 0u);
        umma_commit(tail->bar + 3);
      }
      __syncwarp();
      pending = true;
      ck_wait(tail->bar + 2, finished, a.status, &tail->abort);
      tcgen05_fence_after_sync();
      if (t0 + CQ < length) fetch_bc(t0 + CQ);
      float total = 1.f;
#pragma unroll
      for (int k = 0; k < CQ / 8; ++k) total *= tail->piece[k];
      add_state(S, lanes() + TM_Y0 + t.half * 32, total, tail->v_down + t.half * 32);
      tcgen05_fence_before_sync();
    }
    if (t0 + CQ < length) {
      if (!pending) fetch_bc(t0 + CQ);
      s_most = publish();
    }
    if (pending) {
      ck_wait(tail->bar + 3, finished, a.status, &tail->abort);
      tcgen05_fence_after_sync();
      finished ^= 1;
    }
    if (t0 + CQ < length) fetch_x(t0 + CQ);
  }
  if (pending) store_y((length - 1) / CQ * CQ, (length - 1) % CQ + 1);
  mp_launch_dependents();
  state = tail->state;
  if (state != nullptr && t.row < g.N) {
#pragma unroll
    for (int p = 0; p < 32; ++p)
      if (t.half * 32 + p < pcols) {
        const float2 v = upk(S[p / 2]);
        state[(t.half * 32 + p) * static_cast<long long>(g.N) + t.row] = p & 1 ? v.y : v.x;
      }
  }
  ck_cp_wait<0>();
  tcgen05_fence_before_sync();
  __syncthreads();
  if (t.warp == 0) tmem_dealloc(tail->tmem, TM_COLS);
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
  const Span sp = span_of(a.g.q, a.range, id);
  if (!sp.any || sp.hi >= sp.seq_hi) { mp_launch_dependents(); return; }      // nothing lies behind it
  if (t.warp == 0) tmem_alloc(&tail->tmem, CP);
  const int pcols = min(CP, g.P - p0);
  const __half* x = static_cast<const __half*>(g.x) + static_cast<size_t>(h) * g.P + p0;
  const __half* raw = static_cast<const __half*>(g.raw) + h;
  const __half* Bm = static_cast<const __half*>(g.Bm) + static_cast<size_t>(grp) * g.N;
  const float bias = static_cast<const float*>(g.dt_bias)[h], rate = -expf(static_cast<const float*>(g.A_log)[h]);
  if (threadIdx.x == 0) tail->rate = rate;
  float raw_next = 0.f;
  auto fetch = [&](long long t0) {      // whole chunks: a range that others follow is a multiple of them
    fetch_tile<2>(base + CK_B, Bm + t0 * g.bcp, g.bcp, CQ, g.N);
    fetch_tile<1>(base + CK_X, x + t0 * g.xp, g.xp, CQ, pcols);
    ck_cp_commit();
    raw_next = __half2float(raw[(t0 + t.row) * g.rp]);
  };
  fetch(sp.lo);
  f2 S[16];
  float left = 1.f;
#pragma unroll
  for (int p = 0; p < 16; ++p) S[p] = 0;
  const uint64_t d_bt = umma_smem_desc(base + CK_B, CK_HALF, 1024), d_t = umma_smem_desc(base + CK_T, CK_HALF, 1024);
  constexpr uint32_t id_s = umma_instr_desc(UMMA_FMT_F16, 1, 1, 128, CP), HALF_U = CK_HALF / 16, ROWS_U = 16 * 128 / 16;
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem = tail->tmem, tq = tmem + (static_cast<uint32_t>(t.warp & 3) << 21);
  uint32_t finished = 0;
  const bool odd = !(fabsf(rate) < INFINITY);
  for (long long t0 = sp.lo; t0 < sp.hi; t0 += CQ) {
    ck_cp_wait<0>();
    fence_proxy_async_smem();
    __syncthreads();
    if (tail->abort != 0) break;
    const StepSizes z = step_sizes(raw_next, bias, rate, true, t.lane);
    if (t.half == 0 && (t.lane & 7) == 7) tail->piece[t.row >> 3] = z.piece;
    bool infinite;      // in B: against the two terms of V it would be a NaN
    {
      __half2 b2 = __float2half2_rn(0.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint4 b = ck_ld(base + CK_B + t.half * CK_HALF + ck_at(t.row, k));
        const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) b2 = __hmax2_nan(b2, __habs2(*reinterpret_cast<const __half2*>(&w[e])));
      }
      const float2 f = __half22float2(b2);
      infinite = __any_sync(0xffffffffu, !(f.x < INFINITY && f.y < INFINITY));
    }
    __syncthreads();
    float w = z.dt * z.leave, total = 1.f;
#pragma unroll
    for (int k = 0; k < CQ / 8; ++k) {
      const float d = tail->piece[k];
      total *= d;
      if (k > (t.row >> 3)) w *= d;
    }
    left *= total;
    f2 v[16];
    weigh(v, base + CK_X, t.row, t.half, w);
    column_publish(tail, t, v, tail->most[1], infinite);
    __syncthreads();
    if (odd || cta_most(tail->most[1]) == CK_INFINITE) {
      chunk_plain<false>(ck_smem, tail, t, S, z.dt, CQ, nullptr, 0, pcols, g.N);
    } else {
      column_scales(tail, t, tail->v_down);
      store_terms(base + CK_T, t.row, t.half, v, tail->v_down);
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
      ck_wait(tail->bar + 2, finished, a.status, &tail->abort);
      finished ^= 1;
      tcgen05_fence_after_sync();
      add_state(S, tq + t.half * 32, total, tail->v_down + t.half * 32);
    }
    if (t0 + CQ < sp.hi) {
      __syncthreads();
      fetch(t0 + CQ);
    }
  }
  mp_launch_dependents();
  const size_t at = static_cast<size_t>(id) * units + unit;
#pragma unroll
  for (int p = 0; p < 16; ++p) {
    const float2 v = upk(S[p]);
    a.local[at * CP * CN + (t.half * 32 + 2 * p) * CN + t.row] = v.x;
    a.local[at * CP * CN + (t.half * 32 + 2 * p + 1) * CN + t.row] = v.y;
  }
  // not zero, however many steps: an infinite state stays infinite then, as it does step by step
  if (threadIdx.x == 0) a.decay[at] = fmaxf(left, __int_as_float(1));
  ck_cp_wait<0>();
  tcgen05_fence_before_sync();
  __syncthreads();
  if (t.warp == 0) tmem_dealloc(tmem, CP);
}

// From range to range: what each adds is replaced by what it receives, the first one by the kept state.  A thread has four neighbouring values of a state.
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
  // eight ranges on their way at a time: one after the other is a trip to the L2 each (one prompt of 8191 steps: 114.6 -> 112.1 us)
  constexpr int U = 8;
  float4 ahead = *place(0);      // (place j + 1 is read before it is written: what its range adds goes to the one behind)
  *place(0) = v;
  for (long long j = 0; j + 1 < ranges; j += U) {
    float4 add[U + 1];
    float left[U];
    add[0] = ahead;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j + u + 1 < ranges) left[u] = a.decay[first + (j + u) * units];
      if (j + u + 2 < ranges) add[u + 1] = *place(j + u + 1);
    }
    ahead = add[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j + u + 1 < ranges) {
        v.x = left[u] * v.x + add[u].x;
        v.y = left[u] * v.y + add[u].y;
        v.z = left[u] * v.z + add[u].z;
        v.w = left[u] * v.w + add[u].w;
        *place(j + u + 1) = v;
      }
  }
}

// Steps of a range, 0 for whole sequences.  The host knows how many sequences and rows there are, not how long each is.  Where the sequences'
// heads fill the SMs, whole ones: ranges make every state twice.  Otherwise two CTAs for each of 148 SMs (the scratch function, which goes by the same
// numbers, knows no device), of two chunks at least.
constexpr size_t CK_SMS = 148;
int chunk_range(size_t nseq, size_t rows, size_t units) {
  if (nseq * units >= CK_SMS) return 0;
  const size_t want = 2 * CK_SMS / units;
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
  // Enough for every call of as many sequences and rows or fewer: those that are cut have fewer than CK_SMS units in all, ranges of two chunks or more,
  // and no more of them than `chunk_range` wants.
  const size_t sequences = nseq < (CK_SMS - 1) / units ? nseq : (CK_SMS - 1) / units;
  if (sequences == 0 || rows <= 2 * CQ) return 256;
  const size_t want = 2 * CK_SMS / units, ranges = want < rows / (2 * CQ) ? want : rows / (2 * CQ);
  return (ranges + sequences) * units * (CP * CN + 1) * sizeof(float) + 256;
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
