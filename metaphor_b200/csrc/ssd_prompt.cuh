// What the two forms of the scan over packed prompts share (ssd_prompt.cu: the recurrence; ssd_prompt_chunks.cu: r16 in chunks on the tensor
// cores).
#pragma once

#include "mp_sequences.cuh"

struct PromptArgs {
  const void* x; const void* raw; const void* dt_bias; const void* A_log; const void* Bm; const void* Cm; void* states; void* y;
  size_t xp, rp, bcp, yp;
  Sequences q;
  int H, P, N, G;
};

// Which steps a CTA has: whole sequences (`steps` = 0) or ranges of that many.  Ranges are numbered without a table: sequence s has the numbers from starts[s] / range + s on, which is at least as
// many as it has ranges.
struct Span { int s; long long lo, hi, seq_lo, seq_hi, slot; bool any; };
__device__ __forceinline__ Span span_of(const Sequences& q, int steps, int id) {
  Span r;
  if (steps == 0) {
    r.s = id;
  } else {
    const long long range = steps;
    r.s = warp_last_not_above(q.nseq - 1, id, [&](int i) { return seq_first(q, i) / range + i; });
    if (r.s < 0) { r.s = 0; r.any = false; return r; }
  }
  r.seq_lo = seq_first(q, r.s);
  r.seq_hi = seq_first(q, r.s + 1);
  r.slot = seq_slot(q.slots, q.nslots, r.s);
  if (steps == 0) {
    r.lo = r.seq_lo;
    r.hi = r.seq_hi;
    r.any = r.slot >= 0;
  } else {
    const long long j = id - (r.seq_lo / steps + r.s);
    r.lo = r.seq_lo + j * steps;
    r.hi = min(r.lo + steps, r.seq_hi);
    r.any = r.slot >= 0 && (r.lo < r.seq_hi || j == 0);
  }
  return r;
}

// Whether the chunks take the call (r16): rows in 16-byte pieces, states of at most 128 columns.
bool mp_ssd_prompt_chunks_take(const PromptArgs& g);
void mp_ssd_prompt_chunks(const PromptArgs& g, void* scratch, StreamContext ctx);
size_t mp_ssd_prompt_chunks_scratch(size_t nseq, size_t rows, size_t heads, size_t headdim, size_t dstate);
