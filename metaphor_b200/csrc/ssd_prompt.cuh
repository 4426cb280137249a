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

// Whether the chunks take the call (r16): rows in 16-byte pieces, states of at most 128 columns.
bool mp_ssd_prompt_chunks_take(const PromptArgs& g);
void mp_ssd_prompt_chunks(const PromptArgs& g, void* scratch, StreamContext ctx);
size_t mp_ssd_prompt_chunks_scratch(size_t nseq, size_t rows, size_t heads, size_t headdim, size_t dstate);
