// What a decode step does with the token that was chosen for a sequence: the rules that force a token, the output column,
// and the state that the next step reads. Shared by the token-choice kernels.
#pragma once

#include "common.h"

namespace vk {

// Per-sequence decode state [B] (vk_select_update in include/viktor_hip.h). run may be null without the homopolymer rule;
// cache_base, pos32, seqlens and rpos32 may be null.
struct DecodeState {
  int64_t *tok, *run, *pos;
  const int64_t *cache_base;
  int64_t *out;
  int64_t out_stride, out_cols;
  int32_t *pos32, *seqlens, *rpos32;
  int homo_stop;
  int64_t eos, pad;
};

// One sequence's step with `nxt` chosen, in the reference's order (viktor/engine.py:79-116): EOS after a tail token; the
// homopolymer run counter (homo: a token's flag, read for nxt == prev only) and EOS when the run reaches homo_stop
// tokens; PAD after EOS / PAD. p, prev, run_raw, ocol (the output column), rope (its offset) and base are the sequence's
// state before the step.
__device__ __forceinline__ void advance_state(const DecodeState &s, int64_t b, int64_t nxt, int64_t prev, bool prev_tail,
                                              const uint8_t *homo, int V, int64_t p, int64_t run_raw, int64_t ocol,
                                              int64_t rope, int64_t base) {
  if (prev_tail) nxt = s.eos;
  if (s.homo_stop > 0) {
    const bool same = nxt == prev && nxt >= 0 && nxt < V && homo[nxt];
    const int64_t r = same ? run_raw + 1 : 0;
    s.run[b] = r;
    if (r + 1 >= s.homo_stop) nxt = s.eos;
  }
  if (prev == s.eos || prev == s.pad) nxt = s.pad;
  if (ocol >= 0 && ocol < s.out_cols) s.out[b * s.out_stride + ocol] = nxt;
  s.tok[b] = nxt;
  const int64_t np = p + 1;
  s.pos[b] = np;
  // cache_base: the KV-cache row of position p is p - cache_base[b] (a per-sequence suffix cache)
  const int64_t cp = np - base;
  if (s.pos32) s.pos32[b] = static_cast<int32_t>(cp);
  if (s.seqlens) s.seqlens[b] = static_cast<int32_t>(cp + 1);
  if (s.rpos32) s.rpos32[b] = static_cast<int32_t>(np + rope);
}

}  // namespace vk
