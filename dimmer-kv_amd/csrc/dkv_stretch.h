// The stretches that a row of logits is cut into, in arithmetic that a host compiler takes too.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define DKV_EITHER static __host__ __device__ inline
#else
#define DKV_EITHER static inline
#endif

namespace dkv {

// Stretches of `tokens` that hold `vocab` tokens wherever in a line of `line` elements the row begins.
DKV_EITHER int stretches_of_row(int64_t vocab, int line, int tokens) { return (int)((vocab + line - 1 + tokens - 1) / tokens); }

// The tokens of a stretch whose element 0 is token `first`: below 0 where the row begins inside a line, past the vocabulary
// in the last stretch of a row that begins earlier in its line than the stretches are counted for.
struct TokenRange {
  uint32_t lowest, count;
};
DKV_EITHER TokenRange tokens_of_stretch(int32_t first, int32_t tokens, int32_t vocab) {  // (their sum is below 2^31)
  const int32_t lowest = first > 0 ? first : 0, end = first + tokens < vocab ? first + tokens : vocab;
  return TokenRange{(uint32_t)lowest, (uint32_t)(end > lowest ? end - lowest : 0)};
}

}  // namespace dkv
