// Launch parameters of the token log-probabilities (logprobs.hip).
#pragma once

#include "tv_common.h"

namespace tv {

constexpr int kLogprobTopMax = 64;    // alternatives of a row

struct LogprobParams {
  const void* logits;          // [rows, vocab], row stride in elements
  const int* tokens;           // [rows]
  long long row_stride;
  int rows;
  int vocab;
  int top_k;
  bool aligned;                // rows start at multiples of 16 bytes
  float* logprobs;             // [rows]
  float* entropy;              // [rows]
  int* top_ids;                // [rows, top_k]
  float* top_logprobs;         // [rows, top_k]
  unsigned long long* part_keys;   // [rows, segments, top_k] in order
  float* part;                 // [rows, segments, 3]: maximum, sums without its term
};

// Rows of at most 32 KiB take a work-group of 256 threads; longer ones are cut
// into segments of 128 KiB, one of 1024 threads each.
inline bool logprob_small(int vocab, int elem_bytes) { return (long long)vocab * elem_bytes <= 32768; }
inline int logprob_segments(int vocab, int elem_bytes) {
  return (int)(((long long)vocab * elem_bytes + 131071) / 131072);
}

void launch_logprobs(const LogprobParams& p, int dtype, hipStream_t stream);

}  // namespace tv
