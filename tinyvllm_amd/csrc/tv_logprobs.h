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

// Threads of a work-group, each of 128 bytes of a row: 256 for rows of at most 32
// KiB, 1024 up to 128 KiB (a second launch costs more than the coarser work-groups);
// longer rows are cut into segments of 64 KiB, 512 threads each.
inline int logprob_threads(int vocab, int elem_bytes) {
  const long long bytes = (long long)vocab * elem_bytes;
  return bytes <= 32768 ? 256 : bytes <= 131072 ? 1024 : 512;
}
inline int logprob_segments(int vocab, int elem_bytes) {
  const long long seg = 128LL * logprob_threads(vocab, elem_bytes);
  return (int)(((long long)vocab * elem_bytes + seg - 1) / seg);
}

void launch_logprobs(const LogprobParams& p, int dtype, hipStream_t stream);

}  // namespace tv
