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

// Threads of a work-group, each of 128 bytes of a row: 256, 512 or 1024 for rows of
// at most 32, 64 and 128 KiB, the fewest that hold one whole; longer rows are cut
// into segments of 64 KiB, 512 threads each.  MI355X, us, no top tokens: 512 rows of
// 4096 fp32 256 threads 5.6, 512 6.9, 1024 10.8; 1000 of 32000 bf16 512 threads
// 20.4, 1024 31; 2047 of 128256 bf16 512 threads 113, 1024 120 (with 20 top tokens
// 146 / 165); 16 of 32000 fp32 with 5 top tokens in one piece 9.8, in two of 512
// threads 10.9 (1000 rows 33.1 / 31.6, without top tokens 25.4 / 25.8).
inline int logprob_threads(int vocab, int elem_bytes) {
  const long long bytes = (long long)vocab * elem_bytes;
  return bytes <= 32768 ? 256 : bytes <= 65536 || bytes > 131072 ? 512 : 1024;
}
inline int logprob_segments(int vocab, int elem_bytes) {
  const long long seg = 128LL * logprob_threads(vocab, elem_bytes);
  return (int)(((long long)vocab * elem_bytes + seg - 1) / seg);
}

void launch_logprobs(const LogprobParams& p, int dtype, hipStream_t stream);

}  // namespace tv
