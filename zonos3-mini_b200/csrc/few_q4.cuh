// The attention of few rows over a KV cache of 4 bits: what gqa_chunk_q4's entry point passes on. A unit of its work is one
// request's rows of one KV head, up to few_rows() (token, head) pairs; requests of more rows are the tensor-memory kernel's.
#pragma once

#include "kv_q4.cuh"

namespace zb {
namespace q4 {

struct FewCall {
  PagedBatch kv;  // a cache of 4 bits
  const __nv_bfloat16* q;
  int64_t q_stride;
  int Hq;
  float scale_log2;
  int causal, window, sinks;
  int rows;  // of a request, at most
  bool only;  // no other kernel takes the rest of the batch
  const __nv_bfloat16* gate;
  int64_t gate_stride;
  __nv_bfloat16* out;
  int64_t out_stride;
  float* lse;
  unsigned char* workspace;  // its first kFewFlagBytes zero, and left zero
};

constexpr int64_t kFewFlagBytes = 32768;

// Rows of a request that the kernel takes in a call (0: none): 8 or 16 (token, head) pairs. No request has more new tokens than
// `max_new`.
int few_rows(int hd, int G, int max_new);
int64_t few_workspace_bytes(int B, int N, int Hkv, int hd, int rows, int64_t max_keys);
int launch_few(const FewCall& call, cudaStream_t stream);

}  // namespace q4
}  // namespace zb
