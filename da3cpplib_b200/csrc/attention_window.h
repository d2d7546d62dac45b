// Windowed attention (attention_window.cu): arguments of one call.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace da3b {

// Element strides of a [sequence][token][head][head_dim] tensor, head_dim contiguous.
struct Strides {
  int64_t seq, tok, head;
};

struct AttnWindow {
  const void *q, *k, *v;
  void* out;
  Strides qs, ks, vs, os;
  int bf16;  // element type: 0 f16, 1 bf16
  int nseq, q_len, k_len, heads, kv_heads, head_dim;
  const int *q_lens, *k_lens;  // device, [nseq] each, or null
  // Keys a query at position p sees: j <= p + right and (j >= p - left or j < sinks);
  // left, right: kWindowAll = no limit on that side.
  int left, right, sinks;
  float scale;
};
constexpr int kWindowAll = 1 << 30;

int attention_window(const AttnWindow& a, int* status, cudaStream_t s);

}  // namespace da3b
