// Softmax attention over a window of keys and the first few keys of each sequence.
//
// Query i of a sequence with ql queries and kl keys stands at position p = kl - ql + i
// (the queries are the last ones of the keys) and sees the keys j < kl with
// j <= p + right and (j >= p - left or j < sinks). o = sum_j softmax_j(scale q.k_j) v_j; a
// query that sees nothing gets zeros, rows from ql on are not written.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "attention_window.h"
#include "da3b.h"
#include "ops.h"
#include "ptx.cuh"

namespace da3b {

namespace {

// Reference form: one warp per (query, head), one key at a time, D / 32 dims a lane.
template <typename T, int D>
__global__ void __launch_bounds__(256) k_attn_window(const AttnWindow a) {
  constexpr int E = D / 32;
  const long w = static_cast<long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (w >= static_cast<long>(a.nseq) * a.heads * a.q_len) return;
  const int i = static_cast<int>(w % a.q_len), h = static_cast<int>(w / a.q_len % a.heads);
  const int b = static_cast<int>(w / a.q_len / a.heads);
  const int ql = a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len;
  const int kl = a.k_lens ? min(max(a.k_lens[b], 0), a.k_len) : a.k_len;
  if (i >= ql) return;
  const int hk = h / (a.heads / a.kv_heads), p = kl - ql + i;
  const T* q = static_cast<const T*>(a.q) + b * a.qs.seq + i * a.qs.tok + h * a.qs.head + lane * E;
  const T* k = static_cast<const T*>(a.k) + b * a.ks.seq + hk * a.ks.head + lane * E;
  const T* v = static_cast<const T*>(a.v) + b * a.vs.seq + hk * a.vs.head + lane * E;
  float o[E] = {}, l = 0.f, m = -INFINITY;
  const int hi = min(kl - 1, p + a.right), lo = max(p - a.left, 0);
  const float c = a.scale * 1.4426950408889634f;
  for (int j = 0; j <= hi; ++j) {
    if (j < lo && j >= a.sinks) {
      j = lo - 1;
      continue;
    }
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(static_cast<float>(q[e]), static_cast<float>(k[j * a.ks.tok + e]), s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
    const float alpha = exp2f((m - base) * c), pr = exp2f((s - base) * c);
    m = mn;
    l = l * alpha + pr;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * alpha + pr * static_cast<float>(v[j * a.vs.tok + e]);
  }
  T* out = static_cast<T*>(a.out) + b * a.os.seq + i * a.os.tok + h * a.os.head + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = static_cast<T>(l > 0.f ? o[e] / l : (l == 0.f ? 0.f : l));
}

}  // namespace

int attention_window(const AttnWindow& a, int* status, cudaStream_t s) {
  (void)status;
  const long rows = static_cast<long>(a.nseq) * a.heads * a.q_len;
  const unsigned grid = static_cast<unsigned>((rows + 7) / 8);
  if (a.bf16) {
    if (a.head_dim == 64) k_attn_window<__nv_bfloat16, 64><<<grid, 256, 0, s>>>(a);
    else k_attn_window<__nv_bfloat16, 128><<<grid, 256, 0, s>>>(a);
  } else {
    if (a.head_dim == 64) k_attn_window<__half, 64><<<grid, 256, 0, s>>>(a);
    else k_attn_window<__half, 128><<<grid, 256, 0, s>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // namespace da3b

using namespace da3b;

// Strides of a tensor of the given sizes: multiples of 8 elements, positive (a stride of
// a size of one is never used, and set to one token or head so that nothing depends on it).
static bool take_strides(const int64_t* in, int nseq, int len, int heads, int D, Strides* st) {
  *st = {in[0], in[1], in[2]};
  if (heads == 1) st->head = D;
  if (len == 1) st->tok = static_cast<int64_t>(heads) * D;
  if (nseq == 1) st->seq = static_cast<int64_t>(len) * heads * D;
  const int64_t most = int64_t(1) << 38;  // tensor maps hold strides below 2^40 bytes
  for (int64_t v : {st->seq, st->tok, st->head})
    if (v < D || v % 8 || v >= most) return false;
  return true;
}

extern "C" {

DA3B_API int da3b_attention_window(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                   const void* v, const int64_t* v_strides, void* out, const int64_t* out_strides,
                                   int dtype, int nseq, int q_len, int k_len, int heads, int kv_heads, int head_dim,
                                   const int* q_lens, const int* k_lens, int left, int right, int sinks, float scale,
                                   void* stream) {
  if (!q || !k || !v || !out || !q_strides || !k_strides || !v_strides || !out_strides) return -100;
  if ((dtype != 0 && dtype != 1) || nseq < 0 || q_len < 0 || k_len < 0 || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads || (head_dim != 64 && head_dim != 128) || sinks < 0 || !(scale >= 0.f) || isinf(scale))
    return -100;
  if (q_len > kWindowAll || k_len > kWindowAll) return -1;
  if (nseq == 0 || q_len == 0) return 0;
  AttnWindow a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.bf16 = dtype;
  a.nseq = nseq;
  a.q_len = q_len;
  a.k_len = k_len;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.head_dim = head_dim;
  a.q_lens = q_lens;
  a.k_lens = k_lens;
  a.left = left < 0 || left > kWindowAll ? kWindowAll : left;
  a.right = right < 0 || right > kWindowAll ? kWindowAll : right;
  a.sinks = sinks;
  a.scale = fmaxf(scale, 1e-30f);  // at 0 a masked score (-inf) times it would be NaN
  if (!take_strides(q_strides, nseq, q_len, heads, head_dim, &a.qs) ||
      !take_strides(k_strides, nseq, k_len, kv_heads, head_dim, &a.ks) ||
      !take_strides(v_strides, nseq, k_len, kv_heads, head_dim, &a.vs) ||
      !take_strides(out_strides, nseq, q_len, heads, head_dim, &a.os))
    return -1;
  for (const void* p : {q, k, v, static_cast<const void*>(out)})
    if (reinterpret_cast<uintptr_t>(p) & 15) return -1;
  // 32-bit work counts inside
  if (static_cast<double>(nseq) * heads * q_len > 2147483647.0 * 8) return -1;
  int* st = device_status_word();
  if (!st) return -101;
  return attention_window(a, st, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
