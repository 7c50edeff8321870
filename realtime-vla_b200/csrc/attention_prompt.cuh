// Attention over packed prompts: sequence b owns rows cu_q[b] .. cu_q[b + 1] of q and o and rows cu_k[b] .. cu_k[b + 1] of
// k and v.  With nq, nk its lengths, row i sees the keys j < L_i, where L_i = nk, or min(nk, i + nk - nq + 1) when causal (the
// last row sees every key; keys that stand before the prompt's own are seen by all of its rows):
//     o_i = sum_{j < L_i} p_ij v_j / sum_{j < L_i} p_ij,   p_ij = exp(scale q_i . k_j - max_j)
// A row with L_i <= 0 is zero.  heads / kv_heads consecutive query heads share a key/value head.
#pragma once
#include <cuda_fp16.h>
#include "common.cuh"

struct PromptAttnParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  const int* cu_q;
  const int* cu_k;
  int n_seqs, tokens_q, tokens_k;
  int heads, kv_heads, dim;
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;
  int causal;
  float scale_log2e;
};

// One warp per (row, head), lanes over the head dim, one key after the other.
template <typename T>
__global__ void __launch_bounds__(128) prompt_attention_kernel(const PromptAttnParams p) {
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x, head = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (head >= p.heads) return;
  int b = 0, q0 = 0, q1 = 0;
  for (; b < p.n_seqs; ++b) {
    q0 = min(max(p.cu_q[b], 0), p.tokens_q);
    q1 = min(max(p.cu_q[b + 1], q0), p.tokens_q);
    if (t >= q0 && t < q1) break;
  }
  if (b == p.n_seqs) return;
  const int k0 = min(max(p.cu_k[b], 0), p.tokens_k), k1 = min(max(p.cu_k[b + 1], k0), p.tokens_k);
  const int nk = k1 - k0;
  const int limit = p.causal ? min(nk, t - q0 + nk - (q1 - q0) + 1) : nk;
  const int hk = head / (p.heads / p.kv_heads);
  const T* q = reinterpret_cast<const T*>(p.q) + t * p.q_tok + head * p.q_head;
  const T* k = reinterpret_cast<const T*>(p.k) + k0 * p.k_tok + hk * p.k_head;
  const T* v = reinterpret_cast<const T*>(p.v) + k0 * p.v_tok + hk * p.v_head;
  float qr[8], acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    qr[i] = d < p.dim ? (float)q[d] : 0.f;
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < limit; ++j) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < p.dim) s = fmaf(qr[i], (float)k[j * p.k_tok + lane + 32 * i], s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= p.scale_log2e;
    const float m_new = fmaxf(m, s);
    const float a = exp2f(m - m_new), e = exp2f(s - m_new);
    m = m_new;
    l = l * a + e;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < p.dim) acc[i] = acc[i] * a + e * (float)v[j * p.v_tok + lane + 32 * i];
  }
  T* o = reinterpret_cast<T*>(p.o) + t * p.o_tok + head * p.o_head;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < p.dim) o[lane + 32 * i] = (T)(limit > 0 ? acc[i] / l : 0.f);
}
