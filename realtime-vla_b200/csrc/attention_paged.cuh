// Attention of the newest tokens of every sequence over its cache in pages (e4m3 codes, one scale for each page and head;
// layout in cache_pages.cuh).  q[b][i] is token lens[b] - n + i of sequence b and sees the keys j <= lens[b] - n + i; key j is
// row j % block of page table[b][j / block].  A page id outside the cache is not seen.  A row that sees nothing is zero.
#pragma once
#include "cache_pages.cuh"

struct PagedAttnParams {
  const void* q;
  void* o;
  long long q_seq, q_tok, q_head, o_seq, o_tok, o_head;
  const uint8_t* kc;
  const uint8_t* vc;
  const float* ks;
  const float* vs;
  const int* table;
  long long table_ld;
  const int* lens;
  int n_seqs, n_q, heads, kv_heads, dim;
  int blocks, block, width;
  float scale_log2e;
};

// One warp per (sequence, token, head), lanes over the head dim, one key after the other.
template <typename T>
__global__ void __launch_bounds__(128) paged_attention_kernel(const PagedAttnParams p) {
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.x / p.n_q, i = blockIdx.x % p.n_q, head = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (head >= p.heads) return;
  const int hk = head / (p.heads / p.kv_heads);
  const int len = (int)min(max((long long)p.lens[b], 0ll), (long long)p.width * p.block);
  const int limit = len - p.n_q + 1 + i;
  const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_seq + i * p.q_tok + head * p.q_head;
  float qr[8], acc[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    qr[c] = lane + 32 * c < p.dim ? (float)q[lane + 32 * c] : 0.f;
    acc[c] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < limit; ++j) {
    const int id = p.table[b * p.table_ld + j / p.block];
    if (id < 0 || id >= p.blocks) continue;
    const long long row = ((long long)id * p.kv_heads + hk) * p.block + j % p.block;
    const float ks = p.ks[(long long)id * p.kv_heads + hk], vs = p.vs[(long long)id * p.kv_heads + hk];
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (lane + 32 * c < p.dim) s = fmaf(qr[c], from_e4m3x2(p.kc[row * p.dim + lane + 32 * c]).x, s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= p.scale_log2e * ks;
    const float m_new = fmaxf(m, s);
    const float a = exp2f(m - m_new), e = exp2f(s - m_new);
    m = m_new;
    l = l * a + e;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (lane + 32 * c < p.dim) acc[c] = acc[c] * a + e * vs * from_e4m3x2(p.vc[row * p.dim + lane + 32 * c]).x;
  }
  T* o = reinterpret_cast<T*>(p.o) + b * p.o_seq + i * p.o_tok + head * p.o_head;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (lane + 32 * c < p.dim) o[lane + 32 * c] = (T)(l != 0.f ? acc[c] / l : 0.f);
}
