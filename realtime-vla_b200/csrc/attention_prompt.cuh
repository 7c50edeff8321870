// Attention over packed prompts: sequence b owns rows cu_q[b] .. cu_q[b + 1] of q and o and rows cu_k[b] .. cu_k[b + 1] of
// k and v.  With nq, nk its lengths, row i sees the keys j < L_i, where L_i = nk, or min(nk, i + nk - nq + 1) when causal (the
// last row sees every key; keys that stand before the prompt's own are seen by all of its rows):
//     o_i = sum_{j < L_i} p_ij v_j / sum_{j < L_i} p_ij,   p_ij = exp(scale q_i . k_j - max_j)
// A row with L_i <= 0 is zero.  heads / kv_heads consecutive query heads share a key/value head.
//
// One CTA = one tile of 128 rows: the G = heads / kv_heads query heads of 128 / G consecutive tokens, which share their
// keys, so that short prompts fill tiles too and a causal tile's diagonal is only 128 / G keys wide.  Chunks of 128 (64) keys:
//     S[128 x 128]  = Q . K_chunk^T       tcgen05.mma, both operands K-major in shared memory
//     P             = exp2(S scale - m)   one thread per row, straight from TMEM, written back over S as 16-bit pairs
//     O[128 x dim] += P . V_chunk         tcgen05.mma, A = P in TMEM, B = V as it lies in memory (MN-major), so V needs
//                                         neither a transposed copy nor a pass through registers
// P is rounded to the operands' type, because P V takes both of one type; a row's sum is of the unrounded ones, which costs half a step
// of the type on each probability and no more.  The maximum m a row subtracts is only moved when it grows by more than 2^8 (probabilities then stay below 2^8, sums in
// fp32), so that O in TMEM is rescaled a few times per tile instead of once per chunk.
// Roles: warp 0 = tile lookup and TMA producer, warp 1 = MMA issuer and TMEM owner, warps 2..5 = softmax and epilogue.
// All mbarrier waits are bounded.
#pragma once
#include <type_traits>
#include "cache_pages.cuh"

struct PromptAttnParams {
  CUtensorMap tmQ;   // [token][kv head][group head][dim], box 64 x G x 1 x tokens of a tile
  CUtensorMap tmK;   // [token][kv head][dim], box 64 x 1 x KEYS
  CUtensorMap tmV;   // the same, box 64 x 1 x V_ROWS
  const void* v;
  void* o;
  const int* cu_q;
  const int* cu_k;
  int n_seqs, tokens_q, tokens_k;
  int kv_heads, group, dim;
  int tile_tokens;   // 128 / group
  long long v_tok, v_head, o_tok, o_head;
  int causal;
  float scale_log2e;
};

// Two S buffers, so that the next chunk's S is there when the softmax has finished a chunk.  Up to 128 columns of head dim a
// CTA takes half an SM (96 KB of shared memory, 256 TMEM columns) with chunks of 64 keys, and the two CTAs of an SM
// share its tensor core and its exponentials; wider heads need the whole SM, with chunks of 128 keys whose K and V come in
// halves of 32 KB.
// What bounds it: an MMA of 128 rows and 16 steps of K takes about 85 clocks for N = 64 as for N = 128 and 125 for N = 256, so
// S of 64 keys costs as much as S of 128.  Measured: one causal prompt of 8192, 32 heads on 8 of 128, 482 to 500 us, 1.1 PFLOP/s (566 in
// a long row of calls, when the clock falls); 48 ragged prompts of the same heads 134 us (146).  With chunks of 128 keys there is TMEM for one S buffer a CTA only: 674 and
// 198 us.  32 prompts of 276 to 968, 8 heads on 1 of 256, 138 us, 0.72 PFLOP/s: there the loads before a tile's first MMA and
// the stores behind its last, 11,600 of 25,600 clocks, run under nothing.
template <bool WIDE>
struct PromptCfg {
  static constexpr int BOXES = WIDE ? 4 : 2;              // 64-column boxes of head dim, at most
  static constexpr int KEYS = WIDE ? 128 : 64;            // keys per chunk
  static constexpr int AHEAD = 2;                         // S buffers = chunks of S in flight
  static constexpr int UNITS = WIDE ? 2 : 1;              // ring slots per K or V chunk
  static constexpr int STAGES = WIDE ? 5 : 4;
  static constexpr int V_ROWS = KEYS / UNITS;
  static constexpr int Q_BOX = 128 * 128, K_BOX = KEYS * 128, V_BOX = V_ROWS * 128;   // bytes of 64 columns x rows
  static constexpr int SLOT_BYTES = 2 * K_BOX;            // K: 2 boxes x KEYS; V: BOXES boxes x V_ROWS keys
  static constexpr int Q_BYTES = BOXES * Q_BOX;
  static constexpr int SMEM_BYTES = Q_BYTES + STAGES * SLOT_BYTES + 256 + 1024;
  static constexpr int TMEM_COLS = WIDE ? 512 : 256;      // S buffers, then O
  static constexpr int O_COL = AHEAD * KEYS;
  static constexpr int THREADS = 192;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tm, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(tm), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem desc]; A holds two consecutive K elements per 32-bit column.
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// MN-major operand (rows of K, 64 MN columns of 128 bytes each, 128-byte swizzle): 8-row groups 1024 bytes apart, the next
// 64 columns `box_bytes` further.
__device__ __forceinline__ uint64_t prompt_desc_mn(uint32_t smem_addr, uint32_t box_bytes) {
  return (uint64_t)((smem_addr & 0x3FFFF) >> 4) | ((uint64_t)(box_bytes >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// two fp32 operations an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(PromptCfg<WIDE>::THREADS, WIDE ? 1 : 2) prompt_attention_kernel(const __grid_constant__ PromptAttnParams p) {
  using C = PromptCfg<WIDE>;
  constexpr uint32_t EXP = Bits16<T>::EXP;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
  const uint32_t sQ = raw_addr + pad, sRing = sQ + C::Q_BYTES;
  uint8_t* ring = smem_raw + pad + C::Q_BYTES;
  uint8_t* bar_ptr = ring + C::STAGES * C::SLOT_BYTES;
  const uint32_t bars = sRing + C::STAGES * C::SLOT_BYTES;
  const uint32_t q_full = bars;
  auto full = [&](int s) { return bars + 8 + 16 * s; };
  auto empty = [&](int s) { return bars + 16 + 16 * s; };
  auto s_full = [&](int b) { return bars + 96 + 8 * b; };
  auto p_ready = [&](int b) { return bars + 112 + 8 * b; };
  auto o_done = [&](int b) { return bars + 128 + 8 * b; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_ptr + 160);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bar_ptr + 164);
  volatile int* poison = reinterpret_cast<volatile int*>(bar_ptr + 168);   // a hidden value was not finite
  volatile int* tile_seq = reinterpret_cast<volatile int*>(bar_ptr + 172);
  volatile int* tile_at = reinterpret_cast<volatile int*>(bar_ptr + 176);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.x % p.kv_heads;
  if (warp == 0) {
    pdl_wait();
    // Which tile this CTA is: the sequences' tiles are counted from cu_q on the device, 32 sequences at a time.  A
    // causal sequence hands out its last tiles first, because they have the most keys.
    int idx = blockIdx.x / p.kv_heads, seq = -1, at = 0;
    for (int base = 0; base < p.n_seqs && seq < 0; base += 32) {
      int tiles = 0;
      if (base + lane < p.n_seqs) {
        const int a = min(max(p.cu_q[base + lane], 0), p.tokens_q), e = min(max(p.cu_q[base + lane + 1], a), p.tokens_q);
        tiles = (e - a + p.tile_tokens - 1) / p.tile_tokens;
      }
      int sum = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += u;
      }
      const int total = __shfl_sync(0xffffffffu, sum, 31);
      if (idx < total) {
        const int l = __ffs(__ballot_sync(0xffffffffu, sum > idx)) - 1;
        const int t = idx - __shfl_sync(0xffffffffu, sum - tiles, l);
        seq = base + l;
        at = p.causal ? __shfl_sync(0xffffffffu, tiles, l) - 1 - t : t;
      }
      idx -= total;
    }
    if (lane == 0) {
      *tile_seq = seq;
      *tile_at = at * p.tile_tokens;
    }
  } else if (warp == 1) {
    pdl_wait();          // before the TMEM: a CTA of the kernel before this one may yet have to take its own
    tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
  } else if (threadIdx.x == 64) {
    mbar_init(q_full, 1);
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(s_full(b), 1);
      mbar_init(p_ready(b), 128);
      mbar_init(o_done(b), 1);
    }
    *abort_flag = 0;
    *poison = 0;
    mbar_fence_init();
    tma_prefetch_desc(&p.tmQ);
    tma_prefetch_desc(&p.tmK);
    tma_prefetch_desc(&p.tmV);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int seq = *tile_seq;
  pdl_trigger();       // the TMEM is there: no CTA of the next kernel can take it first and wait for this one
  pdl_wait();

  // Lengths, and the limits of the tile's first and last row (every thread: four words from L1 / L2)
  int q0 = 0, nq = 0, k0 = 0, nk = 0;
  const int tok0 = *tile_at;
  if (seq >= 0) {
    q0 = min(max(p.cu_q[seq], 0), p.tokens_q);
    nq = min(max(p.cu_q[seq + 1], q0), p.tokens_q) - q0;
    k0 = min(max(p.cu_k[seq], 0), p.tokens_k);
    nk = min(max(p.cu_k[seq + 1], k0), p.tokens_k) - k0;
  }
  const int last_tok = min(tok0 + p.tile_tokens, nq) - 1;
  auto limit_of = [&](int tok) { return p.causal ? min(max(tok + nk - nq + 1, 0), nk) : nk; };
  const int lim_min = seq >= 0 ? limit_of(tok0) : 0, lim_max = seq >= 0 ? limit_of(last_tok) : 0;
  const int n_chunks = (lim_max + C::KEYS - 1) / C::KEYS;
  const int boxes = (p.dim + 63) / 64;
  // position of a K or V chunk in the ring's order of use: K_0 .. K_{AHEAD-1}, then V_c, K_{c+AHEAD} in turn
  auto k_pos = [&](int c) { return C::UNITS * (c < C::AHEAD ? c : 2 * c - C::AHEAD + 1); };
  auto v_pos = [&](int c) { return C::UNITS * (min(c + C::AHEAD, n_chunks) + c); };

  if (warp == 0) {
    if (lane == 0 && n_chunks > 0) {
      const int rows = p.group * p.tile_tokens;
      mbar_expect_tx(q_full, boxes * rows * 128);
      for (int x = 0; x < boxes; ++x) tma_load_4d(sQ + x * C::Q_BOX, &p.tmQ, q_full, x * 64, 0, kvh, q0 + tok0);
      bool ok = true;
      auto slot_free = [&](int pos) {
        return pos < C::STAGES || mbar_wait_small(empty(pos % C::STAGES), (uint32_t)(pos / C::STAGES - 1) & 1u, abort_flag);
      };
      const uint64_t pol = policy_evict_last();   // other tiles of this sequence read the same keys
      auto load_k = [&](int c) {
        for (int u = 0; u < C::UNITS && ok; ++u) {
          const int pos = k_pos(c) + u, s = pos % C::STAGES;
          ok = slot_free(pos);
          if (!ok) return;
          const int b0 = u * 2, nb = min(boxes - b0, 2);     // at least one: wider heads than 128 have three boxes or four
          mbar_expect_tx(full(s), nb * C::K_BOX);
          for (int x = 0; x < nb; ++x)
            tma_load_3d(sRing + s * C::SLOT_BYTES + x * C::K_BOX, &p.tmK, full(s), (b0 + x) * 64, kvh, k0 + c * C::KEYS, pol);
        }
      };
      auto load_v = [&](int c) {
        for (int u = 0; u < C::UNITS && ok; ++u) {
          const int pos = v_pos(c) + u, s = pos % C::STAGES;
          ok = slot_free(pos);
          if (!ok) return;
          mbar_expect_tx(full(s), boxes * C::V_BOX);
          for (int x = 0; x < boxes; ++x)
            tma_load_3d(sRing + s * C::SLOT_BYTES + x * C::V_BOX, &p.tmV, full(s), x * 64, kvh, k0 + c * C::KEYS + u * C::V_ROWS, pol);
        }
      };
      for (int c = 0; c < min(C::AHEAD, n_chunks); ++c) load_k(c);
      for (int c = 0; c < n_chunks && ok; ++c) {
        load_v(c);
        if (c + C::AHEAD < n_chunks) load_k(c + C::AHEAD);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && n_chunks > 0) {
      constexpr uint32_t TYPE = std::is_same<T, bf16>::value ? 1u : 0u;      // both operands bf16, or both fp16
      const uint32_t idesc = (1u << 4) | (TYPE << 7) | (TYPE << 10) | (8u << 24);
      const int k_steps = (p.dim + 15) / 16;
      const uint32_t idesc_o = idesc | (1u << 16) | ((uint32_t)(k_steps * 2) << 17);      // N = head dim, B MN-major
      bool ok = mbar_wait_small(q_full, 0, abort_flag);
      // The loops are unrolled over what the tile can hold, with the descriptors as constants from a base: formed step by
      // step, an MMA took this one thread about 140 clocks to issue, more than twice what it runs for.
      const uint64_t q_desc = attn_desc_sw128(sQ), k_desc = attn_desc_sw128(sRing), v_desc = prompt_desc_mn(sRing, C::V_BOX);
      auto wait_units = [&](int pos0) {
        for (int u = 0; u < C::UNITS; ++u) {
          const int pos = pos0 + u;
          ok = ok && mbar_wait_small(full(pos % C::STAGES), (uint32_t)(pos / C::STAGES) & 1u, abort_flag);
        }
      };
      auto issue_s = [&](int c) {
        // the last chunk multiplies only the keys that some row sees, rounded up to 16
        const int keys16 = (min(lim_max - c * C::KEYS, C::KEYS) + 15) / 16;
        const uint32_t idesc_s = idesc | ((uint32_t)(keys16 * 2) << 17), d = tmem + (c % C::AHEAD) * C::KEYS;
#pragma unroll
        for (int u = 0; u < C::UNITS; ++u) {
          const int s = (k_pos(c) + u) % C::STAGES;
          const uint64_t kd = k_desc + s * (C::SLOT_BYTES / 16);
          const int mine = k_steps - u * 8;     // steps of 16 head dims in this slot
          auto step = [&](int ks) {
            umma_bf16(d, q_desc + (u * 2 + ks / 4) * (C::Q_BOX / 16) + 2 * (ks % 4), kd + (ks / 4) * (C::K_BOX / 16) + 2 * (ks % 4), idesc_s, (u | ks) != 0);
          };
          if (mine >= 8) {
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) step(ks);
          } else {
#pragma unroll 1
            for (int ks = 0; ks < mine; ++ks) step(ks);
          }
          umma_commit(empty(s));
        }
        umma_commit(s_full(c % C::AHEAD));
      };
      for (int c = 0; c < min(C::AHEAD, n_chunks) && ok; ++c) {
        wait_units(k_pos(c));
        tc_fence_after();
        if (ok) issue_s(c);
      }
      for (int c = 0; c < n_chunks && ok; ++c) {
        // What the loads bring is waited for first, so that nothing but P stands before the MMAs: V of this chunk, and K of
        // the chunk whose S goes over this one's P (its slot was that of a K whose S is long formed, not of this V).
        const int buf = c % C::AHEAD;
        const bool more = c + C::AHEAD < n_chunks;
        wait_units(v_pos(c));
        if (more) wait_units(k_pos(c + C::AHEAD));
        ok = ok && mbar_wait_small(p_ready(buf), (uint32_t)(c / C::AHEAD) & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const int keys16 = (min(lim_max - c * C::KEYS, C::KEYS) + 15) / 16;
#pragma unroll
        for (int u = 0; u < C::UNITS; ++u) {
          const int s = (v_pos(c) + u) % C::STAGES;
          const uint64_t vd = v_desc + s * (C::SLOT_BYTES / 16);
          const uint32_t p_at = tmem + buf * C::KEYS + u * (C::V_ROWS / 2);
          auto step = [&](int kk) { umma_ts(tmem + C::O_COL, p_at + kk * 8, vd + 128 * kk, idesc_o, (c | u | kk) != 0); };
          if (keys16 >= 4 * u + 4) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) step(kk);
          } else {
#pragma unroll 1
            for (int kk = 0; kk < keys16 - 4 * u; ++kk) step(kk);
          }
          umma_commit(empty(s));
        }
        umma_commit(o_done(c & 1));
        // S of chunk c + AHEAD goes over P of chunk c: the tensor core takes MMAs in the order of their issue
        if (more) issue_s(c + C::AHEAD);
      }
    }
    __syncwarp();
  } else {
    // ---------------- softmax and epilogue: one row per thread ----------------
    const int quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const int tok = tok0 + r / p.group;
    const bool row_ok = seq >= 0 && r < p.group * p.tile_tokens && tok < nq;
    const int limit = row_ok ? limit_of(tok) : 0;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int c = 0; c < n_chunks && ok; ++c) {
      const int buf = c % C::AHEAD;
      ok = __all_sync(0xffffffffu, mbar_wait_small(s_full(buf), (uint32_t)(c / C::AHEAD) & 1u, abort_flag));
      if (!ok) break;
      tc_fence_after();
      const uint32_t ts = tmem + lane_off + buf * C::KEYS;
      float s[C::KEYS];
#pragma unroll
      for (int g = 0; g < C::KEYS / 32; ++g) tmem_ld32(ts + 32 * g, reinterpret_cast<uint32_t*>(s) + 32 * g);
      tmem_ld_wait();
      const int vis = limit - c * C::KEYS;
      if (!__all_sync(0xffffffffu, vis >= C::KEYS)) {
#pragma unroll
        for (int j = 0; j < C::KEYS; ++j)
          if (j >= vis) s[j] = -INFINITY;
      }
      float mx[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) mx[j] = s[j];
#pragma unroll
      for (int j = 8; j < C::KEYS; j += 16)
#pragma unroll
        for (int k = 0; k < 8; ++k) mx[k] = fmaxf(fmaxf(mx[k], s[j + k]), j + 8 + k < C::KEYS ? s[j + 8 + k] : s[j + k]);   // three inputs an instruction
      const float top = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7]))) * p.scale_log2e;
      // the first chunk sets the maximum; later it moves when a row of this warp has outgrown it by 2^8
      if (__any_sync(0xffffffffu, top > m + 8.f)) {
        const float m_new = fmaxf(m, top);
        if (c > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait_small(o_done((c - 1) & 1), (uint32_t)((c - 1) >> 1) & 1u, abort_flag));
          if (!ok) break;
          tc_fence_after();
          const float a = m == m_new ? 1.f : ex2_approx(m - m_new);
          l *= a;
#pragma unroll 1
          for (int d = 0; d < p.dim; d += 32) {
            uint32_t v[32];
            tmem_ld32(tmem + lane_off + C::O_COL + d, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * a);
            tmem_st32(tmem + lane_off + C::O_COL + d, v);
          }
        }
        m = m_new;
      }
      const float sub = m == -INFINITY ? 0.f : m;        // a row that has seen nothing yet
      const float2 scale2 = make_float2(p.scale_log2e, p.scale_log2e), sub2 = make_float2(-sub, -sub);
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int g = 0; g < C::KEYS / 64; ++g) {
        uint32_t w[32];
#pragma unroll
        for (int j = 0; j < 64; j += 2) {
          float2 e = fma2(make_float2(s[64 * g + j], s[64 * g + j + 1]), scale2, sub2);
          e.x = ex2_approx(e.x);
          e.y = ex2_approx(e.y);
          sum[j >> 1 & 1] = add2(sum[j >> 1 & 1], e);
          w[j >> 1] = pack2<T>(e.x, e.y);
        }
        tmem_st32(ts + 32 * g, w);
      }
      l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      if ((c + 1) * C::KEYS > lim_min) {
        // Keys that not every row sees (the causal diagonal) or that none does (behind the last key, up to the MMA's step of
        // 16): their P is zero in the rows that do not see them, but zero times NaN or infinity is NaN.  Such values are
        // cleared in shared memory; the epilogue gives them back to the rows that see them.  S of this chunk and the P V
        // before it are over, so V's slots are past their earlier uses and a look at them cannot take one for this use.
        // After the exponentials, so that the wait for that P V runs under them.
        if (c > 0) ok = __all_sync(0xffffffffu, mbar_wait_small(o_done((c - 1) & 1), (uint32_t)((c - 1) >> 1) & 1u, abort_flag));
        const int at = v_pos(c), s0 = at % C::STAGES, s1 = (at + C::UNITS - 1) % C::STAGES;
#pragma unroll
        for (int u = 0; u < C::UNITS; ++u)
          ok = ok && __all_sync(0xffffffffu, mbar_wait_small(full(u ? s1 : s0), (uint32_t)((at + u) / C::STAGES) & 1u, abort_flag));
        if (!ok) break;
        const int lo = max(lim_min - c * C::KEYS, 0), tail = lim_max - c * C::KEYS, hi = (min(tail, C::KEYS) + 15) / 16 * 16;
        constexpr int PIECES = C::BOXES * 8;           // of a key's row, 16 bytes each
        const int piece = r % PIECES;
        uint8_t* const column = ring + (piece >> 3) * C::V_BOX + (piece & 7) * 16;
        if (piece >> 3 < boxes) {
#pragma unroll 2
          for (int j = lo + r / PIECES; j < hi; j += 128 / PIECES) {
            uint4* const w4 = reinterpret_cast<uint4*>(column + (j < C::V_ROWS ? s0 : s1) * C::SLOT_BYTES + j % C::V_ROWS * 128);
            uint4 w = *w4;
            // the exponents inverted: a half whose bits were all ones is zero, and taking one from it sets its top bit
            auto bad = [](uint32_t b) { return ((~b & EXP * 0x10001u) - 0x10001u) & 0x80008000u; };
            if (j >= tail) {
              *w4 = make_uint4(0u, 0u, 0u, 0u);
            } else if (bad(w.x) | bad(w.y) | bad(w.z) | bad(w.w)) {
              auto clean = [](uint32_t b) {
                return ((b & EXP) == EXP ? 0u : b & 0xffffu) | ((b >> 16 & EXP) == EXP ? 0u : b & 0xffff0000u);
              };
              *w4 = make_uint4(clean(w.x), clean(w.y), clean(w.z), clean(w.w));
              *poison = 1;
            }
          }
        }
        fence_proxy_async_shared();
        __syncwarp();
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_ready(buf));
    }
    if (ok && n_chunks > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait_small(o_done((n_chunks - 1) & 1), (uint32_t)((n_chunks - 1) >> 1) & 1u, abort_flag));
      tc_fence_after();
    }
    if (!ok) l = NAN;                            // a wait ran out: no row is left as it was
    if (seq >= 0) {
      const float inv = l != 0.f ? 1.f / l : 0.f;         // nothing seen: O is zero or was never written
      const bool any_poison = *poison != 0;
      const long long row_at = (long long)(q0 + tok) * p.o_tok + (long long)(kvh * p.group + r % p.group) * p.o_head;
      const uint32_t rows_ok = __ballot_sync(0xffffffffu, row_ok);
      // Through Q's shared memory (its last product is over), so that rows leave as whole lines: stored by the thread that
      // has the row, 16 bytes of 32 rows an instruction, the end of a tile of 256 head dims took 5800 clocks.
#pragma unroll 1
      for (int d = 0; d < p.dim; d += 32) {
        uint32_t v[32];
        if (n_chunks > 0) {
          tmem_ld32(tmem + lane_off + C::O_COL + d, v);
          tmem_ld_wait();
        }
        float f[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] = l != 0.f ? __uint_as_float(v[j]) * inv : 0.f;
        if (any_poison) {
#pragma unroll 1
          for (int key = lim_min; key < limit; ++key) {
            const unsigned short* vr = reinterpret_cast<const unsigned short*>(p.v) + (long long)(k0 + key) * p.v_tok + kvh * p.v_head + d;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (d + j < p.dim && (vr[j] & EXP) == EXP) f[j] += Bits16<T>::value(vr[j]);
          }
          __syncwarp();
        }
#pragma unroll
        for (int j = 0; j < 32; j += 8)
          *reinterpret_cast<uint4*>(smem_raw + pad + ((d + j) >> 6) * C::Q_BOX + r * 128 + ((((d + j) >> 3 & 7) ^ (r & 7)) << 4)) =
              make_uint4(pack2<T>(f[j], f[j + 1]), pack2<T>(f[j + 2], f[j + 3]), pack2<T>(f[j + 4], f[j + 5]), pack2<T>(f[j + 6], f[j + 7]));
      }
      __syncwarp();
      constexpr int LANES = C::BOXES * 8;        // per row, 16 bytes each
      const int piece = lane % LANES;
      const uint8_t* from = smem_raw + pad + (piece >> 3) * C::Q_BOX;
#pragma unroll 4
      for (int k = lane / LANES; k < 32; k += 32 / LANES) {
        const long long at = __shfl_sync(0xffffffffu, row_at, k);
        const int rr = quarter * 32 + k;
        if ((rows_ok >> k & 1) && piece * 8 < p.dim)
          *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.o) + at + piece * 8) =
              *reinterpret_cast<const uint4*>(from + rr * 128 + (((piece & 7) ^ (rr & 7)) << 4));
      }
    }
  }

  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {   // a wait ran out: say so, and let copies in flight land before the shared memory goes to another CTA
    if (threadIdx.x == 0) atomicOr(&cache_ops_status, VLA_ST_WAIT_TIMEOUT);
    for (int i = 0; i < 32; ++i) __nanosleep(1000);
  }
  if (warp == 1) tmem_dealloc(tmem, C::TMEM_COLS);
}
