// A key/value cache in pages of `block` tokens, held as e4m3 with one scale for each (page, head): the maps of the pages
// and the kernel that writes tokens into them.  Cache layout: codes [blocks][kv heads][block][head dim], so that the
// tokens of a head within a page are one contiguous piece; scales fp32 [blocks][kv heads]; value = code * scale.
#pragma once
#include <cuda_fp16.h>
#include "common.cuh"

// Bits VLA_ST_* of the operators in this translation unit: a bounded wait that ran out.
static __device__ int cache_ops_status;

// ---- block tables and slot maps ------------------------------------------------------------------------------------
// Request b holds ctx[b] tokens in have = ceil(ctx / bs) blocks and gets n[b] more; it takes want - have blocks, want =
// ceil((ctx + n) / bs), from the free list, in request order.  Everything follows from two exclusive sums over the
// requests (new tokens, new blocks).
struct PlanParams {
  const int* ctx;
  const int* n_new;
  int n_seqs;
  int* table;            // [n_seqs, table_ld], width columns used
  int width;
  long long table_ld;
  const int* free_ids;
  int n_free;
  const int* first;      // blocks of the free list already given away (null: none)
  int block;
  int total;             // rows of slots / positions
  int* slots;
  int* positions;
  int* cu_new;           // [n_seqs + 1]
  int* seq_lens;
  int* counts;           // next free, blocks missing, sum of new tokens
};

constexpr int PLAN_THREADS = 512;
constexpr int PLAN_MAX_SEQS = 8192;   // two sums of 4 bytes per request in shared memory

// Last index i in [0, n) with a[i] <= x (a ascending, a[0] <= x).
__device__ __forceinline__ int plan_find(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Every CTA forms both sums itself (8 bytes per request, from L2 after the first CTA) instead of waiting for another
// kernel to do it, keeps them in shared memory and then writes its share of the tokens and of the new table entries.
__global__ void __launch_bounds__(PLAN_THREADS) block_plan_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];
  int* cu = plan_smem;                   // [n_seqs + 1] first token row of each request
  int* off = plan_smem + p.n_seqs + 1;   // [n_seqs + 1] first new block of each request
  __shared__ long long warp_sum[2][PLAN_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = p.first ? min(max(*p.first, 0), p.n_free) : 0;
  const int avail = p.n_free - first;
  long long carry_t = 0, carry_b = 0, missing_wide = 0;
  constexpr long long TOP = 0x7fffffff;

  for (int base = 0; base < p.n_seqs; base += PLAN_THREADS) {
    const int b = base + threadIdx.x;
    long long ctx = 0, n = 0;
    if (b < p.n_seqs) {
      ctx = max(p.ctx[b], 0);
      n = max(p.n_new[b], 0);
    }
    const long long have = (ctx + p.block - 1) / p.block, want = (ctx + n + p.block - 1) / p.block;
    const long long need = min(want, (long long)p.width) - min(have, (long long)p.width);
    missing_wide += (want - have) - need;
    long long st = n, sb = need;         // inclusive sums over the warp, then over the CTA
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long ut = __shfl_up_sync(0xffffffffu, st, o), ub = __shfl_up_sync(0xffffffffu, sb, o);
      if (lane >= o) { st += ut; sb += ub; }
    }
    if (lane == 31) { warp_sum[0][warp] = st; warp_sum[1][warp] = sb; }
    __syncthreads();
    long long all_t = 0, all_b = 0, pre_t = 0, pre_b = 0;
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 32; ++w) {
      if (w == warp) { pre_t = all_t; pre_b = all_b; }
      all_t += warp_sum[0][w];
      all_b += warp_sum[1][w];
    }
    const long long t0 = carry_t + pre_t + st - n, b0 = carry_b + pre_b + sb - need;
    if (b < p.n_seqs) {
      cu[b] = (int)min(t0, TOP);
      off[b] = (int)min(b0, TOP);
      if (blockIdx.x == 0) {
        const long long granted = min(max((long long)avail - b0, 0ll), need);
        p.cu_new[b] = (int)min(t0, TOP);
        p.seq_lens[b] = (int)min(min(ctx + n, (min(have, (long long)p.width) + granted) * p.block), TOP);
      }
    }
    carry_t += all_t;
    carry_b += all_b;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    cu[p.n_seqs] = (int)min(carry_t, TOP);
    off[p.n_seqs] = (int)min(carry_b, TOP);
  }
  // blocks that no table column is left for: summed over the CTA for the count of missing blocks
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) missing_wide += __shfl_xor_sync(0xffffffffu, missing_wide, o);
  if (lane == 0) warp_sum[0][warp] = missing_wide;
  __syncthreads();
  const int sum_new = cu[p.n_seqs], sum_need = off[p.n_seqs];
  const int given = min(sum_need, avail);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    long long missing = sum_need - given;
    for (int w = 0; w < PLAN_THREADS / 32; ++w) missing += warp_sum[0][w];
    p.cu_new[p.n_seqs] = sum_new;
    p.counts[0] = first + given;
    p.counts[1] = (int)min(missing, TOP);
    p.counts[2] = sum_new;
  }

  const int worker = blockIdx.x * PLAN_THREADS + threadIdx.x, workers = gridDim.x * PLAN_THREADS;
  // new table entries: the j-th block given away
  for (int j = worker; j < given; j += workers) {
    const int b = plan_find(off, p.n_seqs, j);
    const long long have = ((long long)max(p.ctx[b], 0) + p.block - 1) / p.block;
    p.table[b * p.table_ld + have + (j - off[b])] = p.free_ids[first + j];
  }
  // Slot and position of each token row.  An old block's id is read from the table (nothing in this call writes that
  // entry), a new one's from the free list.  Rows behind the last request get slot -1, position 0.
  // One thread does four consecutive rows, so that the two results leave as 16-byte stores.
  const long long quads = ((long long)p.total + 3) / 4;
  for (long long qd = worker; qd < quads; qd += workers) {
    const int t0 = (int)(qd * 4);
    int slot[4] = {-1, -1, -1, -1}, pos[4] = {0, 0, 0, 0};
    int b = t0 < sum_new ? plan_find(cu, p.n_seqs, t0) : p.n_seqs;
    for (int k = 0; k < 4; ++k) {
      const int t = t0 + k;
      if (t >= sum_new) break;
      while (t >= cu[b + 1]) ++b;        // requests without new tokens are passed over
      const int ctx = max(p.ctx[b], 0);
      const long long at = (long long)ctx + (t - cu[b]);
      const long long blk = at / p.block;
      const long long have = ((long long)ctx + p.block - 1) / p.block;
      int id = -1;
      if (blk < p.width) {
        if (blk < have) id = p.table[b * p.table_ld + blk];
        else if (off[b] + (blk - have) < given) id = p.free_ids[first + off[b] + (blk - have)];
      }
      const long long s = (long long)id * p.block + at % p.block;
      slot[k] = id >= 0 && s <= TOP ? (int)s : -1;
      pos[k] = (int)min(at, TOP);
    }
    if (t0 + 3 < p.total) {
      *reinterpret_cast<int4*>(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
      for (int k = 0; k < 4 && t0 + k < p.total; ++k) {
        p.slots[t0 + k] = slot[k];
        p.positions[t0 + k] = pos[k];
      }
    }
  }
}

// ---- writing tokens into the pages ---------------------------------------------------------------------------------
struct AppendParams {
  const void* x[2];            // keys, values: [tokens, kv heads, head dim]
  long long x_tok[2], x_head[2];
  uint8_t* codes[2];
  float* scale[2];
  const int* slots;
  int tokens, kv_heads, block;
  int window;                  // token rows per CTA
  long long n_slots;           // blocks * block
};

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<bf16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<bf16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// two floats -> two e4m3 codes (a in the low byte): nearest, ties to even, saturating at 448; NaN stays NaN
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
  uint16_t w;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(w) : "f"(b), "f"(a));
  return w;
}
// two e4m3 codes -> two floats (exact)
__device__ __forceinline__ float2 from_e4m3x2(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// The smallest 2^e >= 2^-60 that brings amax to 448 = 1.75 * 2^8 or less, from amax's own exponent and mantissa.
// A power of two makes x / scale exact, and e4m3 keeps the same relative precision whatever the power; so raising a
// block's scale later loses nothing but the last bits of codes that become subnormal.
__device__ __forceinline__ float block_scale(float amax) {
  const int bits = __float_as_int(amax);
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return __int_as_float((max(e, -60) + 127) << 23);
}

constexpr int APPEND_THREADS = 256;

// One warp writes one run (the consecutive token rows of one block) for one head, keys or values: it finds the largest
// magnitude of the run, raises the block's scale to it if it has to, rounds what the block holds again under the new
// scale, and stores the run's codes.  A run belongs to the CTA whose window of token rows it starts in, and has one
// writer, so nothing is atomic and the result does not depend on the order of CTAs.
template <typename T, int D>
__global__ void __launch_bounds__(APPEND_THREADS) cache_append_kernel(const AppendParams p) {
  constexpr int LPR = D / 8;              // lanes per row: 8 elements (16 bytes) each
  constexpr int RPI = 32 / LPR;           // rows per warp instruction
  __shared__ int run_at[32];
  __shared__ int n_runs;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int w0 = blockIdx.x * p.window;
  auto block_of = [&](int slot) { return slot >= 0 && slot < p.n_slots ? slot / p.block : -1; };
  if (warp == 0) {
    const int t = w0 + lane;
    bool start = false;
    if (lane < p.window && t < p.tokens) {
      const int b = block_of(p.slots[t]);
      start = b >= 0 && (t == 0 || block_of(p.slots[t - 1]) != b);
    }
    const uint32_t m = __ballot_sync(0xffffffffu, start);
    if (start) run_at[__popc(m & ((1u << lane) - 1u))] = t;
    if (lane == 0) n_runs = __popc(m);
  }
  __syncthreads();
  const int items = n_runs * p.kv_heads * 2;
  const int sub = lane / LPR, col = (lane % LPR) * 8;
  for (int item = warp; item < items; item += APPEND_THREADS / 32) {
    const int kv = item & 1, head = (item >> 1) % p.kv_heads, t0 = run_at[(item >> 1) / p.kv_heads];
    const T* x = reinterpret_cast<const T*>(p.x[kv]) + head * p.x_head[kv] + col;
    const int blk = block_of(p.slots[t0]);
    float* scale_at = p.scale[kv] + (long long)blk * p.kv_heads + head;
    uint8_t* page = p.codes[kv] + ((long long)blk * p.kv_heads + head) * p.block * D;
    const float old = *scale_at;

    // largest finite magnitude of the run; whether it holds the block's first slot
    float amax = 0.f;
    bool begun = false;
    for (int c = t0;; c += 32) {
      const int slot = c + lane < p.tokens ? p.slots[c + lane] : -1;
      const uint32_t out = __ballot_sync(0xffffffffu, block_of(slot) != blk);
      const int cnt = out ? __ffs(out) - 1 : 32;
      begun |= __any_sync(0xffffffffu, lane < cnt && slot % p.block == 0);
#pragma unroll 4
      for (int r = sub; r < cnt; r += RPI) {
        const uint4 v = *reinterpret_cast<const uint4*>(x + (c + r) * p.x_tok[kv]);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack2<T>(w[i]);
          const float a = fabsf(f.x), b = fabsf(f.y);
          if (a < INFINITY) amax = fmaxf(amax, a);
          if (b < INFINITY) amax = fmaxf(amax, b);
        }
      }
      if (cnt < 32) break;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float need = block_scale(amax);
    const float scale = begun ? need : fmaxf(old, need);
    if (!begun && scale > old) {          // warp-uniform
      const float ratio = old / scale;
      for (int i = lane * 16; i < p.block * D; i += 512) {
        uint4 v = *reinterpret_cast<const uint4*>(page + i);
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 lo = from_e4m3x2(w[k] & 0xffffu), hi = from_e4m3x2(w[k] >> 16);
          w[k] = to_e4m3x2(lo.x * ratio, lo.y * ratio) | to_e4m3x2(hi.x * ratio, hi.y * ratio) << 16;
        }
        *reinterpret_cast<uint4*>(page + i) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    __syncwarp();                         // the run's codes go over the ones that were rounded again
    if (lane == 0 && scale != old) *scale_at = scale;
    const bool power = (__float_as_int(scale) & 0x7fffff) == 0;   // a scale another writer chose may be no power of two
    const float inv = 1.f / scale;
    for (int c = t0;; c += 32) {
      const int slot = c + lane < p.tokens ? p.slots[c + lane] : -1;
      const uint32_t out = __ballot_sync(0xffffffffu, block_of(slot) != blk);
      const int cnt = out ? __ffs(out) - 1 : 32;
      // a slot named twice: the later token has it (the highest lane here, the later chunk across chunks)
      const uint32_t same = __match_any_sync(0xffffffffu, lane < cnt ? slot : -1 - lane);
      const int keep = 31 - __clz(same) == lane && lane < cnt ? slot % p.block : -1;
      for (int r0 = 0; r0 < cnt; r0 += RPI) {
        const int off = __shfl_sync(0xffffffffu, keep, (r0 + sub) & 31);
        if (r0 + sub < cnt && off >= 0) {
          const uint4 v = *reinterpret_cast<const uint4*>(x + (c + r0 + sub) * p.x_tok[kv]);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
          uint32_t q[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(w[i]);
            q[i] = power ? to_e4m3x2(f.x * inv, f.y * inv) : to_e4m3x2(f.x / scale, f.y / scale);
          }
          *reinterpret_cast<uint2*>(page + off * D + col) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
        }
      }
      __syncwarp();
      if (cnt < 32) break;
    }
  }
}
