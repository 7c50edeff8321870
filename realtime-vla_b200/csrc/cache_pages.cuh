// A key/value cache in pages of `block` tokens, held as e4m3 with one scale for each (page, head): the maps of the pages
// and the kernel that writes tokens into them.  Cache layout: codes [blocks][kv heads][block][head dim], so that the
// tokens of a head within a page are one contiguous piece; scales fp32 [blocks][kv heads]; value = code * scale.
#pragma once
#include <cuda_fp16.h>
#include "common.cuh"

// Bits VLA_ST_* of the operators in this translation unit: a bounded wait that ran out.
static __device__ int cache_ops_status;
static __device__ int cache_ops_taken;       // what the last look at it found

// Reads and clears in one step: a bit that is set meanwhile stays for the next look.
static __global__ void cache_status_kernel() { cache_ops_taken = atomicExch(&cache_ops_status, 0); }
// A wait that nothing ends, as the others are when something goes wrong.
static __global__ void cache_wait_kernel(unsigned long long limit_ns) {
  __shared__ __align__(8) uint64_t bar;
  __shared__ int abort_mem;
  mbar_init(smem_u32(&bar), 1);
  mbar_fence_init();
  abort_mem = 0;
  if (!mbar_wait_small(smem_u32(&bar), 0, &abort_mem, limit_ns)) atomicOr(&cache_ops_status, VLA_ST_WAIT_TIMEOUT);
}

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
  unsigned block_recip;  // see plan_div
  int total;             // rows of slots / positions
  int* slots;
  int* positions;
  int* cu_new;           // [n_seqs + 1]
  int* seq_lens;
  int* counts;           // next free, blocks missing, sum of new tokens
};

constexpr int PLAN_THREADS = 512;
constexpr int PLAN_MAX_SEQS = 8192;   // two sums of 4 bytes per request in shared memory

// x / block by the reciprocal floor(2^32 / block) (2^32 - 1 for blocks of 1), which falls short by one at most.  Lengths are
// below 2^31 and sums of two below 2^32, so that this is all in 32 bits.
__device__ __forceinline__ unsigned plan_div(unsigned x, const PlanParams& p) {
  const unsigned q = __umulhi(x, p.block_recip);
  return q + (x - q * p.block >= (unsigned)p.block);
}
__device__ __forceinline__ unsigned plan_blocks(unsigned tokens, const PlanParams& p) {      // ceil(tokens / block)
  const unsigned q = plan_div(tokens, p);
  return q + (q * p.block != tokens);
}
// Last index i in [lo, n) with a[i] <= x (a ascending, a[lo] <= x).
__device__ __forceinline__ int plan_find(const int* a, int lo, int n, int x) {
  int hi = n;
#pragma unroll 1
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}
// inclusive sum over the lanes of a warp
__device__ __forceinline__ long long plan_scan(long long x, int lane) {
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += up;
  }
  return x;
}

// Every CTA forms both sums itself (8 bytes per request, from L2 after the first CTA) instead of waiting for another
// kernel to do it, keeps them in shared memory and then writes its share of the tokens and of the new table entries.
// A few dependent steps on little data: what counts is how much code they run through once (some 8 clocks an instruction
// until it is in the caches), so loops stay loops and there is no division.
// Measured: 256 requests with a new token each 4.8 us (25 KB of code took 6.5), 512 requests with 1 to 2048 new tokens 5.5 us.
__global__ void __launch_bounds__(PLAN_THREADS) block_plan_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ int plan_smem[];
  int* cu = plan_smem;                   // [n_seqs + 1] first token row of each request
  int* off = plan_smem + p.n_seqs + 1;   // [n_seqs + 1] first new block of each request
  __shared__ long long warp_sum[2][PLAN_THREADS / 32], missing_sum[PLAN_THREADS / 32];
  static_assert(PLAN_THREADS / 32 <= 32, "a warp adds up the warps' sums");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  pdl_wait();
  const int first = p.first ? min(max(*p.first, 0), p.n_free) : 0;
  const int avail = p.n_free - first;
  constexpr long long TOP = 0x7fffffff;

  // A thread's requests are consecutive: it adds them up, the sums of all threads are scanned once, and it goes over its
  // requests again from there.
  const int per = (p.n_seqs + PLAN_THREADS - 1) / PLAN_THREADS;
  const int r0 = min((int)threadIdx.x * per, p.n_seqs), r1 = min(r0 + per, p.n_seqs);
  const unsigned width = p.width;
  unsigned ctx = 0, n = 0, have = 0, need = 0, missing_one = 0;
  auto look = [&](int b) {
    ctx = max(p.ctx[b], 0);
    n = max(p.n_new[b], 0);
    have = plan_blocks(ctx, p);
    const unsigned want = plan_blocks(ctx + n, p);
    need = min(want, width) - min(have, width);
    missing_one = (want - have) - need;
  };
  long long t0 = 0, b0 = 0, missing_wide = 0;
#pragma unroll 1
  for (int b = r0; b < r1; ++b) {
    look(b);
    t0 += n;
    b0 += need;
    missing_wide += missing_one;
  }
  long long all[2];
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {          // of tokens, then of blocks: over the warp, then over the CTA
    const long long own = i ? b0 : t0, in_warp = plan_scan(own, lane);
    if (lane == 31) warp_sum[i][warp] = in_warp;
    __syncthreads();
    const long long s = plan_scan(lane < PLAN_THREADS / 32 ? warp_sum[i][lane] : 0, lane);
    const long long before = __shfl_sync(0xffffffffu, s, (warp - 1) & 31), start = (warp ? before : 0) + in_warp - own;
    const long long total = __shfl_sync(0xffffffffu, s, 31);
    if (i) { b0 = start; all[1] = total; } else { t0 = start; all[0] = total; }
  }
#pragma unroll 1
  for (int b = r0; b < r1; ++b) {
    if (per > 1) look(b);
    cu[b] = (int)min(t0, TOP);
    off[b] = (int)min(b0, TOP);
    if (blockIdx.x == 0) {
      const long long granted = min(max((long long)avail - b0, 0ll), (long long)need);
      p.cu_new[b] = (int)min(t0, TOP);
      p.seq_lens[b] = (int)min(min((long long)(ctx + n), ((long long)min(have, width) + granted) * p.block), TOP);
    }
    t0 += n;
    b0 += need;
  }
  if (threadIdx.x == 0) {
    cu[p.n_seqs] = (int)min(all[0], TOP);
    off[p.n_seqs] = (int)min(all[1], TOP);
  }
  __syncthreads();
  const int sum_new = cu[p.n_seqs], sum_need = off[p.n_seqs];
  const int given = min(sum_need, avail);
  if (blockIdx.x == 0) {
    // blocks that no table column is left for are missing, too
    missing_wide = plan_scan(missing_wide, lane);
    if (lane == 31) missing_sum[warp] = missing_wide;
    __syncthreads();
    if (threadIdx.x == 0) {
      long long missing = sum_need - given;
#pragma unroll 1
      for (int w = 0; w < PLAN_THREADS / 32; ++w) missing += missing_sum[w];
      p.cu_new[p.n_seqs] = sum_new;
      p.counts[0] = first + given;
      p.counts[1] = (int)min(missing, TOP);
      p.counts[2] = sum_new;
    }
  }

  const int worker = blockIdx.x * PLAN_THREADS + threadIdx.x, workers = gridDim.x * PLAN_THREADS;
  // new table entries: the j-th block given away
#pragma unroll 1
  for (int j = worker; j < given; j += workers) {
    const int b = plan_find(off, 0, p.n_seqs, j);
    p.table[b * p.table_ld + plan_blocks(max(p.ctx[b], 0), p) + (j - off[b])] = p.free_ids[first + j];
  }
  // Slot and position of each token row.  An old block's id is read from the table (nothing in this call writes that
  // entry), a new one's from the free list.  Rows behind the last request get slot -1, position 0.
  // A warp does consecutive rows, 32 at a time, so that in long prompts a thread's next row is mostly the same request's.
  const long long each = ((long long)p.total + workers - 1) / workers * 32, t_end = min((long long)(worker / 32 + 1) * each, (long long)p.total);
  int b = 0;
#pragma unroll 1
  for (long long t = worker / 32 * each + lane; t < t_end; t += 32) {
    int slot = -1, pos = 0;
    if (t < sum_new) {
      if (t >= cu[b + 1]) b = plan_find(cu, b, p.n_seqs, (int)t);     // the last that begins here: the others have no new tokens
      const unsigned ctx = max(p.ctx[b], 0), at = ctx + (unsigned)((int)t - cu[b]), blk = plan_div(at, p);
      int id = -1;
      if (blk < (unsigned)p.width) {
        const unsigned have = plan_blocks(ctx, p);
        const long long nth = (long long)off[b] + (blk - have);
        if (blk < have) id = p.table[b * p.table_ld + blk];
        else if (nth < given) id = p.free_ids[first + nth];
      }
      const long long s = (long long)id * p.block + (at - blk * p.block);
      if (id >= 0 && s <= TOP) slot = (int)s;
      pos = (int)min(at, (unsigned)TOP);
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
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
  int window;                  // token rows that a warp looks for runs in: 1 .. 16
  uint32_t block_recip;        // ceil(2^32 / (block / 16)); 0 for blocks of 16
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
template <typename T>
struct Bits16;                 // exponent bits of the two 16-bit types, and the value that bits stand for
template <>
struct Bits16<bf16> {
  static constexpr uint32_t EXP = 0x7f80u;
  static __device__ __forceinline__ float value(uint32_t bits) { return __uint_as_float(bits << 16); }
};
template <>
struct Bits16<__half> {
  static constexpr uint32_t EXP = 0x7c00u;
  static __device__ __forceinline__ float value(uint32_t bits) { return __half2float(__ushort_as_half((unsigned short)bits)); }
};
// two floats -> two e4m3 codes (a in the low byte): nearest, ties to even, saturating at 448; NaN stays NaN
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
  uint16_t w;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(w) : "f"(b), "f"(a));
  return w;
}
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  uint32_t w;
  asm("{\n .reg .b16 lo, hi;\n cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n mov.b32 %0, {lo, hi};\n}"
      : "=r"(w) : "f"(a), "f"(b), "f"(c), "f"(d));
  return w;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t m;
  asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  return m;
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

constexpr int APPEND_THREADS = 128;
constexpr int append_ctas(int head_dim) { return head_dim == 256 ? 4 : 7; }      // on an SM at once
constexpr int APPEND_WINDOW = 16;        // token rows a warp looks for runs in, when there are many

// One warp writes the runs (the consecutive token rows of one block) that start in its window of token rows, for one head,
// keys or values: it finds the largest magnitude of a run, raises the block's scale to it if it has to, rounds what the
// block holds again under the new scale, and stores the run's codes.  A run has one writer, so nothing is atomic and the
// result does not depend on the order of warps.
// Bound by memory where there are many tokens, and two trips to memory long where there are few: the slots of a window and
// the row before it come in one load (a lane each), then 16 rows of a run, all in flight, with the block's scale; they stay
// in registers between the maximum and the rounding.  Only runs of more than 16 tokens are read twice.  The window is as
// wide as leaves a warp for every place on the GPU: 4096 rows of 8 heads of 64 take 18.3 us with windows of one row and
// 3.1 us with 16, one new token in each of 256 sequences 4.3 us either way.
// Measured (8 heads of 128, keys and values): 64 new tokens 2.9 us; 24 prompts of 40 to 2048 tokens 21.9 us, 4.5 TB/s of what must be
// read and written; 32k tokens of heads of 256 67 us, 5.8 TB/s.  What the prompts wait for is memory (long scoreboard 4.7 of 11
// stalls an issue, issue slots 42% active): a warp loads nothing while it rounds.
template <typename T, int D>
__global__ void __launch_bounds__(APPEND_THREADS, append_ctas(D)) cache_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int LPR = D / 8;              // lanes per row: 8 elements (16 bytes) each
  constexpr int RPI = 32 / LPR;           // rows per warp instruction
  constexpr int N = 16 / RPI;             // registers of 16 bytes for 16 rows
  constexpr uint32_t EXP = Bits16<T>::EXP * 0x10001u, TOP = 0x80008000u;
  const uint32_t FULL = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const unsigned items = 2u * p.kv_heads, job = blockIdx.x * (APPEND_THREADS / 32) + (threadIdx.x >> 5);
  const unsigned win = job / items, item = job - win * items;
  if ((unsigned long long)win * p.window >= (unsigned)p.tokens) return;
  const unsigned w0 = win * p.window;
  const int kv = item & 1, head = item >> 1;
  const int sub = lane / LPR, col = (lane % LPR) * 8;
  const T* const x = reinterpret_cast<const T*>(kv ? p.x[1] : p.x[0]) + head * (kv ? p.x_head[1] : p.x_head[0]) + col;
  const long long x_tok = kv ? p.x_tok[1] : p.x_tok[0];
  float* const scales = kv ? p.scale[1] : p.scale[0];
  uint8_t* const codes = kv ? p.codes[1] : p.codes[0];

  auto slot_at = [&](unsigned t) { return t < (unsigned)p.tokens ? p.slots[t] : -1; };      // w0 - 1 may be none
  // slot / block, by the reciprocal of block / 16 (exact below 2^27 for divisors of 16 or less); -1 outside the cache
  auto block_of = [&](int slot) {
    if (slot < 0 || slot >= p.n_slots) return -1;
    const uint32_t s16 = (uint32_t)slot >> 4;
    return (int)(p.block_recip ? __umulhi(s16, p.block_recip) : s16);
  };
  pdl_trigger();
  pdl_wait();
  const int slot_w = slot_at(w0 - 1 + lane), blk_w = block_of(slot_w);     // lane 0: the row before the window
  const int blk_before = __shfl_up_sync(FULL, blk_w, 1);
  uint32_t starts = __ballot_sync(FULL, lane >= 1 && lane <= p.window && blk_w >= 0 && blk_w != blk_before);

#pragma unroll 1
  for (; starts; starts &= starts - 1) {
    const int s = __ffs(starts) - 1;                    // the run's first row is w0 - 1 + s
    const unsigned t0 = w0 - 1 + s;
    const int blk = __shfl_sync(FULL, blk_w, s);
    float* const scale_at = scales + (long long)blk * p.kv_heads + head;
    uint8_t* const page = codes + ((long long)blk * p.kv_heads + head) * p.block * D;
    const float old = *scale_at;
    // Slots of a run's rows c .. c + 15 in lanes 0 .. 15; returns how many of them are the run's
    int slot;
    auto look = [&](unsigned c) {
      if (c == t0) slot = __shfl_sync(FULL, slot_w, (s + lane) & 31);     // s + 15 <= 31
      else slot = slot_at(c + (lane & 15));
      const uint32_t out = __ballot_sync(FULL, lane >= 16 || block_of(slot) != blk);
      return __ffs(out) - 1;
    };
    uint4 v[N];
    auto load = [&](unsigned c, int cnt) {
      const T* from = x + (long long)(c + sub) * x_tok;
#pragma unroll
      for (int i = 0; i < N; ++i, from += RPI * x_tok) {
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (i * RPI + sub < cnt) v[i] = *reinterpret_cast<const uint4*>(from);
      }
    };
    // largest finite magnitude of the rows held, as the bits of T: magnitudes compare as integers
    auto magnitude = [&]() {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < N; ++i)
        top = max_u16x2(top, max_u16x2(max_u16x2(v[i].x & ~TOP, v[i].y & ~TOP), max_u16x2(v[i].z & ~TOP, v[i].w & ~TOP)));
      uint32_t most = __reduce_max_sync(FULL, max(top & 0xffffu, top >> 16));
      if (most >= Bits16<T>::EXP) {       // an infinity or a NaN: again without those
        top = 0;
        auto finite = [](uint32_t w) {    // halves whose exponent is all ones become zero
          const uint32_t bad = ((w & ~TOP) + (TOP - EXP)) & TOP;
          return w & ~TOP & ~(bad | (bad - (bad >> 15)));
        };
#pragma unroll
        for (int i = 0; i < N; ++i)
          top = max_u16x2(top, max_u16x2(max_u16x2(finite(v[i].x), finite(v[i].y)), max_u16x2(finite(v[i].z), finite(v[i].w))));
        most = __reduce_max_sync(FULL, max(top & 0xffffu, top >> 16));
      }
      return most;
    };

    bool begun = false, again = false;    // holds the block's first slot; is longer than the 16 rows that registers keep
    uint32_t most = 0;
#pragma unroll 1
    for (unsigned c = t0;; c += 16) {
      const int cnt = look(c);
      if (cnt) {
        load(c, cnt);
        begun |= __any_sync(FULL, lane < cnt && slot == blk * p.block);
        most = max(most, magnitude());
        again |= c != t0;
      }
      if (cnt < 16) break;
      if (c == t0 && s + 16 <= 31 && __shfl_sync(FULL, blk_w, (s + 16) & 31) != blk) break;      // known without a look
    }
    const float need = block_scale(Bits16<T>::value(most));
    const float scale = begun ? need : fmaxf(old, need);
    if (!begun && scale > old) {          // warp-uniform
      const float ratio = old / scale;
      for (int i = lane * 16; i < p.block * D; i += 512) {
        uint4 u = *reinterpret_cast<const uint4*>(page + i);
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
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
    uint8_t* const to_page = page + col;
#pragma unroll 1
    for (unsigned c = t0;; c += 16) {
      const int cnt = look(c);
      if (again) load(c, cnt);
      const int off = slot - blk * p.block, before = __shfl_up_sync(FULL, off, 1);
      int keep = lane < cnt ? off : -1;
      // a slot named twice: the later token has it (the highest lane here, the later piece across pieces)
      if (__any_sync(FULL, lane > 0 && lane < cnt && off <= before)) {
        const uint32_t same = __match_any_sync(FULL, lane < cnt ? slot : -1 - lane);
        if (31 - __clz(same) != lane) keep = -1;
      }
      if (power) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int to = __shfl_sync(FULL, keep, i * RPI + sub);
          auto times = [&](uint32_t w) { return mul2(unpack2<T>(w), make_float2(inv, inv)); };
          const float2 a = times(v[i].x), b = times(v[i].y), f = times(v[i].z), g = times(v[i].w);
          const uint2 q = make_uint2(to_e4m3x4(a.x, a.y, b.x, b.y), to_e4m3x4(f.x, f.y, g.x, g.y));
          if (to >= 0) *reinterpret_cast<uint2*>(to_page + to * D) = q;
        }
      } else {                            // one row at a time, read again: 128 divisions in line were 70 KB of code
#pragma unroll 1
        for (int i = 0; i < cnt; i += RPI) {
          const int to = __shfl_sync(FULL, keep, (i + sub) & 31);
          if (to < 0) continue;
          const uint2* from = reinterpret_cast<const uint2*>(x + (long long)(c + i + sub) * x_tok);
#pragma unroll 1
          for (int k = 0; k < 2; ++k) {
            const uint2 w = from[k];
            const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
            *reinterpret_cast<uint32_t*>(to_page + to * D + 4 * k) = to_e4m3x4(a.x / scale, a.y / scale, b.x / scale, b.y / scale);
          }
        }
      }
      __syncwarp();
      if (!again || cnt < 16) break;
    }
  }
}
