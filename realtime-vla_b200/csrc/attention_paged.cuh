// Attention of the newest tokens of every sequence over its cache in pages (e4m3 codes, one scale for each page and head;
// layout in cache_pages.cuh).  q[b][i] is token lens[b] - n + i of sequence b and sees the keys j <= lens[b] - n + i; key j is
// row j % block of page table[b][j / block].  A page id outside the cache is not seen.  A row that sees nothing is zero.
//
// Bound by the bytes of the cache: each code is read once, for the n * heads / kv_heads rows that share it.  The codes go
// from TMA straight into tcgen05.mma (kind f8f6f4), so no thread ever touches one; what the threads do is the softmax of
// 8 or 16 numbers per token.  For that, the other operand has to be e4m3 as well, without losing what bf16 or fp16
// hold: Q and P are each split into three e4m3 numbers, x = x0 + x1 / 16 + x2 / 256, each the rounding of what is left
// (4 bits a piece, 12 bits in all, down to 2^-25 of the row's largest element).  The pieces are further columns of the MMA's N side, which costs nothing that counts:
//     S[128 tokens x 3R]      = K_tile . (Q0 Q1 Q2)^T       A = K tile, K-major;    R = 8 NT rows
//     O[128 head dims x 3R]  += V_tile^T . (P0 P1 P2)       A = V tile, MN-major: as the page lies in memory
// The page's scale of K multiplies S.  That of V multiplies P: P = 2^(s - m + 7) s_v / 2^L, with m the running maximum of s and
// 2^L a scale that the unit's pages have at most, and the softmax's own sum gets 2^(s - m + 7).  P is a fixed-point number, 2^8 down
// to 2^-18, so that only pages whose scales lie close together (PAGED_SPAN) may share one L: else a page that is scaled for one large
// value, asked for or not, would push the weights of all the others off P's end (with the largest s + log2 s_v as the one
// reference, a page 2^20 above the rest cost 5% of the result, 2^24 all of it).  A tile with scales further apart is done
// group by group (apart, below), one P V for each group of scales with a reference of its own; the sums in tensor memory are fp32 and are moved
// from one reference to the next by whole powers of two.
//
// A unit is (sequence, kv head, block of R rows).  All units are laid out in one line, by groups of 16 tokens with a gap
// for a unit's fixed cost, and the line is cut into equal pieces, one per CTA, whatever the lengths.  A unit cut by a
// piece's border leaves a result for each part in the workspace, which a second kernel joins in a fixed order.
// Roles, all walking the same piece on their own: warp 0 pages and TMA, warp 1 MMA, warp 2 Q pieces of the next unit, warps
// 3..6 softmax, one token (and, at a unit's end, one head dim) per thread.  All mbarrier waits are bounded.  Code that
// runs once per unit is kept in loops: run straight through, it costs about 8 clocks an instruction to fetch.
// Measured: 64 sequences of 64 to 8192 tokens, 32 heads on 8 of 128, 49.5 us, 4.4 TB/s of codes and scales; 4 of 90001 to 131071, 8
// heads on 1 of 256, 51.8 us, 4.5 TB/s; one of 809 tokens 9.5 us.
#pragma once
#include "cache_pages.cuh"

struct PagedAttnParams {
  CUtensorMap tmK;       // codes [blocks][kv heads * block][head dim], box of `box_rows` rows x 128 (64) bytes
  CUtensorMap tmV;
  const void* q;
  void* o;
  long long q_seq, q_tok, q_head, o_seq, o_tok, o_head;
  const uint8_t* vc;
  const float* ks;
  const float* vs;
  const int* table;
  long long table_ld;
  const int* lens;
  int n_seqs, n_q, group, kv_heads;
  int rows;              // n_q * group
  int row_blocks;        // ceil(rows / R)
  int units;             // per sequence: kv_heads * row_blocks
  uint32_t per_page_inv; // ceil(2^32 / (block / 16)), 0 for blocks of 16: see page_of
  int blocks, block, width;
  int box_rows;          // 16, 32, 64 or 128 tokens: the largest that divides the block
  float scale_log2e;
  int whole;             // units are short: pieces are cut between units only, nothing to join
  float* part_o;         // [cta][2][R][D]: result of a unit's first part (slot 1) or a later one (slot 0) by itself
  float2* part_ml;       // [cta][2][R]: its maximum and sum
  int* cut;              // [cta][4]: the unit that starts in this CTA and ends in another: sequence (-1: none), kv head, row block, last CTA
};

constexpr int PAGED_THREADS = 224;
// Fixed cost of a unit, in groups of 16 tokens.  Measured with 8, 12, 16, 20: 200 sequences of 100 to 1500 tokens, 32 heads on 8 of 128,
// 85.8, 82.3, 81.1, 81.1 us; the same with 16 heads on 4 of 64, 43.2, 41.0, 40.5, 41.3; 64 of 64 to 8192 of these, 56.5, 57.0, 57.0, 57.9.
// Heads of 256 with 12, 16, 20, 24: 83 sequences of 217 to 10009, 3 tokens each, 102.1, 102.0, 102.0, 103.7.
constexpr int paged_gap(int head_dim) { return head_dim == 256 ? 20 : 12; }
// Groups (with gaps) per CTA, at least.  With less a piece could hold no tile's start, which the join counts on.  With 8, 16, 32: one
// sequence of 809 tokens, heads of 256, 9.3, 10.6, 13.5 us; 16 of 100 to 4001, 13.9, 13.4, 15.9; of 700 to 900, heads of 64, 12.0, 12.0, 13.8.
constexpr int PAGED_MIN_PIECE = 8;
// Units of at most this many groups are not cut, which spares the join.  512 tokens (32 groups) uncut and cut: 300 sequences of 300, 32 heads
// on 8 of 128, 60.0 and 74.7 us, 64 of 512 20.1 and 23.0, but one of 512 9.4 and 8.9, and with 8 heads on 1 of 256 12.5 and 9.2.  1024 tokens:
// 64 sequences 31.8 and 33.1, 8 of them 23.8 and 12.2, one of 256 head dims 19.5 and 9.5.
constexpr int PAGED_WHOLE = 32;

// Scales of V with one reference 2^L: 2^(L - PAGED_SPAN - 1) < s_v <= 2^L, so that the last piece of P ends 2^-18 below the largest
// probability at the most, and 2^-25 below it where all scales are alike.
constexpr int PAGED_SPAN = 6;
// Scales more than 2^80 below the largest that a part has seen share the lowest reference: with 2^8 of P, 2^9 of the codes and 2^17
// tokens or more, sums relative to less could leave fp32.
constexpr int PAGED_REACH = 80;
constexpr int PAGED_NONE = -1000;        // no page with a scale

template <int D, int NT>
struct PagedCfg {
  static constexpr int R = 8 * NT;                    // rows of a unit
  static constexpr int N = NT == 1 ? 32 : 48;         // MMA columns: three pieces of R rows, a multiple of 16
  static constexpr int HALVES = D == 256 ? 2 : 1;     // 128-byte column blocks of a tile
  static constexpr int ROW_BYTES = D == 64 ? 64 : 128;
  static constexpr int TILE_BYTES = 128 * D;          // 128 tokens of K, or of V
  static constexpr int BLOCK_BYTES = 128 * ROW_BYTES; // one column block of a tile
  static constexpr int SLOTS = D == 64 ? 10 : 6;      // ring of tiles: K and V in turn, each with barriers of its own
  static constexpr int Q_BUFS = D == 128 && NT == 2 ? 1 : 2;
  static constexpr int Q_BYTES = N * D;
  static constexpr int P_BYTES = N * 128;
  static constexpr int SMEM_BYTES = SLOTS * TILE_BYTES + Q_BUFS * Q_BYTES + P_BYTES + 1024;
  static constexpr int PER_SM = D == 256 ? 1 : 2;
  static constexpr int GAP = paged_gap(D);
  static constexpr int S_COL = 0, O_COL = 2 * N;      // two S buffers, then O per column block
  static constexpr int TMEM_COLS = NT == 1 ? 128 : 256;
  static constexpr uint64_t LAYOUT = D == 64 ? 4ull : 2ull;                 // 64- or 128-byte swizzle
  static constexpr uint64_t GROUP_STRIDE = 8 * ROW_BYTES;                   // bytes from 8 rows to the next 8
};

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ uint64_t paged_desc(uint32_t smem_addr, uint64_t lead_bytes, uint64_t stride_bytes, uint64_t layout) {
  return (uint64_t)((smem_addr & 0x3FFFF) >> 4) | (lead_bytes >> 4) << 16 | (stride_bytes >> 4) << 32 | 1ull << 46 | layout << 61;
}
// The three pieces of 8 rows in one lane: columns 0 .. 7 of each of three blocks of `apart` columns.
__device__ __forceinline__ void paged_tmem_ld(uint32_t taddr, int apart, uint32_t (&v)[24]) {
#pragma unroll
  for (int i = 0; i < 3; ++i)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[8 * i]), "=r"(v[8 * i + 1]), "=r"(v[8 * i + 2]), "=r"(v[8 * i + 3]), "=r"(v[8 * i + 4]), "=r"(v[8 * i + 5]),
                   "=r"(v[8 * i + 6]), "=r"(v[8 * i + 7])
                 : "r"(taddr + i * apart)
                 : "memory");
  tmem_ld_wait();
}
// One of them.
__device__ __forceinline__ void paged_tmem_ld8(uint32_t taddr, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(taddr) : "memory");
  tmem_ld_wait();
}
__device__ __forceinline__ void paged_tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
  tmem_st_wait();
}
// Those of two rows.
__device__ __forceinline__ float2 paged_tmem_ld2(uint32_t taddr, int apart) {
  uint32_t v[3][2];
#pragma unroll
  for (int i = 0; i < 3; ++i)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0, %1}, [%2];" : "=r"(v[i][0]), "=r"(v[i][1]) : "r"(taddr + i * apart) : "memory");
  tmem_ld_wait();
  auto sum = [&](int r) { return fmaf(__uint_as_float(v[2][r]), 0x1p-8f, fmaf(__uint_as_float(v[1][r]), 0x1p-4f, __uint_as_float(v[0][r]))); };
  return make_float2(sum(0), sum(1));
}
__device__ __forceinline__ void paged_tmem_st(uint32_t taddr, int apart, const uint32_t (&v)[24]) {
#pragma unroll
  for (int i = 0; i < 3; ++i)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(taddr + i * apart), "r"(v[8 * i]), "r"(v[8 * i + 1]), "r"(v[8 * i + 2]), "r"(v[8 * i + 3]), "r"(v[8 * i + 4]),
                   "r"(v[8 * i + 5]), "r"(v[8 * i + 6]), "r"(v[8 * i + 7])
                 : "memory");
  tmem_st_wait();
}
// the number that three pieces stand for
__device__ __forceinline__ float paged_sum(const uint32_t (&v)[24], int r) {
  return fmaf(__uint_as_float(v[16 + r]), 0x1p-8f, fmaf(__uint_as_float(v[8 + r]), 0x1p-4f, __uint_as_float(v[r])));
}
// mbar_wait with its loop out of line: a kernel of many roles has many waits, and its code has to stay in the caches
__device__ __noinline__ bool paged_wait_loop(uint32_t bar, uint32_t parity, volatile int* abort_flag) { return mbar_wait_small(bar, parity, abort_flag); }
__device__ __forceinline__ bool paged_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return mbar_try_wait(bar, parity) || paged_wait_loop(bar, parity, abort_flag);
}
// whether `on` holds in any of the 128 threads that meet at named barrier `id`
__device__ __forceinline__ bool barrier_any(int id, bool on) {
  uint32_t any;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n barrier.cta.red.or.pred p, %2, 128, q;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(any) : "r"((uint32_t)on), "r"(id) : "memory");
  return any != 0;
}
// largest value of a warp's lanes
__device__ __forceinline__ float warp_max_f32(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The smallest L >= -100 with |x| <= 2^L, and 2^L for -126 <= L <= 127.
__device__ __forceinline__ int scale_level(float x) {
  const int bits = __float_as_int(x) & 0x7fffffff;
  return max((bits >> 23) - 127 + ((bits & 0x7fffff) != 0), -100);
}
__device__ __forceinline__ float power_of_2(int e) { return __int_as_float((e + 127) << 23); }
// x / 2^L for L of scale_level
__device__ __forceinline__ float below_level(float x, int level) { return x * 0.25f * power_of_2(2 - level); }
__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Three e4m3 pieces of two numbers of at most 256: a in the low bytes of c[], b in the high ones.
__device__ __forceinline__ void pieces(float a, float b, uint32_t (&c)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    c[i] = to_e4m3x2(a, b);
    const float2 f = from_e4m3x2(c[i]);
    a = (a - f.x) * 16.f;
    b = (b - f.y) * 16.f;
  }
}
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {   // 0x80 in the bytes that are 0x7f or 0xff
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

__device__ __forceinline__ int paged_len(const PagedAttnParams& p, int b) {
  return (int)min(max((long long)p.lens[b], 0ll), (long long)p.width * p.block);
}
// The page of a sequence that group g of 16 tokens lies in, g / (block / 16): with at most 16 groups a page and g below 2^27,
// the product's error stays below 1 / 32, less than a step of the quotient.
__device__ __forceinline__ int page_of(const PagedAttnParams& p, int g) { return p.per_page_inv ? (int)__umulhi((uint32_t)g, p.per_page_inv) : g; }
// where row rr of (sequence b, kv head h) lies in q / o
__device__ __forceinline__ long long paged_row(const PagedAttnParams& p, int b, int h, int rr, long long seq, long long tok, long long head) {
  return b * seq + (rr / p.group) * tok + (long long)(h * p.group + rr % p.group) * head;
}

// Sums over the CTA's threads before this one, and over all of them.
__device__ __forceinline__ int paged_scan(int v, int* all, int* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < PAGED_THREADS / 32; ++w) {
    const int n = warp_sum[w];
    if (w < warp) before += n;
    total += n;
  }
  __syncthreads();
  *all = total;
  return before + s - v;
}

// The parts of units in one piece of the line, in order.  Every role walks on its own; the state is a few registers.  The
// host refuses sizes whose line could pass 2^31.
template <int GAP>
struct PagedWalk {
  int begin, end;        // the piece
  int at, next_at;       // line position of the unit's first tile, and of the next unit's gap
  int next_b, next_h, next_rb, len;
  int b, h, rb, t0, t1, tiles;   // the part at hand: tiles [t0, t1) of `tiles` of row block rb of kv head h of sequence b

  __device__ __forceinline__ bool next(const PagedAttnParams& p) {
#pragma unroll 1
    while (next_at < end) {
      const int groups = (len + 15) >> 4;
      if (next_h == p.kv_heads || !groups) {   // the line goes on, so there is a further sequence with tokens
        next_h = 0;
        len = paged_len(p, ++next_b);
        continue;
      }
      b = next_b;
      h = next_h;
      rb = next_rb;
      if (++next_rb == p.row_blocks) {
        next_rb = 0;
        ++next_h;
      }
      at = next_at + GAP;
      next_at = at + groups;
      tiles = (groups + 7) >> 3;
      // a border inside a tile belongs to the piece where the tile starts
      t0 = cut(p, begin);
      t1 = cut(p, end);
      if (t0 < t1) return true;
    }
    return false;
  }
  __device__ __forceinline__ int cut(const PagedAttnParams& p, int x) const { return x <= at ? 0 : p.whole ? tiles : min(tiles, (x - at + 7) >> 3); }
};


template <typename T, int D, int NT>
__global__ void __launch_bounds__(PAGED_THREADS, (PagedCfg<D, NT>::PER_SM)) paged_attention_kernel(const __grid_constant__ PagedAttnParams p) {
  using C = PagedCfg<D, NT>;
  constexpr int R = C::R;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_mem[2 * C::SLOTS + 8];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_mem, poison_mem[3];          // poison: a hidden value of the unit was NaN (units in turn)
  __shared__ int again_mem;                         // this tile has a further P V: apart
  __shared__ int found_b, found_base, warp_sum[PAGED_THREADS / 32];
  // of the 8 groups of a tile, written and handed back with its V: scale of K, whether there is a page, scale of V, and highest and lowest
  // level of the scales of V in this tile and up to three beside it (two 16-bit numbers)
  __shared__ float4 page_info[C::SLOTS / 2][8];
  __shared__ float q_scale[2][R];
  // each softmax warp's copy of the scale of Q and the maximum of each row, the same for all its lanes: with two CTAs an SM they are
  // kept there only, with one they are put there for `apart`
  constexpr bool KEPT = C::PER_SM == 2;
  __shared__ float4 row_mem[4][2][R / 4];
  // as well: what O of the part at hand is relative to, O = sum 2^(s - m + 7) s_v / 2^x; the levels from which, y, and up to which, w, x may
  // follow the scales without a look at the scores; the highest level so far, z
  __shared__ int4 level_mem[4];
  __shared__ int late_mem[4];                       // a wait for a tile's scales has run out, here or in another warp
  __shared__ float4 warp_max[R], warp_sums[2][R];   // by row, of the four softmax warps (sums: of odd and even units)
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
  const uint32_t sRing = raw_addr + pad, sQ = sRing + C::SLOTS * C::TILE_BYTES, sP = sQ + C::Q_BUFS * C::Q_BYTES;
  uint8_t* ring = smem_raw + pad;
  uint8_t* q_mem = ring + C::SLOTS * C::TILE_BYTES;
  uint8_t* p_mem = q_mem + C::Q_BUFS * C::Q_BYTES;
  const uint32_t bars = smem_u32(bar_mem);
  // K of tile c lies in slot 2c, V in slot 2c + 1, modulo the ring; a slot is used for the (c / HALF)-th time
  constexpr int HALF = C::SLOTS / 2, B0 = 2 * C::SLOTS;
  auto full = [&](int s) { return bars + 8 * s; };
  auto empty = [&](int s) { return bars + 8 * (C::SLOTS + s); };
  auto s_full = [&](int b) { return bars + 8 * (B0 + b); };
  const uint32_t p_ready = bars + 8 * (B0 + 2), o_done = bars + 8 * (B0 + 3);
  auto q_ready = [&](int b) { return bars + 8 * (B0 + 4 + b); };
  auto q_empty = [&](int b) { return bars + 8 * (B0 + 6 + b); };
  volatile int* abort_flag = &abort_mem;
  volatile int* poison = poison_mem;
  volatile int* again_flag = &again_mem;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int s = 0; s < C::SLOTS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(s_full(b), 1);
      mbar_init(q_ready(b), 1);
      mbar_init(q_empty(b), 1 + 4);
    }
    mbar_init(p_ready, 128);
    mbar_init(o_done, 1);
    abort_mem = again_mem = late_mem[0] = late_mem[1] = late_mem[2] = late_mem[3] = 0;
    poison_mem[0] = poison_mem[1] = poison_mem[2] = 0;
    mbar_fence_init();
    tma_prefetch_desc(&p.tmK);
    tma_prefetch_desc(&p.tmV);
  }
  pdl_wait();
  // behind the wait: a CTA of the kernel before this one may yet have to take its own, and this one would hold it up for good
  if (warp == 1) tmem_alloc(smem_u32(&tmem_slot), C::TMEM_COLS);

  // rows of sequences without tokens
#pragma unroll 1
  for (int b = blockIdx.x; b < p.n_seqs; b += gridDim.x) {
    if (paged_len(p, b)) continue;
#pragma unroll 1
    for (int x = threadIdx.x; x < p.kv_heads * p.rows * D; x += PAGED_THREADS)
      reinterpret_cast<T*>(p.o)[paged_row(p, b, x / (p.rows * D), x / D % p.rows, p.o_seq, p.o_tok, p.o_head) + x % D] = (T)0.f;
  }
  // this CTA's piece of the line, and the sequence it starts in
  PagedWalk<C::GAP> start;
  start.begin = 0;
  start.end = 0;
  int piece = 0, sum = 0;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    // the first pass forms the length of the line; with one round of sequences it also has each one's place in it
#pragma unroll 1
    for (int base = 0, rounds = (p.n_seqs + PAGED_THREADS - 1) / PAGED_THREADS; rounds > 0; --rounds, base += PAGED_THREADS) {
      const int b = base + threadIdx.x;
      const int groups = b < p.n_seqs ? (paged_len(p, b) + 15) >> 4 : 0;
      const int n = groups ? (groups + C::GAP) * p.units : 0;
      int all;
      const int at = sum + paged_scan(n, &all, warp_sum);
      sum += all;
      if (pass == 0 && rounds == 1) {
        piece = max((int)((uint32_t)sum / gridDim.x) + 1, PAGED_MIN_PIECE);
        start.begin = (int)min((long long)blockIdx.x * piece, (long long)sum);
        start.end = min(start.begin + piece, sum);
      }
      if ((pass == 1 || base == 0 && rounds == 1) && at <= start.begin && start.begin < at + n) {
        found_b = b;
        found_base = at;
      }
    }
    if (p.n_seqs <= PAGED_THREADS) break;
    sum = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  if (start.begin < start.end) {
    start.next_b = found_b;
    start.len = paged_len(p, found_b);
    const int one = ((start.len + 15) >> 4) + C::GAP, u = (start.begin - found_base) / one;
    start.next_h = u / p.row_blocks;
    start.next_rb = u - start.next_h * p.row_blocks;
    start.next_at = found_base + u * one;
  } else {
    start.next_at = start.end;               // no part
  }

  if (warp == 0) {
    // ---- pages and TMA: lane (j, g) looks after group g of the j-th of four tiles.  Ids are fetched one batch ahead,
    // across units, and scales while the batch before goes out, so that neither latency stands between two loads. ----
    PagedWalk<C::GAP> w = start;
    struct Batch { int b, h, len, tile, n; int id; float ks, vs; };
    Batch now, next;
    now.n = 0;
    int c = 0, tile = 0, levels = 0;
    bool ok = true, more = w.next(p);
    if (more) tile = w.t0;
    const uint64_t pol = policy_evict_normal();
    const int per_box = p.box_rows / 16;
#pragma unroll 1
    do {
      next.n = 0;
      next.id = -1;
      if (more) {
        next.b = w.b; next.h = w.h; next.len = w.len; next.tile = tile;
        next.n = min(4, w.t1 - tile);
        tile += next.n;
        if ((lane >> 3) < next.n) {
          const int group = next.tile * 8 + lane;
          if (group * 16 < next.len) next.id = p.table[next.b * p.table_ld + page_of(p, group)];
        }
        if (tile == w.t1) {
          more = w.next(p);
          if (more) tile = w.t0;
        }
      }
#pragma unroll 1
      for (int j = 0; j < now.n && ok; ++j, ++c) {
        const int s = 2 * (c % HALF);
        const uint32_t freed = (uint32_t)(c / HALF - 1) & 1u;
        const bool here = lane >> 3 == j;
        const int g = lane & 7, group = (now.tile + j) * 8 + g;
        const bool load = here && now.id >= 0 && g % per_box == 0;
        const int bytes = __popc(__ballot_sync(0xffffffffu, load)) * p.box_rows * D;
        const int row = now.h * p.block + group * 16 - page_of(p, group) * p.block;
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          if (c >= HALF) ok = ok && __all_sync(0xffffffffu, paged_wait(empty(s + kv), freed, abort_flag));
          if (!ok) break;
          if (load) {
            const uint32_t dst = sRing + (s + kv) * C::TILE_BYTES + g * 16 * C::ROW_BYTES;
#pragma unroll
            for (int x = 0; x < C::HALVES; ++x)
              tma_load_3d(dst + x * C::BLOCK_BYTES, kv ? &p.tmV : &p.tmK, full(s + kv), x * 128, row, now.id, pol);
          }
          if (kv == 1) {                        // the scales may come in later than the loads go out
            const bool on = now.id >= 0, finite = on && fabsf(now.vs) < INFINITY;
            const float vs = finite ? now.vs : 0.f;
            if (j == 0) {                       // over the batch, which is quicker than each tile's own and does as well
              const int level = scale_level(vs), hi = __reduce_max_sync(0xffffffffu, vs != 0.f ? level : PAGED_NONE);
              levels = hi << 16 | (__reduce_min_sync(0xffffffffu, vs != 0.f ? level : -PAGED_NONE) & 0xffff);
            }
            // a scale of V that is not finite makes the tokens' scores NaN, and so every row that sees one
            if (here) page_info[c % HALF][g] = make_float4(!on ? 0.f : finite ? now.ks : NAN, on ? 1.f : 0.f, vs, __int_as_float(levels));
          }
          __syncwarp();                         // page_info goes out with lane 0's arrival
          if (lane == 0) mbar_expect_tx(full(s + kv), bytes);
        }
      }
      // the batch that is next: its ids are here by now, its scales are asked for
      now = next;
      if (now.id >= p.blocks) now.id = -1;
      if (now.n && now.id >= 0) {
        now.ks = p.ks[(long long)now.id * p.kv_heads + now.h];
        now.vs = p.vs[(long long)now.id * p.kv_heads + now.h];
      }
    } while (ok && now.n);
  } else if (warp == 1) {
    // ---- MMA: S up to one tile ahead of P V, each issued as soon as its operands are there ----
    if (lane == 0) {
      const uint32_t idesc = (1u << 4) | ((uint32_t)(C::N / 8) << 17) | (8u << 24);       // e4m3 x e4m3 -> fp32, M = 128
      const uint32_t idesc_pv = idesc | (1u << 15);                                        // A MN-major
      PagedWalk<C::GAP> w = start;
      int tile = 0, cs = 0, cp = 0, pv = 0, seg = -1;     // pv: P V so far, of which a tile has one, or another odd number
      bool more = true, turn = true;            // turn: the next S is a unit's first
      // of the tiles whose P V is to come, at most two, even and odd: MMA steps of 32 tokens, negative for a unit's first
      int steps_of[2] = {0, 0};
      const uint64_t k_desc = paged_desc(sRing, 16, C::GROUP_STRIDE, C::LAYOUT), q_desc = paged_desc(sQ, 16, C::GROUP_STRIDE, C::LAYOUT);
      // 64 head dims: M's second half runs on into what lies behind, and is not used
      const uint64_t v_desc = paged_desc(sRing, D == 64 ? C::TILE_BYTES : 16, C::GROUP_STRIDE, C::LAYOUT), p_desc = paged_desc(sP, 16, 1024, 2);
      uint64_t t_idle = 0;
      uint32_t idle = 0;
#pragma unroll 1
      for (;;) {
        bool did = false;
        if (turn && more) {
          more = w.next(p);
          tile = w.t0;
          ++seg;
          turn = false;
        }
        if (!more && cp == cs) break;
        if (more && cs <= cp + 1) {            // S of tile cp + 1 goes over that of cp - 1, whose P has been taken
          const int s = 2 * (cs % HALF), qb = seg % C::Q_BUFS;
          if (mbar_test(full(s), (uint32_t)(cs / HALF) & 1u) && (tile != w.t0 || mbar_test(q_ready(qb), (uint32_t)(seg / C::Q_BUFS) & 1u))) {
            tc_fence_after();
            const uint64_t kd = k_desc + s * (C::TILE_BYTES / 16), qd = q_desc + qb * (C::Q_BYTES / 16);
#pragma unroll
            for (int x = 0; x < C::HALVES; ++x)
#pragma unroll
              for (int k = 0; k < C::ROW_BYTES / 32; ++k)
                umma_f8(tmem + C::S_COL + (cs & 1) * C::N, kd + x * (C::BLOCK_BYTES / 16) + 2 * k, qd + x * (C::N * 8) + 2 * k, idesc, (x | k) != 0);
            umma_commit(empty(s));
            umma_commit(s_full(cs & 1));
            const int steps = (min(w.len - tile * 128, 128) + 31) >> 5;
            steps_of[cs & 1] = tile == w.t0 ? -steps : steps;
            ++cs;
            if (++tile == w.t1) {
              umma_commit(q_empty(qb));        // this unit's Q is no longer read
              turn = true;
            }
            did = true;
          }
        }
        if (cp < cs) {
          const int s = 2 * (cp % HALF) + 1;
          if (mbar_test(p_ready, (uint32_t)pv & 1u) && mbar_test(full(s), (uint32_t)(cp / HALF) & 1u)) {
            tc_fence_after();
            const bool again = *again_flag;
            const uint64_t vd = v_desc + s * (C::TILE_BYTES / 16);
            const int steps = steps_of[cp & 1];
#pragma unroll
            for (int x = 0; x < C::HALVES; ++x)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < abs(steps))
                  umma_f8(tmem + C::O_COL + x * C::N, vd + x * (C::BLOCK_BYTES / 16) + k * (32 * C::ROW_BYTES / 16), p_desc + 2 * k, idesc_pv, steps > 0 || k != 0);
            if (!again) umma_commit(empty(s));
            umma_commit(o_done);
            ++pv;
            if (again) steps_of[cp & 1] = abs(steps);
            else ++cp;
            did = true;
          }
        }
        if (did) {
          idle = 0;
        } else if ((++idle & 255) == 0) {      // the clock is read seldom: a look at it costs more than one at the barriers
          const uint64_t now = globaltimer_ns();
          if (idle == 256) t_idle = now;
          if (*abort_flag || now - t_idle > VLA_WAIT_LIMIT_NS) {
            *abort_flag = 1;
            break;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // ---- Q pieces: each row times the power of two that brings its largest magnitude to [2^7, 2^8) ----
    PagedWalk<C::GAP> w = start;
#pragma unroll 1
    for (int seg = 0; w.next(p); ++seg) {
      const int qb = seg % C::Q_BUFS, h = w.h, r0 = w.rb * R;
      constexpr int E = D / 64;               // pairs of elements per lane and row
      uint32_t rows[R][E];                    // all in flight at once; they move up as the loop takes the first
      const int i0 = r0 ? r0 / p.group : 0;
      int g = r0 - i0 * p.group;
      const T* src = reinterpret_cast<const T*>(p.q) + w.b * p.q_seq + i0 * p.q_tok + (long long)(h * p.group + g) * p.q_head + lane * (2 * E);
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 0; i < E; ++i) rows[r][i] = 0u;
        if (r0 + r < p.rows) {
          if (E == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(src);
            rows[r][0] = v.x; rows[r][1 % E] = v.y; rows[r][2 % E] = v.z; rows[r][3 % E] = v.w;
          } else if (E == 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(src);
            rows[r][0] = v.x; rows[r][1 % E] = v.y;
          } else {
            rows[r][0] = *reinterpret_cast<const uint32_t*>(src);
          }
        }
        src += p.q_head;
        if (++g == p.group) {
          g = 0;
          src += p.q_tok - p.group * p.q_head;
        }
      }
      if (seg >= C::Q_BUFS && !__all_sync(0xffffffffu, paged_wait(q_empty(qb), (uint32_t)(seg / C::Q_BUFS - 1) & 1u, abort_flag))) break;
      // Two rows at a time: a row is a chain of some 450 clocks, and short sequences wait for them.  3 sequences of 69 to 276, 5
      // tokens each of 64 heads on 8, took 1.2 us less than with one; four at a time 0.2 less again, but more where there are 8 rows.
#pragma unroll 1
      for (int r = 0; r < R; r += 2) {
        float2 f[2][E];
        float top[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          top[j] = 0.f;
#pragma unroll
          for (int i = 0; i < E; ++i) {
            f[j][i] = unpack2<T>(rows[j][i]);
            top[j] = fmaxf(top[j], fmaxf(fabsf(f[j][i].x), fabsf(f[j][i].y)));
          }
        }
#pragma unroll
        for (int k = 0; k + 2 < R; ++k)
#pragma unroll
          for (int i = 0; i < E; ++i) rows[k][i] = rows[k + 2][i];
#pragma unroll
        for (int j = 0; j < 2; ++j) top[j] = warp_max_f32(top[j]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int e = (__float_as_int(top[j]) >> 23) - 127 - 7;
          // zeros, the smallest numbers and infinities stay as they are; the scores of a row with an infinity are NaN
          const bool plain = top[j] == 0.f || !(top[j] < INFINITY) || e < -126;
          const float up = plain ? 1.f : __int_as_float((127 - e) << 23);
          if (lane == 0) q_scale[qb][r + j] = (plain ? 1.f : __int_as_float((127 + e) << 23)) * (top[j] < INFINITY ? p.scale_log2e : NAN);
          uint32_t c[E][3];
#pragma unroll
          for (int i = 0; i < E; ++i) pieces(f[j][i].x * up, f[j][i].y * up, c[i]);
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            const int n = k * R + r + j, at = lane * (2 * E);          // byte of the row
            uint8_t* dst = q_mem + qb * C::Q_BYTES + (at / 128) * C::N * 128 + n * C::ROW_BYTES +
                           (((at % 128 / 16) ^ (D == 64 ? n >> 1 & 3 : n & 7)) << 4) + at % 16;
            if (E == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(c[0][k] | c[1 % E][k] << 16, c[2 % E][k] | c[3 % E][k] << 16);
            else if (E == 2) *reinterpret_cast<uint32_t*>(dst) = c[0][k] | c[1 % E][k] << 16;
            else *reinterpret_cast<uint16_t*>(dst) = (uint16_t)c[0][k];
          }
        }
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready(qb));
    }
  } else {
    // ---- softmax: thread = token of the tile; at a unit's end, thread = head dim.  A wait that runs out raises the abort
    // flag and the loop goes on with whatever is there, because the 128 threads meet at barriers; what decides which barriers those are
    // is the same in all of them: the walk, and the pages' scales, once nobody's wait for them has run out. ----
    const int quarter = warp & 3, tid = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      paged_wait(bar, parity, abort_flag);
      __syncwarp();
    };
    // a part, with head, first row, and that row's query and group head
    struct Part { int b, h, rb, len, t0, t1, tiles, at, r0, i0, g0; };
    PagedWalk<C::GAP> walk = start;
    auto take = [&](Part& x) {
      if (!walk.next(p)) return false;
      x.b = walk.b; x.h = walk.h; x.rb = walk.rb; x.len = walk.len; x.t0 = walk.t0; x.t1 = walk.t1; x.tiles = walk.tiles; x.at = walk.at;
      x.r0 = x.rb * R;
      x.i0 = x.r0 ? x.r0 / p.group : 0;
      x.g0 = x.r0 - x.i0 * p.group;
      return true;
    };
    Part w, w_next;
    w.t0 = w.t1 = 0;
    // m and qs are kept there and read where they are needed: in 128 registers a thread more is spilled than the 56 to 80 bytes that
    // 16 rows still cost, and 9 sequences of 2940 to 16102, 8 tokens each of 28 heads on 4 of 128, take 84 us instead of 72.
    auto from_mem = [&](int what, float (&v)[R]) {
      if constexpr (KEPT) {
#pragma unroll
        for (int r = 0; r < R; r += 4) {
          const float4 f = row_mem[quarter][what][r / 4];
          v[r] = f.x; v[r + 1] = f.y; v[r + 2] = f.z; v[r + 3] = f.w;
        }
      }
    };
    auto to_mem = [&](int what, const float (&v)[R]) {
      __syncwarp();
      if (lane == 0) {
#pragma unroll
        for (int r = 0; r < R; r += 4) row_mem[quarter][what][r / 4] = make_float4(v[r], v[r + 1], v[r + 2], v[r + 3]);
      }
      __syncwarp();
    };
    const uint32_t o_at = tmem + lane_off + C::O_COL;
    uint8_t* const p_col = p_mem + (tid & 15);
    auto put = [&](int r, float a, float b) {      // P of rows r, r + 1
      uint32_t pc[3];
      pieces(a, b, pc);
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const int n = k * R + r;
        p_col[n * 128 + (((tid >> 4) ^ (n & 7)) << 4)] = (uint8_t)pc[k];
        p_col[(n + 1) * 128 + (((tid >> 4) ^ ((n + 1) & 7)) << 4)] = (uint8_t)(pc[k] >> 8);
      }
    };
    auto move = [&](int by) {                    // O *= 2^by, by that of lane r for row r
#pragma unroll 1
      for (int y = 0; y < C::HALVES * 3 * R; y += 8) {         // 8 rows of one piece
        const uint32_t at = o_at + y / (3 * R) * C::N + y % (3 * R);
        uint32_t o[8];
        paged_tmem_ld8(at, o);
#pragma unroll
        for (int r = 0; r < 8; ++r)
          o[r] = __float_as_uint(__uint_as_float(o[r]) * power_of_2(min(max(__shfl_sync(0xffffffffu, by, y % R + r), -126), 127)));
        paged_tmem_st8(at, o);
      }
    };
    // The reference follows a tile whose highest scale is somewhat larger.  Lower ones need no move.
    auto follow = [&](int c, int hi, int lo, bool first) {
      int4* const lv = &level_mem[quarter];
      if (lv->y == -PAGED_NONE || hi <= lv->x || hi > lv->w || lo < hi - PAGED_SPAN) return false;
      const int by = lv->x - hi;
      if (c > 0) wait(o_done, (uint32_t)(c - 1) & 1u);
      tc_fence_after();
      if (!first) move(by);
      if (lane == 0) *lv = make_int4(hi, hi - PAGED_SPAN, max(lv->z, hi), lv->w);
      __syncwarp();
      return true;
    };
    // P of a tile whose scales of V lie further apart, or elsewhere than those that the part's reference is made for.  Tokens are
    // taken by groups of levels, from the highest down, each with a reference that fits the products 2^s s_v of that group alone:
    // that of row r is 2^(m - g + L), with a whole number g >= 0 in lane r.  P V runs once for each group, over the same V; between
    // two, O is moved by whole powers of two.  In the end O is relative to 2^(m + x) again, where x is made for the level of a
    // group that holds next to the largest probabilities in all rows; where there is none and the maxima have just moved, no
    // level is known to fit, and the next tile comes here as well.  The number of P V is odd, with an empty one if need be, so
    // that the phases of the barriers stay those of one a tile.  Rare, so that it is kept in loops that need few registers: S is read
    // again row by row (as a function of its own, with the call in the loop over tiles, all other tiles took half as long again).
    // 64 sequences of 64 to 8192 tokens, 32 heads on 8 of 128: 50 us with scales within 2^5, 272 with a scale of its own out of 2^9 for
    // each page, 466 out of 2^60; 4 of 90001 to 131071, 8 heads on 1 of 256: 52, 171 and 256.
    auto apart = [&](int c, int tok, int len, int lim_min, int g0, bool first, bool moved) {
      const float4* const infos = page_info[c % HALF];
      int4* const lv = &level_mem[quarter];
      auto level_of = [&](float v) { return v != 0.f ? scale_level(v) : PAGED_NONE; };
      auto highest = [&](int under) {              // of the tile's levels
        int most = PAGED_NONE;
#pragma unroll 1
        for (int k = 0; k < 8; ++k) {
          const int l = level_of(infos[k].z);
          if (l < under) most = max(most, l);
        }
        return most;
      };
      auto scores = [&](int r) {                   // of rows r, r + 1
        float2 x = paged_tmem_ld2(tmem + lane_off + C::S_COL + (c & 1) * C::N + r, R);
        const float* qs = reinterpret_cast<const float*>(row_mem[quarter][0]);
        const float4 info = infos[tid >> 4];
        x.x *= qs[r] * info.x;
        x.y *= qs[r + 1] * info.x;
        if (info.y == 0.f || tok >= min(len, lim_min + (g0 + r) / p.group)) x.x = -INFINITY;
        if (info.y == 0.f || tok >= min(len, lim_min + (g0 + r + 1) / p.group)) x.y = -INFINITY;
        return x;
      };
      const float* const maxima = reinterpret_cast<const float*>(row_mem[quarter][1]);
      auto least = [&]() { return lv->z - PAGED_REACH; };          // no reference below 2^(m + least): the sums have to stay within fp32
      int level = highest(1 - PAGED_NONE), under = 1 - PAGED_NONE, at = lv->x, g = 0, fits = PAGED_NONE, pass = 0;
      if (lane == 0) lv->z = max(lv->z, level);
#pragma unroll 1
      for (;; ++pass) {
        named_barrier_sync(1, 128);                // warp_max has been read
        const int from = level - PAGED_SPAN, ref = level == PAGED_NONE ? at : max(level, least());
        const float vs = infos[tid >> 4].z;
        const int mine = level_of(vs);
        const float f = mine < under && mine >= from && mine != PAGED_NONE ? below_level(vs, ref) : 0.f;
        const float up = f != 0.f ? lg2_approx(fabsf(f)) : -INFINITY;
#pragma unroll 1
        for (int r = 0; r < R; r += 2) {
          const float2 x = scores(r);
          const float a = warp_max_f32(x.x + up), b = warp_max_f32(x.y + up);
          if (lane == 0) {
            reinterpret_cast<float*>(&warp_max[r])[quarter] = a;
            reinterpret_cast<float*>(&warp_max[r + 1])[quarter] = b;
          }
        }
        const int next = level == PAGED_NONE ? PAGED_NONE : highest(from);
        const bool again = next != PAGED_NONE || (pass & 1);
        named_barrier_sync(1, 128);
        const float4 tops = warp_max[lane % R];
        const float own_m = maxima[lane % R];
        const float below = own_m - fmaxf(fmaxf(tops.x, tops.y), fmaxf(tops.z, tops.w));       // NaN: the row has seen nothing
        const bool near = __all_sync(0xffffffffu, own_m == -INFINITY || below <= PAGED_SPAN + 1.f);
        if (near && fits == PAGED_NONE) fits = level;
        int to = below < (float)PAGED_REACH ? max((int)floorf(below) + 1, 0) : below < INFINITY ? PAGED_REACH : 0;
        to = level == PAGED_NONE ? g : min(to, ref - least());
        const int by = to - g + at - ref;
        g = to;
        at = ref;
        if (c + pass > 0) wait(o_done, (uint32_t)(c + pass - 1) & 1u);     // the P V before has read P, and O is complete
        tc_fence_after();
        if (!(first && pass == 0)) move(by);
#pragma unroll 1
        for (int r = 0; r < R; r += 2) {
          const float2 x = scores(r);
          const float m0 = maxima[r], m1 = maxima[r + 1];
          const float up0 = (float)(__shfl_sync(0xffffffffu, g, r) + 7), up1 = (float)(__shfl_sync(0xffffffffu, g, r + 1) + 7);
          put(r, f * ex2_approx(x.x - (m0 == -INFINITY ? 0.f : m0) + up0), f * ex2_approx(x.y - (m1 == -INFINITY ? 0.f : m1) + up1));
        }
        if (tid == 0) *again_flag = again;         // the MMA looks at it behind p_ready
        fence_proxy_async_shared();
        tc_fence_before();
        mbar_arrive(p_ready);
        if (!again) break;
        under = from;
        level = next;
      }
      const int home = max(fits != PAGED_NONE ? fits : lv->x, least());
      if (lane == 0) {                             // the others have read it: barriers
        if (fits != PAGED_NONE) {
          lv->y = fits - PAGED_SPAN;
          lv->w = fits + PAGED_SPAN;
        } else if (moved) {
          lv->y = -PAGED_NONE;
        }
      }
      wait(o_done, (uint32_t)(c + pass) & 1u);
      tc_fence_after();
      move(at - g - home);
      if (lane == 0) lv->x = home;
      __syncwarp();
    };
    int c = 0, cut_b = -1;
    // one pass per unit, after a first that only looks up the unit to begin with
#pragma unroll 1
    for (int seg = -1;; ++seg) {
      const int h = w.h, r0 = w.r0, i0 = w.i0, g0 = w.g0;
      const int lim_min = w.len - p.n_q + 1 + i0;               // the first row sees the fewest keys
      float qs[R], m[R], l[R];
#pragma unroll 1
      for (int tile = w.t0; tile < w.t1; ++tile, ++c) {
        const int s = 2 * (c % HALF), tok = tile * 128 + tid;
        const bool late = !paged_wait(full(s + 1), (uint32_t)(c / HALF) & 1u, abort_flag);
        __syncwarp();
        const float4 info = page_info[c % HALF][tid >> 4];
        const bool edge = tile * 128 + 128 > lim_min;
        if (edge || !__all_sync(0xffffffffu, info.y != 0.f)) {
          // A row of V that no row of this unit sees is cleared; where only some see it, a NaN in it is, and the end of
          // the unit gives it back: P is zero there, but zero times NaN is NaN.
          uint8_t* row = ring + (s + 1) * C::TILE_BYTES + tid * C::ROW_BYTES;
          const bool none = tok >= w.len || info.y == 0.f;
          if ((none || tok >= lim_min) && tid < (min(w.len - tile * 128, 128) + 31) / 32 * 32) {   // of what P V reads
#pragma unroll 2
            for (int x = 0; x < D / 16; ++x) {
              uint4* at = reinterpret_cast<uint4*>(row + (x / 8) * C::BLOCK_BYTES + (((x & 7) ^ (D == 64 ? tid >> 1 & 3 : tid & 7)) << 4));
              uint4 v = *at;
              const uint4 bad = make_uint4(nan_bytes(v.x), nan_bytes(v.y), nan_bytes(v.z), nan_bytes(v.w));
              if (none) {
                *at = make_uint4(0u, 0u, 0u, 0u);
              } else if (bad.x | bad.y | bad.z | bad.w) {
                v.x &= ~((bad.x >> 7) * 0xffu); v.y &= ~((bad.y >> 7) * 0xffu);     // 0x80 -> 0xff over the byte
                v.z &= ~((bad.z >> 7) * 0xffu); v.w &= ~((bad.w >> 7) * 0xffu);
                *at = v;
                poison[seg % 3] = 1;
              }
            }
          }
          __syncwarp();
        }
        if (tile == w.t0) {                      // a part begins with the level of its first tile, if there is one for all of it
          const int hi = __float_as_int(info.w) >> 16, lo = (int)(short)__float_as_int(info.w), at = max(hi, -100);
          if (lane == 0) level_mem[quarter] = make_int4(at, hi - lo <= PAGED_SPAN ? at - PAGED_SPAN : -PAGED_NONE, at, at + PAGED_SPAN);
          __syncwarp();
        }
        const int2 lv = *reinterpret_cast<const int2*>(&level_mem[quarter]);
        // the same in all threads, unless a wait for the scales has run out, of which all know by the barrier below: they have to go one way
        const bool out = __float_as_int(info.w) >> 16 > lv.x || (int)(short)__float_as_int(info.w) < lv.y;
        wait(s_full(c & 1), (uint32_t)(c >> 1) & 1u);
        tc_fence_after();
        if (tile == w.t0) {
          wait(q_ready(seg % C::Q_BUFS), (uint32_t)(seg / C::Q_BUFS) & 1u);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            qs[r] = q_scale[seg % C::Q_BUFS][r];
            m[r] = -INFINITY;
            l[r] = 0.f;
          }
          if (KEPT) {
            to_mem(0, qs);
            to_mem(1, m);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(q_empty(seg % C::Q_BUFS));
        }
        from_mem(0, qs);
        float x[R];                              // s
#pragma unroll
        for (int r8 = 0; r8 < R; r8 += 8) {
          uint32_t v[24];
          paged_tmem_ld(tmem + lane_off + C::S_COL + (c & 1) * C::N + r8, R, v);
#pragma unroll
          for (int r = 0; r < 8; ++r) x[r8 + r] = info.y == 0.f ? -INFINITY : paged_sum(v, r) * (qs[r8 + r] * info.x);
        }
        if (edge) {
          int lim = min(w.len, lim_min), left = p.group - g0;   // rows of a query follow one another
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if (tok >= lim) x[r] = -INFINITY;
            if (--left == 0) {
              left = p.group;
              lim = min(w.len, lim + 1);
            }
          }
        }
        from_mem(1, m);
        bool grow = late, moved = false;
#pragma unroll
        for (int r = 0; r < R; ++r) grow |= x[r] > m[r] + 1.f;
        // The subtracted maximum moves when a token has outgrown it by more than 2: P stays below 2 * 2^7, in e4m3's range.
        if (tile == w.t0 || barrier_any(1, grow)) {
          moved = true;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float top = warp_max_f32(x[r]);
            if (lane == 0) reinterpret_cast<float*>(&warp_max[r])[quarter] = top;
          }
          if (tile > w.t0) wait(o_done, (uint32_t)(c - 1) & 1u);
          tc_fence_after();
          if (barrier_any(1, late)) late_mem[quarter] = 1;
          float a[R];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float4 tops = warp_max[r];
            const float top = fmaxf(m[r], fmaxf(fmaxf(tops.x, tops.y), fmaxf(tops.z, tops.w)));
            a[r] = top == m[r] ? 1.f : ex2_approx(m[r] - top);
            m[r] = top;
            l[r] *= a[r];
          }
          if (KEPT) to_mem(1, m);
          if (tile > w.t0) {
#pragma unroll 1
            for (int y = 0; y < C::HALVES; ++y) {
#pragma unroll
              for (int r8 = 0; r8 < R; r8 += 8) {
                uint32_t o[24];
                paged_tmem_ld(tmem + lane_off + C::O_COL + y * C::N + r8, R, o);
#pragma unroll
                for (int i = 0; i < 24; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a[r8 + i % 8]);
                paged_tmem_st(tmem + lane_off + C::O_COL + y * C::N + r8, R, o);
              }
            }
          }
        }
        from_mem(1, m);
        if (__builtin_expect(out, 0)) {
          const int levels = __float_as_int(page_info[c % HALF][tid >> 4].w);
          if (!late_mem[quarter] && !follow(c, levels >> 16, (int)(short)levels, tile == w.t0)) {
#pragma unroll
            for (int r = 0; r < R; ++r) l[r] += ex2_approx(x[r] - (m[r] == -INFINITY ? 0.f : m[r]) + 7.f);
            if (!KEPT) {
              to_mem(0, qs);
              to_mem(1, m);
            }
            apart(c, tok, w.len, lim_min, g0, tile == w.t0, moved);
            continue;
          }
        }
        // read again instead of kept: registers are short here
        const float f = below_level(page_info[c % HALF][tid >> 4].z, level_mem[quarter].x);
        if (c > 0) wait(o_done, (uint32_t)(c - 1) & 1u);   // P of the tile before has been read
#pragma unroll
        for (int r = 0; r < R; r += 2) {
          float e[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            e[k] = ex2_approx(x[r + k] - (m[r + k] == -INFINITY ? 0.f : m[r + k]) + 7.f);
            l[r + k] += e[k];
          }
          put(r, e[0] * f, e[1] * f);
        }
        fence_proxy_async_shared();
        tc_fence_before();
        mbar_arrive(p_ready);
      }

      // ---- the unit's end: out = O / l ----
      if (seg >= 0) {
        // sums over a warp's lanes: each exchange halves the rows a lane looks after, so R + 1 or so exchanges do for all
#pragma unroll
        for (int half = R / 2, bit = 16; half >= 1; half >>= 1, bit >>= 1) {
#pragma unroll
          for (int r = 0; r < half; ++r) {
            const bool up = lane & bit;
            const float give = up ? l[r] : l[r + half], keep = up ? l[r + half] : l[r];
            l[r] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
          }
        }
#pragma unroll
        for (int bit = 16 / R; bit > 0; bit >>= 1) l[0] += __shfl_xor_sync(0xffffffffu, l[0], bit);
        // a quarter of the sum: see `at`; NaN where a wait has run out
        if (lane % (32 / R) == 0) reinterpret_cast<float*>(&warp_sums[seg & 1][lane / (32 / R)])[quarter] = *abort_flag ? NAN : l[0] * 0.25f;
      }
      const bool more = take(w_next);            // while the last P V runs
      if (seg >= 0) {
        wait(o_done, (uint32_t)(c - 1) & 1u);
        tc_fence_after();
        named_barrier_sync(1, 128);
        const int slot = w.t0 == 0 ? (w.t1 == w.tiles ? -1 : 1) : 0;
        // A flag is read here, after this barrier, by all; cleared a unit later, and written two units later at the
        // earliest: there are barriers between.  The same goes for warp_sums, which two units share in turn.
        const bool bad = poison[seg % 3] != 0;
        if (tid == 0) poison[(seg + 2) % 3] = 0;
        const long long o_at = slot < 0 ? w.b * p.o_seq + i0 * p.o_tok + (long long)(h * p.group + g0) * p.o_head : 0;
        const long long turn = p.o_tok - (p.group - 1) * p.o_head;     // from a query's last head to the next query's first
#pragma unroll 1
        for (int y = 0; y < C::HALVES; ++y) {
          float val[R];
#pragma unroll
          for (int r8 = 0; r8 < R; r8 += 8) {
            uint32_t o[24];
            paged_tmem_ld(tmem + lane_off + C::O_COL + y * C::N + r8, R, o);
#pragma unroll
            for (int r = 0; r < 8; ++r) val[r8 + r] = paged_sum(o, r);
          }
          const int d = y * 128 + tid;
          if (d >= D) break;
          uint32_t nans = *abort_flag ? ~0u : 0u;  // rows that see a NaN in this head dim, or that the last wait left incomplete
          if (bad) {
#pragma unroll 1
            for (int tok = max(lim_min, w.t0 * 128); tok < min(w.len, w.t1 * 128); ++tok) {
              const int id = p.table[w.b * p.table_ld + page_of(p, tok >> 4)];
              if (id >= 0 && id < p.blocks && (p.vc[(((long long)id * p.kv_heads + h) * p.block + tok % p.block) * D + d] & 0x7f) == 0x7f) {
#pragma unroll 1
                for (int r = 0; r < R; ++r) nans |= (uint32_t)(tok < w.len - p.n_q + 1 + (r0 + r) / p.group) << r;
              }
            }
          }
          const int n_rows = min(R, p.rows - r0);
          const float at = power_of_2(level_mem[quarter].x - 2);  // 2^x / 4, because x may be 128
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (nans >> r & 1) val[r] = NAN;
          if (slot < 0) {
            T* dst = reinterpret_cast<T*>(p.o) + o_at + d;
            int left = p.group - g0;
#pragma unroll
            for (int r = 0; r < R; ++r) {
              const float4 sums = warp_sums[seg & 1][r];
              const float sum = (sums.x + sums.y) + (sums.z + sums.w);
              if (r < n_rows) *dst = (T)(sum == 0.f ? 0.f : val[r] * (rcp_approx(sum) * at));       // 0: nothing seen
              --left;
              dst += left ? p.o_head : turn;
              left = left ? left : p.group;
            }
          } else {
            from_mem(1, m);
            float* part = p.part_o + ((long long)blockIdx.x * 2 + slot) * (R * D) + d;
            float2* part_ml = p.part_ml + ((long long)blockIdx.x * 2 + slot) * R;
#pragma unroll
            for (int r = 0; r < R; ++r) {
              const float4 sums = warp_sums[seg & 1][r];
              const float sum = (sums.x + sums.y) + (sums.z + sums.w);
              if (r < n_rows) part[r * D] = sum == 0.f ? 0.f : val[r] * (rcp_approx(sum) * at);
              if (d == r) part_ml[r] = make_float2(m[r], sum * 0x1p-38f);      // the join's products with it stay finite
            }
          }
        }
        __syncwarp();
        tc_fence_before();
        if (slot == 1) cut_b = w.b;                // the piece's last unit
      }
      if (!more) break;
      w = w_next;
    }
    if (tid == 0 && !p.whole)
      *reinterpret_cast<int4*>(p.cut + 4 * blockIdx.x) = make_int4(cut_b, w.h, w.rb, cut_b < 0 ? 0 : (w.at + 8 * (w.tiles - 1)) / piece);
  }

  // ---- teardown ----
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  if (abort_mem) {   // a wait ran out: say so, and let copies in flight land before the shared memory goes to another CTA
    if (threadIdx.x == 0) atomicOr(&cache_ops_status, VLA_ST_WAIT_TIMEOUT);
#pragma unroll 1
    for (int i = 0; i < 32; ++i) __nanosleep(1000);
  }
  if (warp == 1) tmem_dealloc(tmem, C::TMEM_COLS);
}

// Joins the parts of the units that were cut, each with its share of the unit's sum: block (c, y) does two or four rows of the unit that starts in piece c.  A row's
// parts are dealt out to groups of D / 4 threads, which take four head dims each; the groups' sums are then added in order.
// Half and twice the rows a block: heads of 256, 4 sequences of 90001 to 131071, 46.2 and 52.9 us (48.4 so), 16 of 3000 to 9000 with 2
// tokens each, 25.9 and 26.0 (25.2); heads of 64, 16 of 100 to 4001 with 4 tokens each, 18.7 and 17.5 (17.1); of 128, 51.2, 53.5 (51.9).
constexpr int PAGED_JOIN_THREADS = 512;
template <int D>
constexpr int PAGED_JOIN_ROWS = D == 256 ? 2 : 4;
template <typename T, int D, int NT>
__global__ void __launch_bounds__(PAGED_JOIN_THREADS) paged_join_kernel(const __grid_constant__ PagedAttnParams p) {
  constexpr int R = 8 * NT, ROWS = PAGED_JOIN_ROWS<D>, LANES = D / 4, GROUPS = PAGED_JOIN_THREADS / (LANES * ROWS);
  __shared__ float4 sums[GROUPS][ROWS][LANES];
  __shared__ float2 group_ml[GROUPS][ROWS];
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x;
  const int4 cut = *reinterpret_cast<const int4*>(p.cut + 4 * c);
  if (cut.x < 0) return;
  const int n = cut.w - c + 1, lane = threadIdx.x % LANES, row = threadIdx.x / LANES % ROWS, group = threadIdx.x / (LANES * ROWS);
  const int r = blockIdx.y * ROWS + row, rr = cut.z * R + r;
  const bool on = r < R && rr < p.rows;          // rows of the last block beyond the unit's were not written
  auto at = [&](int i) { return ((long long)(c + i) * 2 + (i == 0 ? 1 : 0)) * R + r; };
  auto weight = [](float m, float top) { return m == top ? 1.f : ex2_approx(m - top); };
  float m = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = group; i < (on ? n : 0); i += GROUPS) {
    const float2 ml = p.part_ml[at(i)];
    const float4 v = *reinterpret_cast<const float4*>(p.part_o + at(i) * D + 4 * lane);
    const float top = fmaxf(m, ml.x), a = weight(m, top), b = weight(ml.x, top);
    m = top;
    const float weigh = ml.y * b;
    sum = sum * a + weigh;
    acc.x = acc.x * a + v.x * weigh;
    acc.y = acc.y * a + v.y * weigh;
    acc.z = acc.z * a + v.z * weigh;
    acc.w = acc.w * a + v.w * weigh;
  }
  sums[group][row][lane] = acc;
  if (lane == 0) group_ml[group][row] = make_float2(m, sum);
  __syncthreads();
  if (group || !on) return;
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) top = fmaxf(top, group_ml[k][row].x);
  sum = 0.f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) {
    const float2 ml = group_ml[k][row];
    const float4 v = sums[k][row][lane];
    const float b = weight(ml.x, top);
    sum += ml.y * b;
    acc.x += v.x * b;
    acc.y += v.y * b;
    acc.z += v.z * b;
    acc.w += v.w * b;
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  uint2* dst = reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.o) + paged_row(p, cut.x, cut.y, rr, p.o_seq, p.o_tok, p.o_head) + 4 * lane);
  *dst = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
}
