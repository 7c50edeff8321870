// Attention of the newest tokens of every sequence over its cache in pages (e4m3 codes, one scale for each page and head;
// layout in cache_pages.cuh).  q[b][i] is token lens[b] - n + i of sequence b and sees the keys j <= lens[b] - n + i; key j is
// row j % block of page table[b][j / block].  A page id outside the cache is not seen.  A row that sees nothing is zero.
//
// Bound by the bytes of the cache: each code is read once and used by the n * heads / kv_heads rows that share it.
// Codes become fp16 without rounding (e4m3 has 4 bits of significand and 2^-9 .. 448 for a range), so the products run on
// mma.m16n8k16 with fp16 operands and fp32 sums; at 8 rows per key the tensor work is a few per cent of what even
// that path can do while the codes stream in.  Keys and values are the 16-wide operand (tokens, then head dims), the rows
// the 8-wide one, so that 8 rows, the heads of the Gemma prefix, leave nothing idle:
//     S^T[16 tokens x 8 rows]  = K . Q^T          O^T[head dims x 8 rows] += s_v (V^T . P^T)
// The page's scale of K multiplies S, that of V the product's fp32 result, both after the sums.
// A warp works alone on tiles of 16 tokens (never more than one page) with cp.async into its own ring of tiles; the 8
// warps of a CTA take the tiles of a unit in turn and join their sums at its end.
//
// A unit is (sequence, kv head, block of 8 NT rows).  With few or long sequences the tiles of all units are laid out in one
// line and cut into equal pieces, one per CTA, whatever the lengths; a unit cut by a piece's border leaves partial sums in
// the workspace, which a second kernel joins in a fixed order.
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
  int n_seqs, n_q, group, kv_heads;
  int rows;              // n_q * group
  int row_blocks;        // ceil(rows / (8 NT))
  int blocks, block, width;
  float scale_log2e;
  int split;             // 0: CTA c does unit c; 1: pieces of the line of tiles
  float* part_o;         // [cta][2][8 NT][D]: sums of a unit's first piece (slot 1) or a later one (slot 0)
  float2* part_ml;       // [cta][2][8 NT]: maximum and sum
  int* cut;              // [cta][4]: the unit that starts in this CTA and ends in another: sequence (-1: none), rest, last CTA
};

constexpr int PAGED_THREADS = 256;
constexpr int PAGED_WARPS = PAGED_THREADS / 32;
constexpr int PAGED_MIN_TILES = 16;      // tiles per CTA, at least

template <int D, int NT>
struct PagedCfg {
  static constexpr int TILE_BYTES = 16 * D;                            // of K, and of V
  static constexpr int STAGES = D == 64 ? 4 : 3;
  static constexpr int RING_BYTES = PAGED_WARPS * STAGES * 2 * TILE_BYTES;
  static constexpr int RSTRIDE = D + 8;                                // floats per row of a warp's sums
  static constexpr int JOIN_BYTES = PAGED_WARPS * 8 * NT * RSTRIDE * 4;   // over the ring, once its tiles are used up
  static constexpr int Q_BYTES = 8 * NT * D * 2;
  static constexpr int KSTEPS = D / 16;
  static constexpr bool Q_REGS = D * NT <= 128 || (D == 256 && NT == 1);
  static constexpr int PER_SM = D == 256 ? 1 : 2;
  static constexpr int BODY_BYTES = RING_BYTES > JOIN_BYTES ? RING_BYTES : JOIN_BYTES;
  static constexpr int SMEM_BYTES = BODY_BYTES + Q_BYTES;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;             // nothing is read where n is 0; the 16 bytes become zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
// two e4m3 codes -> two fp16 values, exact
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
  return h;
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Byte of 16-byte piece c of row r in a tile of rows of D bytes.  The pieces of a row are exchanged so that the K reads (8
// rows, every second piece) and the V reads (every second row, 8 pieces) of a warp hit distinct banks.
template <int D>
__device__ __forceinline__ int tile_at(int r, int c) {
  return D == 64 ? r * D + ((c ^ (r >> 1 & 3)) << 4) : r * D + (((c & ~7) | ((c ^ r) & 7)) << 4);
}
__device__ __forceinline__ bool has_nan(uint32_t w) {   // any of four e4m3 codes is 0x7f or 0xff
  return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
}

__device__ __forceinline__ int paged_len(const PagedAttnParams& p, int b) {
  return (int)min(max((long long)p.lens[b], 0ll), (long long)p.width * p.block);
}
__device__ __forceinline__ int paged_tiles(const PagedAttnParams& p, int b) { return (paged_len(p, b) + 15) / 16; }

// where row rr of (sequence b, kv head h) lies in q / o
__device__ __forceinline__ long long paged_row(const PagedAttnParams& p, int b, int h, int rr, long long seq, long long tok, long long head) {
  return b * seq + (rr / p.group) * tok + (long long)(h * p.group + rr % p.group) * head;
}

// Sums over the CTA's threads before this one, and over all of them.
__device__ __forceinline__ long long block_scan(long long v, long long* all, long long* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < PAGED_WARPS; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  __syncthreads();
  *all = total;
  return before + s - v;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(PAGED_THREADS, (PagedCfg<D, NT>::PER_SM)) paged_attention_kernel(const PagedAttnParams p) {
  using C = PagedCfg<D, NT>;
  constexpr int ROWS = 8 * NT;
  extern __shared__ __align__(128) uint8_t paged_smem[];
  float* join = reinterpret_cast<float*>(paged_smem);
  uint2* q_frag = reinterpret_cast<uint2*>(paged_smem + C::BODY_BYTES);   // [NT][KSTEPS][32]
  __shared__ float q_scale[ROWS];
  __shared__ float2 warp_ml[PAGED_WARPS][ROWS];
  __shared__ long long warp_sum[PAGED_WARPS];
  __shared__ int found_b;
  __shared__ long long found_base;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(paged_smem) + warp * (C::STAGES * 2 * C::TILE_BYTES);
  const int units = p.kv_heads * p.row_blocks;      // per sequence

  // ---- one unit's tiles [t0, t1) ----
  auto segment = [&](int b, int u, int t0, int t1, int part_slot) {
    const int h = u / p.row_blocks, r0 = (u % p.row_blocks) * ROWS;
    const int len = paged_len(p, b);
    const int* table = p.table + b * p.table_ld;

    // tiles of this warp: t0 + warp, + 8, ...; lane i knows the page and scales of the i-th of 32 of them
    const int mine = max(0, (t1 - t0 - warp + PAGED_WARPS - 1) / PAGED_WARPS);
    auto look = [&](int first, int& id, float& ks, float& vs) {
      id = -1;
      ks = vs = 0.f;
      if (first + lane < mine) {
        id = table[(t0 + warp + (first + lane) * PAGED_WARPS) * 16 / p.block];
        if (id < 0 || id >= p.blocks) id = -1;
        else {
          ks = p.ks[(long long)id * p.kv_heads + h];
          vs = p.vs[(long long)id * p.kv_heads + h];
        }
      }
    };
    int id_now, id_next;
    float ks_now, vs_now, ks_next, vs_next;
    look(0, id_now, ks_now, vs_now);
    look(32, id_next, ks_next, vs_next);
    auto issue = [&](int i, int batch) {
      if (i < mine) {
        const int id = __shfl_sync(0xffffffffu, i >> 5 == batch ? id_now : id_next, i & 31);
        const int tok = (t0 + warp + i * PAGED_WARPS) * 16;
        const long long at = id < 0 ? 0 : (((long long)id * p.kv_heads + h) * p.block + tok % p.block) * D;
        const uint32_t dst = ring + (i % C::STAGES) * 2 * C::TILE_BYTES;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          const int piece = k * 32 + lane;
          const uint32_t to = dst + tile_at<D>(piece / (D / 16), piece % (D / 16));
          cp_async16(to, p.kc + at + piece * 16, id >= 0);
          cp_async16(to + C::TILE_BYTES, p.vc + at + piece * 16, id >= 0);
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int i = 0; i < C::STAGES - 1; ++i) issue(i, 0);

    // Q as fp16 fragments for all warps.  A row is multiplied by the power of two that brings its largest magnitude to
    // [2^14, 2^15): bf16's 8 bits fit fp16's 11, and only what is 2^-28 of the row's largest begins to lose bits.
    // MMA (half a, piece s, word j) pairs K's bytes 4j .. 4j + 3 of piece 8a + 2t + s (D = 64: piece t) with the same head
    // dims of Q.
    for (int nt = warp; nt < NT; nt += PAGED_WARPS) {
      const int rr = r0 + nt * 8 + g;
      const T* src = reinterpret_cast<const T*>(p.q) + (rr < p.rows ? paged_row(p, b, h, rr, p.q_seq, p.q_tok, p.q_head) : 0);
      constexpr int PIECES = D / 64;         // 16-element pieces per lane
      uint32_t w[PIECES][8];
      float top = 0.f;
#pragma unroll
      for (int x = 0; x < PIECES; ++x) {
        const int d = D == 64 ? 16 * t : 128 * (x >> 1) + 32 * t + 16 * (x & 1);
        uint4 v0 = make_uint4(0u, 0u, 0u, 0u), v1 = v0;
        if (rr < p.rows) {
          v0 = *reinterpret_cast<const uint4*>(src + d);
          v1 = *reinterpret_cast<const uint4*>(src + d + 8);
        }
        const uint32_t vv[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[x][e] = vv[e];
          const float2 f = unpack2<T>(vv[e]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = (__float_as_int(top) >> 23) - 127 - 14;                       // top in [2^(e+14), 2^(e+15))
      const bool plain = top == 0.f || !(top < INFINITY) || e < -126 || e > 126;  // zeros, infinities, the edges of the range
      const float up = plain ? 1.f : __int_as_float((127 - e) << 23);
      if (t == 0) q_scale[nt * 8 + g] = (plain ? 1.f : __int_as_float((127 + e) << 23)) * p.scale_log2e;
#pragma unroll
      for (int x = 0; x < PIECES; ++x)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f0 = unpack2<T>(w[x][2 * j]), f1 = unpack2<T>(w[x][2 * j + 1]);
          const __half2 h0 = __floats2half2_rn(f0.x * up, f0.y * up), h1 = __floats2half2_rn(f1.x * up, f1.y * up);
          q_frag[(nt * C::KSTEPS + x * 4 + j) * 32 + lane] =
              make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
        }
    }
    __syncthreads();
    uint2 qr[C::Q_REGS ? NT * C::KSTEPS : 1];
    if (C::Q_REGS) {
#pragma unroll
      for (int i = 0; i < (C::Q_REGS ? NT * C::KSTEPS : 1); ++i) qr[i] = q_frag[i * 32 + lane];
    }
    float sc[NT][2];
    int lim[NT][2];                          // keys that the rows of this lane's columns see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = nt * 8 + 2 * t + c;
        sc[nt][c] = q_scale[r];
        lim[nt][c] = r0 + r < p.rows ? len - p.n_q + 1 + (r0 + r) / p.group : len;
      }
    const int lim_min = len - p.n_q + 1 + r0 / p.group;

    float o[NT][D / 16][4];                  // [.][(half a, word j, e)]: head dims 128a + 16g + 4j + 2e, + 1 (D = 64: 8g + 4j + 2e)
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int f = 0; f < D / 16; ++f) o[nt][f][0] = o[nt][f][1] = o[nt][f][2] = o[nt][f][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }

    for (int i = 0; i < mine; ++i) {
      if (i && (i & 31) == 0) {
        id_now = id_next; ks_now = ks_next; vs_now = vs_next;
        look(i + 32, id_next, ks_next, vs_next);
      }
      cp_wait<C::STAGES - 2>();
      __syncwarp();
      issue(i + C::STAGES - 1, i >> 5);
      const int id = __shfl_sync(0xffffffffu, id_now, i & 31);
      const float ks = __shfl_sync(0xffffffffu, ks_now, i & 31), vs = __shfl_sync(0xffffffffu, vs_now, i & 31);
      const int tok = (t0 + warp + i * PAGED_WARPS) * 16;
      const uint32_t sk = ring + (i % C::STAGES) * 2 * C::TILE_BYTES, sv = sk + C::TILE_BYTES;

      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int x = 0; x < D / 64; ++x) {
        const int piece = D == 64 ? t : 8 * (x >> 1) + 2 * t + (x & 1);
        const uint4 a = lds128(sk + tile_at<D>(g, piece)), c = lds128(sk + tile_at<D>(g + 8, piece));
        const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wc[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t fr[4] = {e4m3x2_f16x2(wa[j]), e4m3x2_f16x2(wc[j]), e4m3x2_f16x2(wa[j] >> 16), e4m3x2_f16x2(wc[j] >> 16)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint2 qq = C::Q_REGS ? qr[nt * C::KSTEPS + x * 4 + j] : q_frag[(nt * C::KSTEPS + x * 4 + j) * 32 + lane];
            mma_f16(s[nt], fr, qq.x, qq.y);
          }
        }
      }
      const bool edge = tok + 16 > lim_min || id < 0;        // warp-uniform: some row does not see some token
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nt][e] *= sc[nt][e & 1] * ks;
          if (edge && (id < 0 || tok + g + 4 * (e & 2) >= lim[nt][e & 1])) s[nt][e] = -INFINITY;
          grow |= s[nt][e] > m[nt][e & 1] + 8.f;
        }
      // The subtracted maximum moves when a score has outgrown it by 2^8: probabilities stay below that, within fp16.
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = fmaxf(m[nt][c], fmaxf(s[nt][c], s[nt][c + 2]));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            const float a = top == m[nt][c] ? 1.f : ex2_approx(m[nt][c] - top);
            m[nt][c] = top;
            l[nt][c] *= a;
#pragma unroll
            for (int f = 0; f < D / 16; ++f) {
              o[nt][f][c] *= a;
              o[nt][f][c + 2] *= a;
            }
          }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float e[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float sub = m[nt][k & 1] == -INFINITY ? 0.f : m[nt][k & 1];
          e[k] = ex2_approx(s[nt][k] - sub);
          l[nt][k & 1] += e[k];
        }
        const __half2 h0 = __floats2half2_rn(e[0], e[1]), h1 = __floats2half2_rn(e[2], e[3]);
        pb[nt][0] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&h0));
        pb[nt][1] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&h1));
      }
      // O^T += s_v (V^T P^T), tokens 2t, 2t + 1, 2t + 8, 2t + 9 of each lane.  `seen`: tokens from there on are cleared;
      // `query` >= 0: only the columns of that query are added.
      auto pv = [&](auto careful, int seen, int query) {
        constexpr int VW = D == 64 ? 2 : 4;                  // words per row and lane
        bool nan = false;
#pragma unroll
        for (int a = 0; a < (D == 256 ? 2 : 1); ++a) {
          uint32_t w[4][VW];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = 2 * t + (k & 1) + 4 * (k & 2);
            if (D == 64) {
              const uint2 v = lds64(sv + tile_at<D>(row, g >> 1) + 8 * (g & 1));
              w[k][0] = v.x; w[k][1] = v.y;
            } else {
              const uint4 v = lds128(sv + tile_at<D>(row, 8 * a + g));
              w[k][0] = v.x; w[k][1] = v.y; w[k][VW - 2] = v.z; w[k][VW - 1] = v.w;
            }
            if (decltype(careful)::value && tok + row >= seen) {
#pragma unroll
              for (int j = 0; j < VW; ++j) w[k][j] = 0u;
            }
          }
#pragma unroll
          for (int j = 0; j < VW; ++j) {
            if (decltype(careful)::value && query < 0) nan |= has_nan(w[0][j]) || has_nan(w[1][j]) || has_nan(w[2][j]) || has_nan(w[3][j]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t x = __byte_perm(w[0][j], w[1][j], e ? 0x7362 : 0x5140), y = __byte_perm(w[2][j], w[3][j], e ? 0x7362 : 0x5140);
              const uint32_t fr[4] = {e4m3x2_f16x2(x), e4m3x2_f16x2(x >> 16), e4m3x2_f16x2(y), e4m3x2_f16x2(y >> 16)};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                mma_f16(c, fr, pb[nt][0], pb[nt][1]);
                float* acc = o[nt][a * 8 + j * 2 + e];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  if (!decltype(careful)::value || query < 0 || (r0 + nt * 8 + 2 * t + (k & 1)) / p.group == query) acc[k] = fmaf(vs, c[k], acc[k]);
              }
            }
          }
        }
        return nan;
      };
      if (!edge) {
        pv(std::false_type{}, 0, -1);
      } else if (p.n_q == 1) {
        pv(std::true_type{}, len, -1);
      } else {
        // Tokens that only later queries see: a NaN among their values would reach the others as 0 * NaN.  Then each
        // query is multiplied with its own tokens alone.
        bool nan = false;
        for (int k = lane; k < D; k += 32) {
          const int row = k / (D / 16);
          const uint4 v = lds128(sv + tile_at<D>(row, k % (D / 16)));
          nan |= tok + row >= lim_min && tok + row < len && (has_nan(v.x) || has_nan(v.y) || has_nan(v.z) || has_nan(v.w));
        }
        if (!__any_sync(0xffffffffu, nan)) {
          pv(std::true_type{}, len, -1);
        } else {
          const int q_end = min((r0 + ROWS - 1) / p.group, p.n_q - 1);
          for (int query = r0 / p.group; query <= q_end; ++query) pv(std::true_type{}, len - p.n_q + 1 + query, query);
        }
      }
    }
    cp_wait<0>();

    // ---- join the warps' sums: out = sum_w 2^(m_w - M) o_w / sum_w 2^(m_w - M) l_w ----
    __syncthreads();                         // every warp is through with its ring
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], x);
        if (g == 0) warp_ml[warp][nt * 8 + 2 * t + c] = make_float2(m[nt][c], l[nt][c]);
      }
      if (mine > 0) {
#pragma unroll
        for (int f = 0; f < D / 16; ++f)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            *reinterpret_cast<float2*>(join + (warp * ROWS + nt * 8 + 2 * t + c) * C::RSTRIDE + f * 16 + g * 2) =
                make_float2(o[nt][f][c], o[nt][f][c + 2]);
      }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < ROWS * (D / 2); x += PAGED_THREADS) {
      const int r = x / (D / 2), d = (x % (D / 2)) * 2, rr = r0 + r;
      if (rr >= p.rows) continue;
      // head dim d lies at fragment f, lane group gg
      const int gg = D == 64 ? d / 8 : d % 128 / 16, f = D == 64 ? d % 8 / 2 : d / 128 * 8 + d % 16 / 2;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < PAGED_WARPS; ++w) top = fmaxf(top, warp_ml[w][r].x);
      float2 acc = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < PAGED_WARPS; ++w) {
        const float2 ml = warp_ml[w][r];
        if (ml.x != -INFINITY || ml.y != 0.f) {   // otherwise this warp has seen nothing of this row
          const float a = ml.x == top ? 1.f : ex2_approx(ml.x - top);
          const float2 v = *reinterpret_cast<const float2*>(join + (w * ROWS + r) * C::RSTRIDE + f * 16 + gg * 2);
          acc.x = fmaf(a, v.x, acc.x);
          acc.y = fmaf(a, v.y, acc.y);
          sum = fmaf(a, ml.y, sum);
        }
      }
      if (part_slot < 0) {
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        T* dst = reinterpret_cast<T*>(p.o) + paged_row(p, b, h, rr, p.o_seq, p.o_tok, p.o_head) + d;
        dst[0] = (T)(acc.x * inv);
        dst[1] = (T)(acc.y * inv);
      } else {
        const long long at = ((long long)blockIdx.x * 2 + part_slot) * ROWS + r;
        *reinterpret_cast<float2*>(p.part_o + at * D + d) = acc;
        if (d == 0) p.part_ml[at] = make_float2(top, sum);
      }
    }
    __syncthreads();                         // before the next unit's tiles go over the sums
  };
  auto zero = [&](int b, int h0, int h1) {
    for (int x = threadIdx.x; x < (h1 - h0) * p.rows * D; x += PAGED_THREADS) {
      const int h = h0 + x / (p.rows * D), rr = x / D % p.rows;
      reinterpret_cast<T*>(p.o)[paged_row(p, b, h, rr, p.o_seq, p.o_tok, p.o_head) + x % D] = (T)0.f;
    }
  };

  if (!p.split) {
    const int b = blockIdx.x / units, u = blockIdx.x % units;
    const int tiles = paged_tiles(p, b);
    if (tiles) segment(b, u, 0, tiles, -1);
    else if (u % p.row_blocks == 0) zero(b, u / p.row_blocks, u / p.row_blocks + 1);
    return;
  }
  for (int b = blockIdx.x; b < p.n_seqs; b += gridDim.x)
    if (paged_tiles(p, b) == 0) zero(b, 0, p.kv_heads);

  // This CTA's piece of the line of tiles, and the sequence it starts in
  long long total = 0;
  for (int base = 0; base < p.n_seqs; base += PAGED_THREADS) {
    const int b = base + threadIdx.x;
    long long all;
    block_scan(b < p.n_seqs ? (long long)paged_tiles(p, b) * units : 0, &all, warp_sum);
    total += all;
  }
  const long long piece = max((total + gridDim.x - 1) / gridDim.x, (long long)PAGED_MIN_TILES);
  const long long begin = blockIdx.x * piece, end = min(begin + piece, total);
  int cut_b = -1, cut_u = 0, cut_last = 0;
  if (begin < end) {
    long long sum = 0;
    for (int base = 0; base < p.n_seqs && sum <= begin; base += PAGED_THREADS) {
      const int b = base + threadIdx.x;
      const long long n = b < p.n_seqs ? (long long)paged_tiles(p, b) * units : 0;
      long long all;
      const long long at = sum + block_scan(n, &all, warp_sum);
      if (at <= begin && begin < at + n) {
        found_b = b;
        found_base = at;
      }
      sum += all;
    }
    __syncthreads();
    int b = found_b;
    long long base = found_base, pos = begin;
    while (pos < end) {
      const int tiles = paged_tiles(p, b);
      const long long n = (long long)tiles * units;
      if (pos >= base + n) {                 // on to the next sequence that has tokens
        base += n;
        ++b;
        continue;
      }
      const int u = (int)((pos - base) / tiles), t0 = (int)((pos - base) % tiles);
      const int t1 = (int)min((long long)tiles, t0 + (end - pos));
      const long long unit_at = base + (long long)u * tiles;
      const bool first = unit_at >= begin, last = unit_at + tiles <= end;
      segment(b, u, t0, t1, first && last ? -1 : first ? 1 : 0);
      if (first && !last) {
        cut_b = b;
        cut_u = u;
        cut_last = (int)((unit_at + tiles - 1) / piece);
      }
      pos += t1 - t0;
    }
  }
  if (threadIdx.x == 0) *reinterpret_cast<int4*>(p.cut + 4 * blockIdx.x) = make_int4(cut_b, cut_u, cut_last, 0);
  pdl_trigger();
}

// Joins the partial sums of the units that were cut: block (c, r) does row r of the unit that starts in piece c, one thread per
// head dim, the pieces in order.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(D) paged_join_kernel(const PagedAttnParams p) {
  constexpr int ROWS = 8 * NT;
  pdl_wait();
  const int c = blockIdx.x, r = blockIdx.y, d = threadIdx.x;
  const int4 cut = *reinterpret_cast<const int4*>(p.cut + 4 * c);
  if (cut.x < 0) return;
  const int h = cut.y / p.row_blocks, rr = (cut.y % p.row_blocks) * ROWS + r;
  if (rr >= p.rows) return;
  const int n = cut.z - c + 1;
  auto at = [&](int i) { return ((long long)(c + i) * 2 + (i == 0 ? 1 : 0)) * ROWS + r; };
  float top = -INFINITY;
  for (int i = 0; i < n; ++i) top = fmaxf(top, p.part_ml[at(i)].x);
  float acc = 0.f, sum = 0.f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float2 ml = p.part_ml[at(i)];
    const float v = p.part_o[at(i) * D + d];
    if (ml.x != -INFINITY || ml.y != 0.f) {
      const float a = ml.x == top ? 1.f : ex2_approx(ml.x - top);
      acc = fmaf(a, v, acc);
      sum = fmaf(a, ml.y, sum);
    }
  }
  reinterpret_cast<T*>(p.o)[paged_row(p, cut.x, h, rr, p.o_seq, p.o_tok, p.o_head) + d] = (T)(sum != 0.f ? acc / sum : 0.f);
}
