// C entry points of the operators around a key/value cache in pages (include/vla_b200.h): argument checks, launches.
// All of them only enqueue work on the caller's stream: no allocation, no synchronisation, nothing kept between calls, so
// they can be captured into a graph and called from several threads and streams at once.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <type_traits>

#include "../../include/vla_b200.h"
#include "attention_paged.cuh"
#include "attention_prompt.cuh"
#include "cache_pages.cuh"
#include "host.cuh"

namespace {

int refuse(int code, const char* fmt, ...) {
  char buf[320];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  try {
    g_last_error = buf;
  } catch (...) {   // no memory for the message: the code still says what happened
  }
  return code;
}

int launched(const char* who, cudaError_t e) {
  if (e == cudaSuccess) return VLA_OK;
  (void)cudaGetLastError();            // it has been told; the library's next call must not find it
  return refuse(VLA_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}

// No C++ exception leaves a C entry point.
template <typename F>
int guarded(const char* who, F f) {
  try {
    return f();
  } catch (...) {
    return refuse(VLA_ERR_STATE, "%s: out of host memory", who);
  }
}

int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// 16-byte rows: base and strides of a 16-bit tensor that is read in vectors of eight
bool vectors(const void* p, long long a, long long b) { return aligned(p, 16) && a % 8 == 0 && b % 8 == 0; }

constexpr long long INT_TOP = 0x7fffffff;

// Tensor map of a tensor whose innermost dimension, given first, is contiguous (strides in elements of `size` bytes), for
// boxes of rows of 128 or 64 bytes with the swizzle of that width.  The stride of a dimension of size one is free in the
// caller's tensor and made valid here.
template <int N>
bool tensor_map(CUtensorMap* tm, const void* base, int size, CUtensorMapDataType type, const long long (&dims)[N], const long long (&strides)[N - 1],
                const int (&box)[N]) {
  EncodeTiledFn fn = get_encode_fn();            // the callers have looked
  cuuint64_t gd[N], gs[N - 1];
  cuuint32_t bx[N], es[N];
  for (int i = 0; i < N; ++i) {
    gd[i] = (cuuint64_t)dims[i];
    bx[i] = (cuuint32_t)box[i];
    es[i] = 1;
    if (i > 0) gs[i - 1] = (cuuint64_t)(dims[i] > 1 ? strides[i - 1] : dims[0]) * size;
  }
  return fn(tm, type, N, const_cast<void*>(base), gd, gs, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            box[0] * size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How the calls of vla_op_paged_attention are shared out, from the sizes that the host knows (not the lengths).
struct PagedShape {
  int rows, nt, row_blocks;
  long long ctas;
  bool whole;              // units are short enough not to be cut
  size_t workspace;        // bytes; 0: nothing to join
};
PagedShape paged_shape(const vla_paged_attn_desc* d) {
  PagedShape s;
  const long long rows = (long long)d->n_q * (d->heads / d->kv_heads);
  s.rows = (int)std::min(rows, INT_TOP);
  s.nt = s.rows > 8 ? 2 : 1;
  s.row_blocks = (int)((rows + 8 * s.nt - 1) / (8 * s.nt));
  const long long units = (long long)d->n_seqs * d->kv_heads * s.row_blocks;
  const long long groups = (long long)d->width * d->block_size / 16;            // of 16 tokens in a unit, at most
  const long long room = (long long)sm_count() * (d->head_dim == 256 ? 1 : 2);  // CTAs that run at once
  s.whole = groups <= PAGED_WHOLE;
  s.ctas = std::min(room, s.whole ? units : (units * (groups + paged_gap(d->head_dim)) + PAGED_MIN_PIECE - 1) / PAGED_MIN_PIECE);
  const size_t rows_kept = (size_t)s.ctas * 2 * 8 * s.nt;
  s.workspace = s.whole ? 0 : rows_kept * ((size_t)d->head_dim * sizeof(float) + sizeof(float2)) + (size_t)s.ctas * 4 * sizeof(int);
  return s;
}

// Sizes and types of a vla_paged_attn_desc; what passes keeps paged_shape within 64 bits
int paged_check(const char* who, const vla_paged_attn_desc* d) {
  if (!d) return refuse(VLA_ERR_STATE, "%s: null descriptor", who);
  if (d->n_seqs < 0 || d->n_q < 1 || d->heads < 1 || d->kv_heads < 1 || d->num_blocks < 1 || d->width < 0 || d->table_stride < d->width)
    return refuse(VLA_ERR_SHAPE, "%s: bad sizes", who);
  if (d->heads % d->kv_heads) return refuse(VLA_ERR_SHAPE, "%s: heads must be a multiple of kv_heads", who);
  if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256) return refuse(VLA_ERR_SHAPE, "%s: head_dim must be 64, 128 or 256", who);
  if (d->block_size < 16 || d->block_size % 16 || d->block_size > 256) return refuse(VLA_ERR_SHAPE, "%s: block_size must be a multiple of 16 up to 256", who);
  if ((long long)d->width * d->block_size > INT_TOP - 16 || (long long)d->num_blocks * d->block_size > INT_TOP || (long long)d->n_q * d->heads > 1 << 20)
    return refuse(VLA_ERR_LIMIT, "%s: more than 2^31 - 17 tokens, or 2^20 rows of a sequence", who);
  if (d->dtype != VLA_BF16 && d->dtype != VLA_F16) return refuse(VLA_ERR_SHAPE, "%s: q must be bf16 or f16", who);
  if (!(d->scale > 0.f) || d->scale > 3e38f) return refuse(VLA_ERR_SHAPE, "%s: scale must be positive and finite", who);
  // in floating point, because the products may leave 64 bits
  const double rows = (double)d->n_q * (d->heads / d->kv_heads), row_blocks = std::ceil(rows / (rows > 8 ? 16 : 8));
  if ((double)d->n_seqs * d->kv_heads * row_blocks * ((double)d->width * d->block_size / 16 + paged_gap(d->head_dim)) > 2e9)
    return refuse(VLA_ERR_LIMIT, "%s: more than 2e9 groups of 16 tokens in the table's rows, times key/value heads and blocks of 8 or 16 rows", who);
  return VLA_OK;
}

}  // namespace

extern "C" {

int vla_op_block_plan(const vla_block_plan_desc* d, void* stream) {
  const char* who = "vla_op_block_plan";
  return guarded(who, [&]() -> int {
    if (!d) return refuse(VLA_ERR_STATE, "%s: null descriptor", who);
    if (d->n_seqs < 0 || d->n_seqs > PLAN_MAX_SEQS) return refuse(VLA_ERR_LIMIT, "%s: %d requests, at most %d are served", who, d->n_seqs, PLAN_MAX_SEQS);
    if (d->block_size < 1 || d->width < 0 || d->n_free < 0 || d->total_new < 0 || d->table_stride < d->width)
      return refuse(VLA_ERR_SHAPE, "%s: negative size, or a table stride below its width", who);
    if (!d->cu_new || !d->counts) return refuse(VLA_ERR_STATE, "%s: null output", who);
    if (d->n_seqs && (!d->context_lens || !d->new_lens || !d->seq_lens)) return refuse(VLA_ERR_STATE, "%s: null lengths", who);
    if (d->n_seqs && d->width && !d->block_table) return refuse(VLA_ERR_STATE, "%s: null block table", who);
    if (d->n_free && !d->free_blocks) return refuse(VLA_ERR_STATE, "%s: null free list", who);
    if (d->total_new && (!d->slots || !d->positions)) return refuse(VLA_ERR_STATE, "%s: null slots or positions", who);
    if (!aligned(d->slots, 16) || !aligned(d->positions, 16)) return refuse(VLA_ERR_SHAPE, "%s: slots and positions must start on 16 bytes", who);
    PlanParams p;
    p.ctx = d->context_lens; p.n_new = d->new_lens; p.n_seqs = d->n_seqs;
    p.table = d->block_table; p.width = d->width; p.table_ld = d->table_stride;
    p.free_ids = d->free_blocks; p.n_free = d->n_free; p.first = d->first_free;
    p.block = d->block_size; p.total = d->total_new;
    p.block_recip = (unsigned)std::min<unsigned long long>((1ull << 32) / d->block_size, 0xffffffffull);
    p.slots = d->slots; p.positions = d->positions; p.cu_new = d->cu_new; p.seq_lens = d->seq_lens; p.counts = d->counts;
    const size_t smem = (size_t)(2 * d->n_seqs + 2) * sizeof(int);
    if (smem > 40 * 1024)
      if (cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(block_plan_kernel), (2 * PLAN_MAX_SEQS + 2) * (int)sizeof(int)); e != cudaSuccess)
        return launched(who, e);
    // one row a thread, or a CTA on each SM: with four rows a thread 140k rows of 512 requests take 6.2 us instead of 5.2
    const int ctas = std::min((std::max(std::max(d->total_new, d->n_seqs), 1) - 1) / PLAN_THREADS + 1, sm_count());
    return launched(who, launch_ex(block_plan_kernel, dim3(ctas), dim3(PLAN_THREADS), smem, reinterpret_cast<cudaStream_t>(stream), 1, true, p));
  });
}

int vla_op_cache_append(const vla_cache_append_desc* d, void* stream) {
  const char* who = "vla_op_cache_append";
  return guarded(who, [&]() -> int {
    if (!d) return refuse(VLA_ERR_STATE, "%s: null descriptor", who);
    if (d->tokens < 0 || d->kv_heads < 1 || d->num_blocks < 1) return refuse(VLA_ERR_SHAPE, "%s: bad sizes", who);
    if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256) return refuse(VLA_ERR_SHAPE, "%s: head_dim must be 64, 128 or 256", who);
    if (d->block_size < 16 || d->block_size % 16 || d->block_size > 256) return refuse(VLA_ERR_SHAPE, "%s: block_size must be a multiple of 16 up to 256", who);
    if ((long long)d->num_blocks * d->block_size > INT_TOP) return refuse(VLA_ERR_LIMIT, "%s: more than 2^31 - 1 slots", who);
    if (d->dtype != VLA_BF16 && d->dtype != VLA_F16) return refuse(VLA_ERR_SHAPE, "%s: keys and values must be bf16 or f16", who);
    if (!d->k_codes || !d->v_codes || !d->k_scale || !d->v_scale) return refuse(VLA_ERR_STATE, "%s: null cache", who);
    if (!aligned(d->k_codes, 16) || !aligned(d->v_codes, 16)) return refuse(VLA_ERR_SHAPE, "%s: the cache must start on 16 bytes", who);
    if (d->tokens == 0) return VLA_OK;
    if (!d->k || !d->v || !d->slots) return refuse(VLA_ERR_STATE, "%s: null keys, values or slots", who);
    if (!vectors(d->k, d->k_tok_stride, d->k_head_stride) || !vectors(d->v, d->v_tok_stride, d->v_head_stride))
      return refuse(VLA_ERR_SHAPE, "%s: rows of k and v must start on 16 bytes", who);
    AppendParams p;
    p.x[0] = d->k; p.x[1] = d->v;
    p.x_tok[0] = d->k_tok_stride; p.x_tok[1] = d->v_tok_stride; p.x_head[0] = d->k_head_stride; p.x_head[1] = d->v_head_stride;
    p.codes[0] = reinterpret_cast<uint8_t*>(d->k_codes); p.codes[1] = reinterpret_cast<uint8_t*>(d->v_codes);
    p.scale[0] = d->k_scale; p.scale[1] = d->v_scale;
    p.slots = d->slots; p.tokens = d->tokens; p.kv_heads = d->kv_heads; p.block = d->block_size;
    p.n_slots = (long long)d->num_blocks * d->block_size;
    p.block_recip = d->block_size == 16 ? 0 : (uint32_t)(((1ull << 32) + d->block_size / 16 - 1) / (d->block_size / 16));
    const long long per_cta = APPEND_THREADS / 32, items = 2ll * d->kv_heads;
    // As many warps as run at once, and no more: a warp whose window starts no run is launched for nothing.  16,000 tokens of a head
    // of 256 take 4.6 us; with room for 28 warps an SM, of which 16 are there, 6.3.
    const long long at_once = (long long)append_ctas(d->head_dim) * per_cta * sm_count();
    for (p.window = 1; p.window < APPEND_WINDOW && d->tokens / p.window * items > at_once;) p.window *= 2;
    const long long jobs = ((long long)d->tokens + p.window - 1) / p.window * items;
    if (jobs > INT_TOP) return refuse(VLA_ERR_LIMIT, "%s: too many tokens and heads", who);
    const dim3 grid((unsigned)((jobs + per_cta - 1) / per_cta));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    auto go = [&](auto kern) { return launched(who, launch_ex(kern, grid, dim3(APPEND_THREADS), 0, st, 1, true, p)); };
    if (d->dtype == VLA_BF16)
      return d->head_dim == 64 ? go(cache_append_kernel<bf16, 64>) : d->head_dim == 128 ? go(cache_append_kernel<bf16, 128>) : go(cache_append_kernel<bf16, 256>);
    return d->head_dim == 64 ? go(cache_append_kernel<__half, 64>) : d->head_dim == 128 ? go(cache_append_kernel<__half, 128>) : go(cache_append_kernel<__half, 256>);
  });
}

int vla_op_paged_attention_workspace(const vla_paged_attn_desc* d, size_t* bytes) {
  const char* who = "vla_op_paged_attention_workspace";
  return guarded(who, [&]() -> int {
    if (int rc = paged_check(who, d)) return rc;
    if (!bytes) return refuse(VLA_ERR_STATE, "%s: null argument", who);
    *bytes = d->n_seqs ? paged_shape(d).workspace : 0;
    return VLA_OK;
  });
}

int vla_op_paged_attention(const vla_paged_attn_desc* d, void* stream) {
  const char* who = "vla_op_paged_attention";
  return guarded(who, [&]() -> int {
    if (int rc = paged_check(who, d)) return rc;
    if (d->n_seqs == 0) return VLA_OK;
    if (!d->q || !d->o || !d->k_codes || !d->v_codes || !d->k_scale || !d->v_scale || !d->seq_lens || (d->width && !d->block_table))
      return refuse(VLA_ERR_STATE, "%s: null argument", who);
    if (!aligned(d->k_codes, 16) || !aligned(d->v_codes, 16)) return refuse(VLA_ERR_SHAPE, "%s: the cache must start on 16 bytes", who);
    if (!vectors(d->q, d->q_seq_stride, d->q_tok_stride) || d->q_head_stride % 8 || !vectors(d->o, d->o_seq_stride, d->o_tok_stride) || d->o_head_stride % 8)
      return refuse(VLA_ERR_SHAPE, "%s: rows of q and o must start on 16 bytes", who);
    const PagedShape s = paged_shape(d);
    if (s.workspace && (!d->workspace || d->workspace_bytes < s.workspace || !aligned(d->workspace, 16)))
      return refuse(VLA_ERR_STATE, "%s: a workspace of %zu bytes on a 16-byte boundary is needed", who, s.workspace);
    if (!get_encode_fn()) return refuse(VLA_ERR_CUDA, "%s: the CUDA driver that encodes tensor maps is not there", who);
    PagedAttnParams p;
    p.q = d->q; p.o = d->o;
    p.q_seq = d->q_seq_stride; p.q_tok = d->q_tok_stride; p.q_head = d->q_head_stride;
    p.o_seq = d->o_seq_stride; p.o_tok = d->o_tok_stride; p.o_head = d->o_head_stride;
    p.vc = reinterpret_cast<const uint8_t*>(d->v_codes);
    p.ks = d->k_scale; p.vs = d->v_scale;
    p.table = d->block_table; p.table_ld = d->table_stride; p.lens = d->seq_lens;
    p.n_seqs = d->n_seqs; p.n_q = d->n_q; p.group = d->heads / d->kv_heads; p.kv_heads = d->kv_heads;
    p.rows = s.rows; p.row_blocks = s.row_blocks; p.units = d->kv_heads * s.row_blocks;
    p.per_page_inv = d->block_size == 16 ? 0u : (uint32_t)(((1ull << 32) + d->block_size / 16 - 1) / (d->block_size / 16));
    p.blocks = d->num_blocks; p.block = d->block_size; p.width = d->width;
    p.scale_log2e = d->scale * 1.4426950408889634f;
    p.whole = s.whole;
    p.box_rows = d->block_size % 128 == 0 ? 128 : d->block_size % 64 == 0 ? 64 : d->block_size % 32 == 0 ? 32 : 16;
    const long long dim = d->head_dim, page = (long long)d->kv_heads * d->block_size;
    const int width = std::min(d->head_dim, 128);
    if (!tensor_map(&p.tmK, d->k_codes, 1, CU_TENSOR_MAP_DATA_TYPE_UINT8, {dim, page, d->num_blocks}, {dim, page * dim}, {width, p.box_rows, 1}) ||
        !tensor_map(&p.tmV, d->v_codes, 1, CU_TENSOR_MAP_DATA_TYPE_UINT8, {dim, page, d->num_blocks}, {dim, page * dim}, {width, p.box_rows, 1}))
      return refuse(VLA_ERR_SHAPE, "%s: the cache cannot be described by a tensor map", who);
    p.part_o = reinterpret_cast<float*>(d->workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + s.ctas * 2 * 8 * s.nt * d->head_dim);
    p.cut = reinterpret_cast<int*>(p.part_ml + s.ctas * 2 * 8 * s.nt);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    auto go = [&](auto type, auto dim, auto nt) -> int {
      using T = decltype(type);
      constexpr int D = decltype(dim)::value, NT = decltype(nt)::value;
      auto kern = paged_attention_kernel<T, D, NT>;
      cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), PagedCfg<D, NT>::SMEM_BYTES);
      if (e == cudaSuccess) e = launch_ex(kern, dim3((unsigned)s.ctas), dim3(PAGED_THREADS), PagedCfg<D, NT>::SMEM_BYTES, st, 1, true, p);
      if (e == cudaSuccess && !p.whole) e = launch_ex(paged_join_kernel<T, D, NT>, dim3((unsigned)s.ctas, (std::min(8 * NT, s.rows) + PAGED_JOIN_ROWS<D> - 1) / PAGED_JOIN_ROWS<D>), dim3(PAGED_JOIN_THREADS), 0, st, 1, true, p);
      return launched(who, e);
    };
    auto with = [&](auto type, auto dim) -> int {
      return s.nt == 1 ? go(type, dim, std::integral_constant<int, 1>{}) : go(type, dim, std::integral_constant<int, 2>{});
    };
    auto by_dim = [&](auto type) -> int {
      return d->head_dim == 64 ? with(type, std::integral_constant<int, 64>{})
             : d->head_dim == 128 ? with(type, std::integral_constant<int, 128>{}) : with(type, std::integral_constant<int, 256>{});
    };
    return d->dtype == VLA_BF16 ? by_dim(bf16{}) : by_dim(__half{});
  });
}

int vla_op_prompt_attention(const vla_prompt_attn_desc* d, void* stream) {
  const char* who = "vla_op_prompt_attention";
  return guarded(who, [&]() -> int {
    if (!d) return refuse(VLA_ERR_STATE, "%s: null descriptor", who);
    if (d->n_seqs < 0 || d->tokens_q < 0 || d->tokens_k < 0 || d->heads < 1 || d->kv_heads < 1) return refuse(VLA_ERR_SHAPE, "%s: bad sizes", who);
    if (d->heads % d->kv_heads) return refuse(VLA_ERR_SHAPE, "%s: heads must be a multiple of kv_heads", who);
    if (d->heads / d->kv_heads > 128) return refuse(VLA_ERR_LIMIT, "%s: at most 128 query heads share a key/value head", who);
    if (d->head_dim < 8 || d->head_dim % 8 || d->head_dim > 256) return refuse(VLA_ERR_SHAPE, "%s: head_dim must be a multiple of 8 up to 256", who);
    if (d->dtype != VLA_BF16 && d->dtype != VLA_F16) return refuse(VLA_ERR_SHAPE, "%s: q, k and v must be bf16 or f16", who);
    if (!(d->scale > 0.f) || d->scale > 3e38f) return refuse(VLA_ERR_SHAPE, "%s: scale must be positive and finite", who);
    if (d->n_seqs == 0 || d->tokens_q == 0) return VLA_OK;
    if (!d->q || !d->o || !d->cu_q || !d->cu_k || (d->tokens_k && (!d->k || !d->v))) return refuse(VLA_ERR_STATE, "%s: null argument", who);
    if (!vectors(d->q, d->q_tok_stride, d->q_head_stride) || !vectors(d->k, d->k_tok_stride, d->k_head_stride) ||
        !vectors(d->v, d->v_tok_stride, d->v_head_stride) || !vectors(d->o, d->o_tok_stride, d->o_head_stride))
      return refuse(VLA_ERR_SHAPE, "%s: rows of q, k, v and o must start on 16 bytes", who);
    if (!get_encode_fn()) return refuse(VLA_ERR_CUDA, "%s: the CUDA driver that encodes tensor maps is not there", who);
    PromptAttnParams p;
    p.v = d->v; p.o = d->o; p.cu_q = d->cu_q; p.cu_k = d->cu_k;
    p.n_seqs = d->n_seqs; p.tokens_q = d->tokens_q; p.tokens_k = d->tokens_k;
    p.kv_heads = d->kv_heads; p.group = d->heads / d->kv_heads; p.dim = d->head_dim;
    p.tile_tokens = 128 / p.group;
    p.v_tok = d->v_tok_stride; p.v_head = d->v_head_stride; p.o_tok = d->o_tok_stride; p.o_head = d->o_head_stride;
    p.causal = d->causal ? 1 : 0;
    p.scale_log2e = d->scale * 1.4426950408889634f;
    const bool wide = d->head_dim > 128;
    // without keys the maps are never used: any valid tensor stands in
    const void* k = d->tokens_k ? d->k : d->q;
    const void* v = d->tokens_k ? d->v : d->q;
    const long long nk = std::max(d->tokens_k, 1), dim = d->head_dim;
    const CUtensorMapDataType type = d->dtype == VLA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    bool made = tensor_map(&p.tmQ, d->q, 2, type, {dim, p.group, d->kv_heads, d->tokens_q}, {d->q_head_stride, p.group * d->q_head_stride, d->q_tok_stride},
                         {64, p.group, 1, p.tile_tokens});
    made = made && tensor_map(&p.tmK, k, 2, type, {dim, d->kv_heads, nk}, {d->k_head_stride, d->k_tok_stride}, {64, 1, wide ? PromptCfg<true>::KEYS : PromptCfg<false>::KEYS});
    made = made && tensor_map(&p.tmV, v, 2, type, {dim, d->kv_heads, nk}, {d->v_head_stride, d->v_tok_stride}, {64, 1, 64});
    if (!made) return refuse(VLA_ERR_SHAPE, "%s: the strides of q, k or v cannot be described by a tensor map", who);
    const long long tiles = d->tokens_q / p.tile_tokens + d->n_seqs;     // at most one tile of each sequence is not full
    if (tiles * d->kv_heads > INT_TOP) return refuse(VLA_ERR_LIMIT, "%s: too many tiles", who);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    auto go = [&](auto kern, int smem) -> int {
      if (cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kern), smem); e != cudaSuccess) return launched(who, e);
      return launched(who, launch_ex(kern, dim3((unsigned)(tiles * d->kv_heads)), dim3(PromptCfg<false>::THREADS), smem, st, 1, true, p));
    };
    if (d->dtype == VLA_BF16)
      return wide ? go(prompt_attention_kernel<bf16, true>, PromptCfg<true>::SMEM_BYTES) : go(prompt_attention_kernel<bf16, false>, PromptCfg<false>::SMEM_BYTES);
    return wide ? go(prompt_attention_kernel<__half, true>, PromptCfg<true>::SMEM_BYTES) : go(prompt_attention_kernel<__half, false>, PromptCfg<false>::SMEM_BYTES);
  });
}

int vla_op_cache_status(int* out) {
  const char* who = "vla_op_cache_status";
  return guarded(who, [&]() -> int {
    if (!out) return refuse(VLA_ERR_STATE, "%s: null argument", who);
    static std::mutex mu;                  // one look at a time: each has its answer in the same place
    std::lock_guard<std::mutex> lock(mu);
    cudaError_t e = cudaDeviceSynchronize();             // streams that do not wait for the default one as well
    if (e == cudaSuccess) {
      cache_status_kernel<<<1, 1>>>();
      e = cudaGetLastError();
    }
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(out, cache_ops_taken, sizeof(int));
    return launched(who, e);
  });
}

int vla_op_cache_wait_expire(int limit_us, void* stream) {
  const char* who = "vla_op_cache_wait_expire";
  return guarded(who, [&]() -> int {
    if (limit_us < 1 || limit_us > 1000000) return refuse(VLA_ERR_LIMIT, "%s: the limit must be 1 to 1000000 microseconds", who);
    return launched(who, launch_ex(cache_wait_kernel, dim3(1), dim3(1), 0, reinterpret_cast<cudaStream_t>(stream), 1, false, limit_us * 1000ull));
  });
}

}  // extern "C"
