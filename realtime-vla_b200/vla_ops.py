"""Python callers of the single-operator C-ABI entry points (vla_op_*): kernel-level parity tests and
micro-benchmarks call the kernels through these.

The operators around a key/value cache in pages (block_plan, cache_append, paged_attention, prompt_attention) are for
programs that serve sequences of different lengths: they take torch tensors, enqueue on the current stream of the tensors'
device and return without synchronising, so they can be captured into a CUDA graph.  They run forward only."""
import ctypes as C
import functools
import struct
from typing import NamedTuple

import torch

import _capi


def _p(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def gemm(x, w, *, w2=None, bias=None, epi=0, act=0, res=None, gate=None, res_mod=0, split=0, bn=0, pair=0, tok_tile=0, iters=0,
         qkv=None):
    """x bf16 [tokens,K], w bf16 [K,N] (checkpoint layout). Returns the epilogue's output tensor(s)."""
    lib = _capi.lib()
    tokens, K = x.shape
    N = w.shape[1]
    d = _capi.GemmDesc()
    d.x, d.tokens, d.K, d.w, d.w2, d.N = _p(x), tokens, K, _p(w), _p(w2), N
    d.bias, d.epi, d.act = _p(bias), epi, act
    d.split, d.bn, d.iters, d.pair, d.tok_tile = split, bn, iters, pair, tok_tile
    ms = C.c_float(0)
    d.ms_per_iter = C.pointer(ms)
    out = None
    if epi == 0:
        out = torch.full((tokens, N), float("nan"), dtype=torch.bfloat16, device=x.device)
        d.out_bf16, d.ld_out = _p(out), N
    elif epi == 1:
        out = res.clone() if (res is not None and res_mod == 0) else torch.zeros(tokens, N, device=x.device)
        d.out_f32 = _p(out)
        d.res = _p(out) if (res is not None and res_mod == 0) else _p(res)
        d.gate, d.res_mod = _p(gate), res_mod
    else:
        q = torch.zeros(tokens, 2048, dtype=torch.bfloat16, device=x.device)
        rows = qkv["kv_rows"]
        kc = torch.zeros(rows, 256, dtype=torch.bfloat16, device=x.device)
        vc = torch.zeros(rows, 256, dtype=torch.bfloat16, device=x.device)
        vt_ld = (rows + 7) // 8 * 8
        vt = torch.zeros(256, vt_ld, dtype=torch.bfloat16, device=x.device)
        d.q, d.kcache, d.vcache, d.vt, d.vt_ld = _p(q), _p(kc), _p(vc), _p(vt), vt_ld
        d.pos_off, d.rows_per_obs = qkv["pos_off"], qkv["rows_per_obs"]
        d.kv_obs_stride, d.kv_row_off = qkv["kv_obs_stride"], qkv["kv_row_off"]
        out = (q, kc, vc, vt)
    rc = lib.vla_op_gemm(C.byref(d), None)
    _capi.check(rc)
    torch.cuda.synchronize()
    return (out, ms.value) if iters else out


def attention(q, k, v, *, ldq, ldk, ldv, ldo, o, groups_outer=1, groups_inner=1, strides=(0,) * 8, n_q, n_keys, head_dim,
              prefix_alloc=None, valid_prefix=None, restrict_rows=0, scale, ksplit=0, iters=0):
    lib = _capi.lib()
    d = _capi.AttnDesc()
    d.q, d.k, d.v, d.o = _p(q), _p(k), _p(v), _p(o)
    d.ldq, d.ldk, d.ldv, d.ldo = ldq, ldk, ldv, ldo
    d.groups_outer, d.groups_inner = groups_outer, groups_inner
    d.q_go, d.q_gi, d.k_go, d.k_gi, d.v_go, d.v_gi, d.o_go, d.o_gi = strides
    d.n_q, d.n_keys, d.head_dim = n_q, n_keys, head_dim
    d.prefix_alloc = n_keys if prefix_alloc is None else prefix_alloc
    d.valid_prefix = d.prefix_alloc if valid_prefix is None else valid_prefix
    d.restrict_rows, d.scale, d.ksplit, d.iters = restrict_rows, scale, ksplit, iters
    ms = C.c_float(0)
    d.ms_per_iter = C.pointer(ms)
    _capi.check(lib.vla_op_attention(C.byref(d), None))
    torch.cuda.synchronize()
    return ms.value


def attention_tc(q, k, v, *, n_keys=None, prefix_alloc=None, valid_prefix=None, restrict_rows=0, scale, ksplit=0, iters=0):
    """tcgen05 attention: q [n_q,256], k/v [k_rows,256] bf16 (v is transposed here into the layout the kernel reads)."""
    lib = _capi.lib()
    n_q, k_rows = q.shape[0], k.shape[0]
    n_keys = k_rows if n_keys is None else n_keys
    vt_ld = (k_rows + 7) // 8 * 8
    vt = torch.zeros(256, vt_ld, dtype=torch.bfloat16, device=q.device)
    vt[:, :k_rows] = v.t()
    o = torch.zeros(n_q, 256, dtype=torch.bfloat16, device=q.device)
    d = _capi.AttnTcDesc()
    d.q, d.k, d.vt, d.o = _p(q), _p(k), _p(vt), _p(o)
    d.n_q, d.n_keys, d.k_rows, d.vt_ld = n_q, n_keys, k_rows, vt_ld
    d.prefix_alloc = n_keys if prefix_alloc is None else prefix_alloc
    d.valid_prefix = d.prefix_alloc if valid_prefix is None else valid_prefix
    d.restrict_rows, d.scale, d.ksplit, d.iters = restrict_rows, scale, ksplit, iters
    ms = C.c_float(0)
    d.ms_per_iter = C.pointer(ms)
    _capi.check(lib.vla_op_attention_tc(C.byref(d), None))
    torch.cuda.synchronize()
    return (o, ms.value) if iters else o


def norm(x, mode, w=None, b=None):
    lib = _capi.lib()
    rows, D = x.shape
    y = torch.empty(rows, D, dtype=torch.bfloat16, device=x.device)
    _capi.check(lib.vla_op_norm(_p(x), _p(y), rows, D, mode, _p(w), _p(b), None))
    return y


def vit_attention_tc(qkv, *, scale, iters=0):
    """SigLIP attention on tcgen05: qkv bf16 [views*256, 3456] -> bf16 [views*256, 1152]."""
    lib = _capi.lib()
    views = qkv.shape[0] // 256
    out = torch.full((views * 256, 1152), float("nan"), dtype=torch.bfloat16, device=qkv.device)
    ms = C.c_float(0)
    stream = torch.cuda.current_stream(qkv.device).cuda_stream
    _capi.check(lib.vla_op_vit_attention_tc(_p(qkv), _p(out), views, float(scale), iters, C.byref(ms), C.c_void_p(stream)))
    return (out, ms.value) if iters else out


# ---- a key/value cache in pages, held in 8 bits -----------------------------------------------------------------------
_PLAN, _APPEND = _capi.packer(_capi.BlockPlanDesc), _capi.packer(_capi.CacheAppendDesc)
_PAGED, _PROMPT = _capi.packer(_capi.PagedAttnDesc), _capi.packer(_capi.PromptAttnDesc)
_DTYPES = {torch.bfloat16: _capi.VLA_BF16, torch.float16: _capi.VLA_F16}


class KvCache(NamedTuple):
    """Pages of tokens as e4m3 codes with one scale for each page and head; a value is code * scale."""
    k: torch.Tensor          # float8_e4m3fn [blocks, kv_heads, block_size, head_dim]
    v: torch.Tensor
    k_scale: torch.Tensor    # float32 [blocks, kv_heads]
    v_scale: torch.Tensor


class BlockPlan(NamedTuple):
    slots: torch.Tensor       # int32 [total_new]: block * block_size + offset of each new token, -1: none
    positions: torch.Tensor   # int32 [total_new]: position in its sequence
    cu_new: torch.Tensor      # int32 [n + 1]: first row of each request
    seq_lens: torch.Tensor    # int32 [n]: tokens of each request that have a slot
    counts: torch.Tensor      # int32 [3]: next free index, blocks missing, sum of new tokens


def kv_cache(blocks, kv_heads, block_size, head_dim, device=None):
    """An empty cache (all pages zero)."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    codes = [torch.zeros(blocks, kv_heads, block_size, head_dim, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
             for _ in range(2)]
    scales = [torch.zeros(blocks, kv_heads, device=device) for _ in range(2)]
    return KvCache(*codes, *scales)


# The checks below run on every call of operators that take a few microseconds, so messages are formed only on refusal.
def _refuse(text, *args):
    raise _capi.VlaError("vla_ops: " + text % args)


def _tell(t):
    return "%s %s on %s" % (t.dtype, tuple(t.shape), t.device)


def _on_gpu(t, name):
    if not t.is_cuda:
        _refuse("%s must be on a GPU; there is no CPU path", name)
    return t.device


def _whole(t, name, device, dim=1):
    """Address of an int32 tensor of `dim` dimensions on `device` with contiguous rows."""
    if t.dtype is not torch.int32 or t.dim() != dim or t.device != device or (t.stride(-1) != 1 and t.shape[-1] > 1):
        _refuse("%s must be int32 with %d dimension(s), contiguous rows, on %s; got %s", name, dim, device, _tell(t))
    return t.data_ptr()


def _rows(t, name, device, dtype, dim):
    """Address of a 16-bit tensor of `dim` dimensions on `device` whose last one is contiguous."""
    if t.dtype is not dtype or t.dim() != dim or t.device != device or (t.stride(-1) != 1 and t.shape[-1] > 1):
        _refuse("%s must be %s with %d dimensions, the last one contiguous, on %s; got %s", name, dtype, dim, device, _tell(t))
    if t.requires_grad and torch.is_grad_enabled():
        _refuse("%s requires a gradient; this operator has no backward pass", name)
    return t.data_ptr()


def _cache(cache, device):
    """Addresses of the four tensors of a cache."""
    k, v, ks, vs = cache
    shape, f8, f32 = k.shape, torch.float8_e4m3fn, torch.float32
    if not (k.dtype is f8 and v.dtype is f8 and ks.dtype is f32 and vs.dtype is f32 and len(shape) == 4 and v.shape == shape
            and ks.shape == shape[:2] and vs.shape == shape[:2] and k.device == device and v.device == device
            and ks.device == device and vs.device == device and k.is_contiguous() and v.is_contiguous()
            and ks.is_contiguous() and vs.is_contiguous()):
        _refuse("a cache is float8_e4m3fn codes [blocks, kv_heads, block_size, head_dim] twice and float32 scales [blocks, kv_heads] "
                "twice, all contiguous and on %s; got %s, %s, %s, %s", device, *map(_tell, cache))
    return k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr()


def _type(t, name):
    code = _DTYPES.get(t.dtype)
    if code is None:
        _refuse("%s must be bfloat16 or float16, got %s", name, t.dtype)
    return code


def _enqueue(fn, pack, device, *fields):
    try:
        desc = pack(*fields)
    except (struct.error, OverflowError) as e:
        _refuse("a size is too large (%s)", e)
    stream = torch._C._cuda_getCurrentRawStream(device.index)      # current_stream(device).cuda_stream in 0.1 instead of 2.2 us
    if torch._C._cuda_getDevice() == device.index:
        rc = fn(desc, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(desc, stream)
    if rc:
        _capi.check(rc)


def block_plan(context_lens, new_lens, block_table, free_blocks, *, block_size, total_new, first_free=None):
    """Pages and slots for the new tokens of every request, from the lengths alone, on the device.

    context_lens, new_lens int32 [n]; block_table int32 [n, width], updated in place with the blocks each request gets;
    free_blocks int32 [f], taken in order from index first_free (int32 [1] on the device, e.g. counts[:1] of the call
    before; None: 0).  total_new is the number of rows of slots and positions (the sum of new_lens, or more for a padded
    batch).  Returns a BlockPlan; counts[1] > 0 says that blocks were missing and some tokens have slot -1."""
    dev = _on_gpu(context_lens, "context_lens")
    n = context_lens.shape[0]
    if new_lens.shape[0] != n or block_table.shape[0] != n or (first_free is not None and first_free.numel() != 1):
        _refuse("context_lens, new_lens, block_table (and first_free) do not fit each other")
    if total_new < 0:
        _refuse("total_new is negative")
    pad = -total_new % 4                   # one allocation, of which slots and positions start on 16 bytes
    out = context_lens.new_empty(2 * (total_new + pad) + 2 * n + 4)
    if pad:
        slots, _, positions, _, cu, lens, counts = out.split_with_sizes([total_new, pad, total_new, pad, n + 1, n, 3])
    else:
        slots, positions, cu, lens, counts = out.split_with_sizes([total_new, total_new, n + 1, n, 3])
    _enqueue(_capi.lib().vla_op_block_plan, _PLAN, dev,
             _whole(context_lens, "context_lens", dev), _whole(new_lens, "new_lens", dev), n, _whole(block_table, "block_table", dev, 2), block_table.shape[1],
             block_table.stride(0) if n > 1 else block_table.shape[1],
             _whole(free_blocks, "free_blocks", dev), free_blocks.shape[0],
             0 if first_free is None else _whole(first_free, "first_free", dev), block_size, total_new,
             slots.data_ptr(), positions.data_ptr(), cu.data_ptr(), lens.data_ptr(), counts.data_ptr())
    return BlockPlan(slots, positions, cu, lens, counts)


def cache_append(k, v, cache, slots):
    """Keys and values (bf16 or fp16 [tokens, kv_heads, head_dim]) into the cache at slots (int32 [tokens]), in place.

    Slots outside the cache are skipped; the tokens of one block must be consecutive rows.  A block whose first slot is written
    starts anew; another block's scale grows where the new tokens need it and its codes are rounded again."""
    dev = _on_gpu(k, "k")
    code = _type(k, "k")
    codes = _cache(cache, dev)
    blocks, heads, block, dim = cache.k.shape
    pk, pv = _rows(k, "k", dev, k.dtype, 3), _rows(v, "v", dev, k.dtype, 3)
    if k.shape != v.shape or k.shape[1:] != (heads, dim) or slots.shape[0] != k.shape[0]:
        _refuse("k %s, v %s and slots %s do not fit the cache %s", *(tuple(x.shape) for x in (k, v, slots, cache.k)))
    _enqueue(_capi.lib().vla_op_cache_append, _APPEND, dev, pk, pv, _whole(slots, "slots", dev), k.shape[0],
             *k.stride()[:2], *v.stride()[:2], *codes, blocks, heads, block, dim, code)


@functools.lru_cache(maxsize=1024)
def _paged_workspace(device, *sizes):
    """Bytes of workspace, which follow from the sizes (and the device's number of SMs)."""
    d, need = _capi.PagedAttnDesc(), C.c_size_t()
    d.n_seqs, d.n_q, d.heads, d.kv_heads, d.head_dim, d.num_blocks, d.block_size, d.width = sizes
    d.table_stride, d.scale = d.width, 1.0
    with torch.cuda.device(device):
        _capi.check(_capi.lib().vla_op_paged_attention_workspace(C.byref(d), C.byref(need)))
    return need.value


def paged_attention(q, cache, block_table, seq_lens, *, scale=None, out=None):
    """Attention of the newest tokens of every sequence over the cache.

    q bf16 or fp16 [n, tokens, heads, head_dim]: the last tokens of each sequence, whose keys are in the cache already;
    each sees itself and what is before it.  block_table int32 [n, width], seq_lens int32 [n].  scale: head_dim ** -0.5
    unless given.  Returns out, or a new tensor like q; a row that sees nothing is zero."""
    dev = _on_gpu(q, "q")
    code = _type(q, "q")
    codes = _cache(cache, dev)
    blocks, kv_heads, block, dim = cache.k.shape
    pq = _rows(q, "q", dev, q.dtype, 4)
    n, tokens, heads, _ = q.shape
    if q.shape[3] != dim or block_table.shape[0] != n or seq_lens.shape[0] != n:
        _refuse("q %s, block_table %s, seq_lens %s and cache %s do not fit each other",
                *(tuple(x.shape) for x in (q, block_table, seq_lens, cache.k)))
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape:
        _refuse("out must have the shape of q")
    table = _whole(block_table, "block_table", dev, 2)
    width = block_table.shape[1]
    need = _paged_workspace(dev, n, tokens, heads, kv_heads, dim, blocks, block, width)
    # the workspace is this call's own; the allocator orders its reuse on the stream
    space = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _enqueue(_capi.lib().vla_op_paged_attention, _PAGED, dev, pq, _rows(out, "out", dev, q.dtype, 4), *q.stride()[:3], *out.stride()[:3],
             *codes, table, block_table.stride(0) if n > 1 else width, _whole(seq_lens, "seq_lens", dev),
             n, tokens, heads, kv_heads, dim, blocks, block, width, dim ** -0.5 if scale is None else scale, code,
             space.data_ptr() if need else 0, need)
    return out


def prompt_attention(q, k, v, cu_q, cu_k=None, *, causal=True, scale=None, out=None):
    """Attention over packed prompts of different lengths.

    q bf16 or fp16 [tokens, heads, head_dim], k and v [keys, kv_heads, head_dim]; sequence b owns rows cu_q[b] .. cu_q[b + 1] of
    q and cu_k[b] .. cu_k[b + 1] of k and v (int32 [n + 1] on the device, ascending; cu_k: as cu_q unless given).  causal: the last row
    of a sequence sees all its keys, each row before it one less; otherwise every row sees all.  Returns out, or a new
    tensor like q; a row that sees nothing is zero, rows behind the last sequence are not written."""
    dev = _on_gpu(q, "q")
    code = _type(q, "q")
    if cu_k is None:
        cu_k = cu_q
    t = q.dtype
    pq, pk, pv = _rows(q, "q", dev, t, 3), _rows(k, "k", dev, t, 3), _rows(v, "v", dev, t, 3)
    tokens, heads, dim = q.shape
    if k.shape != v.shape or k.shape[2] != dim or cu_q.shape != cu_k.shape or cu_q.shape[0] < 1:
        _refuse("q %s, k %s, v %s, cu_q %s and cu_k %s do not fit each other", *(tuple(x.shape) for x in (q, k, v, cu_q, cu_k)))
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape:
        _refuse("out must have the shape of q")
    _enqueue(_capi.lib().vla_op_prompt_attention, _PROMPT, dev, pq, pk, pv, _rows(out, "out", dev, t, 3),
             _whole(cu_q, "cu_q", dev), _whole(cu_k, "cu_k", dev), cu_q.shape[0] - 1, tokens, k.shape[0], heads, k.shape[1], dim,
             *q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *out.stride()[:2],
             1 if causal else 0, dim ** -0.5 if scale is None else scale, code)
    return out
