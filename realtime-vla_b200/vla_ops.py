"""Python callers of the single-operator C-ABI entry points (vla_op_*): kernel-level parity tests and
micro-benchmarks call the kernels through these.

The operators around a key/value cache in pages (block_plan, cache_append, paged_attention, prompt_attention) are for
programs that serve sequences of different lengths: they take torch tensors, enqueue on the current stream of the tensors'
device and return without synchronising, so they can be captured into a CUDA graph.  They run forward only.  Waits inside their
kernels are bounded; cache_status() says whether one ran out."""
import ctypes as C
from typing import NamedTuple

import torch

import _capi

try:
    import _vla_ops as _native          # csrc/binding.cpp
except ImportError as _e:               # not built, or for another torch or Python: the callers through ctypes do without it
    class _NotBuilt:
        def __init__(self, why):
            self._why = why

        def __getattr__(self, name):
            raise _capi.VlaError("vla_ops: %s needs the built library (python realtime-vla_b200/build.py); there is no CPU path (%s)" % (name, self._why))

    _native = _NotBuilt(str(_e))


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


def block_plan(context_lens, new_lens, block_table, free_blocks, *, block_size, total_new, first_free=None):
    """Pages and slots for the new tokens of every request, from the lengths alone, on the device.

    context_lens, new_lens int32 [n]; block_table int32 [n, width], updated in place with the blocks each request gets;
    free_blocks int32 [f], taken in order from index first_free (int32 [1] on the device, e.g. counts[:1] of the call
    before; None: 0).  total_new is the number of rows of slots and positions (the sum of new_lens, or more for a padded
    batch).  Returns a BlockPlan; counts[1] > 0 says that blocks were missing and some tokens have slot -1."""
    return BlockPlan(*_native.block_plan(context_lens, new_lens, block_table, free_blocks, block_size, total_new, first_free))


def cache_append(k, v, cache, slots):
    """Keys and values (bf16 or fp16 [tokens, kv_heads, head_dim]) into the cache at slots (int32 [tokens]), in place.

    Slots outside the cache are skipped; the tokens of one block must be consecutive rows, with no other or skipped row between
    them (what such a block holds afterwards is not defined).  A block whose first slot is written starts anew; another
    block's scale grows where the new tokens need it and its codes are rounded again."""
    _native.cache_append(k, v, cache, slots)


def paged_attention(q, cache, block_table, seq_lens, *, scale=None, out=None):
    """Attention of the newest tokens of every sequence over the cache.

    q bf16 or fp16 [n, tokens, heads, head_dim]: the last tokens of each sequence, whose keys are in the cache already;
    each sees itself and what is before it.  Fewer new tokens than that: they stand at the end of the row.  block_table int32 [n, width], seq_lens int32 [n].  scale: head_dim ** -0.5
    unless given.  Returns out (which may be q), or a new tensor like q; a row that sees nothing is zero."""
    return _native.paged_attention(q, cache, block_table, seq_lens, scale, out)


def prompt_attention(q, k, v, cu_q, cu_k=None, *, causal=True, scale=None, out=None):
    """Attention over packed prompts of different lengths.  It sees k and v alone: tokens behind a cached context take paged_attention.

    q bf16 or fp16 [tokens, heads, head_dim], k and v [keys, kv_heads, head_dim]; sequence b owns rows cu_q[b] .. cu_q[b + 1] of
    q and cu_k[b] .. cu_k[b + 1] of k and v (int32 [n + 1] on the device, ascending; cu_k: as cu_q unless given).  causal: the last row
    of a sequence sees all its keys, each row before it one less; otherwise every row sees all.  Returns out (which may be q
    but must not overlap k or v), or a new tensor like q; a row that sees nothing is zero, rows behind the last sequence are not written."""
    return _native.prompt_attention(q, k, v, cu_q, cu_k, causal, scale, out)


def cache_status(device=None):
    """Whether the operators around the cache have run to their end on a device since the last call of this: 0, or bit 0 set where a
    bounded wait inside a kernel ran out and the output of some call is not to be trusted.  Waits for all work on the device;
    a serving loop calls it where it waits anyway, and not while a stream is captured."""
    word = C.c_int(0)
    with torch.cuda.device(device):
        _capi.check(_capi.lib().vla_op_cache_status(C.byref(word)))
    return word.value
