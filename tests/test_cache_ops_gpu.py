"""The operators around a key/value cache in pages, on a B200, against their definitions in 64 bits: block tables and slot
maps, the cache writer, attention over the cache, attention over packed prompts, and a serving loop of all four.

Whole numbers, scales and e4m3 codes have to be equal (scales are powers of two, so every quotient is exact and each
code is rounded once).  Attention is held to what its roundings can do, with A = sum_j p_j |v_j| / sum_j p_j:
  * probabilities rounded to the operands' 16-bit type t move the result by at most half(t) * A;
  * a probability below fp16's normal range (2^-14) is off by up to 2^-25 of the row's largest, n keys by n * 2^-25 * max|v|;
  * fp32 scores are off by at most (dim + 8) 2^-24 scale sum|q||k| each, which moves probabilities by that relatively and,
    numerator and denominator together, the result by twice that times A;
  * exponentials and sums in fp32: 2^-20 * A covers them for these lengths (sums of n terms in blocks: a few 2^-24 each);
  * the output's own rounding is half(t) * |o|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda")


def half(t):
    return torch.finfo(t).eps / 2


def starts(lens, d):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(d)


# ---- attention over packed prompts --------------------------------------------------------------------------------------

def attend(q, k, v, limit, scale):
    """q [n, heads, dim], k, v [m, kv, dim] -> (o, bound) in 64 bits; row i sees keys j < limit[i] (or a mask [n, m])."""
    n, heads, dim = q.shape
    kv = k.shape[1]
    t = q.dtype
    qd = q.double().reshape(n, kv, heads // kv, dim)
    kd, vd = k.double(), v.double()
    vis = limit if limit.dim() == 2 else torch.arange(k.shape[0], device=q.device)[None] < limit[:, None]
    kd = torch.where(vis.any(0)[:, None, None], kd, 0.0)          # what no row sees may hold anything
    s = torch.einsum("nhgd,mhd->hgnm", qd, kd) * scale
    mag = torch.einsum("nhgd,mhd->hgnm", qd.abs(), kd.abs()) * scale
    s = s.masked_fill(~vis, float("-inf"))
    top = s.amax(-1, keepdim=True) if k.shape[0] else torch.zeros(*s.shape[:3], 1, device=q.device, dtype=s.dtype)
    p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, 1.0, l)
    # masked values contribute nothing whatever they hold
    fine = torch.isfinite(vd)
    o = torch.einsum("hgnm,mhd->nhgd", p, torch.where(fine, vd, 0.0))
    poison = torch.einsum("hgnm,mhd->nhgd", (p > 0).double(), (~fine).double()) > 0
    vabs = torch.where(fine, vd.abs(), 0.0)
    a = torch.einsum("hgnm,mhd->nhgd", p, vabs)
    ds = (dim + 8) * 2.0 ** -24 * torch.where(vis, mag, 0.0).amax(-1) if k.shape[0] else torch.zeros_like(l[..., 0])
    ds = ds.permute(2, 0, 1)[..., None]
    vmax = vabs.amax() if k.shape[0] else 0.0
    bound = a * (half(t) + 2 * ds + 2.0 ** -20) + half(t) * o.abs() + k.shape[0] * 2.0 ** -25 * vmax
    # outputs below fp16's normal range are rounded to its smallest step
    bound = bound + (2.0 ** -25 if t == torch.float16 else 0.0)
    o = torch.where(poison, float("nan"), o)
    return o.reshape(n, heads, dim), bound.reshape(n, heads, dim)


def held(got, want, bound, what=""):
    got = got.double()
    bad = torch.isnan(want)
    assert not torch.isfinite(got[bad]).any(), what + ": a visible non-finite value vanished"
    got, want, bound = got[~bad], want[~bad], bound[~bad]
    assert torch.isfinite(got).all(), what + ": non-finite output"
    off = ((got - want).abs() - bound)
    assert (off <= 0).all(), "%s: %g beyond the bound %g" % (what, off.max().item(), bound.flatten()[off.argmax()].item())


def check_prompts(q, k, v, cu_q, cu_k, out, causal, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    a, b = cu_q.tolist(), cu_k.tolist()
    for i in range(len(a) - 1):
        n, m = a[i + 1] - a[i], b[i + 1] - b[i]
        if not n:
            continue
        rows = torch.arange(n, device=q.device)
        limit = (rows + m - n + 1).clamp(0, m) if causal else torch.full_like(rows, m)
        want, bound = attend(q[a[i]:a[i + 1]], k[b[i]:b[i + 1]], v[b[i]:b[i + 1]], limit, scale)
        held(out[a[i]:a[i + 1]], want, bound, "sequence %d (%d rows, %d keys)" % (i, n, m))


def prompts(seed, lens_q, lens_k, heads, kv, dim, t, d, spread=1.0):
    g = torch.Generator(device=d).manual_seed(seed)
    mk = lambda *s: (torch.randn(*s, generator=g, device=d) * spread).to(t)      # noqa: E731
    return mk(sum(lens_q), heads, dim), mk(sum(lens_k), kv, dim), mk(sum(lens_k), kv, dim), starts(lens_q, d), starts(lens_k, d)


LENS = [(1,), (20,), (0, 1, 0, 17, 0), (127, 128, 129), (16, 15, 33, 2), (255, 1, 300), (641,)]


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 256), (4, 2, 128), (16, 16, 72), (8, 2, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_lengths(lens, heads, kv, dim, causal):
    import vla_ops
    d = dev()
    q, k, v, cu, _ = prompts(1, lens, lens, heads, kv, dim, torch.bfloat16, d)
    check_prompts(q, k, v, cu, cu, vla_ops.prompt_attention(q, k, v, cu, causal=causal), causal)


@pytest.mark.parametrize("heads,kv,dim", [(7, 1, 128), (3, 3, 8), (6, 2, 96), (5, 1, 200), (128, 1, 64), (28, 4, 128), (2, 1, 136),
                                          (9, 9, 256), (40, 2, 24), (100, 1, 40)])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_prompt_heads_and_types(heads, kv, dim, t):
    import vla_ops
    d = dev()
    q, k, v, cq, ck = prompts(2, (37, 150, 4), (37, 190, 300), heads, kv, dim, t, d)
    check_prompts(q, k, v, cq, ck, vla_ops.prompt_attention(q, k, v, cq, ck), True)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens_q,lens_k", [((5, 140, 3), (300, 140, 0)), ((60, 200), (10, 131)), ((130, 1, 7), (2, 0, 129)),
                                           ((1, 1, 1, 1), (128, 129, 256, 1000))])
def test_prompt_keys_unlike_queries(dim, lens_q, lens_k):
    """More keys than queries (a context stands before), fewer (rows that see nothing), none."""
    import vla_ops
    d = dev()
    q, k, v, cq, ck = prompts(3, lens_q, lens_k, 8, 2, dim, torch.bfloat16, d)
    for causal in (True, False):
        check_prompts(q, k, v, cq, ck, vla_ops.prompt_attention(q, k, v, cq, ck, causal=causal), causal)


@pytest.mark.parametrize("heads,kv,dim", [(16, 8, 128), (8, 8, 64), (8, 4, 256)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_many_sequences(heads, kv, dim, causal):
    """Far more tiles than SMs: every CTA takes many, of one chunk and of several, with one live tile and with two."""
    import vla_ops
    d = dev()
    lens = [(37 * i) % 61 for i in range(300)] + [700, 1, 260]
    keys = [n + (i % 5) * 70 for i, n in enumerate(lens)]
    q, k, v, cq, ck = prompts(7, lens, keys, heads, kv, dim, torch.bfloat16, d)
    for _ in range(3):
        out = vla_ops.prompt_attention(q, k, v, cq, ck, causal=causal)
    check_prompts(q, k, v, cq, ck, out, causal)


@pytest.mark.parametrize("spread", [0.05, 6.0])
@pytest.mark.parametrize("dim", [64, 256])
def test_prompt_flat_and_sharp_rows(spread, dim):
    """Rows whose maximum hardly moves and rows whose maximum keeps growing along the keys; a scale of its own."""
    import vla_ops
    d = dev()
    q, k, v, cu, _ = prompts(4, (520, 300), (520, 300), 8, 1, dim, torch.bfloat16, d, spread)
    ramp = torch.linspace(0.1, 3.0, 820, device=d)[:, None, None]
    k = (k.float() * ramp).to(torch.bfloat16)
    out = vla_ops.prompt_attention(q, k, v, cu, scale=0.11)
    check_prompts(q, k, v, cu, cu, out, True, 0.11)


@pytest.mark.parametrize("dim", [72, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_unseen_rows_may_hold_anything(dim, causal):
    """NaN and infinities behind the last sequence, in a neighbour, and in later tokens do not reach a row; rows of out
    behind the last sequence stay."""
    import vla_ops
    d = dev()
    lens = (50, 131, 9)
    q, k, v, cu, _ = prompts(5, lens + (40,), lens + (40,), 8, 2, dim, torch.bfloat16, d)
    cu = cu[:-1].contiguous()
    q[190:], k[190:], v[190:] = float("nan"), float("nan"), float("inf")
    k[181:190], v[181:190] = float("nan"), float("nan")           # the third sequence is not well: its own rows only
    v[49, 0, 3], k[49, 1] = float("inf"), float("inf")           # the first sequence's last token, and the second's middle
    v[120, 1, 0], v[119, 0, dim - 1] = float("nan"), float("-inf")
    out = torch.full_like(q, 7.0)
    got = vla_ops.prompt_attention(q, k, v, cu, causal=causal, out=out)
    assert got is out and (out[190:] == 7.0).all()
    assert torch.isnan(out[181:190].double()).all()
    if causal:
        check_prompts(q[:49], k[:49], v[:49], starts((49,), d), starts((49,), d), out[:49], True)
        n = 120 - 50
        check_prompts(q[50:50 + n], k[50:50 + n], v[50:50 + n], starts((n,), d), starts((n,), d), out[50:50 + n], True)
    else:
        assert torch.isfinite(out[50:181, :4, :dim - 1].double()).all()      # the second sequence's first key/value head
        assert not torch.isfinite(out[50:181, :4, dim - 1].double()).any()


def test_prompt_strided_and_fused():
    """q, k and v as slices of one projection's output, out as a slice of a wider tensor."""
    import vla_ops
    d = dev()
    g = torch.Generator(device=d).manual_seed(6)
    heads, kv, dim, lens = 8, 2, 128, (70, 200)
    x = torch.randn(270, (heads + 2 * kv) * dim + 64, generator=g, device=d).to(torch.bfloat16)
    q = x[:, :heads * dim].unflatten(1, (heads, dim))
    k = x[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim))
    v = x[:, (heads + kv) * dim:(heads + 2 * kv) * dim].unflatten(1, (kv, dim))
    wide = torch.zeros(270, 3, heads, dim, dtype=torch.bfloat16, device=d)
    cu = starts(lens, d)
    vla_ops.prompt_attention(q, k, v, cu, out=wide[:, 1])
    check_prompts(q, k, v, cu, cu, wide[:, 1], True)
    assert (wide[:, 0] == 0).all() and (wide[:, 2] == 0).all()
    # heads before tokens
    qt, kt, vt = (y.transpose(0, 1).contiguous().transpose(0, 1) for y in (q, k, v))
    check_prompts(q, k, v, cu, cu, vla_ops.prompt_attention(qt, kt, vt, cu), True)


# ---- the cache ------------------------------------------------------------------------------------------------------------

def e4m3(x):
    """Nearest e4m3 value in 64 bits, ties to even, saturating, NaN stays."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(2.0 ** -6, 448.0))) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def need_scale(amax):
    e = -60
    while 448.0 * 2.0 ** e < amax:
        e += 1
    return 2.0 ** e


def write(x, codes, scale, slots):
    """The writer's definition, block by block, in 64 bits on the host -> (codes, scale)."""
    blocks, heads, block, _ = codes.shape
    codes, scale, x = codes.double().cpu(), scale.double().cpu(), x.double().cpu()
    at = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < blocks * block:
            at.setdefault(s // block, []).append((t, s % block))
    for b, toks in at.items():
        for h in range(heads):
            rows = x[[t for t, _ in toks], h]
            need = need_scale(torch.where(torch.isfinite(rows), rows.abs(), 0.0).max().item())
            if any(o == 0 for _, o in toks):
                scale[b, h] = need
            elif need > scale[b, h]:
                codes[b, h] = e4m3(codes[b, h] * (scale[b, h] / need))
                scale[b, h] = need
            for t, o in toks:
                codes[b, h, o] = e4m3(x[t, h] / scale[b, h])
    return codes, scale


def random_cache(seed, blocks, heads, block, dim, d):
    import vla_ops
    g = torch.Generator(device=d).manual_seed(seed)
    codes = [(torch.randn(blocks, heads, block, dim, generator=g, device=d) * 100).clamp(-448, 448).to(F8) for _ in range(2)]
    scales = [torch.exp2(torch.randint(-9, -5, (blocks, heads), generator=g, device=d).float()) for _ in range(2)]
    return vla_ops.KvCache(*codes, *scales)


def clone(c):
    return type(c)(*(x.clone() for x in c))


def equal_codes(got, want):
    got = got.double().cpu()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    assert same.all(), "%d codes differ" % int((~same).sum())


def check_append(k, v, cache, slots):
    import vla_ops
    old = clone(cache)
    vla_ops.cache_append(k, v, cache, slots)
    for x, c, s, c0, s0 in ((k, cache.k, cache.k_scale, old.k, old.k_scale), (v, cache.v, cache.v_scale, old.v, old.v_scale)):
        codes, scale = write(x, c0, s0, slots)
        assert torch.equal(s.double().cpu(), scale)
        equal_codes(c, codes)


@pytest.mark.parametrize("heads,dim,block", [(1, 256, 16), (2, 128, 64), (3, 64, 48), (8, 128, 16), (1, 64, 256)])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_append(heads, dim, block, t):
    """Runs that start a block, sit inside one, fill several and part of a last; sizes that make scales grow and not."""
    d = dev()
    cache = random_cache(11, 12, heads, block, dim, d)
    g = torch.Generator(device=d).manual_seed(12)
    slots = list(range(3 * block + 5, 3 * block + 6)) + list(range(7 * block + block - 2, 8 * block + 3))
    slots += list(range(0, 2 * block + 1)) + [10 * block] + [11 * block + block - 1]
    n = len(slots)
    size = torch.exp2(torch.randint(-12, 9, (n, heads, 1), generator=g, device=d).float())
    k = (torch.randn(n, heads, dim, generator=g, device=d) * size).to(t)
    v = (torch.randn(n, heads, dim, generator=g, device=d) * size.flip(0)).to(t)
    check_append(k, v, cache, torch.tensor(slots, dtype=torch.int32, device=d))


@pytest.mark.parametrize("tokens", [1, 4097, 5000])
def test_append_many_rows(tokens):
    """Both sides of the rule that gives a CTA one token row or a window of them."""
    d = dev()
    block = 16
    blocks = tokens // block + 3
    cache = random_cache(13, blocks, 2, block, 64, d)
    g = torch.Generator(device=d).manual_seed(14)
    order = torch.randperm(blocks - 1, generator=torch.Generator().manual_seed(1)).tolist()
    slots = [order[(5 + i) // block] * block + (5 + i) % block for i in range(tokens)]
    k = torch.randn(tokens, 2, 64, generator=g, device=d).to(torch.bfloat16)
    check_append(k, k * 3, cache, torch.tensor(slots, dtype=torch.int32, device=d))


def test_append_skips_and_odd_values():
    """Slots outside the cache, zero rows, subnormal and huge values, NaN and infinities, a slot named twice, strides."""
    d = dev()
    heads, dim, block = 2, 128, 16
    cache = random_cache(15, 6, heads, block, dim, d)
    slots = [-1, 6 * 16, 2 ** 31 - 1, 0, 1, 2, 33, 33, 34, -5, 80, 81, 82, 50]
    n = len(slots)
    x = torch.randn(n, 3 * heads, dim, device=d, generator=torch.Generator(device=d).manual_seed(16)).to(torch.bfloat16)
    x[3] = 0
    x[4, :, 5], x[5, :, 6], x[5, :, 7] = float("nan"), float("inf"), float("-inf")
    x[10], x[11, :, 0] = x[10] * 1e-30, 3e38
    x[13] *= 1e-38
    k, v = x[:, :heads], x[:, heads:2 * heads]
    check_append(k, v, cache, torch.tensor(slots, dtype=torch.int32, device=d))
    # a block of zeros alone has the smallest scale, and the next token raises it
    import vla_ops
    cache = vla_ops.kv_cache(2, 1, 16, 64, d)
    z = torch.zeros(1, 1, 64, dtype=torch.float16, device=d)
    check_append(z, z, cache, torch.tensor([16], dtype=torch.int32, device=d))
    assert cache.k_scale[1, 0].item() == 2.0 ** -60
    check_append(z + 3, z - 5, cache, torch.tensor([17], dtype=torch.int32, device=d))


def test_append_one_by_one_is_append_at_once():
    """Scales are powers of two: growing them on the way changes only what falls below e4m3's normal range."""
    import vla_ops
    d = dev()
    g = torch.Generator(device=d).manual_seed(17)
    k = (torch.randn(16, 1, 64, generator=g, device=d).abs() + 0.5).to(torch.bfloat16) * torch.arange(1, 17, device=d)[:, None, None]
    whole, step = vla_ops.kv_cache(1, 1, 16, 64, d), vla_ops.kv_cache(1, 1, 16, 64, d)
    slots = torch.arange(16, dtype=torch.int32, device=d)
    vla_ops.cache_append(k, -k, whole, slots)
    for i in range(16):
        vla_ops.cache_append(k[i:i + 1], -k[i:i + 1], step, slots[i:i + 1])
    for a, b in zip(whole, step):
        assert torch.equal(a.float(), b.float())


def check_paged(q, cache, table, lens, out, scale=None):
    scale = q.shape[3] ** -0.5 if scale is None else scale
    blocks, kv, block, dim = cache.k.shape
    n = q.shape[1]
    for b, m in enumerate(lens.tolist()):
        m = max(0, min(m, table.shape[1] * block))
        ids = table[b, :(m + block - 1) // block].long()
        good = (ids >= 0) & (ids < blocks)
        safe = torch.where(good, ids, 0)
        k = (cache.k.view(torch.uint8)[safe].view(F8).double() * cache.k_scale[safe].double()[:, :, None, None]).transpose(1, 2).reshape(-1, kv, dim)[:m]
        v = (cache.v.view(torch.uint8)[safe].view(F8).double() * cache.v_scale[safe].double()[:, :, None, None]).transpose(1, 2).reshape(-1, kv, dim)[:m]
        j = torch.arange(m, device=q.device)
        vis = (j[None] <= m - n + torch.arange(n, device=q.device)[:, None]) & good.repeat_interleave(block)[:m][None]
        want, bound = attend(q[b], k, v, vis, scale)
        held(out[b], want, bound, "sequence %d of %d tokens" % (b, m))


def pages(seed, lens, queries, heads, kv, dim, block, t, d, spare=2, width=None):
    g = torch.Generator(device=d).manual_seed(seed)
    used = [(m + block - 1) // block for m in lens]
    total = sum(used) + spare
    cache = random_cache(seed + 1, total, kv, block, dim, d)
    width = max(used + [1]) if width is None else width
    ids = torch.randperm(total, generator=g, device=d).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=d)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = ids[at:at + u]
        at += u
    q = torch.randn(len(lens), queries, heads, dim, generator=g, device=d).to(t)
    return q, cache, table, torch.tensor(lens, dtype=torch.int32, device=d)


@pytest.mark.parametrize("lens", [(1,), (0, 1, 16, 17), (15, 100, 1000, 33), (809,), (3000, 5, 129)])
@pytest.mark.parametrize("heads,kv,dim,block", [(8, 1, 256, 16), (32, 8, 128, 16), (16, 4, 64, 32), (2, 2, 128, 48), (8, 2, 256, 128)])
def test_paged_lengths(lens, heads, kv, dim, block):
    import vla_ops
    d = dev()
    q, cache, table, n = pages(21, lens, 1, heads, kv, dim, block, torch.bfloat16, d)
    check_paged(q, cache, table, n, vla_ops.paged_attention(q, cache, table, n))


@pytest.mark.parametrize("queries", [1, 2, 3, 4, 8, 17])
@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 256), (28, 4, 128), (6, 6, 64), (64, 2, 128), (12, 1, 256)])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_paged_queries_and_heads(queries, heads, kv, dim, t):
    """Several newest tokens, more of them than a sequence holds, groups that are no power of two."""
    import vla_ops
    d = dev()
    q, cache, table, n = pages(22, (40, 2, 300, 0, 17, 64), queries, heads, kv, dim, 16, t, d)
    check_paged(q, cache, table, n, vla_ops.paged_attention(q, cache, table, n, scale=0.2), 0.2)


@pytest.mark.parametrize("count,longest,width", [(1, 20000, None), (3, 9000, 4000), (40, 700, None), (150, 260, 600), (300, 40, None)])
@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 256), (8, 2, 128)])
def test_paged_split_over_the_keys(count, longest, width, heads, kv, dim):
    """Few long sequences, many short ones, a table far wider than the lengths: every way the keys are shared out."""
    import vla_ops
    d = dev()
    lens = [longest] + [(7919 * i) % longest for i in range(1, count)]
    q, cache, table, n = pages(23, lens, 1, heads, kv, dim, 16, torch.bfloat16, d, width=width)
    check_paged(q, cache, table, n, vla_ops.paged_attention(q, cache, table, n))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("queries", [1, 3])
def test_paged_unseen_tokens_may_hold_anything(dim, queries):
    """NaN codes behind a sequence's end and in later queries' own tokens, NaN scales of unused pages, ids outside the cache."""
    import vla_ops
    d = dev()
    q, cache, table, n = pages(24, (37, 100, 16, 70), queries, 8, 2, dim, 16, torch.bfloat16, d, width=9)
    codes = [c.view(torch.uint8) for c in (cache.k, cache.v)]
    for b, m in enumerate((37, 100, 16, 70)):
        last = table[b, (m - 1) // 16]
        for c in codes:
            c[last, :, (m - 1) % 16 + 1:] = 0x7f
    for c, s in zip(codes, (cache.k_scale, cache.v_scale)):
        unused = sorted(set(range(len(c))) - set(table[table >= 0].tolist()))
        c[unused] = 0xff
        s[unused] = float("nan")
    table[1, 2], table[3, 0], table[3, 4] = -7, 10 ** 9, len(codes[0])
    check_paged(q, cache, table, n, vla_ops.paged_attention(q, cache, table, n))
    # a NaN in the newest token reaches the newest query alone
    if queries == 3:
        last = table[0, 36 // 16]
        for c in codes:
            c[last, 0, 36 % 16] = 0x7f
        got = vla_ops.paged_attention(q, cache, table, n)
        assert torch.isnan(got[0, 2, :4].double()).all() and torch.isfinite(got[0, :2].double()).all() and torch.isfinite(got[0, 2, 4:].double()).all()
        keep = [0, 1, 2, 3]
        check_paged(q[keep][:, :2], cache, table, torch.tensor([36, 99, 15, 69], dtype=torch.int32, device=d), got[:, :2])


def test_paged_all_ids_bad_and_lengths_out_of_range():
    import vla_ops
    d = dev()
    q, cache, table, n = pages(25, (64, 64, 64), 1, 8, 1, 128, 16, torch.bfloat16, d)
    table[0] = -1
    lens = torch.tensor([64, 10 ** 9, -4], dtype=torch.int32, device=d)      # longer than the table, negative
    got = vla_ops.paged_attention(q, cache, table, lens)
    assert (got[0] == 0).all() and (got[2] == 0).all()
    check_paged(q, cache, table, lens, got)


def test_paged_sharp_rows_and_spread_scales():
    """One key that takes all, values whose pages differ by many powers of two, keys of an ordinary (not power of two) scale."""
    import vla_ops
    d = dev()
    q, cache, table, n = pages(26, (900, 333), 1, 8, 1, 256, 16, torch.bfloat16, d)
    g = torch.Generator(device=d).manual_seed(3)
    cache.v_scale.copy_(torch.exp2(torch.randint(-30, 12, cache.v_scale.shape, generator=g, device=d).float()))
    cache.k_scale.copy_(torch.rand(cache.k_scale.shape, generator=g, device=d) * 0.05)
    check_paged(q, cache, table, n, vla_ops.paged_attention(q, cache, table, n))
    check_paged(q * 8, cache, table, n, vla_ops.paged_attention(q * 8, cache, table, n))


def test_paged_strided_and_out():
    import vla_ops
    d = dev()
    q, cache, table, n = pages(27, (50, 80), 3, 8, 2, 128, 16, torch.bfloat16, d)
    wide = torch.zeros(2, 3, 3 * 8, 128, dtype=torch.bfloat16, device=d)
    wide[:, :, 8:16] = q
    out = torch.full((3, 2, 8, 128), 5.0, dtype=torch.bfloat16, device=d)
    padded = torch.full((2, 40), -1, dtype=torch.int32, device=d)
    padded[:, :table.shape[1]] = table
    got = vla_ops.paged_attention(wide[:, :, 8:16], cache, padded[:, :table.shape[1]], n, out=out.transpose(0, 1))
    check_paged(q, cache, table, n, got)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes of codes: writing and reading its last blocks."""
    import vla_ops
    d = dev()
    blocks, kv, block, dim = 34000, 8, 64, 256                 # 4.46e9 bytes of keys
    if torch.cuda.mem_get_info()[0] < 14e9:
        pytest.skip("needs 14 GB")
    cache = vla_ops.kv_cache(blocks, kv, block, dim, d)
    g = torch.Generator(device=d).manual_seed(28)
    ids = [33999, 33998, 0, 16500]
    k = torch.randn(200, kv, dim, generator=g, device=d).to(torch.bfloat16)
    v = torch.randn(200, kv, dim, generator=g, device=d).to(torch.bfloat16)
    slots = torch.tensor([ids[i // block] * block + i % block for i in range(200)], dtype=torch.int32, device=d)
    vla_ops.cache_append(k, v, cache, slots)
    small = vla_ops.KvCache(*(x.view(torch.uint8)[ids].view(F8) for x in cache[:2]), *(x[ids] for x in cache[2:]))
    again = vla_ops.kv_cache(4, kv, block, dim, d)
    vla_ops.cache_append(k, v, again, torch.arange(200, dtype=torch.int32, device=d))
    assert torch.equal(small.k.float(), again.k.float()) and torch.equal(small.v_scale, again.v_scale)
    q = torch.randn(1, 1, 8, dim, generator=g, device=d).to(torch.bfloat16)
    n = torch.tensor([200], dtype=torch.int32, device=d)
    table = torch.tensor([ids], dtype=torch.int32, device=d)
    check_paged(q, again, torch.arange(4, dtype=torch.int32, device=d)[None], n, vla_ops.paged_attention(q, cache, table, n))


# ---- block tables and slot maps ---------------------------------------------------------------------------------------------

def plan(ctx, new, table, free, first, block, total):
    """The definition, request by request, on the host."""
    table = [r[:] for r in table]
    width = len(table[0]) if table else 0
    slots, pos, cu, lens, at, missing = [], [], [0], [], first, 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        have = -(-c // block)
        for i in range(have, -(-(c + n) // block)):
            if i < width and at < len(free):
                table[b][i] = free[at]
                at += 1
            else:
                missing += 1
        held_ = 0
        for i in range(c + n):
            blk = i // block
            ok = blk < width and table[b][blk] >= 0
            held_ += ok
            if i >= c:
                slots.append(table[b][blk] * block + i % block if ok else -1)
                pos.append(i)
        lens.append(held_)
        cu.append(cu[-1] + n)
    slots, pos = (slots + [-1] * total)[:total], (pos + [0] * total)[:total]
    return {"slots": slots, "positions": pos, "cu_new": cu, "seq_lens": lens, "counts": [at, missing, cu[-1]], "table": table}


def check_plan(ctx, new, width, block, total=None, n_free=None, first=None, seed=0):
    import vla_ops
    d = dev()
    r = torch.Generator().manual_seed(seed)
    have = [min(-(-max(c, 0) // block), width) for c in ctx]
    need = sum(-(-(max(c, 0) + max(n, 0)) // block) for c, n in zip(ctx, new))
    ids = torch.randperm(sum(have) + need + 4, generator=r).tolist()
    table, at = [], 0
    for h in have:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    free = ids[at:]
    free = free if n_free is None else free[:n_free]
    total = sum(max(n, 0) for n in new) if total is None else total
    want = plan(ctx, new, table, free, first or 0, block, total)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=d)      # noqa: E731
    tab = i32(table) if table else torch.zeros(0, width, dtype=torch.int32, device=d)
    got = vla_ops.block_plan(i32(ctx), i32(new), tab, i32(free), block_size=block, total_new=total,
                             first_free=None if first is None else i32([first]))
    for name, w in want.items():
        g = tab if name == "table" else getattr(got, name)
        assert g.tolist() == w, name


@pytest.mark.parametrize("block", [1, 16, 48, 128])
@pytest.mark.parametrize("ctx,new", [([0], [1]), ([0], [0]), ([15, 16, 17, 0], [1, 1, 1, 1]), ([0, 100, 31], [33, 0, 130]), ([], []),
                                     ([7] * 40, [0, 3] * 20), ([0, 0, 5000], [0, 0, 1])])
def test_plan(block, ctx, new):
    width = max([-(-(c + n) // block) for c, n in zip(ctx, new)] + [1])
    check_plan(ctx, new, width, block)
    check_plan(ctx, new, width + 3, block, total=sum(new) + 7, first=2)


@pytest.mark.parametrize("n", [511, 512, 513, 1500, 8192])
def test_plan_many_requests(n):
    ctx, new = [(37 * i) % 90 for i in range(n)], [(11 * i) % 7 for i in range(n)]
    check_plan(ctx, new, 7, 16, first=1)


def test_plan_long_prompts():
    check_plan([0, 9, 0], [40000, 3, 25001], 2600, 16, first=0)


def test_plan_without_enough_blocks():
    """The free list ends inside a request, the table is too narrow, fewer rows than new tokens, lengths below zero."""
    check_plan([10, 0, 0], [40, 40, 40], 4, 16, n_free=4)
    check_plan([10, 0, 0], [40, 40, 40], 4, 16, n_free=0)
    check_plan([10, 0, 20], [40, 40, 5], 2, 16, first=1)
    check_plan([5, 5], [30, 30], 4, 16, total=41)
    check_plan([-3, 4, 8], [20, -9, 3], 4, 16)


# ---- together -----------------------------------------------------------------------------------------------------------

def serve(d, heads, kv, dim, block, lens, steps, stream=None):
    """A batch of prompts and then single tokens through all four operators -> per step (q, k, v, out)."""
    import vla_ops
    g = torch.Generator(device=d).manual_seed(31)
    n = len(lens)
    cache = vla_ops.kv_cache(64, kv, block, dim, d)
    table = torch.full((n, 24), -1, dtype=torch.int32, device=d)
    free = torch.randperm(64, generator=g, device=d).to(torch.int32)
    ctx, first, said = torch.zeros(n, dtype=torch.int32, device=d), None, []
    for step in range(steps):
        new = torch.tensor(lens if step == 0 else [1] * n, dtype=torch.int32, device=d)
        rows = sum(lens) if step == 0 else n
        q = torch.randn(rows, heads, dim, generator=g, device=d).to(torch.bfloat16)
        k = torch.randn(rows, kv, dim, generator=g, device=d).to(torch.bfloat16) * (1 + step)
        v = torch.randn(rows, kv, dim, generator=g, device=d).to(torch.bfloat16) * (1 + step)
        p = vla_ops.block_plan(ctx, new, table, free, block_size=block, total_new=rows, first_free=first)
        vla_ops.cache_append(k, v, cache, p.slots)
        if step == 0:
            out = vla_ops.prompt_attention(q, k, v, p.cu_new)
        else:
            out = vla_ops.paged_attention(q[:, None], cache, table, p.seq_lens)[:, 0]
        said.append((q, k, v, out, p))
        ctx, first = p.seq_lens, p.counts[:1]
    return said, cache, table


@pytest.mark.parametrize("heads,kv,dim,block", [(8, 1, 256, 16), (8, 2, 128, 32), (4, 4, 64, 16)])
def test_serving_loop(heads, kv, dim, block):
    d = dev()
    lens = (40, 1, 129, 17)
    said, cache, table = serve(d, heads, kv, dim, block, lens, 6)
    q, k, v, out, p = said[0]
    check_prompts(q, k, v, p.cu_new, p.cu_new, out, True)
    q, _, _, out, p = said[-1]
    assert p.seq_lens.tolist() == [m + 5 for m in lens] and p.counts[1].item() == 0
    check_paged(q[:, None], cache, table, p.seq_lens, out[:, None])
    # the cache holds what was given: keys within half a step of e4m3 under their block's scale
    b, m = 2, lens[2]
    held_k = torch.cat([said[0][1][41:41 + m]] + [s[1][b:b + 1] for s in said[1:]]).double()
    ids = table[b, :(m + 5 + block - 1) // block].long()
    sc = cache.k_scale[ids].double().repeat_interleave(block, 0)[:m + 5]
    codes = cache.k.view(torch.uint8)[ids].view(F8).double().transpose(1, 2).reshape(-1, kv, dim)[:m + 5]
    # one rounding to 2^-4 relative (2^-10 of the scale below the normal range) per time a block's scale grew, at most 5 more
    err = (codes * sc[..., None] - held_k).abs()
    assert (err <= held_k.abs() * 2.0 ** -4 + 6 * 2.0 ** -10 * sc[..., None]).all()


def test_other_streams_and_graph():
    """The same decoding step eagerly, on another stream, and captured and replayed with new inputs in the same buffers."""
    import vla_ops
    d = dev()
    q, cache, table, n = pages(33, (300, 64, 1500, 9), 1, 8, 1, 256, 16, torch.bfloat16, d, width=100)
    free = torch.arange(10, dtype=torch.int32, device=d)
    ctx, one = n - 1, torch.ones_like(n)
    k, v = torch.randn(2, 4, 1, 256, device=d, generator=torch.Generator(device=d).manual_seed(5)).to(torch.bfloat16).unbind(0)
    pq, pk, pv, cu, _ = prompts(34, (30, 200), (30, 200), 8, 1, 256, torch.bfloat16, d)

    def step(c, t):
        p = vla_ops.block_plan(ctx, one, t, free, block_size=16, total_new=4)
        vla_ops.cache_append(k, v, c, p.slots)
        return p, vla_ops.paged_attention(q, c, t, p.seq_lens), vla_ops.prompt_attention(pq, pk, pv, cu)

    c0, t0 = clone(cache), table.clone()
    _, want, want_p = step(c0, t0)
    check_paged(q, c0, t0, n, want)
    check_prompts(pq, pk, pv, cu, cu, want_p, True)
    c1, t1 = clone(cache), table.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _, got, got_p = step(c1, t1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(got_p, want_p)
    c2, t2 = clone(cache), table.clone()
    graphs = []
    for _ in range(2):                     # two graphs live at once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(c2, t2)
        graphs.append((graph, res))
    for x, y in zip(c2, cache):
        x.view(torch.uint8).copy_(y.view(torch.uint8))
    t2.copy_(table)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, (_, got, got_p) in graphs:
        assert torch.equal(got, want) and torch.equal(got_p, want_p)
    q.copy_(q.flip(0))
    graphs[0][0].replay()
    check_paged(q, c2, t2, n, graphs[0][1][1])


def test_two_calls_are_bit_equal():
    import vla_ops
    d = dev()
    q, cache, table, n = pages(35, (5000, 31, 700), 1, 32, 8, 128, 16, torch.float16, d)
    assert torch.equal(vla_ops.paged_attention(q, cache, table, n), vla_ops.paged_attention(q, cache, table, n))
    pq, pk, pv, cu, _ = prompts(36, (300, 700), (300, 700), 16, 4, 128, torch.float16, d)
    assert torch.equal(vla_ops.prompt_attention(pq, pk, pv, cu), vla_ops.prompt_attention(pq, pk, pv, cu))


def test_refusals_on_the_gpu():
    """What the wrapper refuses before anything is launched."""
    import _capi
    import vla_ops
    d = dev()
    q, cache, table, n = pages(37, (20, 30), 1, 8, 2, 128, 16, torch.bfloat16, d)
    bad = [lambda: vla_ops.paged_attention(q.float(), cache, table, n),
           lambda: vla_ops.paged_attention(q[:, :, :7], cache, table, n),
           lambda: vla_ops.paged_attention(q[..., :64], cache, table, n),
           lambda: vla_ops.paged_attention(q, cache, table.long(), n),
           lambda: vla_ops.paged_attention(q, cache, table, n[:1]),
           lambda: vla_ops.paged_attention(q, cache, table, n.cpu()),
           lambda: vla_ops.paged_attention(q, cache, table, n, scale=-1.0),
           lambda: vla_ops.paged_attention(q, cache, table, n, scale=float("nan")),
           lambda: vla_ops.paged_attention(q, cache._replace(k=cache.k.float()), table, n),
           lambda: vla_ops.paged_attention(q, cache, table, n, out=q.float()),
           lambda: vla_ops.paged_attention(q.requires_grad_(True), cache, table, n),
           lambda: vla_ops.prompt_attention(q[0], q[0, :, :3], q[0, :, :3], n),
           lambda: vla_ops.prompt_attention(q[0].detach()[..., :4], q[0].detach()[..., :4], q[0].detach()[..., :4], n),
           lambda: vla_ops.prompt_attention(q.detach().flatten()[1:1 + 1024].view(1, 8, 128), q[0].detach(), q[0].detach(), n),
           lambda: vla_ops.cache_append(q[0].detach(), q[0].detach(), cache, n),
           lambda: vla_ops.cache_append(q[0, :, :2].detach(), q[0, :, :2].detach(), cache, n),
           lambda: vla_ops.block_plan(n, n, table, table, block_size=16, total_new=3),
           lambda: vla_ops.block_plan(n, n, table, n, block_size=0, total_new=3)]
    for i, call in enumerate(bad):
        with pytest.raises(_capi.VlaError):
            call()
            raise AssertionError("call %d was not refused" % i)


def test_expanded_output_is_refused():
    import _capi
    import vla_ops
    d = dev()
    q, cache, table, n = pages(38, (20, 30), 1, 8, 2, 128, 16, torch.bfloat16, d)
    cu = torch.tensor([0, 2], dtype=torch.int32, device=d)
    for call in (lambda: vla_ops.paged_attention(q, cache, table, n, out=q[:, :, :1].clone().expand(-1, -1, 8, -1)),
                 lambda: vla_ops.prompt_attention(q[:, 0], q[:, 0], q[:, 0], cu, out=q[:1, 0].clone().expand(2, -1, -1))):
        with pytest.raises(_capi.VlaError, match="expanded"):
            call()


@pytest.mark.parametrize("block", [1, 3, 7, 16, 48, 1000, 2 ** 20 + 1, 2 ** 31 - 1])
def test_plan_far_positions(block):
    """Lengths up to the last that 32 bits hold; the table has room for the first pages only, and no page is free."""
    import vla_ops
    d = dev()
    top, width = 2 ** 31 - 1, 3
    ctx = [top, top - 5, 2 ** 30, top // block * block, 2 * block - 1 if block < 2 ** 29 else 7]
    new = [3, 5, 1, 2, 2]
    table = [[5 * b + i for i in range(width)] for b in range(5)]
    slots, pos, lens, missing = [], [], [], 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        have, want = -(-c // block), -(-(c + n) // block)
        missing += want - have
        lens.append(min(c + n, min(have, width) * block, top))
        for at in range(c, c + n):
            blk = at // block
            s = table[b][blk] * block + at % block if blk < min(have, width) else -1
            slots.append(s if s <= top else -1)
            pos.append(min(at, top))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=d)      # noqa: E731
    tab = i32(table)
    got = vla_ops.block_plan(i32(ctx), i32(new), tab, i32([]), block_size=block, total_new=sum(new))
    assert got.slots.tolist() == slots and got.positions.tolist() == pos and got.seq_lens.tolist() == lens
    assert got.counts.tolist() == [0, missing, sum(new)] and got.cu_new.tolist() == [0, 3, 8, 9, 11, 13] and tab.tolist() == table


FIRST_CALLS = """
import torch, vla_ops
d = torch.device("cuda", 0)
q, k = torch.randn(20, 8, 256, device=d).bfloat16(), torch.randn(20, 1, 256, device=d).bfloat16()
none, new = torch.zeros(1, dtype=torch.int32, device=d), torch.full((1,), 20, dtype=torch.int32, device=d)
cache, table = vla_ops.kv_cache(300, 1, 16, 256), torch.zeros(1, 200, dtype=torch.int32, device=d)
free = torch.arange(250, dtype=torch.int32, device=d)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
def run():
    p = vla_ops.block_plan(none, new, table, free, block_size=16, total_new=20)
    vla_ops.cache_append(k, k, cache, p.slots)
    return vla_ops.prompt_attention(q, k, k, p.cu_new), vla_ops.paged_attention(q[None, -1:], cache, table, p.seq_lens)
with torch.cuda.graph(graph):
    got = run()
graph.replay()
want = run()
assert all(torch.equal(a, b) for a, b in zip(got, want)) and float(got[0].float().abs().sum()) > 0
print("same")
"""


def test_first_calls_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys

    import vla_ops
    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.abspath(vla_ops.__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


def test_two_threads():
    """Each with its own stream and tensors; both get what one alone gets."""
    import threading

    import vla_ops
    d = dev()
    jobs = [pages(40 + i, (3000, 17, 900 + i), 1, 8, 2, 128, 16, torch.bfloat16, d) for i in range(2)]
    want = [vla_ops.paged_attention(q, cache, table, n) for q, cache, table, n in jobs]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        q, cache, table, n = jobs[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(vla_ops.paged_attention(q, cache, table, n))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(len(got[i]) == 20 and all(torch.equal(x, want[i]) for x in got[i]) for i in range(2))
