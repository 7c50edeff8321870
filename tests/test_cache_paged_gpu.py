"""Attention over the cache in pages, on a B200, held to what its own roundings can do.

With p_j the probabilities, v_j = code_j * scale_j the values that a row sees and A = sum_j p_j |v_j|:
  * a probability is held in three e4m3 pieces of 4 bits each, so it is off by at most 2^-12 of itself;
  * the last piece ends at 2^-18 (and what is smaller is off by itself at most) where the largest is at least 2^7, and the scales
    of the values that are summed up with one reference differ by 2^7 at most: sum_j min(p_j, 2^-18 max p) |v_j|, and 2^-25 where all
    scales are one;
  * fp32 scores are off by at most ds_j = (dim + 8) 2^-24 scale sum|q||k|, which moves a probability by that relatively: the
    numerator by sum_j p_j ds_j |v_j|, the denominator by sum_j p_j ds_j of itself;
  * exponentials are off by 2^-22 of themselves, a product with the scale by 2^-24: 2^-20 * A for those above and below;
  * sums of m products in fp32, 32 at a time, truncated: (m / 32 + 40) 2^-23 * A;
  * the output's own rounding is half(t) * |o|, in fp16 2^-25 at least."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda")


def values(codes, scale, ids):
    """The tokens of the pages `ids` in 64 bits: [tokens, kv heads, dim]."""
    x = codes.view(torch.uint8)[ids].view(F8).double() * scale[ids].double()[:, :, None, None]
    return x.transpose(1, 2).reshape(-1, codes.shape[1], codes.shape[3])


def attend(q, k, v, vis, scale, end):
    """q [n, heads, dim], k, v [m, kv, dim] in 64 bits, vis [n, m] -> (o, bound)."""
    n, heads, dim = q.shape
    m, kv = k.shape[:2]
    qd = q.double().reshape(n, kv, heads // kv, dim)
    s = torch.einsum("nhgd,mhd->hgnm", qd, k) * scale
    ds = torch.einsum("nhgd,mhd->hgnm", qd.abs(), k.abs()) * (scale * (dim + 8) * 2.0 ** -24)
    s = s.masked_fill(~vis, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, 1.0, l)
    weigh = lambda w, x: torch.einsum("hgnm,mhd->nhgd", w, x)      # noqa: E731
    o, a = weigh(p, v), weigh(p, v.abs())
    t = q.dtype
    bound = a * (2.0 ** -12 + 2.0 ** -20 + (m / 32 + 40) * 2.0 ** -23) + weigh(torch.minimum(p, end * p.amax(-1, keepdim=True)), v.abs())
    bound += weigh(p * ds, v.abs()) + a * (p * ds).sum(-1).permute(2, 0, 1)[..., None] + torch.finfo(t).eps / 2 * o.abs()
    return o.reshape(n, heads, dim), (bound + (2.0 ** -25 if t == torch.float16 else 0.0)).reshape(n, heads, dim)


def check(q, cache, table, lens, out, scale=None, end=2.0 ** -18):
    scale = q.shape[3] ** -0.5 if scale is None else scale
    block, n = cache.k.shape[2], q.shape[1]
    worst = 0.0
    for b, m in enumerate(lens.tolist()):
        if m == 0:
            assert (out[b] == 0).all()
            continue
        ids = table[b, :(m + block - 1) // block].long()
        k, v = values(cache.k, cache.k_scale, ids)[:m], values(cache.v, cache.v_scale, ids)[:m]
        vis = torch.arange(m, device=q.device)[None] <= m - n + torch.arange(n, device=q.device)[:, None]
        want, bound = attend(q[b], k, v, vis, scale, end)
        got = out[b].double()
        assert torch.isfinite(got).all()
        off = (got - want).abs()
        worst = max(worst, (off / bound.clamp_min(1e-300)).max().item())
        assert (off <= bound).all(), "sequence %d of %d tokens: %g of the bound" % (b, m, worst)
    return worst


def pages(seed, lens, queries, heads, kv, dim, block, t, spread=0):
    """Sequences in pages that are strewn over a cache; `spread`: the scales of V are powers of two that far apart."""
    import vla_ops
    d = dev()
    g = torch.Generator(device=d).manual_seed(seed)
    used = [(m + block - 1) // block for m in lens]
    total = sum(used) + 2
    codes = [(torch.randn(total, kv, block, dim, generator=g, device=d) * 100).clamp(-448, 448).to(F8) for _ in range(2)]
    ks = torch.full((total, kv), 2.0 ** -7, device=d)
    vs = torch.exp2(torch.randint(-8, spread - 7, (total, kv), generator=g, device=d).float())
    ids = torch.randperm(total, generator=g, device=d).to(torch.int32)
    table = torch.full((len(lens), max(used + [1])), -1, dtype=torch.int32, device=d)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = ids[at:at + u]
        at += u
    q = torch.randn(len(lens), queries, heads, dim, generator=g, device=d).to(t)
    return q, vla_ops.KvCache(*codes, ks, vs), table, torch.tensor(lens, dtype=torch.int32, device=d)


def raw(codes):
    return codes.view(torch.uint8)


LAYOUTS = [(8, 1, 256, 1), (32, 8, 128, 1), (8, 2, 128, 3), (16, 4, 64, 5), (12, 1, 256, 2)]


# ---- scales of V that are far apart ---------------------------------------------------------------------------------------

def far(q, cache, up):
    """Channel 0 is up in every query and zero in every key: a key with a negative number there is far from all queries."""
    q[..., 0] = up
    raw(cache.k)[..., 0] = 0


@pytest.mark.parametrize("heads,kv,dim,queries", LAYOUTS)
@pytest.mark.parametrize("ratio", [5, 7, 10, 16, 24, 40, 70])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_a_page_raised_by_a_value_that_nobody_asks_for(heads, kv, dim, queries, ratio, where):
    """One page's scale of V is 2^ratio above the others': a single row of it is large, and its key is far from every query, or it
    stands behind the sequence's end.  The page's other rows are as asked for as any, and are held as small numbers or zeros."""
    import vla_ops
    lens = (1500, 90, 300)                                     # the last pages are not full
    q, cache, table, n = pages(51, lens, queries, heads, kv, dim, 16, torch.bfloat16)
    far(q, cache, 30.0)
    for b, m in enumerate(lens):
        at = {"first": 0, "middle": m // 32, "last": (m - 1) // 16}[where]
        page = int(table[b, at])
        big = m % 16 if where == "last" else 7
        cache.v_scale[page] *= 2.0 ** ratio
        raw(cache.v)[page] = raw((cache.v[page].float() * 2.0 ** -ratio).to(F8))
        raw(cache.v)[page, :, big] = 0x7e                      # 448
        cache.k_scale[page] *= 64.0
        raw(cache.k)[page] = raw((cache.k[page].float() / 64).to(F8))
        raw(cache.k)[page, :, big] = 0
        raw(cache.k)[page, :, big, 0] = 0xfe                   # -448: a score of -400 and less
    check(q, cache, table, n, vla_ops.paged_attention(q, cache, table, n))


@pytest.mark.parametrize("heads,kv,dim,queries", LAYOUTS)
@pytest.mark.parametrize("spread", [3, 9, 30, 60])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_scales_all_over(heads, kv, dim, queries, spread, t):
    """Every page has a scale of its own, within 2^spread; flat rows, and rows that ask for few tokens."""
    import vla_ops
    q, cache, table, n = pages(52, (700, 33, 5000, 129, 1), queries, heads, kv, dim, 32, t, spread)
    cache.v_scale.mul_(2.0 ** -max(0, spread - 14))            # the largest within fp16's range
    for up in (1, 6):
        check(q * up, cache, table, n, vla_ops.paged_attention(q * up, cache, table, n))


@pytest.mark.parametrize("heads,kv,dim,queries", LAYOUTS)
def test_scales_of_few_kinds(heads, kv, dim, queries):
    """Long runs of pages of one scale and then of another, pages of zeros, scales that are no power of two or negative."""
    import vla_ops
    q, cache, table, n = pages(53, (3000, 260, 64), queries, heads, kv, dim, 16, torch.bfloat16)
    for b in range(3):
        row = table[b][table[b] >= 0].long()
        run = torch.arange(len(row), device=q.device)
        cache.v_scale[row] = torch.where((run // 40 % 2 == 0)[:, None], 2.0 ** -8, 3.0 * 2.0 ** 6).expand(-1, kv).contiguous()
        cache.v_scale[row[::7]] *= -1.0
        raw(cache.v)[row[3::11]] = 0
        cache.v_scale[row[3::11]] = 2.0 ** -60
        cache.v_scale[row[3::33]] = 0.0
    check(q, cache, table, n, vla_ops.paged_attention(q, cache, table, n))


@pytest.mark.parametrize("ratio", [12, 20, 26])
def test_a_large_value_with_a_small_probability_counts(ratio):
    """The other way about: the page with the large scale has a probability of 2^-ratio, and gives as much as all the others."""
    import vla_ops
    q, cache, table, n = pages(54, (1000,), 1, 8, 1, 128, 16, torch.bfloat16)
    far(q, cache, 60.0)
    page = int(table[0, 30])
    # -60 * code * 2^-7 * 128^-0.5 is -ratio * ln 2
    raw(cache.k)[page] = raw(torch.zeros(1, device=q.device).to(F8))
    raw(cache.k)[page, :, :, 0] = raw(torch.tensor([-ratio * 16.733], device=q.device).to(F8))
    cache.v_scale[page] *= 2.0 ** ratio
    check(q, cache, table, n, vla_ops.paged_attention(q, cache, table, n))


def test_scales_far_apart_in_cut_units_and_graphs():
    """Few long sequences, whose units are cut between CTAs: parts with references of their own are joined; replayed, too."""
    import vla_ops
    q, cache, table, n = pages(55, (20000, 9000), 1, 8, 1, 256, 16, torch.float16, 40)
    cache.v_scale.mul_(2.0 ** -26)
    want = vla_ops.paged_attention(q, cache, table, n)
    check(q, cache, table, n, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = vla_ops.paged_attention(q, cache, table, n)
    for _ in range(2):
        got.zero_()
        graph.replay()
        assert torch.equal(got, want)


def test_not_a_number_in_a_far_scale():
    """A visible page whose scale of V is NaN or infinite makes the row not finite; an unseen one does not."""
    import vla_ops
    q, cache, table, n = pages(56, (400, 400), 1, 8, 1, 128, 16, torch.bfloat16, 20)
    for bad in (float("nan"), float("inf")):
        c = vla_ops.KvCache(*(x.clone() for x in cache))
        c.v_scale[int(table[1, 5])] = bad
        got = vla_ops.paged_attention(q, c, table, n)
        assert not torch.isfinite(got[1].double()).any()
        check(q[:1], c, table[:1], n[:1], got[:1])


# ---- every token once -------------------------------------------------------------------------------------------------------

def one_hot(cache, table, lens):
    """V of a token is one number, in the head dim that its tile of 128 has: a result is the probability of each tile."""
    blocks, kv, block, dim = cache.v.shape
    raw(cache.v)[:] = 0
    for b, m in enumerate(lens.tolist()):
        t = torch.arange(m, device=table.device)
        page = table[b, t // block].long()
        raw(cache.v)[page[:, None], torch.arange(kv, device=page.device)[None], (t % block)[:, None], (t // 128 % dim)[:, None]] = 0x38     # 1
    cache.v_scale.fill_(2.0 ** -3)


@pytest.mark.parametrize("lens", [(20000,), (9000, 131, 4097, 1, 12800), (300, 513, 129, 0, 1025, 511, 512)])
@pytest.mark.parametrize("heads,kv,dim,queries", LAYOUTS + [(16, 16, 64, 1), (28, 4, 128, 8)])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_every_tile_counts_once(lens, heads, kv, dim, queries, t):
    """A tile that a piece's border loses, or that two pieces take, shows in its own head dim (or in one it shares with few others)."""
    import vla_ops
    q, cache, table, n = pages(57, lens, queries, heads, kv, dim, 16, t)
    one_hot(cache, table, n)
    check(q, cache, table, n, vla_ops.paged_attention(q, cache, table, n), end=2.0 ** -25)


@pytest.mark.parametrize("heads,kv,dim,queries,t", [(8, 1, 256, 1, torch.bfloat16), (8, 1, 256, 3, torch.float16), (8, 2, 128, 1, torch.float16)])
def test_every_tile_counts_once_in_long_contexts(heads, kv, dim, queries, t):
    import vla_ops
    q, cache, table, n = pages(58, (131071, 90001), queries, heads, kv, dim, 64, t)
    one_hot(cache, table, n)
    check(q, cache, table, n, vla_ops.paged_attention(q, cache, table, n), end=2.0 ** -25)


@pytest.mark.parametrize("ahead", [10, 17, 22])
def test_many_faint_tokens_beside_a_loud_one(ahead):
    """One key stands 2^ahead above the largest of 60000 others, which together still count."""
    import vla_ops
    q, cache, table, n = pages(59, (60000,), 1, 8, 1, 128, 16, torch.float16)
    far(q, cache, 60.0)
    one_hot(cache, table, n)
    page = int(table[0, 1000])
    raw(cache.k)[page, 0, 3] = raw(torch.zeros(1, device=q.device).to(F8))
    raw(cache.k)[page, 0, 3, 0] = raw(torch.tensor([(ahead + 4) * 16.733], device=q.device).to(F8))      # as above, the other way
    check(q, cache, table, n, vla_ops.paged_attention(q, cache, table, n), end=2.0 ** -25)


@pytest.mark.parametrize("block", [16, 32, 48, 64, 80, 96, 112, 128, 144, 176, 192, 208, 240, 256])
@pytest.mark.parametrize("heads,kv,dim,queries", [(8, 1, 256, 1), (8, 2, 128, 3), (16, 4, 64, 5)])
def test_pages_of_every_size(block, heads, kv, dim, queries):
    """Pages that end inside a tile and boxes of 16, 32, 64 and 128 rows."""
    import vla_ops
    lens = (block - 1, block, block + 1, 3 * block + 5, 2000)
    q, cache, table, n = pages(60, lens, queries, heads, kv, dim, block, torch.bfloat16, 3)
    check(q, cache, table, n, vla_ops.paged_attention(q, cache, table, n))
    one_hot(cache, table, n)
    check(q, cache, table, n, vla_ops.paged_attention(q, cache, table, n), end=2.0 ** -25)


# ---- refusals ---------------------------------------------------------------------------------------------------------------

def test_each_refusal_says_why():
    """Every call with one thing wrong, and the words for it."""
    import _capi
    import vla_ops
    q, cache, table, n = pages(61, (20, 30), 1, 8, 2, 128, 16, torch.bfloat16)
    x = q[:, 0]
    k = torch.zeros(2, 2, 128, dtype=torch.bfloat16, device=q.device)
    slots, cu = torch.arange(2, dtype=torch.int32, device=q.device), torch.tensor([0, 1, 2], dtype=torch.int32, device=q.device)
    odd = torch.zeros(2 * 8 * 128 + 1, dtype=torch.bfloat16, device=q.device)[1:].view(2, 1, 8, 128)
    paged, prompt, append, plan = vla_ops.paged_attention, vla_ops.prompt_attention, vla_ops.cache_append, vla_ops.block_plan
    paged(q, cache, table, n)
    prompt(x, k, k, cu)
    append(k, k, cache, slots)
    plan(n, n, table.clone(), n, block_size=16, total_new=50)
    for words, call in [
            ("bfloat16 or float16", lambda: paged(q.float(), cache, table, n)),
            ("multiple of kv_heads", lambda: paged(q[:, :, :7], cache, table, n)),
            ("do not fit", lambda: paged(q[..., :64], cache, table, n)),
            ("last one contiguous", lambda: paged(q.transpose(2, 3), cache, table, n)),
            ("block_table must be int32", lambda: paged(q, cache, table.long(), n)),
            ("do not fit", lambda: paged(q, cache, table, n[:1])),
            ("seq_lens must be int32", lambda: paged(q, cache, table, n.cpu())),
            ("scale must be", lambda: paged(q, cache, table, n, scale=-1.0)),
            ("scale must be", lambda: paged(q, cache, table, n, scale=float("nan"))),
            ("a cache is", lambda: paged(q, cache._replace(k=cache.k.float()), table, n)),
            ("a cache is", lambda: paged(q, cache._replace(v_scale=cache.v_scale[:, :1]), table, n)),
            ("cache must be", lambda: paged(q, list(cache), table, n)),
            ("out must be", lambda: paged(q, cache, table, n, out=q.float())),
            ("shape of q", lambda: paged(q, cache, table, n, out=torch.empty(2, 1, 7, 128, dtype=q.dtype, device=q.device))),
            ("requires a gradient", lambda: paged(q.detach().clone().requires_grad_(), cache, table, n)),
            ("start on 16 bytes", lambda: paged(odd, cache, table, n)),
            ("multiple of kv_heads", lambda: prompt(x[:, :7], k, k, cu)),
            ("multiple of kv_heads", lambda: prompt(x, torch.zeros(2, 3, 128, dtype=q.dtype, device=q.device), torch.zeros(2, 3, 128, dtype=q.dtype, device=q.device), cu)),
            ("head_dim must be", lambda: prompt(x[..., :4], k[..., :4], k[..., :4], cu)),
            ("k must be", lambda: prompt(x, k.half(), k, cu)),
            ("do not fit", lambda: prompt(x, k, k[:1], cu)),
            ("do not fit", lambda: prompt(x, k, k, cu, cu[:2])),
            ("cu_q must be int32", lambda: prompt(x, k, k, cu.float())),
            ("start on 16 bytes", lambda: prompt(odd[:, 0], k, k, cu)),
            ("requires a gradient", lambda: prompt(x, k.clone().requires_grad_(), k, cu)),
            ("do not fit the cache", lambda: append(x, x, cache, slots)),
            ("do not fit the cache", lambda: append(k, k, cache, slots[:1])),
            ("slots must be int32", lambda: append(k, k, cache, slots.long())),
            ("k must be bfloat16", lambda: append(k.float(), k.float(), cache, slots)),
            ("v must be", lambda: append(k, k.half(), cache, slots)),
            ("requires a gradient", lambda: append(k.clone().requires_grad_(), k, cache, slots)),
            ("free_blocks must be int32", lambda: plan(n, n, table, table, block_size=16, total_new=3)),
            ("do not fit", lambda: plan(n, n[:1], table, n, block_size=16, total_new=3)),
            ("negative size", lambda: plan(n, n, table, n, block_size=0, total_new=3)),
            ("total_new is negative", lambda: plan(n, n, table, n, block_size=16, total_new=-1)),
            ("too large", lambda: plan(n, n, table, n, block_size=16, total_new=2 ** 31)),
            ("one element", lambda: plan(n, n, table, n, block_size=16, total_new=3, first_free=n))]:
        with pytest.raises(_capi.VlaError, match=words):
            call()


# ---- a second turn ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 256), (8, 2, 128)])
def test_second_turn_of_different_lengths(heads, kv, dim):
    """Prompts, then further tokens behind them, a different number for each sequence: plan, append, and attention over the cache with
    the queries of each sequence at the end of its row, as the documentation lays it out.  Every token sees its sequence's cache
    up to itself."""
    import vla_ops
    g = torch.Generator(device=dev()).manual_seed(63)
    first, then, block = (40, 1, 129, 17), (5, 33, 0, 12), 16
    cache = vla_ops.kv_cache(40, kv, block, dim)
    table = torch.full((4, 12), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(40, generator=g, device="cuda").to(torch.int32)
    lens, taken = torch.zeros(4, dtype=torch.int32, device="cuda"), None
    for turn in (first, then):
        new = torch.tensor(turn, dtype=torch.int32, device="cuda")
        q = torch.randn(sum(turn), heads, dim, generator=g, device="cuda").bfloat16()
        k, v = torch.randn(2, sum(turn), kv, dim, generator=g, device="cuda").bfloat16().unbind(0)
        plan = vla_ops.block_plan(lens, new, table, free, block_size=block, total_new=sum(turn), first_free=taken)
        vla_ops.cache_append(k, v, cache, plan.slots)
        lens, taken = plan.seq_lens, plan.counts[:1]
    most = max(then)
    row = plan.cu_new[1:, None] - most + torch.arange(most, device="cuda")                  # [sequences, most]; negative: padding
    out = vla_ops.paged_attention(q[row.clamp_min(0)], cache, table, plan.seq_lens)
    out = out[torch.arange(most, device="cuda") >= most - new[:, None]]                     # [sum of new tokens, heads, dim]
    assert out.shape == q.shape and plan.seq_lens.tolist() == [a + b for a, b in zip(first, then)]
    cu = plan.cu_new.tolist()
    for b in range(4):
        if then[b]:
            one = slice(b, b + 1)
            check(q[None, cu[b]:cu[b + 1]], cache, table[one], plan.seq_lens[one], out[None, cu[b]:cu[b + 1]])
