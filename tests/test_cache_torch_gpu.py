"""The operators around a key/value cache in pages among torch's own: gradients that they would lose, and tensors that they change."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import vla_ops
    return vla_ops


def made(ops):
    g = torch.Generator(device="cuda").manual_seed(61)
    cache = ops.kv_cache(4, 2, 16, 64)
    x = torch.randn(20, 2, 64, generator=g, device="cuda").bfloat16()
    slots = torch.arange(20, dtype=torch.int32, device="cuda")
    ops.cache_append(x, x, cache, slots)
    q = torch.randn(1, 1, 8, 64, generator=g, device="cuda").bfloat16()
    table, lens = torch.arange(4, dtype=torch.int32, device="cuda")[None], torch.full((1,), 20, dtype=torch.int32, device="cuda")
    return cache, x, slots, q, table, lens


def calls(ops, cache, x, slots, q, table, lens):
    """Each operator with one tensor of its arguments exchanged by f."""
    cu = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    ident = lambda t: t                                                                  # noqa: E731
    part = lambda name, f: cache._replace(**{name: f(getattr(cache, name))})             # noqa: E731
    return {
        "q": lambda f=ident: ops.paged_attention(f(q), cache, table, lens),
        "k_scale": lambda f=ident: ops.paged_attention(q, part("k_scale", f), table, lens),
        "v_scale": lambda f=ident: ops.paged_attention(q, part("v_scale", f), table, lens),
        "append k": lambda f=ident: ops.cache_append(f(x), x, cache, slots),
        "append v": lambda f=ident: ops.cache_append(x, f(x), cache, slots),
        "append v_scale": lambda f=ident: ops.cache_append(x, x, part("v_scale", f), slots),
        "prompt q": lambda f=ident: ops.prompt_attention(f(x), x, x, cu),
        "prompt k": lambda f=ident: ops.prompt_attention(x, f(x), x, cu),
        "prompt v": lambda f=ident: ops.prompt_attention(x, x, f(x), cu),
        "out": lambda f=ident: ops.prompt_attention(x, x, x, cu, out=f(torch.empty_like(x))),
    }


NAMES = ["q", "k_scale", "v_scale", "append k", "append v", "append v_scale", "prompt q", "prompt k", "prompt v", "out"]


@pytest.mark.parametrize("name", NAMES)
def test_tangents_and_gradients_are_refused_not_lost(ops, name):
    import _capi
    call = calls(ops, *made(ops))[name]
    call()
    with fwd.dual_level():
        with pytest.raises(_capi.VlaError, match="gradient|tangent"):
            call(lambda t: fwd.make_dual(t, torch.ones_like(t)))
    grown = lambda t: t.detach().clone().requires_grad_()           # noqa: E731
    with pytest.raises(_capi.VlaError, match="gradient"):
        call(grown)
    with torch.no_grad():
        call(grown)                                                  # nobody asks for one


def test_what_is_written_has_a_new_version(ops):
    cache, x, slots, q, table, lens = made(ops)
    before = [t._version for t in cache]
    ops.cache_append(x, x, cache, slots)
    assert all(t._version > b for t, b in zip(cache, before))
    before = [t._version for t in (*cache, q, table, lens, x)]
    out = torch.empty_like(q)
    version = out._version
    ops.paged_attention(q, cache, table, lens, out=out)
    assert out._version > version and [t._version for t in (*cache, q, table, lens, x)] == before
    wide = torch.empty(20, 2, 2, 64, dtype=torch.bfloat16, device="cuda")
    version = wide._version
    ops.prompt_attention(x, x, x, torch.tensor([0, 20], dtype=torch.int32, device="cuda"), out=wide[:, 1])
    assert wide._version > version                                   # a view's base as well
    version = table._version
    ops.block_plan(lens, torch.ones_like(lens), table, torch.zeros(1, dtype=torch.int32, device="cuda"), block_size=16, total_new=1)
    assert table._version > version


def test_a_backward_pass_over_changed_scales_is_refused_by_torch(ops):
    cache, x, slots, *_ = made(ops)
    w = torch.ones_like(cache.v_scale).requires_grad_()
    loss = (w * cache.v_scale).sum()                                 # keeps v_scale
    ops.cache_append(x * 64, x * 64, cache, slots)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_tensors_of_inference_mode_may_be_written_anywhere(ops):
    with torch.inference_mode():
        cache, x, slots, q, table, lens = made(ops)
        out = torch.empty_like(q)
        want = ops.paged_attention(q, cache, table, lens).clone()
    ops.cache_append(x, x, cache, slots)
    ops.paged_attention(q, cache, table, lens, out=out)
    assert torch.equal(out, want)


def test_out_may_be_q_and_nothing_else_that_is_read(ops):
    """Written over q an output is what it is elsewhere; over k or v, or across q, it is refused: other rows still read those."""
    import _capi
    g = torch.Generator(device="cuda").manual_seed(62)
    q, k, v = (torch.randn(700, 4, 128, generator=g, device="cuda").bfloat16() for _ in range(3))
    cu = torch.tensor([0, 300, 301, 700], dtype=torch.int32, device="cuda")
    want = ops.prompt_attention(q, k, v, cu)
    for out in (k, v, k.view(-1).view(700, 4, 128)):
        with pytest.raises(_capi.VlaError, match="overlap"):
            ops.prompt_attention(q, k, v, cu, out=out)
    wide = torch.empty(701, 4, 128, device="cuda", dtype=torch.bfloat16)
    wide[:700] = q
    with pytest.raises(_capi.VlaError, match="overlap"):
        ops.prompt_attention(wide[:700], k, v, cu, out=wide[1:])
    fused = torch.cat([q, k, v], 1)                      # [700, 12, 128]: one projection's output, written over its own q
    fq, fk, fv = fused[:, :4], fused[:, 4:8], fused[:, 8:]
    for out in (fk, fv, fused[:, 2:6], fused[:, 7:11]):
        with pytest.raises(_capi.VlaError, match="overlap"):
            ops.prompt_attention(fq, fk, fv, cu, out=out)
    assert torch.equal(ops.prompt_attention(fq, fk, fv, cu, out=fq), want) and torch.equal(fk, k) and torch.equal(fv, v)
    got = q.clone()
    assert torch.equal(ops.prompt_attention(got, k, v, cu, out=got), want)
    # attention over a cache: units that are cut between CTAs read q several times
    cache = ops.kv_cache(600, 2, 16, 128)
    x = torch.randn(9000, 2, 128, generator=g, device="cuda").bfloat16()
    ops.cache_append(x, x, cache, torch.arange(9000, dtype=torch.int32, device="cuda"))
    table = torch.arange(600, dtype=torch.int32, device="cuda")[None].expand(3, -1).contiguous()
    lens = torch.tensor([9000, 40, 0], dtype=torch.int32, device="cuda")
    q = torch.randn(3, 3, 8, 128, generator=g, device="cuda").bfloat16()
    want = ops.paged_attention(q, cache, table, lens)
    got = q.clone()
    assert torch.equal(ops.paged_attention(got, cache, table, lens, out=got), want)
    wide = torch.zeros(4, 3, 8, 128, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(_capi.VlaError, match="overlap"):
        ops.paged_attention(wide[:3], cache, table, lens, out=wide[1:])


def test_strides_of_dimensions_of_one_do_not_matter(ops):
    """A single token, sequence or head out of a tensor of odd width: nothing is ever that stride away from it."""
    cache, x, slots, q, table, lens = made(ops)
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    odd = lambda t: torch.cat([t.flatten(), t.new_zeros(3)]).as_strided(t.shape, [1003 if n == 1 else s for n, s in zip(t.shape, t.stride())])   # noqa: E731
    one = x[:1].contiguous()
    assert odd(one).stride(0) == 1003 and torch.equal(odd(one), one)
    want = ops.prompt_attention(one, one, one, cu)
    assert torch.equal(ops.prompt_attention(odd(one), odd(one), odd(one), cu, out=odd(torch.empty_like(one))), want)
    single = x[:20, :1].contiguous()
    cu20 = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.prompt_attention(odd(single), odd(single), odd(single), cu20), ops.prompt_attention(single, single, single, cu20))
    want = ops.paged_attention(q, cache, table, lens)
    assert torch.equal(ops.paged_attention(odd(q), cache, table, lens, out=odd(torch.empty_like(q))), want)
    a, b = ops.kv_cache(4, 2, 16, 64), ops.kv_cache(4, 2, 16, 64)
    ops.cache_append(one, one, a, slots[:1])
    ops.cache_append(odd(one), odd(one), b, slots[:1])
    assert all(torch.equal(s.float(), t.float()) for s, t in zip(a, b))
