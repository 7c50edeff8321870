"""Cases of the operators around a key/value cache held in pages: the maps of the pages (`block_plan`), the writer that
keeps keys and values in 8 bits (`cache_append`), attention over that cache for the newest tokens of every sequence
(`paged_attention`) and attention over whole packed prompts (`prompt_attention`).

`run` computes a case in elementary torch operations in 32 bits, or, where `own` is true, through `vla_ops`.
Head layouts: 8 query heads on one key/value head of 256 is the prefix model of this repository, 16 heads of 72 its vision
tower; the others are generic grouped layouts.  Lengths: 256 tokens per camera view plus a prompt, up to long contexts.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
SCALE_FLOOR = 2.0 ** -60        # smallest scale of a block in the cache


def _ops():
    pkg = os.path.join(os.getcwd(), "realtime-vla_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import vla_ops
    return vla_ops


# ---- cases ------------------------------------------------------------------------------------------------------------

def _prompt(name, count, shortest, longest, heads, kv_heads, dim, dtype, causal, context=0):
    """`count` prompts of shortest..longest tokens; `context`: up to that many keys stand before each prompt's own."""
    return {"name": name, "op": "prompt_attention", "count": count, "shortest": shortest, "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "causal": causal, "context": context}


def _paged(name, count, shortest, longest, queries, heads, kv_heads, dim, block, dtype):
    """`count` sequences of shortest..longest cached tokens, the last `queries` of which ask."""
    return {"name": name, "op": "paged_attention", "count": count, "shortest": shortest, "longest": longest, "queries": queries,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block, "dtype": dtype}


def _append(name, count, shortest, longest, kv_heads, dim, block, dtype, fresh):
    """`count` sequences append shortest..longest tokens each; `fresh`: at the start of a block, else somewhere inside one."""
    return {"name": name, "op": "cache_append", "count": count, "shortest": shortest, "longest": longest, "kv_heads": kv_heads,
            "dim": dim, "block": block, "dtype": dtype, "fresh": fresh}


def _plan(name, count, shortest, longest, context, block):
    """`count` requests of up to `context` cached tokens get shortest..longest new ones."""
    return {"name": name, "op": "block_plan", "count": count, "shortest": shortest, "longest": longest, "context": context,
            "block": block}


def listed():
    return [
        # one instruction of 20 tokens: the call's latency is what counts
        _prompt("prompt of one instruction", 1, 20, 20, 8, 1, 256, "bf16", True),
        # the prefixes of 32 observations with one to three views and prompts of their own, every token sees every other
        _prompt("prefixes of 32 observations", 32, 276, 968, 8, 1, 256, "bf16", False),
        # a serving batch: short and long prompts packed, some of them the later part of a prompt that has begun
        _prompt("packed ragged prompts", 48, 1, 1201, 32, 8, 128, "fp16", True, 400),
        # one long document
        _prompt("one long prompt", 1, 8192, 8192, 32, 8, 128, "bf16", True),
        # one robot's next text token behind three views and an instruction
        _paged("next token of one robot", 1, 809, 809, 1, 8, 1, 256, 16, "bf16"),
        # a serving batch of short and long conversations
        _paged("next tokens of a batch", 64, 64, 8192, 1, 32, 8, 128, 16, "bf16"),
        # a few very long contexts
        _paged("next tokens of long contexts", 4, 90001, 131071, 1, 8, 1, 256, 64, "bf16"),
        # several proposed tokens verified at once
        _paged("proposed tokens verified", 16, 100, 4001, 4, 16, 4, 64, 32, "fp16"),
        # each sequence of a batch adds its newest token to a block that is in use
        _append("newest tokens of a batch", 64, 1, 1, 8, 128, 16, "bf16", False),
        # the prompts of a batch enter the cache
        _append("prompts of a batch", 24, 40, 2048, 8, 128, 16, "bf16", True),
        # the maps of one step of decoding
        _plan("maps of a decoding step", 256, 1, 1, 4096, 16),
        # the maps of many new prompts
        _plan("maps of new prompts", 512, 1, 2048, 0, 32),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))


_PROMPT_MOST = 32 * 8192 * 8192 * 128            # heads x scores x dim, padded to the longest
_PAGED_MOST = 64 * 8192 * 8 * 128                # keys x heads x dim, padded to the longest
_BYTES_MOST, _FLOPS_MOST = 2.3e8, 5.4e11         # of one call, as the largest listed ones have


def draw(rng):
    while True:
        c = _drawn(rng)
        w = work(c)
        if w["bytes"] <= _BYTES_MOST and w["flops"] <= _FLOPS_MOST:
            return c


def _drawn(rng):
    op = rng.choice(["prompt_attention", "paged_attention", "cache_append", "block_plan"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "prompt_attention":
        heads, kv_heads, dim = rng.choice([(8, 1, 256), (32, 8, 128), (16, 16, 72), (16, 4, 64), (28, 4, 128), (12, 3, 96)])
        longest = _log(rng, 1, 8192)
        count = _log(rng, 1, max(1, min(64, _PROMPT_MOST // (4 * heads * dim * longest * longest))))
        context = rng.choice([0, 0, _log(rng, 1, longest)])
        c = _prompt("", count, rng.randint(1, longest), longest, heads, kv_heads, dim, dtype, rng.random() < 0.7, context)
    elif op == "paged_attention":
        heads, kv_heads, dim = rng.choice([(8, 1, 256), (32, 8, 128), (16, 4, 64), (28, 4, 128), (64, 8, 128), (16, 16, 64)])
        longest = _log(rng, 1, 131072)
        count = _log(rng, 1, max(1, min(256, _PAGED_MOST // (longest * kv_heads * dim))))
        c = _paged("", count, rng.randint(1, longest), longest, rng.choice([1, 1, 2, 3, 5, 8]), heads, kv_heads, dim,
                   rng.choice([16, 32, 64, 128]), dtype)
    elif op == "cache_append":
        kv_heads, dim = rng.choice([(1, 256), (8, 128), (4, 64), (3, 128)])
        longest = _log(rng, 1, 2048)
        c = _append("", _log(rng, 1, max(1, min(256, 40000 // longest))), rng.randint(1, longest), longest, kv_heads, dim,
                    rng.choice([16, 32, 64, 128]), dtype, rng.random() < 0.5)
    else:
        longest = _log(rng, 1, 4096)
        c = _plan("", _log(rng, 1, max(1, min(2048, 200000 // longest))), rng.randint(1, longest), longest, _log(rng, 1, 8192),
                  rng.choice([16, 32, 64, 128]))
    del c["name"]
    return c


def _lengths(case):
    """The sequences' lengths: spread over the logarithm, the longest among them; they belong to the case."""
    r = random.Random(1000003 * case["count"] + 1009 * case["longest"] + case["shortest"])
    return [case["longest"]] + [_log(r, case["shortest"], case["longest"]) for _ in range(case["count"] - 1)]


def _contexts(case):
    """The tokens that stand before each sequence's new ones."""
    r = random.Random(7 * case["count"] + case["longest"])
    return [r.randint(0, case["context"]) for _ in range(case["count"])]


def _blocks(tokens, block):
    return -(-tokens // block)


def work(case):
    lens = _lengths(case)
    op = case["op"]
    if op == "prompt_attention":
        more = _contexts(case)
        keys = [n + c for n, c in zip(lens, more)]
        pairs = sum(n * k - (n * (n - 1) // 2 if case["causal"] else 0) for n, k in zip(lens, keys))
        tok, key = sum(lens), sum(keys)
        return {"bytes": 2 * case["dim"] * (2 * tok * case["heads"] + 2 * key * case["kv_heads"]) + 8 * (case["count"] + 1),
                "flops": 4 * case["dim"] * case["heads"] * pairs}
    if op == "paged_attention":
        n, h = case["queries"], case["kv_heads"]
        pages = sum(_blocks(k, case["block"]) for k in lens)
        return {"bytes": 2 * case["dim"] * h * sum(lens) + pages * (8 * h + 4) + 4 * case["count"]
                + 4 * case["count"] * n * case["heads"] * case["dim"],
                "flops": 4 * case["dim"] * case["heads"] * sum(max(0, k - n + 1 + i) for k in lens for i in range(n))}
    if op == "cache_append":
        tok = sum(lens)
        pages = sum(_blocks(n, case["block"]) for n in lens)
        return {"bytes": tok * (case["kv_heads"] * case["dim"] * 2 * (2 + 1) + 4) + pages * 8 * case["kv_heads"],
                "flops": tok * case["kv_heads"] * case["dim"] * 2 * 2}
    more = _contexts(case)
    new = sum(_blocks(c + n, case["block"]) - _blocks(c, case["block"]) for n, c in zip(lens, more))
    return {"bytes": 8 * sum(lens) + 8 * new + 16 * case["count"], "flops": 4 * sum(lens)}


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _power_scale(amax):
    """The smallest power of two that brings amax to 448 or less."""
    m, e = torch.frexp(amax.float())
    e = torch.where(amax > 0, e - 9 + (m > 0.875), -1000).clamp_min(int(math.log2(SCALE_FLOOR)))
    return ((e + 127) << 23).view(torch.float32)


def _codes(x, scale):
    """x in 8 bits: [blocks, heads, tokens, dim] with a scale for each block and head."""
    return (x / scale[:, :, None, None]).clamp(-F8_MAX, F8_MAX).to(F8)


def _cache(g, blocks, heads, block, dim):
    """A cache full of tokens: keys with a few strong channels, as rotary attention makes them, values around one."""
    d = "cuda"
    channel = torch.exp(0.7 * torch.randn(heads, 1, dim, generator=g, device=d))
    k = torch.randn(blocks, heads, block, dim, generator=g, device=d) * channel
    v = torch.randn(blocks, heads, block, dim, generator=g, device=d)
    ks, vs = _power_scale(k.abs().amax((2, 3))), _power_scale(v.abs().amax((2, 3)))
    return {"k": _codes(k, ks), "v": _codes(v, vs), "k_scale": ks, "v_scale": vs}


def _starts(lens):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    lens = _lengths(case)
    r.shuffle(lens)                       # the sequences stand in another order for every seed
    op = case["op"]
    s = {"op": op, "case": case}
    if op == "prompt_attention":
        t = TYPES[case["dtype"]]
        keys = [n + c for n, c in zip(lens, _contexts(case))]
        s["longest_q"], s["longest_k"] = max(lens), max(keys)
        s["cu_q"], s["cu_k"] = _starts(lens), _starts(keys)
        s["q"] = torch.randn(sum(lens), case["heads"], case["dim"], generator=g, device="cuda").to(t)
        s["k"] = torch.randn(sum(keys), case["kv_heads"], case["dim"], generator=g, device="cuda").to(t)
        s["v"] = torch.randn(sum(keys), case["kv_heads"], case["dim"], generator=g, device="cuda").to(t)
    elif op == "paged_attention":
        width = _blocks(case["longest"], case["block"])
        used = [_blocks(n, case["block"]) for n in lens]
        total = sum(used) + 3
        s["cache"] = _cache(g, total, case["kv_heads"], case["block"], case["dim"])
        ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        at = _starts(used)[:-1, None] + torch.arange(width, device="cuda")[None]
        s["table"] = torch.where(torch.arange(width, device="cuda")[None] < torch.tensor(used, device="cuda")[:, None],
                                 ids[at.clamp_max(total - 1)], -1).to(torch.int32).contiguous()
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["q"] = torch.randn(case["count"], case["queries"], case["heads"], case["dim"], generator=g, device="cuda").to(
            TYPES[case["dtype"]])
    elif op == "cache_append":
        t, block = TYPES[case["dtype"]], case["block"]
        first = [0 if case["fresh"] else r.randint(1, block - 1) for _ in lens]
        used = [_blocks(f + n, block) for f, n in zip(first, lens)]
        total = sum(_blocks(n, block) + (not case["fresh"]) for n in lens) + 3
        s["cache"] = _cache(g, total, case["kv_heads"], block, case["dim"])
        ids = torch.randperm(total, generator=g, device="cuda").tolist()
        slots, at = [], 0
        for f, n, u in zip(first, lens, used):
            slots += [ids[at + (f + i) // block] * block + (f + i) % block for i in range(n)]
            at += u
        s["slots"] = torch.tensor(slots, dtype=torch.int32).cuda()
        # the newest tokens' size changes from layer to layer and token to token
        size = torch.exp(torch.randn(sum(lens), case["kv_heads"], 1, generator=g, device="cuda"))
        s["k"] = (torch.randn(sum(lens), case["kv_heads"], case["dim"], generator=g, device="cuda") * size).to(t)
        s["v"] = (torch.randn(sum(lens), case["kv_heads"], case["dim"], generator=g, device="cuda") * size).to(t)
    else:
        block, more = case["block"], _contexts(case)
        r.shuffle(more)
        have = [_blocks(c, block) for c in more]
        width = _blocks(case["context"] + case["longest"], block) + 2
        total = sum(have) + sum(_blocks(n, block) + 1 for n in lens) + 5
        ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        at = _starts(have)[:-1, None] + torch.arange(width, device="cuda")[None]
        s["table"] = torch.where(torch.arange(width, device="cuda")[None] < torch.tensor(have, device="cuda")[:, None],
                                 ids[at.clamp_max(total - 1)], -1).to(torch.int32).contiguous()
        s["free"] = ids[sum(have):].contiguous()
        s["first"] = torch.tensor([2], dtype=torch.int32, device="cuda")       # two blocks went to others before
        s["context"] = torch.tensor(more, dtype=torch.int32, device="cuda")
        s["new"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["total"] = sum(lens)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------

def _masked_attention(scores, visible, values):
    """softmax(scores) @ values over the visible keys; rows that see nothing give zeros.  Works in place on scores."""
    scores.masked_fill_(~visible, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = scores.sum(-1, keepdim=True)
    return torch.matmul(scores, values) / torch.where(total == 0, torch.ones_like(total), total)


def _plain_prompt(s):
    q, k, v, case = s["q"], s["k"], s["v"], s["case"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    nq, nk = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    iq, ik = torch.arange(s["longest_q"], device=q.device), torch.arange(s["longest_k"], device=q.device)
    at_q = (cu_q[:-1, None] + iq[None]).clamp_max(q.shape[0] - 1)
    at_k = (cu_k[:-1, None] + ik[None]).clamp_max(k.shape[0] - 1)
    qp = q.float()[at_q].reshape(-1, iq.numel(), kv, heads // kv, dim).permute(0, 2, 3, 1, 4)     # [seq, kv, group, q, dim]
    kp = k.float()[at_k].permute(0, 2, 3, 1)[:, :, None]                                          # [seq, kv, 1, dim, k]
    vp = v.float()[at_k].permute(0, 2, 1, 3)[:, :, None]
    visible = ik[None, None] < nk[:, None, None]
    if case["causal"]:
        visible = visible & (ik[None, None] <= iq[None, :, None] + (nk - nq)[:, None, None])
    o = _masked_attention(torch.matmul(qp * dim ** -0.5, kp), visible[:, None, None], vp)
    o = o.permute(0, 3, 1, 2, 4).reshape(-1, heads, dim)                                          # [seq * q, heads, dim]
    token = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(cu_q[1:], token, right=True)
    return o[seq * iq.numel() + token - cu_q[seq]].to(q.dtype)


def _plain_paged(s):
    q, c, case = s["q"], s["cache"], s["case"]
    count, n, heads, dim = q.shape
    kv = case["kv_heads"]
    at = s["table"].long().clamp_min(0)
    keys = (c["k"].float() * c["k_scale"][:, :, None, None])[at].transpose(1, 2).reshape(count, kv, -1, dim)
    vals = (c["v"].float() * c["v_scale"][:, :, None, None])[at].transpose(1, 2).reshape(count, kv, -1, dim)
    qp = (q.float() * dim ** -0.5).reshape(count, n, kv, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(count, kv, -1, dim)
    i = torch.arange(n, device=q.device).repeat_interleave(heads // kv)
    j = torch.arange(keys.shape[2], device=q.device)
    visible = j[None, None] <= (s["lens"].long()[:, None] - n + i[None])[:, :, None]
    o = _masked_attention(torch.matmul(qp, keys.transpose(-1, -2)), visible[:, None], vals)
    return o.reshape(count, kv, n, heads // kv, dim).transpose(1, 2).reshape(count, n, heads, dim).to(q.dtype)


def _plain_write(x, codes, scale, slots):
    blocks, heads, block, dim = codes.shape
    at, off = slots.long() // block, slots.long() % block
    amax = x.float().abs().amax(-1)
    need = torch.zeros_like(scale).index_reduce(0, at, _power_scale(amax), "amax")
    touched = torch.zeros(blocks, dtype=torch.bool, device=x.device).index_fill(0, at, True)[:, None]
    begun = torch.zeros(blocks, device=x.device).index_reduce(0, at, (off == 0).float(), "amax")[:, None] > 0
    new = torch.where(touched, torch.maximum(torch.where(begun, torch.zeros_like(scale), scale), need), scale)
    ratio = torch.where(touched & ~begun, scale / new, torch.ones_like(scale))
    kept = (codes.float() * ratio[:, :, None, None]).to(F8)
    kept.view(torch.uint8)[at, :, off] = (x.float() / new[at][:, :, None]).clamp(-F8_MAX, F8_MAX).to(F8).view(torch.uint8)
    return kept, new


def _plain_append(s):
    c = s["cache"]
    k, ks = _plain_write(s["k"], c["k"], c["k_scale"], s["slots"])
    v, vs = _plain_write(s["v"], c["v"], c["v_scale"], s["slots"])
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}


def _plain_plan(s):
    ctx, new, table, free = s["context"].long(), s["new"].long(), s["table"], s["free"]
    block, first = s["case"]["block"], s["first"].long()
    width = table.shape[1]
    have, want = (ctx + block - 1) // block, (ctx + new + block - 1) // block
    need = want.clamp_max(width) - have.clamp_max(width)
    before = need.cumsum(0) - need
    granted = torch.minimum((free.numel() - first - before).clamp_min(0), need)
    cu = torch.cat([torch.zeros_like(ctx[:1]), new.cumsum(0)])
    lens = torch.minimum(ctx + new, (have.clamp_max(width) + granted) * block)
    row = torch.arange(width, device=ctx.device)[None] - have[:, None]
    fresh = free[(first + before[:, None] + row).clamp(0, free.numel() - 1)]
    table = torch.where((row >= 0) & (row < granted[:, None]), fresh, table)
    t = torch.arange(s["total"], device=ctx.device)
    seq = torch.searchsorted(cu[1:], t, right=True)
    pos = ctx[seq] + t - cu[seq]
    slots = torch.where(pos < lens[seq], table[seq, (pos // block).clamp_max(width - 1)].long() * block + pos % block, -1)
    counts = torch.cat([first + granted.sum(), (want - have - granted).sum().reshape(1), cu[-1:]])
    whole = torch.int32
    return {"slots": slots.to(whole), "positions": pos.to(whole), "cu_new": cu.to(whole), "seq_lens": lens.to(whole),
            "counts": counts.to(whole), "table": table}


def run(state):
    op = state["op"]
    if own:
        ops = _ops()
        if op == "prompt_attention":
            return ops.prompt_attention(state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"],
                                        causal=state["case"]["causal"])
        if op == "block_plan":
            plan = ops.block_plan(state["context"], state["new"], state["table"], state["free"],
                                  block_size=state["case"]["block"], total_new=state["total"], first_free=state["first"])
            return {"slots": plan.slots, "positions": plan.positions, "cu_new": plan.cu_new, "seq_lens": plan.seq_lens,
                    "counts": plan.counts, "table": state["table"]}
        cache = ops.KvCache(**state["cache"])
        if op == "paged_attention":
            return ops.paged_attention(state["q"], cache, state["table"], state["lens"])
        ops.cache_append(state["k"], state["v"], cache, state["slots"])
        return state["cache"]
    return {"prompt_attention": _plain_prompt, "paged_attention": _plain_paged, "cache_append": _plain_append,
            "block_plan": _plain_plan}[op](state)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def _exact_rows(q, k, v, limit):
    """One sequence: q [n, heads, dim], k and v [keys, kv heads, dim], row i sees the first limit[i] keys."""
    n, heads, dim = q.shape
    out = torch.zeros(n, heads, dim, dtype=torch.float64, device=q.device)
    hidden = torch.arange(k.shape[0], device=q.device)[None] >= limit[:, None]
    some = (limit > 0)[:, None]
    for h in range(heads):
        kh, vh = k[:, h * k.shape[1] // heads].double(), v[:, h * k.shape[1] // heads].double()
        p = torch.softmax((q[:, h].double() @ kh.T / math.sqrt(dim)).masked_fill_(hidden & some, -math.inf), 1)
        out[:, h] = torch.where(some, p @ vh, 0.0)
    return out


def _exact_e4m3(x):
    """The value of e4m3 next to x, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-F8_MAX, F8_MAX)


def _exact_write(x, codes, scale, slots):
    block = codes.shape[2]
    codes, scale, x = codes.double(), scale.double(), x.double()
    at, off = slots.long() // block, slots.long() % block
    top = torch.zeros_like(scale)
    top.scatter_reduce_(0, at[:, None].expand(-1, scale.shape[1]), x.abs().amax(-1), "amax")
    named = torch.bincount(at, minlength=len(scale))[:, None] > 0
    begun = torch.bincount(at[off == 0], minlength=len(scale))[:, None] > 0
    powers = torch.tensor([2.0 ** i for i in range(int(math.log2(SCALE_FLOOR)), 130)], dtype=torch.float64, device=x.device)
    need = powers[torch.searchsorted(powers * F8_MAX, top.contiguous())]
    new = torch.where(named, torch.where(begun, need, torch.maximum(need, scale)), scale)
    grown = (named & ~begun & (new > scale))[:, :, None, None]
    codes = torch.where(grown, _exact_e4m3(codes * (scale / new)[:, :, None, None]), codes)
    codes[at, :, off] = _exact_e4m3(x / new[at][:, :, None])
    return codes, new


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "block_plan":
        return None                       # whole numbers
    if s["op"] == "cache_append":
        c = s["cache"]
        k, ks = _exact_write(s["k"], c["k"], c["k_scale"], s["slots"])
        v, vs = _exact_write(s["v"], c["v"], c["v_scale"], s["slots"])
        return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}
    out = []
    if s["op"] == "prompt_attention":
        cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
        for b in range(case["count"]):
            n, m = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
            limit = torch.arange(n, device="cuda") + (m - n + 1) if case["causal"] else torch.full((n,), m, device="cuda")
            out.append(_exact_rows(s["q"][cu_q[b]:cu_q[b + 1]], s["k"][cu_k[b]:cu_k[b + 1]], s["v"][cu_k[b]:cu_k[b + 1]], limit))
        return torch.cat(out)
    c, n = s["cache"], case["queries"]
    for b, m in enumerate(s["lens"].tolist()):
        ids = s["table"][b, :_blocks(m, case["block"])].long()
        k = (c["k"][ids].double() * c["k_scale"][ids].double()[:, :, None, None]).transpose(1, 2).flatten(0, 1)[:m]
        v = (c["v"][ids].double() * c["v_scale"][ids].double()[:, :, None, None]).transpose(1, 2).flatten(0, 1)[:m]
        out.append(_exact_rows(s["q"][b], k, v, torch.arange(n, device="cuda") + (m - n + 1)))
    return torch.stack(out)
