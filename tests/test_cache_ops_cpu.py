"""What the C entry points and the wrappers of the operators around a key/value cache in pages refuse, without a GPU: every
refusal comes before a launch, with a code and a message."""
import ctypes as C
import os

import pytest
import torch

import _capi
import vla_ops

needs_library = pytest.mark.skipif(not os.path.exists(_capi.LIB_PATH), reason="library not built")
P = 4096          # an address for arguments that are only checked, never followed


def call(name, desc):
    lib = _capi.lib()
    rc = getattr(lib, name)(C.byref(desc) if desc is not None else None, None)
    return rc, lib.vla_last_error(None).decode()


def plan_desc(**kw):
    d = _capi.BlockPlanDesc(P, P, 2, P, 4, 4, P, 8, None, 16, 5, P, P, P, P, P)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def append_desc(**kw):
    d = _capi.CacheAppendDesc(P, P, P, 3, 256, 128, 256, 128, P, P, P, P, 8, 2, 16, 128, _capi.VLA_BF16)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def paged_desc(**kw):
    d = _capi.PagedAttnDesc(P, P, 1024, 1024, 128, 1024, 1024, 128, P, P, P, P, P, 4, P, 2, 1, 8, 2, 128, 8, 16, 4, 0.1, _capi.VLA_BF16)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def prompt_desc(**kw):
    d = _capi.PromptAttnDesc(P, P, P, P, P, P, 2, 9, 9, 8, 2, 128, 1024, 128, 256, 128, 256, 128, 1024, 128, 1, 0.1, _capi.VLA_BF16)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


STATE, SHAPE, LIMIT = 4, 3, 5
CASES = [
    ("vla_op_block_plan", plan_desc, [
        (STATE, dict(context_lens=None)), (STATE, dict(block_table=None)), (STATE, dict(free_blocks=None)), (STATE, dict(slots=None)),
        (STATE, dict(counts=None)), (STATE, dict(seq_lens=None)), (SHAPE, dict(block_size=0)), (SHAPE, dict(total_new=-1)),
        (SHAPE, dict(table_stride=3)), (SHAPE, dict(slots=P + 4)), (LIMIT, dict(n_seqs=8193)), (LIMIT, dict(n_seqs=-1))]),
    ("vla_op_cache_append", append_desc, [
        (STATE, dict(k=None)), (STATE, dict(slots=None)), (STATE, dict(v_codes=None)), (STATE, dict(k_scale=None)), (SHAPE, dict(tokens=-1)),
        (SHAPE, dict(head_dim=96)), (SHAPE, dict(head_dim=0)), (SHAPE, dict(block_size=8)), (SHAPE, dict(block_size=272)),
        (SHAPE, dict(dtype=_capi.VLA_F32)), (SHAPE, dict(k=P + 2)), (SHAPE, dict(v_tok_stride=257)), (SHAPE, dict(k_codes=P + 8)),
        (SHAPE, dict(kv_heads=0)), (LIMIT, dict(num_blocks=2 ** 27))]),
    ("vla_op_paged_attention", paged_desc, [
        (STATE, dict(q=None)), (STATE, dict(o=None)), (STATE, dict(block_table=None)), (STATE, dict(seq_lens=None)), (STATE, dict(v_scale=None)),
        (SHAPE, dict(heads=7)), (SHAPE, dict(heads=0)), (SHAPE, dict(kv_heads=0)), (SHAPE, dict(n_q=0)), (SHAPE, dict(head_dim=72)),
        (SHAPE, dict(block_size=24)), (SHAPE, dict(dtype=_capi.VLA_F32)), (SHAPE, dict(scale=0.0)), (SHAPE, dict(scale=float("nan"))),
        (SHAPE, dict(scale=float("inf"))), (SHAPE, dict(q=P + 8)), (SHAPE, dict(o_head_stride=4)), (SHAPE, dict(table_stride=3)),
        (SHAPE, dict(num_blocks=0)), (LIMIT, dict(n_q=2 ** 20)), (LIMIT, dict(width=2 ** 28, table_stride=2 ** 28))]),
    ("vla_op_prompt_attention", prompt_desc, [
        (STATE, dict(q=None)), (STATE, dict(v=None)), (STATE, dict(cu_k=None)), (STATE, dict(o=None)), (SHAPE, dict(heads=3)),
        (SHAPE, dict(head_dim=4)), (SHAPE, dict(head_dim=264)), (SHAPE, dict(head_dim=100)), (SHAPE, dict(tokens_q=-1)), (SHAPE, dict(n_seqs=-2)),
        (SHAPE, dict(dtype=7)), (SHAPE, dict(scale=-1.0)), (SHAPE, dict(k=P + 4)), (SHAPE, dict(v_tok_stride=4)), (LIMIT, dict(heads=129, kv_heads=1))]),
]


@needs_library
@pytest.mark.parametrize("name,make,code,change", [(n, m, c, k) for n, m, cases in CASES for c, k in cases])
def test_entry_points_refuse(name, make, code, change):
    rc, text = call(name, make(**change))
    assert rc == code and name in text


@needs_library
def test_paged_workspace():
    """Nothing where one CTA does a unit; else what the sizes ask for, and the call refuses less or none."""
    need = C.c_size_t(1)
    f = _capi.lib().vla_op_paged_attention_workspace
    assert f(C.byref(paged_desc()), C.byref(need)) == 0 and need.value == 0
    long = paged_desc(width=200, table_stride=200)
    assert f(C.byref(long), C.byref(need)) == 0 and need.value > 0
    for kw in (dict(), dict(workspace=P, workspace_bytes=need.value - 1), dict(workspace=P + 4, workspace_bytes=need.value)):
        rc, text = call("vla_op_paged_attention", paged_desc(width=200, table_stride=200, **kw))
        assert rc == STATE and "workspace" in text
    assert f(C.byref(paged_desc(heads=7)), C.byref(need)) == SHAPE
    assert f(None, C.byref(need)) == STATE and f(C.byref(long), None) == STATE


@needs_library
@pytest.mark.parametrize("name", [c[0] for c in CASES])
def test_null_descriptor(name):
    assert call(name, None)[0] == STATE


@needs_library
@pytest.mark.parametrize("name,desc", [("vla_op_cache_append", append_desc(tokens=0, k=None, v=None, slots=None)),
                                       ("vla_op_paged_attention", paged_desc(n_seqs=0, q=None)),
                                       ("vla_op_prompt_attention", prompt_desc(n_seqs=0)), ("vla_op_prompt_attention", prompt_desc(tokens_q=0, q=None))])
def test_nothing_to_do_is_no_error(name, desc):
    assert call(name, desc)[0] == 0


def test_wrappers_refuse_the_cpu():
    q, i = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    cache = vla_ops.kv_cache(2, 2, 16, 64, "cpu")
    assert cache.k.shape == (2, 2, 16, 64) and cache.k.dtype == torch.float8_e4m3fn and cache.v_scale.shape == (2, 2)
    for f in (lambda: vla_ops.prompt_attention(q, q, q, i), lambda: vla_ops.paged_attention(q[None], cache, i[None], i[:1]),
              lambda: vla_ops.cache_append(q[:, :2], q[:, :2], cache, i), lambda: vla_ops.block_plan(i, i, i[None], i, block_size=16, total_new=0)):
        with pytest.raises(_capi.VlaError, match="no CPU path"):
            f()


@needs_library
def test_wrappers_refuse_what_is_no_tensor():
    i = torch.zeros(2, dtype=torch.int32)
    for f in (lambda: vla_ops.prompt_attention(None, i, i, i), lambda: vla_ops.paged_attention([1.0], None, i, i),
              lambda: vla_ops.cache_append(3, i, None, i), lambda: vla_ops.block_plan("x", i, i, i, block_size=16, total_new=0)):
        with pytest.raises(_capi.VlaError, match="must be a tensor"):
            f()


@needs_library
def test_status_refusals():
    lib = _capi.lib()
    assert lib.vla_op_cache_status(None) == STATE and "null" in lib.vla_last_error(None).decode()
    for limit in (0, -1, 1000001):
        assert lib.vla_op_cache_wait_expire(limit, None) == LIMIT and "microseconds" in lib.vla_last_error(None).decode()


IMPORTS = """
import torch, _capi, vla_ops
assert all(callable(getattr(vla_ops, f)) for f in ("gemm", "attention", "norm", "attention_tc"))
i = torch.zeros(1, dtype=torch.int32)
try:
    vla_ops.block_plan(i, i, i[None], i, block_size=16, total_new=0)
except _capi.VlaError as e:
    print("refused:", e)
"""


def test_a_binding_that_does_not_load_leaves_the_rest(tmp_path):
    """A file of another torch, another Python or half a build: what goes through ctypes alone is still there, and the operators that
    need the binding say why they are not."""
    import subprocess
    import sys
    (tmp_path / "_vla_ops.so").write_bytes(b"no shared object")
    package = os.path.dirname(os.path.abspath(vla_ops.__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([str(tmp_path), package]))
    done = subprocess.run([sys.executable, "-c", IMPORTS], env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "refused:" in done.stdout and "_vla_ops.so" in done.stdout, done.stderr[-2000:]


def test_the_binding_is_rebuilt_for_another_torch_or_python(monkeypatch):
    import build
    made_for = build._made_for()
    assert made_for and build._made_for() == made_for
    monkeypatch.setattr(build, "_stale", lambda target, inputs: False)
    monkeypatch.setattr(build, "_read", lambda path: made_for)
    assert not build._binding_stale()
    monkeypatch.setattr(build, "_read", lambda path: made_for.replace("torch", "torch 0 "))
    assert build._binding_stale()


def test_building_needs_no_torch_for_the_c_library(monkeypatch, capsys):
    """Without torch, or when only the C library is asked for, nothing is said to be missing and no binding is tried."""
    import build
    ran = []
    monkeypatch.setattr(build, "_stale", lambda target, inputs: target == build.BINDING)
    monkeypatch.setattr(build.subprocess, "run", lambda command, **kw: ran.append(command))
    assert build.needs_build() and not build.needs_build(binding=False)
    assert build.build(binding=False) == build.LIB and not ran
    monkeypatch.setattr(build, "find_spec", lambda name: None)
    assert not build.needs_build()
    assert build.build() == build.LIB and not ran
    assert build.build(force=False) == build.LIB
    monkeypatch.setattr(build, "_stale", lambda target, inputs: True)
    monkeypatch.setattr(build.subprocess, "Popen", lambda command, **kw: type("Done", (), {"wait": lambda self: 0})())
    build.build()
    assert len(ran) == 1 and ran[0][-1].endswith(".o") and "no torch" in capsys.readouterr().err


def test_a_binding_that_does_not_compile_names_the_library_that_is_there(monkeypatch):
    import build

    def run(command, **kw):
        if command[0] == "g++":
            raise build.subprocess.CalledProcessError(1, command)

    monkeypatch.setattr(build, "_stale", lambda target, inputs: target == build.BINDING)
    monkeypatch.setattr(build.subprocess, "run", run)
    with pytest.raises(RuntimeError, match="libvla_b200.so is complete"):
        build.build()


@needs_library
@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are only good where nothing can be launched")
def test_first_calls_from_several_threads_without_a_driver():
    """Every one of them says that there is no driver, and none blames the strides."""
    import threading
    said = []

    def first():
        for name, desc in (("vla_op_prompt_attention", prompt_desc()), ("vla_op_paged_attention", paged_desc())):
            said.append(call(name, desc))

    threads = [threading.Thread(target=first) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(said) == 16 and all(rc == 1 and "driver" in text for rc, text in said)


@needs_library
@pytest.mark.parametrize("change", [dict(n_seqs=2 ** 31 - 1, n_q=1, heads=2 ** 20, kv_heads=2 ** 20, width=2 ** 20, table_stride=2 ** 20),
                                    dict(n_seqs=2 ** 31 - 1, n_q=2 ** 13, heads=2 ** 7, kv_heads=2 ** 7, width=2 ** 26, table_stride=2 ** 26),
                                    dict(n_seqs=2 ** 30, heads=8, kv_heads=8, width=2 ** 26, table_stride=2 ** 26)])
def test_sizes_whose_products_leave_64_bits(change):
    """Refused by the question for the workspace as by the call, before any product is formed."""
    need = C.c_size_t(77)
    desc = paged_desc(**change)
    assert _capi.lib().vla_op_paged_attention_workspace(C.byref(desc), C.byref(need)) == LIMIT and need.value == 77
    assert call("vla_op_paged_attention", desc)[0] == LIMIT
