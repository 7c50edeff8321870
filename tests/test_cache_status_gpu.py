"""The status word of the operators around a key/value cache in pages: a bounded wait that runs out on any stream is seen, once."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def expire(us, stream):
    import _capi
    _capi.check(_capi.lib().vla_op_cache_wait_expire(us, stream.cuda_stream))


@pytest.fixture
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import vla_ops
    vla_ops.cache_status()
    return vla_ops


def test_nothing_has_run_out(ops):
    assert ops.cache_status() == 0 and ops.cache_status("cuda") == 0 and ops.cache_status(torch.device("cuda", 0)) == 0


def test_a_wait_that_runs_out_is_seen_once(ops):
    expire(1000, torch.cuda.current_stream())
    assert ops.cache_status() == 1
    assert ops.cache_status() == 0


def test_a_wait_on_a_side_stream_is_waited_for(ops):
    """torch's side streams do not wait for the default stream, nor it for them: the word is read after their work all the same."""
    side = torch.cuda.Stream()
    for _ in range(3):
        expire(200000, side)
        assert ops.cache_status() == 1
    assert ops.cache_status() == 0


def test_operators_work_after_it(ops):
    q = torch.randn(20, 8, 128, device="cuda").bfloat16()
    cu = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    want = ops.prompt_attention(q, q, q, cu)
    expire(1000, torch.cuda.current_stream())
    assert torch.equal(ops.prompt_attention(q, q, q, cu), want)
    assert ops.cache_status() == 1
    assert ops.cache_status() == 0


def test_replayed_waits_are_seen(ops):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        expire(1000, torch.cuda.current_stream())
    assert ops.cache_status() == 0
    for _ in range(2):
        graph.replay()
        assert ops.cache_status() == 1


REFUSED_LAUNCH = """
import torch, _capi, vla_ops
x, slots = torch.ones(4, 1, 64, device="cuda").bfloat16(), torch.arange(4, dtype=torch.int32, device="cuda")
cache = vla_ops.kv_cache(1, 1, 16, 64)
torch.cuda.synchronize()
refused = False
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        try:
            torch.cuda.synchronize()                 # ends the capture
        except RuntimeError:
            pass
        try:
            vla_ops.cache_append(x, x, cache, slots)
        except _capi.VlaError:
            refused = True
except RuntimeError:
    pass
assert refused
assert vla_ops.cache_status() == 0
vla_ops.cache_append(x, x, cache, slots)
assert cache.k[0, 0, :4].float().abs().min() > 0
print("works")
"""


def test_a_launch_that_is_refused_leaves_no_error_behind(ops):
    """A launch into a capture that has become invalid is refused; the library's next call does not find that error."""
    import os
    import subprocess
    import sys
    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.abspath(ops.__file__)))
    done = subprocess.run([sys.executable, "-c", REFUSED_LAUNCH], env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "works" in done.stdout, done.stderr[-2000:]
