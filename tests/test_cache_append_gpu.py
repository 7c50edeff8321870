"""The cache writer, on a B200, at token counts on all sides of the rule that widens a warp's window of token rows: codes and scales equal
to the definition, block by block, in 64 bits."""
import pytest
import torch

from tests.test_cache_ops_gpu import check_append, random_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dim,tokens", [(1, 256, n) for n in (1100, 1190, 2400, 4800, 9500, 19500)] + [(2, 256, 700), (8, 128, 300), (8, 128, 1100)])
@pytest.mark.parametrize("first", [0, 11])
def test_windows_of_every_width(heads, dim, tokens, first):
    """Windows of 1, 2, 4, 8 and 16 rows; runs that begin in one window and end in the next, and blocks begun by another call."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    d, block = torch.device("cuda"), 16
    blocks = (first + tokens) // block + 3
    cache = random_cache(71, blocks, heads, block, dim, d)
    g = torch.Generator(device=d).manual_seed(72)
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(3)).tolist()
    slots = [order[(first + i) // block] * block + (first + i) % block for i in range(tokens)]
    size = torch.exp2(torch.randint(-6, 7, (tokens, heads, 1), generator=g, device=d).float())
    k = (torch.randn(tokens, heads, dim, generator=g, device=d) * size).to(torch.bfloat16)
    check_append(k, k.flip(0), cache, torch.tensor(slots, dtype=torch.int32, device=d))
