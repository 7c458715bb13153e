"""Paged attention where its arithmetic is near its limits, against values known in closed form."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
ROUND = {BF: 2.0 ** -8, F16: 2.0 ** -11}


def one_text(dev, kv, rows, **kw):
    """A cache of ``rows`` sequences that all hold the same tokens, kv [2, kv_heads, tokens, dim]."""
    from xcalibur_b200 import PagedKVCache

    _, heads, n, dim = kv.shape
    ps = 32
    pages = -(-n // ps)
    pool = torch.zeros((2, heads, pages * ps, dim), dtype=kv.dtype, device=dev)
    pool.view(torch.uint8)[:, :, :n] = kv.to(dev).view(torch.uint8)
    pool = pool.view(2, heads, pages, ps, dim).transpose(1, 2).contiguous()[None]
    table = torch.arange(pages, dtype=torch.int32, device=dev).expand(rows, pages).contiguous()
    return PagedKVCache.from_tensors(pool, table, torch.full((rows,), n, dtype=torch.int32, device=dev), **kw)


@pytest.mark.parametrize("dt,cdt", [(BF, BF), (F16, F16), (BF, F8), (F16, F8)])
@pytest.mark.parametrize("group", [1, 20, 128])
@pytest.mark.parametrize("gap", [12.0, 16.0, 18.0])
def test_small_probabilities_beside_a_large_one(cuda_device, dt, cdt, group, gap):
    """The first token takes nearly all weight and holds nothing: the result is what the others hold, each with a weight
    of e^-gap.

    A weight is off by 2^-10 of itself at most (half an f16 step of 2^-24 against a weight of 2^-15 or more), and the
    32-bit sums and exponentials by 2^-13; the result is rounded once."""
    n, rows = 513, 300
    kv = torch.zeros((2, 1, n, 128))
    kv[0, 0, 0, 0] = gap / 4
    kv[1, 0, 1:] = 64.0
    cache = one_text(cuda_device, kv.to(cdt), rows)
    q = torch.zeros((rows, group, 128), dtype=dt, device=cuda_device)
    q[..., 0] = 4.0
    out, lse = cache.attend(0, q, scale=1.0, return_lse=True)
    rest = (n - 1) * math.exp(-gap)
    want = 64.0 * rest / (1 + rest)
    assert (out.double() - want).abs().max() <= want * (2.0 ** -10 + 2.0 ** -13 + ROUND[dt])
    assert (lse.double() - gap - math.log1p(rest)).abs().max() <= 2.0 ** -20 + n * 2.0 ** -23 + 2.0 ** -21 * gap
