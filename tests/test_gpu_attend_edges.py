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


@pytest.mark.parametrize("dt,cdt", [(BF, BF), (F16, F16), (BF, F8), (F16, F8)])
@pytest.mark.parametrize("new", [1, 3])
def test_error_is_that_of_the_outputs_rounding(cuda_device, dt, cdt, new):
    """The error against 64 bits, root of the mean square, beside that of the exact result rounded once.

    Both are sums of many independent roundings.  Probabilities in two parts, scores and sums in 32 bits add less than
    2^-15 to an output rounded to 2^-12.8 (f16) or more; in one f16 part (bf16 queries over e4m3) 2^-12.8 to 2^-9.8: less
    than 3 % in quadrature either way.  One f16 part under an f16 output would add as much as its rounding (up to 41 %)."""
    gen = torch.Generator().manual_seed(7)
    kv = torch.randn((2, 2, 700, 128), generator=gen)
    scales = {}
    if cdt == F8:
        kv = kv * 16
        scales = {n: torch.tensor([s, 2 * s], device=cuda_device) for n, s in (("k_scale", 0.05), ("v_scale", 0.07))}
    kv = kv.to(cdt)
    cache = one_text(cuda_device, kv, 40, **scales)
    q = torch.randn((40, new, 16, 128), generator=gen).to(dt).to(cuda_device)
    out = cache.attend(0, q).double()
    k, v = kv.double().to(cuda_device)
    if scales:
        k, v = (x * s.double()[:, None, None] for x, s in zip((k, v), scales.values()))
    score = torch.einsum("blhgd,hnd->blhgn", q.double().view(40, new, 2, 8, 128), k) * 128 ** -0.5
    at = torch.arange(700, device=cuda_device)
    hidden = at > 700 - new + torch.arange(new, device=cuda_device)[:, None]
    p = score.masked_fill(hidden[None, :, None, None], -math.inf).softmax(-1)
    want = torch.einsum("blhgn,hnd->blhgd", p, v).reshape(40, new, 16, 128)
    once = (want.to(dt).double() - want).square().mean().sqrt()
    assert (out - want).square().mean().sqrt() <= 1.03 * once


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("group,new,dim,n", [(8, 1, 128, 40), (8, 1, 128, 20000), (5, 4, 80, 700), (128, 1, 128, 700),
                                             (64, 4, 64, 9000), (16, 2, 256, 300), (64, 1, 256, 300)])
def test_infinite_values_that_are_seen(cuda_device, dt, group, new, dim, n):
    """Weights are positive, so an infinite value makes its dimension infinite, values of both signs or a NaN make it
    NaN, wherever they stand and however the sequence is split; the other dimensions do not change."""
    gen = torch.Generator().manual_seed(n)
    kv = torch.randn((2, 2, n, dim), generator=gen).to(dt)
    q = torch.randn((3, new, 2 * group, dim), generator=gen).to(dt).to(cuda_device)
    plain = one_text(cuda_device, kv, 3).attend(0, q)
    where = [0, n // 3, n // 2 + 5, n - new]
    for i, at in enumerate(where):
        kv[1, 1, at, 8 * i % dim] = math.inf
        kv[1, 1, at, 8 * i % dim + 1] = -math.inf
        kv[1, 1, at, 8 * i % dim + 3] = math.nan
        kv[1, 1, at, 8 * i % dim + 6] = math.inf
    kv[1, 1, n // 4, 6] = -math.inf
    out, lse = one_text(cuda_device, kv, 3).attend(0, q, return_lse=True)
    want = plain.clone()
    for i in range(len(where)):
        d = 8 * i % dim
        want[:, :, group:, d] = math.inf
        want[:, :, group:, d + 1] = -math.inf
        want[:, :, group:, d + 3] = math.nan
        want[:, :, group:, d + 6] = math.nan if d == 0 else math.inf
    # other dimensions: rows of a tile that holds such values may be summed in another order
    torch.testing.assert_close(out, want, rtol=2 * ROUND[dt], atol=2.0 ** -10, equal_nan=True)
    assert torch.isfinite(lse).all()


@pytest.mark.parametrize("dt", [BF, F16])
def test_infinite_values_outside_the_window(cuda_device, dt):
    """The single token sees what its window holds; NaN and infinities in other heads, before it or past it stay out."""
    n, window = 900, 64
    kv = torch.randn((2, 1, n, 128), generator=torch.Generator().manual_seed(1)).to(dt)
    kv[1, 0, n - window, 0] = math.inf
    kv[1, 0, n - window - 1, :2] = -math.inf
    kv[1, 0, :100] = math.nan
    q = torch.randn((1, 8, 128), generator=torch.Generator().manual_seed(2)).to(dt).to(cuda_device)
    out = one_text(cuda_device, kv, 1).attend(0, q, window=window)
    assert (out[..., 0] == math.inf).all() and torch.isfinite(out[..., 1:]).all()


@pytest.mark.parametrize("dt,cdt", [(BF, BF), (F16, F8)])
def test_a_scale_that_is_not_a_number_is_not_hidden(cuda_device, dt, cdt):
    kv = torch.randn((2, 2, 70, 64), generator=torch.Generator().manual_seed(1)).to(cdt)
    q = torch.randn((1, 2, 8, 64), generator=torch.Generator().manual_seed(2)).to(dt).to(cuda_device)
    out, lse = one_text(cuda_device, kv, 1).attend(0, q, scale=math.nan, return_lse=True)
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    if cdt == F8:
        cache = one_text(cuda_device, kv, 1, k_scale=torch.tensor([1.0, math.nan], device=cuda_device))
        out = cache.attend(0, q)
        assert torch.isfinite(out[:, :, :4]).all() and torch.isnan(out[:, :, 4:]).all()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 40])
def test_a_window_longer_than_any_sequence(cuda_device, window):
    kv = torch.randn((2, 1, 3, 64), generator=torch.Generator().manual_seed(1)).to(BF)
    cache = one_text(cuda_device, kv, 2)
    q = torch.randn((2, 9, 4, 64), generator=torch.Generator().manual_seed(2)).to(BF).to(cuda_device)
    out, lse = cache.attend(0, q, window=window, return_lse=True)  # the first six tokens see nothing
    want, wlse = cache.attend(0, q, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    assert not out[:, :6].any() and (lse[:, :6] == -math.inf).all()


@pytest.mark.parametrize("dt", [BF, F16])
def test_values_that_are_all_infinite(cuda_device, dt):
    """Every output is looked up, in whole and in split sequences, and one of another sign anywhere makes it NaN."""
    n, group = 5000, 6
    kv = torch.randn((2, 2, n, 96), generator=torch.Generator().manual_seed(1)).to(dt)
    kv[1] = -math.inf
    kv[1, 1, 4321, 95] = math.inf
    q = torch.randn((40, 2, 2 * group, 96), generator=torch.Generator().manual_seed(2)).to(dt).to(cuda_device)
    cache = one_text(cuda_device, kv, 40)
    for rows in (40, 2):
        out = cache.attend(0, q[:rows])
        assert (out[:, :, :group] == -math.inf).all() and (out[:, :, group:, :95] == -math.inf).all()
        assert torch.isnan(out[:, :, group:, 95]).all()
    assert cache.check_device_status() == 0
