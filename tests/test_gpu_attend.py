"""Paged attention against its plain 64-bit form: types, head layouts, lengths from nothing to thousands, odd page
sizes, masks that leave a row empty, and whatever may lie in places that are not seen."""
import math

import pytest
import torch

from tests import _attn_ref as ref

pytestmark = pytest.mark.gpu

BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def make(dev, lens, kv_heads, dim, ps, dtype, *, layers=1, spare=3, seed=0, poison=True):
    """A cache with the given lengths over shuffled pages; slots past a length and free pages hold NaN."""
    from xcalibur_b200 import PagedKVCache

    gen = torch.Generator().manual_seed(seed)
    each = [-(-n // ps) for n in lens]
    pages = sum(each) + spare
    ids = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((len(lens), max(each + [1]) + 1), -1, dtype=torch.int32)
    kv = torch.randn((layers, 2, pages, kv_heads, ps, dim), generator=gen)
    live = torch.zeros(pages, ps, dtype=torch.bool)
    for s, n in enumerate(each):
        for j in range(n):
            table[s, j] = ids.pop()
            live[table[s, j], : min(ps, lens[s] - j * ps)] = True
    scales = {}
    if dtype == F8:
        kv = kv * 16
        scales = {n: (torch.rand(kv_heads, generator=gen) + 0.5) / 16 for n in ("k_scale", "v_scale")}
    if poison:
        kv = kv.masked_fill(~live[None, None, :, None, :, None], math.nan)
    cache = PagedKVCache.from_tensors(kv.to(dtype).to(dev), table.to(dev),
                                      torch.tensor(lens, dtype=torch.int32, device=dev),
                                      **{n: x.to(dev) for n, x in scales.items()})
    return cache


def queries(dev, batch, new, heads, dim, dtype, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn((batch, new, heads, dim), generator=gen).to(dtype).to(dev)


def check(cache, q, out, lse, **kw):
    w_out, w_lse, t_out, t_lse = ref.attend(cache.kv, cache.page_table, cache.seq_lens, q, k_scale=cache.k_scale,
                                            v_scale=cache.v_scale, **kw)
    ref.assert_within(out, w_out, t_out)
    ref.assert_within(lse, w_lse, t_lse)


CASES = [
    # q_heads, kv_heads, dim, page, q dtype, cache dtype, new, window, lens
    (32, 4, 128, 64, BF, BF, 1, 0, [1, 64, 65, 777, 0, 5000, 128, 127]),
    (5, 5, 64, 16, F16, F16, 1, 0, [17, 1, 300]),
    (14, 2, 80, 24, BF, BF, 3, 100, [0, 1, 2, 3, 150, 1031]),
    (16, 1, 256, 32, BF, BF, 2, 0, [1, 31, 33, 700]),
    (40, 8, 96, 1, F16, F16, 1, 0, [3, 130, 0]),
    (64, 8, 128, 64, BF, F8, 1, 0, [1, 2000, 63, 64, 0, 700]),
    (12, 4, 80, 24, F16, F8, 4, 33, [2, 4, 5, 200]),
    (8, 2, 64, 128, BF, F8, 2, 0, [1, 129, 1000]),
    (6, 2, 256, 48, F16, F8, 1, 0, [500, 3]),
    (6, 2, 192, 16, BF, BF, 1, 50, [500, 3, 50, 51]),
    (128, 8, 128, 64, BF, BF, 8, 0, [5, 8, 9, 900]),           # 128 rows of a head: one tile
    (64, 2, 64, 32, F16, F16, 8, 200, [7, 700]),               # 256 rows: two tiles
    (16, 1, 256, 64, F16, F16, 8, 0, [3, 600]),                # 128 rows at the widest head: two tiles
    (33, 3, 128, 64, BF, F8, 5, 0, [1, 400]),                  # 55 rows of 64
    (36, 2, 128, 64, BF, F8, 7, 64, [6, 500]),                 # 126 rows of 128, 8-bit
    (24, 8, 16, 8, BF, BF, 1, 0, [100, 9]),                    # narrow heads
    (4, 4, 128, 16, BF, BF, 200, 0, [150, 333]),               # a prompt's chunk as queries
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-p{c[3]}-n{c[6]}-w{c[7]}")
def test_attend_matches_plain_form(cuda_device, case):
    hq, hkv, dim, ps, dt, cdt, new, window, lens = case
    cache = make(cuda_device, lens, hkv, dim, ps, cdt)
    q = queries(cuda_device, len(lens), new, hq, dim, dt)
    out, lse = cache.attend(0, q, window=window, return_lse=True)
    check(cache, q, out, lse, window=window)
    assert cache.check_device_status() == 0


@pytest.mark.parametrize("case", [
    (8, 2, 128, 4, BF, BF, 1, 0, [1, 4, 5, 250]),
    (8, 2, 128, 12, F16, F16, 2, 30, [2, 12, 13, 411]),
    (8, 1, 64, 20, BF, F8, 1, 0, [19, 20, 21, 900]),
    (16, 2, 128, 20, BF, F8, 3, 0, [3, 40, 41, 1300]),         # 24 rows of 32, 8-bit
    (24, 2, 96, 7, F16, F8, 2, 90, [2, 7, 0, 513]),            # 24 rows, a page that is no power of two
    (4, 4, 48, 5, BF, F8, 1, 3, [1, 2, 3, 4, 6, 100]),
], ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-p{c[3]}-n{c[6]}-w{c[7]}")
def test_attend_over_odd_pages(cuda_device, case):
    test_attend_matches_plain_form(cuda_device, case)


@pytest.mark.parametrize("new", [1, 3])
def test_many_ragged_8_bit_sequences(cuda_device, new):
    lens = [(i * 97) % 900 for i in range(200)]
    cache = make(cuda_device, lens, 2, 128, 32, F8)
    q = queries(cuda_device, len(lens), new, 16, 128, BF)
    out, lse = cache.attend(0, q, return_lse=True)
    check(cache, q, out, lse)
    again, lse2 = cache.attend(0, q, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("cdt", [BF, F8])
def test_long_sequences_split_over_the_gpu(cuda_device, cdt):
    cache = make(cuda_device, [40000, 3, 12345], 2, 128, 64, cdt)
    q = queries(cuda_device, 3, 1, 16, 128, BF)
    out, lse = cache.attend(0, q, return_lse=True)
    check(cache, q, out, lse)
    again, lse2 = cache.attend(0, q, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2), "the order of joins must not depend on timing"


def test_many_short_sequences(cuda_device):
    lens = [(i * 37) % 90 for i in range(600)]
    cache = make(cuda_device, lens, 1, 64, 16, BF)
    q = queries(cuda_device, len(lens), 1, 3, 64, BF)
    out, lse = cache.attend(0, q, return_lse=True)
    check(cache, q, out, lse)


def test_single_token_form_strides_scale_layers_and_sequence_ids(cuda_device):
    dev = cuda_device
    cache = make(dev, [100, 40, 7, 260], 2, 128, 32, BF, layers=3)
    wide = queries(dev, 5, 1, 12, 128, BF)          # queries are the first 8 heads of a wider projection
    q = wide[:, 0, :8]
    seqs = torch.tensor([3, 1, 1, 0, 2], dtype=torch.int32, device=dev)
    out, lse = cache.attend(2, q, seqs=seqs, scale=0.3, return_lse=True)
    assert out.shape == (5, 8, 128) and lse.shape == (5, 8)
    check(cache, q.unsqueeze(1), out.unsqueeze(1), lse.unsqueeze(1), layer=2, seqs=seqs, scale=0.3)
    given = torch.empty_like(out)
    assert cache.attend(2, q, seqs=seqs, scale=0.3, out=given) is given and torch.equal(given, out)
    odd = torch.empty(5 * 8 * 128 + 1, dtype=BF, device=dev)[1:].view(5, 8, 128)   # not 16-byte aligned: copied
    odd.copy_(q)
    assert torch.equal(cache.attend(2, odd, seqs=seqs, scale=0.3), out)


def test_unknown_sequences_and_missing_pages(cuda_device):
    from xcalibur_b200 import _lib

    dev = cuda_device
    cache = make(dev, [100, 90, 50], 2, 64, 16, F16)
    q = queries(dev, 4, 1, 4, 64, F16)
    seqs = torch.tensor([0, 7, 2, -1], dtype=torch.int32, device=dev)
    out, lse = cache.attend(0, q, seqs=seqs, return_lse=True)
    check(cache, q, out, lse, seqs=seqs)
    assert cache.check_device_status() == _lib.XCB_STATUS_BAD_SEQ
    cache.page_table[0, 2] = -1                      # a page given back from the middle
    cache.page_table[1, 0] = cache.num_pages         # an id past the pool
    cache.page_table[2, :] = -1                      # nothing left
    out, lse = cache.attend(0, q[:3], return_lse=True)
    check(cache, q[:3], out, lse)
    assert torch.all(out[2] == 0) and torch.all(lse[2] == -math.inf)
    assert cache.check_device_status() == _lib.XCB_STATUS_BAD_PAGE
    cache.seq_lens[1] = -5
    assert torch.all(cache.attend(0, q[:3])[1] == 0)
    cache.seq_lens[1] = 2 ** 31 - 1                  # longer than its row of the table
    cache.attend(0, q[:3])
    assert cache.check_device_status() & _lib.XCB_STATUS_BAD_PAGE


@pytest.mark.parametrize("dt,cdt", [(BF, BF), (F16, F16), (BF, F8)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_hidden_from_a_token_does_not_reach_it(cuda_device, dt, cdt, bad):
    """Draft tokens see the ones before them only: a value that is not finite in a later one, or before the window,
    stays out."""
    if cdt == F8 and math.isinf(bad):
        pytest.skip("e4m3 has no infinities")
    new, window, n = 4, 40, 150
    cache = make(cuda_device, [n], 2, 128, 16, cdt)
    raw = cache.kv
    vals = raw.float()
    page = lambda pos: int(cache.page_table[0, pos // 16])  # noqa: E731
    for pos in (n - 1, n - new + 1 - window):  # the last token; the oldest one that only the first draft sees
        vals[0, 1, page(pos), :, pos % 16, 5] = bad
        vals[0, 0, page(pos), :, pos % 16, 7] = bad
    cache.kv.copy_(vals.to(cdt))
    q = queries(cuda_device, 1, new, 8, 128, dt)
    out = cache.attend(0, q, window=window)
    clean = make(cuda_device, [n], 2, 128, 16, cdt)
    want, _, tol, _ = ref.attend(clean.kv, clean.page_table, clean.seq_lens, q, window=window, k_scale=clean.k_scale,
                                 v_scale=clean.v_scale)
    ref.assert_within(out[:, 1:3], want[:, 1:3], tol[:, 1:3])
    assert not torch.isfinite(out[:, 0]).all() and not torch.isfinite(out[:, 3]).all()


@pytest.mark.parametrize("size", [1e-30, 3e3])
def test_scores_of_any_size(cuda_device, size):
    """Vanishing queries give the mean of the values, huge ones the value of the best key."""
    cache = make(cuda_device, [300, 5], 2, 128, 64, BF)
    q = (queries(cuda_device, 2, 1, 16, 128, BF).float() * size).to(BF)
    out, lse = cache.attend(0, q, return_lse=True)
    check(cache, q, out, lse)
    cache8 = make(cuda_device, [300, 5], 2, 128, 64, F8)
    out, lse = cache8.attend(0, q, return_lse=True)
    check(cache8, q, out, lse)


def test_cache_past_32_bit_offsets(cuda_device):
    """Pages whose byte offset in the keys' plane is above 2^32."""
    from xcalibur_b200 import PagedKVCache

    dev, ps, dim, heads = cuda_device, 64, 128, 2
    pages = (1 << 32) // (heads * ps * dim * 2) + 40
    kv = torch.empty((1, 2, pages, heads, ps, dim), dtype=BF, device=dev)
    table = torch.arange(pages - 1, pages - 33, -1, dtype=torch.int32, device=dev).view(2, 16)
    kv[:, :, table.flatten().long()] = torch.randn((1, 2, 32, heads, ps, dim), device=dev,
                                                   generator=torch.Generator(dev).manual_seed(3)).to(BF)
    cache = PagedKVCache.from_tensors(kv, table, torch.tensor([1000, 16], dtype=torch.int32, device=dev))
    q = queries(dev, 2, 1, 8, dim, BF)
    out, lse = cache.attend(0, q, return_lse=True)
    check(cache, q, out, lse)


def test_other_stream_and_graph(cuda_device):
    dev = cuda_device
    cache = make(dev, [4000, 100], 2, 128, 64, BF)
    q = queries(dev, 2, 1, 8, 128, BF)
    want = cache.attend(0, q)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = cache.attend(0, q)
        graph_out = torch.empty_like(want)
        cache.attend(0, q, out=graph_out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        graph_out.zero_()
        with torch.cuda.graph(graph, stream=side):
            cache.attend(0, q, out=graph_out)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize(dev)
    assert torch.equal(got, want) and torch.equal(graph_out, want)


def test_parts_join_by_their_lse(cuda_device):
    """Two caches that hold the halves of a context give the whole when joined with the returned sums."""
    dev = cuda_device
    whole = make(dev, [640], 2, 128, 64, BF)
    q = queries(dev, 1, 1, 8, 128, BF)
    want, wlse = whole.attend(0, q, return_lse=True)
    parts = []
    for rows in (slice(0, 4), slice(4, 10)):
        part = type(whole).from_tensors(whole.kv, whole.page_table[:, rows].contiguous(),
                                        torch.tensor([(rows.stop - rows.start) * 64], dtype=torch.int32, device=dev))
        parts.append(part.attend(0, q, return_lse=True))
    lse = torch.stack([p[1] for p in parts]).double()
    total = lse.logsumexp(0)
    joined = sum(p[0].double() * (l - total).exp()[..., None] for p, l in zip(parts, lse))
    assert (total - wlse.double()).abs().max() < 1e-4
    assert (joined - want.double()).abs().max() <= 3 * 2.0 ** -8 * want.double().abs().max()


def test_refusals(cuda_device):
    from xcalibur_b200 import PagedKVCache

    dev = cuda_device
    cache = make(dev, [10, 20], 2, 64, 16, BF)
    q = queries(dev, 2, 1, 4, 64, BF)
    for bad, kw in [(q.cpu(), {}), (q.float(), {}), (q.half(), {}), (q[..., :32], {}), (q[:, :, :3], {}),
                    (q[:, :0], {}), (q[0, 0], {}), (torch.cat([q, q]), {}), (q, {"window": -1}),
                    (q, {"seqs": torch.zeros(3, dtype=torch.int32, device=dev)}),
                    (q, {"seqs": torch.zeros(2, dtype=torch.int64, device=dev)}),
                    (q, {"out": torch.empty_like(q)[..., :32]}), (q, {"out": torch.empty_like(q).half()})]:
        with pytest.raises(ValueError):
            cache.attend(0, bad, **kw)
    for layer in (-1, 1):
        with pytest.raises(ValueError):
            cache.attend(layer, q)
    assert cache.attend(0, q[:0]).shape == (0, 1, 4, 64)
    with pytest.raises(ValueError):
        PagedKVCache(1, 4, 2, 16, 60, max_seqs=2, max_pages=4, device=dev)
    with pytest.raises(ValueError):
        PagedKVCache(1, 4, 2, 16, 72, max_seqs=2, max_pages=4, dtype=F8, device=dev)
    with pytest.raises(ValueError):
        PagedKVCache(1, 4, 2, 16, 64, max_seqs=2, max_pages=4, dtype=torch.float32, device=dev)
    with pytest.raises(ValueError):
        PagedKVCache(1, 4, 2, 16, 64, max_seqs=2, max_pages=4, device=dev, k_scale=torch.ones(2, device=dev))


def test_a_scale_that_changes_in_place(cuda_device):
    cache = make(cuda_device, [70], 1, 64, 16, BF)
    q = queries(cuda_device, 1, 1, 2, 64, BF)
    scale = torch.tensor(0.125)
    first = cache.attend(0, q, scale=scale)
    scale.mul_(4)
    assert torch.equal(cache.attend(0, q, scale=scale), cache.attend(0, q, scale=0.5))
    assert torch.equal(first, cache.attend(0, q, scale=0.125))
