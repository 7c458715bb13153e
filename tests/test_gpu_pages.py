"""Page bookkeeping against a one-sequence-at-a-time model: tables, lengths and counts exactly, copies bit for bit."""
import random

import pytest
import torch

from tests._attn_ref import Pages

pytestmark = pytest.mark.gpu


def make(dev, *, layers=2, pages=64, heads=2, ps=16, dim=64, seqs=8, width=8, dtype=torch.bfloat16):
    from xcalibur_b200 import PagedKVCache

    cache = PagedKVCache(layers, pages, heads, ps, dim, max_seqs=seqs, max_pages=width, dtype=dtype, device=dev)
    raw = cache.kv.view(torch.uint8 if dtype == torch.float8_e4m3fn else torch.int16)
    raw.copy_(torch.randint(-100, 100, raw.shape, device=dev, generator=torch.Generator(dev).manual_seed(1)))
    return cache, raw


def ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def model(cache):
    return Pages(cache.page_table.cpu(), cache.seq_lens.cpu(), cache.refcounts.cpu(), cache.page_size)


def check(cache, m, raw, before):
    assert cache.page_table.tolist() == m.table
    assert cache.seq_lens.tolist() == m.lens
    assert cache.refcounts.tolist() == m.refs
    want = before.clone()
    for a, b, n in m.copies:
        want[:, :, b, :, :n] = before[:, :, a, :, :n]
    assert torch.equal(raw, want)
    # every page is held as often as the tables say
    held = [0] * cache.num_pages
    for row, n in zip(m.table, m.lens):
        for p in row[: -(-n // cache.page_size)]:
            held[p] += 1
    assert held == m.refs


@pytest.mark.parametrize("dtype,ps,dim,seed", [(torch.bfloat16, 16, 64, 0), (torch.float8_e4m3fn, 24, 48, 1),
                                               (torch.float16, 1, 8, 2), (torch.bfloat16, 64, 128, 3)])
def test_random_histories(cuda_device, dtype, ps, dim, seed):
    from xcalibur_b200 import _lib

    dev, rng = cuda_device, random.Random(seed)
    cache, raw = make(dev, pages=70, ps=ps, dim=dim, seqs=12, width=9, dtype=dtype)
    for step in range(60):
        m, before = model(cache), raw.clone()
        op = rng.choice(["extend", "extend", "extend", "fork", "truncate", "free", "compact"])
        some = rng.sample(range(12), rng.randrange(1, 12))
        want = 0
        if op == "extend":
            if rng.random() < 0.2:
                some[-1] = rng.choice([-1, 12, some[0]])
                some = some + [3] if len(some) < 12 and 3 not in some else some
            new = [rng.choice([0, 1, 1, 2, ps, 3 * ps + 1, rng.randrange(9 * ps)]) for _ in some]
            bad, short = m.extend(some, new)
            cache.extend(ints(dev, some), ints(dev, new))
            want = (_lib.XCB_STATUS_BAD_SEQ if bad else 0) | (_lib.XCB_STATUS_NO_PAGES if short else 0)
        elif op == "fork":
            src = [rng.randrange(12) for _ in some]
            bad = m.fork(src, some)
            cache.fork(ints(dev, src), ints(dev, some))
            want = _lib.XCB_STATUS_BAD_SEQ if bad else 0
        elif op == "truncate":
            to = [rng.randrange(m.lens[s] + 1) if rng.random() < 0.9 else m.lens[s] + 1 for s in some]
            bad = m.truncate(some, to)
            cache.truncate(ints(dev, some), ints(dev, to))
            want = _lib.XCB_STATUS_BAD_SEQ if bad else 0
        elif op == "free":
            m.truncate(some, [0] * len(some))
            cache.free(ints(dev, some))
        else:
            m.compact()
            cache.compact()
        check(cache, m, raw, before)
        assert cache.check_device_status() == want, (step, op)


def test_who_keeps_a_shared_page(cuda_device):
    dev = cuda_device
    cache, raw = make(dev)
    cache.extend(ints(dev, [0]), ints(dev, [20]))
    cache.fork(ints(dev, [0, 0]), ints(dev, [1, 2]))
    assert cache.page_table[:3, :2].tolist() == [[0, 1]] * 3 and cache.refcounts[:2].tolist() == [3, 3]
    m, before = model(cache), raw.clone()
    assert m.extend([2, 0, 1], [1, 1, 1]) == (False, False)
    cache.extend(ints(dev, [2, 0, 1]), ints(dev, [1, 1, 1]))     # all holders grow: the first listed keeps the page
    check(cache, m, raw, before)
    assert cache.page_table[:3, 1].tolist() == [2, 3, 1]
    cache.fork(ints(dev, [0]), ints(dev, [3]))
    m, before = model(cache), raw.clone()
    assert m.extend([3], [1]) == (False, False)
    cache.extend(ints(dev, [3]), ints(dev, [1]))                 # one of two holders grows: it gets the copy
    check(cache, m, raw, before)
    assert int(cache.page_table[3, 1]) == 4 and int(cache.refcounts[3]) == 1


def test_too_few_pages_change_nothing(cuda_device):
    from xcalibur_b200 import _lib

    dev = cuda_device
    cache, raw = make(dev, pages=4, seqs=3)
    cache.extend(ints(dev, [0, 1]), ints(dev, [20, 16]))
    m, before = model(cache), raw.clone()
    assert m.extend([0, 1], [13, 17]) == (False, True)
    cache.extend(ints(dev, [0, 1]), ints(dev, [13, 17]))
    check(cache, m, raw, before)
    assert cache.check_device_status() == _lib.XCB_STATUS_NO_PAGES
    m.extend([0], [13])
    cache.extend(ints(dev, [0]), ints(dev, [13]))                # the call before left no trace
    check(cache, m, raw, before)
    assert cache.check_device_status() == 0


def test_large_pool_and_many_sequences(cuda_device):
    """More sequences than a block has threads, more pages than one scan step, and growths of hundreds of pages."""
    dev, rng = cuda_device, random.Random(4)
    cache, raw = make(dev, layers=1, pages=60000, heads=1, ps=4, dim=8, seqs=2500, width=400)
    m, before = model(cache), raw.clone()
    every = list(range(2500))
    rng.shuffle(every)
    new = [rng.choice([1, 3, 30, 200]) for _ in every]
    new[7] = 1600
    assert m.extend(every, new) == (False, False)
    cache.extend(ints(dev, every), ints(dev, new))
    check(cache, m, raw, before)
    some = rng.sample(every, 1200)
    m.truncate(some, [0] * 1200)
    cache.free(ints(dev, some))
    check(cache, m, raw, before)
    m, before = model(cache), raw.clone()
    m.compact()
    cache.compact()
    check(cache, m, raw, before)
    m, before = model(cache), raw.clone()
    left = [s for s in every if s not in set(some)]
    m.fork(left[:1200], some)
    cache.fork(ints(dev, left[:1200]), ints(dev, some))
    assert m.extend(every, [1] * 2500) == (False, False)
    cache.extend(ints(dev, every), ints(dev, [1] * 2500))
    check(cache, m, raw, before)
    assert cache.check_device_status() == 0


def test_copy_pages(cuda_device):
    from xcalibur_b200 import _lib

    dev = cuda_device
    cache, raw = make(dev, layers=3, heads=3, ps=40, dim=136)
    before = raw.clone()
    cache.copy_pages(ints(dev, [3, 9, 3]), ints(dev, [60, 0, 11]))
    want = before.clone()
    for a, b in ((3, 60), (9, 0), (3, 11)):
        want[:, :, b] = before[:, :, a]
    assert torch.equal(raw, want) and cache.check_device_status() == 0
    cache.copy_pages(ints(dev, [64, 1, -1, 2]), ints(dev, [5, -1, 6, 64]))
    assert torch.equal(raw, want) and cache.check_device_status() == _lib.XCB_STATUS_BAD_PAGE


def test_refusals(cuda_device):
    from xcalibur_b200 import PagedKVCache

    dev = cuda_device
    cache, _ = make(dev)
    good = ints(dev, [0, 1])
    for bad in (good.long(), good.cpu(), good.view(2, 1), ints(dev, list(range(9)))):
        with pytest.raises(ValueError):
            cache.free(bad)
    for f in (cache.extend, cache.fork, cache.truncate, cache.copy_pages):
        with pytest.raises(ValueError):
            f(good, good[:1])
    cache.extend(good[:0], good[:0])
    cache.free(good[:0])
    with pytest.raises(ValueError):
        PagedKVCache.from_tensors(cache.kv, cache.page_table.long(), cache.seq_lens)
    with pytest.raises(ValueError):
        PagedKVCache.from_tensors(cache.kv[:, :1], cache.page_table, cache.seq_lens)
    with pytest.raises(ValueError):
        PagedKVCache.from_tensors(cache.kv, cache.page_table[:, :-1], cache.seq_lens)


def test_first_extend_in_a_graph_and_calls_outside_it(cuda_device):
    """A capture that makes the workspace does not leave one behind that only the graph has set up."""
    from xcalibur_b200 import PagedKVCache

    cache = PagedKVCache(1, 8, 1, 4, 16, max_seqs=2, max_pages=4, device=cuda_device)
    seqs = torch.tensor([0, 1], dtype=torch.int32, device=cuda_device)
    three = torch.full_like(seqs, 3)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cache.extend(seqs, three)
    with torch.cuda.stream(side):
        cache.extend(seqs, three)
        graph.replay()
        cache.extend(seqs, three)
        graph.replay()
    side.synchronize()
    assert cache.check_device_status() == 0
    assert cache.seq_lens.tolist() == [12, 12]
    assert sorted(cache.page_table[:, :3].flatten().tolist()) == [0, 1, 2, 3, 4, 5]
