"""Every form of the attention kernel (types, head widths, numbers of warps a tile's rows take), prompts of several row
tiles, and all calls of a step in a CUDA graph."""
import pytest
import torch

from tests.test_gpu_attend import check, make, queries

pytestmark = pytest.mark.gpu

BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.mark.parametrize("group,new", [(7, 1), (10, 2), (11, 5), (25, 4)], ids=["7rows", "20rows", "55rows", "100rows"])
@pytest.mark.parametrize("dim", [64, 48, 128, 112, 256, 176])
@pytest.mark.parametrize("dt,cdt", [(BF, BF), (F16, F16), (BF, F8), (F16, F8)], ids=["bf16", "f16", "bf16-e4m3", "f16-e4m3"])
def test_every_form(cuda_device, dt, cdt, dim, group, new):
    lens = [1, 0, 33, 500, 129]
    cache = make(cuda_device, lens, 2, dim, 24, cdt, seed=dim + group)
    q = queries(cuda_device, len(lens), new, 2 * group, dim, dt)
    out, lse = cache.attend(0, q, return_lse=True)
    check(cache, q, out, lse)
    assert cache.check_device_status() == 0


@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("dim,group,new", [(128, 8, 70), (64, 5, 81), (256, 3, 50), (80, 1, 300)])
@pytest.mark.parametrize("dt,cdt", [(BF, BF), (F16, F16), (BF, F8), (F16, F8)], ids=["bf16", "f16", "bf16-e4m3", "f16-e4m3"])
def test_prompts_of_several_tiles(cuda_device, dt, cdt, dim, group, new, window):
    lens = [new, 333, new - 7]                       # from nothing, after other tokens, longer than what is held
    cache = make(cuda_device, lens, 2, dim, 16, cdt, seed=new)
    q = queries(cuda_device, len(lens), new, 2 * group, dim, dt)
    out, lse = cache.attend(0, q, window=window, return_lse=True)
    check(cache, q, out, lse, window=window)
    again = cache.attend(0, q, window=window)
    assert torch.equal(out, again)


@pytest.mark.parametrize("cdt", [BF, F8])
def test_a_whole_step_in_a_graph(cuda_device, cdt):
    """extend, append, attend, fork, growth with copies, truncate, free and compact, captured together and replayed."""
    from xcalibur_b200 import PagedKVCache, Rope

    dev = cuda_device
    gen = torch.Generator().manual_seed(0)
    two, third, grow = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 1], [2], [3]))
    one = torch.ones_like(two)
    zero = torch.zeros_like(third)
    rope = Rope(64, device=dev)
    qkv = torch.randn((2, 2, 12, 64), generator=gen).to(BF).to(dev)
    w = torch.rand(64, generator=gen).to(BF).to(dev)

    def cache():
        c = PagedKVCache(2, 40, 2, 8, 64, max_seqs=4, max_pages=9, dtype=cdt, device=dev)
        c.kv.view(torch.uint8).zero_()
        c.extend(two, torch.tensor([21, 8], dtype=torch.int32, device=dev))
        return c

    def step(c, outs):
        c.extend(two, one)
        for layer in range(2):
            q, k, v = qkv[layer].split([8, 2, 2], dim=1)
            q = c.append(layer, q, k, v, c.seq_lens[:2] - 1, two, rope, q_weight=w, k_weight=w)
            c.attend(layer, q, seqs=two, out=outs[layer])
        c.fork(two[:1], third)
        c.extend(third, grow)
        q, k, v = qkv[0, :1].expand(3, -1, -1).split([8, 2, 2], dim=1)
        c.append(0, q, k, v, c.seq_lens[2] - 3 + torch.arange(3, dtype=torch.int32, device=dev), third.expand(3), rope)
        c.truncate(third, c.seq_lens[2:3] - 2)
        c.attend(1, q[:1], seqs=third, out=outs[2])
        c.free(third)
        c.compact()

    def empty():
        return [torch.zeros((n, 8, 64), dtype=BF, device=dev) for n in (2, 2, 1)]

    eager, captured, want, got = cache(), cache(), empty(), empty()
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured, got)
    for _ in range(3):
        step(eager, want)
        graph.replay()
        torch.cuda.synchronize(dev)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(a.any() for a in got)
        for name in ("page_table", "seq_lens", "refcounts"):
            assert torch.equal(getattr(captured, name), getattr(eager, name)), name
        assert torch.equal(captured.kv.view(torch.uint8), eager.kv.view(torch.uint8))
    assert eager.seq_lens.tolist() == [24, 11, 0, 0]
    assert eager.check_device_status() == 0 and captured.check_device_status() == 0
