"""What calls on a cache keep and share: workspaces, checked forms, state."""
import pytest
import torch

from tests import _attn_ref as ref
from tests.test_gpu_attend import make, queries

pytestmark = pytest.mark.gpu

BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def test_workspaces_do_not_grow_with_the_lengths_of_prompts(cuda_device):
    """Each number of new tokens is another form of call, of which a server sees hundreds; their scratch is shared."""
    dev = cuda_device
    cache = make(dev, [400], 1, 128, 64, BF)
    q = queries(dev, 1, 300, 8, 128, BF)
    cache.attend(0, q)
    torch.cuda.synchronize(dev)
    before = torch.cuda.memory_allocated(dev)
    for new in range(1, 300):
        cache.attend(0, q[:, :new])
    # one buffer for 1, 2, 4 and 8 warps of rows each, 148 blocks of two parts of 16 rows of 128 floats a warp at most
    assert len(cache._attn_ws) <= 4
    assert torch.cuda.memory_allocated(dev) - before <= (1 + 2 + 4) * 160 * 2 * 16 * 132 * 4


def test_a_workspace_holds_anything_at_first(cuda_device):
    dev = cuda_device
    lens = [3000, 1, 0, 777]
    cache = make(dev, lens, 2, 128, 64, BF)
    for new in (1, 5, 40):
        q = queries(dev, len(lens), new, 16, 128, BF)
        cache.attend(0, q)
        for ws in cache._attn_ws.values():
            ws.fill_(0xff)
        out, lse = cache.attend(0, q, return_lse=True)
        want, wlse, tol, ltol = ref.attend(cache.kv, cache.page_table, cache.seq_lens, q)
        ref.assert_within(out, want, tol)
        ref.assert_within(lse, wlse, ltol)


def test_captures_of_page_calls_keep_no_memory(cuda_device):
    """A server captures its steps again and again; each capture of a page call kept scratch of the pool's size."""
    from xcalibur_b200 import PagedKVCache

    dev = cuda_device
    cache = PagedKVCache(1, 200000, 1, 1, 8, max_seqs=2, max_pages=4, device=dev)
    seqs = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    none = torch.zeros_like(seqs)
    side = torch.cuda.Stream(dev)
    torch.cuda.synchronize(dev)

    def capture():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            cache.extend(seqs, none)
            cache.compact()
        graph.replay()
        torch.cuda.synchronize(dev)

    capture()
    before = torch.cuda.memory_allocated(dev)
    for _ in range(5):
        capture()
    assert torch.cuda.memory_allocated(dev) - before < 1 << 20  # the scratch is 5.6 MB
    assert cache.check_device_status() == 0


def test_norm_of_a_head_whose_mean_square_is_below_the_normal_range(cuda_device):
    """1e-38 is a 32-bit number, and without an epsilon its root divides."""
    from xcalibur_b200 import Rope, qk_norm_rope

    gen = torch.Generator().manual_seed(0)
    q = (torch.randint(0, 2, (5, 3, 128), generator=gen) * 2 - 1).mul(1e-19).to(BF).to(cuda_device)
    w = (1 + 0.1 * torch.randn(128, generator=gen)).to(BF).to(cuda_device)
    at = torch.arange(5, dtype=torch.int32, device=cuda_device)
    rope = Rope(64, device=cuda_device)
    got, _ = qk_norm_rope(q, None, at, rope, q_weight=w, eps=0.0)
    want, tol = ref.rope(q, at, rope.frequencies, 64, weight=w, eps=0.0)
    ref.assert_within(got, want, ref.rounded_tol(want, tol, BF))


def test_a_form_of_call_is_checked_once_for_all_layers(cuda_device):
    """The checked forms are kept up to a number; with one for each layer, a deep model's had room for few others."""
    from xcalibur_b200 import Rope

    dev = cuda_device
    cache = make(dev, [20, 33], 2, 64, 16, BF, layers=5)
    q = queries(dev, 2, 1, 4, 64, BF)
    rope = Rope(64, device=dev)
    at, seqs = cache.seq_lens - 1, torch.arange(2, dtype=torch.int32, device=dev)
    new = torch.randn((2, 5, 2, 64), generator=torch.Generator().manual_seed(4)).to(BF).to(dev)
    before = cache.kv.clone()
    for layer in range(5):
        q2 = cache.append(layer, q[:, 0], new[:, layer], new[:, layer], at, seqs, rope)
        out = cache.attend(layer, q2)
        want, _, tol, _ = ref.attend(cache.kv, cache.page_table, cache.seq_lens, q2[:, None], layer=layer)
        ref.assert_within(out[:, None], want, tol)
        for s in range(2):
            p = int(cache.page_table[s, int(at[s]) // 16])
            assert torch.equal(cache.kv[layer, 1, p, :, int(at[s]) % 16], new[s, layer])
        # the layers that follow are untouched
        raw = cache.kv[layer + 1:].view(torch.int16)
        assert torch.equal(raw, before[layer + 1:].view(torch.int16))
    assert len(cache._plans) == 1 and len(cache._rope_plans) == 1
    for layer in (-1, 5):
        with pytest.raises(ValueError):
            cache.append(layer, q[:, 0], new[:, 0], new[:, 0], at, seqs, rope)
        with pytest.raises(ValueError):
            cache.attend(layer, q)


def test_counts_of_a_callers_table(cuda_device):
    """Entries past a sequence's last page, zeros in many a table, are not held pages."""
    from xcalibur_b200 import PagedKVCache

    dev = cuda_device
    kv = torch.zeros((1, 2, 6, 1, 4, 8), dtype=BF, device=dev)
    table = torch.tensor([[0, 1, 0, 0], [0, 0, 0, 0], [0, 2, 9, -1], [3, 0, 0, 0]], dtype=torch.int32, device=dev)
    lens = torch.tensor([5, 0, 10, 4], dtype=torch.int32, device=dev)
    cache = PagedKVCache.from_tensors(kv, table, lens)
    assert cache.refcounts.tolist() == [2, 1, 1, 1, 0, 0]
    cache.free(torch.tensor([0, 3], dtype=torch.int32, device=dev))
    assert cache.refcounts.tolist() == [1, 0, 1, 0, 0, 0]
    for bad in (lens[:3], lens.long(), lens[:, None], lens.cpu()):
        with pytest.raises(ValueError):
            PagedKVCache.from_tensors(kv, table, bad)
    with pytest.raises(ValueError):
        PagedKVCache.from_tensors(kv, table[0], lens)


def test_another_tensor_cannot_take_the_states_place(cuda_device):
    """The kernels go by the tensors' addresses: one that was assigned would have been passed over in silence."""
    cache = make(cuda_device, [20], 2, 64, 16, F8)
    q = queries(cuda_device, 1, 1, 4, 64, BF)
    for name in ("kv", "page_table", "seq_lens", "refcounts", "k_scale", "v_scale", "status"):
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(cache, name).clone())
    saved = cache.seq_lens.clone()
    want = cache.attend(0, q)
    cache.seq_lens.fill_(3)
    assert not torch.equal(cache.attend(0, q), want)
    cache.seq_lens.copy_(saved)
    assert torch.equal(cache.attend(0, q), want)


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 2e-38])
def test_norm_with_a_vanishing_epsilon(cuda_device, dt, eps):
    from xcalibur_b200 import Rope, qk_norm_rope

    gen = torch.Generator().manual_seed(3)
    q = (torch.randn((4, 3, 96), generator=gen) * 2e-7).to(dt).to(cuda_device)
    w = (1 + 0.1 * torch.randn(96, generator=gen)).to(dt).to(cuda_device)
    at = torch.arange(4, dtype=torch.int32, device=cuda_device)
    rope = Rope(96, device=cuda_device)
    got, _ = qk_norm_rope(q, None, at, rope, q_weight=w, eps=eps)
    want, tol = ref.rope(q, at, rope.frequencies, 96, weight=w, eps=eps)
    ref.assert_within(got, want, ref.rounded_tol(want, tol, dt))
    if eps:  # without one, zeros divide zero
        assert not qk_norm_rope(torch.zeros_like(q), None, at, rope, q_weight=w, eps=eps)[0].any()
