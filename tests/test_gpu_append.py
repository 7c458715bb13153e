"""Norm, rotation and store of new tokens against the plain 64-bit form."""
import pytest
import torch

from tests import _attn_ref as ref

pytestmark = pytest.mark.gpu

BF, F16, F8, F32 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float32


def rows(dev, tokens, hq, hkv, dim, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    qkv = torch.randn((tokens, hq + 2 * hkv, dim), generator=gen).to(dtype).to(dev)
    return qkv.split([hq, hkv, hkv], dim=1)


def weights(dev, dim, dtype, seed=5):
    gen = torch.Generator().manual_seed(seed)
    return [(1 + 0.2 * torch.randn(dim, generator=gen)).to(dtype).to(dev) for _ in range(2)]


CASES = [
    # tokens, q_heads, kv_heads, dim, rotary, interleaved, dtype, norm, weight dtype
    (1, 32, 4, 128, 128, False, BF, True, BF),
    (5, 4, 4, 64, 64, True, F16, True, F16),
    (300, 7, 1, 80, 32, False, F16, False, F16),
    (33, 5, 5, 80, 20, False, BF, True, F32),      # pairs 10 apart
    (33, 5, 5, 80, 20, True, BF, True, F32),
    (2000, 16, 2, 128, 64, True, BF, True, BF),
    (700, 6, 2, 256, 256, False, BF, True, BF),
    (65, 3, 1, 192, 2, False, F16, True, F16),
    (3, 1, 1, 8, 8, False, BF, True, BF),
    (40, 2, 2, 24, 0, False, BF, True, BF),        # norm alone
    (700, 64, 8, 96, 96, False, F16, True, F16),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"t{c[0]}-h{c[1]}.{c[2]}-d{c[3]}-r{c[4]}-i{int(c[5])}")
def test_qk_norm_rope(cuda_device, case):
    from xcalibur_b200 import Rope, qk_norm_rope

    tokens, hq, hkv, dim, rot, inter, dt, norm, wdt = case
    dev = cuda_device
    q, k, _ = rows(dev, tokens, hq, hkv, dim, dt)
    wq, wk = weights(dev, dim, wdt) if norm else (None, None)
    pos = (torch.arange(tokens, dtype=torch.int32, device=dev) * 131) % 200000
    rope = Rope(rot, base=1e6, interleaved=inter, device=dev)
    q2, k2 = qk_norm_rope(q, k, pos, rope, q_weight=wq, k_weight=wk, eps=1e-5)
    for got, x, w in ((q2, q, wq), (k2, k, wk)):
        want, tol = ref.rope(x, pos, rope.frequencies, rot, interleaved=inter, weight=w, eps=1e-5)
        ref.assert_within(got, want, ref.rounded_tol(want, tol, dt))
    # in place, on the strided views
    kept = q.clone()
    qk_norm_rope(q, k, pos, rope, q_weight=wq, k_weight=wk, eps=1e-5, q_out=q, k_out=k)
    assert torch.equal(q, q2) and torch.equal(k, k2)
    q.copy_(kept)
    # queries alone; one norm alone; weights as 1 + w
    alone, none = qk_norm_rope(q, None, pos, rope, q_weight=wq, eps=1e-5)
    assert none is None and torch.equal(alone, q2)


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": 8.0}, {"type": "ntk", "factor": 4.0},
                                     {"type": "yarn", "factor": 4.0, "original": 4096}])
def test_scaled_rotations_and_weight_offset(cuda_device, scaling):
    from xcalibur_b200 import Rope, qk_norm_rope

    dev = cuda_device
    q, k, _ = rows(dev, 64, 4, 2, 128, F16)
    wq, wk = (w - 1 for w in weights(dev, 128, F32))
    rope = Rope(128, base=10000.0, scaling=scaling, device=dev)
    pos = torch.arange(64, dtype=torch.int32, device=dev) * 2047
    q2, k2 = qk_norm_rope(q, k, pos, rope, q_weight=wq, k_weight=wk, weight_offset=1.0)
    for got, x, w in ((q2, q, wq), (k2, k, wk)):
        want, tol = ref.rope(x, pos, rope.frequencies, 128, weight=w, offset=1.0, mscale=rope.mscale)
        ref.assert_within(got, want, ref.rounded_tol(want, tol, F16))


def test_positions_up_to_31_bits(cuda_device):
    """The angle is exact modulo a turn, so the last positions are as good as the first."""
    from xcalibur_b200 import Rope, qk_norm_rope

    dev = cuda_device
    q, _, _ = rows(dev, 6, 2, 1, 64, F16)
    rope = Rope(64, device=dev)
    pos = torch.tensor([0, 1, -7, 2 ** 20 + 1, 2 ** 31 - 1, 10 ** 9], dtype=torch.int32, device=dev)
    got, _ = qk_norm_rope(q, None, pos, rope)
    want, tol = ref.rope(q, pos, rope.frequencies, 64)
    # the reference's own angle in 64 bits is off by up to 2^31 * 2^-52 turns of radians
    ref.assert_within(got, want, ref.rounded_tol(want, tol + 2.0 ** -20, F16))


def expected_cache(cache, before, pos, seqs, k, v):
    """The cache's values after the store, in 64 bits, and which slots are new."""
    kv = before.double().cpu()
    new = torch.zeros(kv.shape[2], kv.shape[4], dtype=torch.bool)
    for i, (p, s) in enumerate(zip(pos.tolist(), seqs.tolist())):
        if s < 0:
            continue
        page = int(cache.page_table[s, p // cache.page_size])
        kv[1, 0, page, :, p % cache.page_size] = k[i]
        kv[1, 1, page, :, p % cache.page_size] = v[i]
        new[page, p % cache.page_size] = True
    return kv, new


@pytest.mark.parametrize("dt,cdt", [(BF, BF), (F16, F16), (BF, F8), (F16, F8)])
@pytest.mark.parametrize("tokens,hkv,dim,ps", [(3, 2, 128, 16), (150, 4, 80, 24), (1500, 1, 64, 64)])
def test_append(cuda_device, dt, cdt, tokens, hkv, dim, ps):
    from xcalibur_b200 import PagedKVCache, Rope

    dev = cuda_device
    hq = hkv * 3
    n_seq = 3
    each = -(-tokens // n_seq)
    width = -(-(each + 100) // ps) + 1
    scales = {n: torch.tensor([0.01 * (i + 1) + 0.005 * j for i in range(hkv)], device=dev)
              for j, n in enumerate(("k_scale", "v_scale"))} if cdt == F8 else {}
    cache = PagedKVCache(2, n_seq * width + 2, hkv, ps, dim, max_seqs=n_seq, max_pages=width, dtype=cdt, device=dev,
                         **scales)
    cache.kv.copy_(torch.ones(1, device=dev).to(cdt).expand_as(cache.kv))
    cache.page_table.copy_(torch.randperm(n_seq * width, generator=torch.Generator().manual_seed(2)).view(n_seq, width))
    q, k, v = rows(dev, tokens, hq, hkv, dim, dt)
    wq, wk = weights(dev, dim, dt)
    seqs = torch.arange(tokens, dtype=torch.int32, device=dev) % n_seq
    pos = torch.arange(tokens, dtype=torch.int32, device=dev) // n_seq + 70
    seqs[1] = -1                                     # padding
    rope = Rope(dim // 2, interleaved=True, device=dev)
    before = cache.kv.clone()
    got = cache.append(1, q, k, v, pos, seqs, rope, q_weight=wq, k_weight=wk)
    want, tol = ref.rope(q, pos, rope.frequencies, dim // 2, interleaved=True, weight=wq)
    ref.assert_within(got, want, ref.rounded_tol(want, tol, dt))
    wk_, tk = ref.rope(k, pos, rope.frequencies, dim // 2, interleaved=True, weight=wk)
    wv = v.double().cpu()
    unit = [1.0, 1.0]
    if cdt == F8:
        unit = [scales[n].double().cpu()[:, None] for n in ("k_scale", "v_scale")]
    kv, new = expected_cache(cache, before, pos, seqs, wk_ / unit[0], wv / unit[1])
    tols, _ = expected_cache(cache, torch.zeros_like(before), pos, seqs, tk / unit[0], torch.zeros_like(wv))
    after = cache.kv.double().cpu()
    fresh = new[None, None, :, None, :, None].expand_as(after).clone()
    fresh[0] = False                                 # the other layer is untouched
    assert torch.equal(after[~fresh], before.double().cpu()[~fresh])
    if cdt == F8:
        kv = kv.clamp(-448, 448)
        bound = ref.e4m3_tol(kv, tols, 1.0)
    else:
        bound = ref.rounded_tol(kv, tols, cdt)
    ref.assert_within(after[fresh], kv[fresh], bound[fresh])
    assert cache.check_device_status() == 0


def test_e4m3_store_saturates_and_keeps_nan(cuda_device):
    from xcalibur_b200 import PagedKVCache, Rope

    dev = cuda_device
    cache = PagedKVCache(1, 1, 1, 16, 32, max_seqs=1, max_pages=1, dtype=F8, device=dev)
    cache.page_table.zero_()
    q = torch.zeros(1, 1, 32, dtype=BF, device=dev)
    k = q.clone()
    v = q.clone()
    v[0, 0, :6] = torch.tensor([500.0, -1e30, float("inf"), float("-inf"), float("nan"), 0.3])
    at = torch.zeros(1, dtype=torch.int32, device=dev)
    cache.append(0, q, k, v, at, at, Rope(0, device=dev))
    got = cache.kv[0, 1, 0, 0, 0, :6].float().cpu()
    assert got[:4].tolist() == [448.0, -448.0, 448.0, -448.0] and torch.isnan(got[4]) and got[5] == 0.3125


@pytest.mark.parametrize("rot, interleaved", [(32, False), (12, False), (32, True), (12, True)])
def test_what_does_not_turn_stays_as_it_is(cuda_device, rot, interleaved):
    from xcalibur_b200 import Rope, qk_norm_rope

    dev = cuda_device
    q, _, _ = rows(dev, 9, 3, 1, 64, BF)
    q[:, 1, 40] = float("inf")
    q[:, 2, 63] = float("-inf")
    q[:, 0, 33] = float("nan")
    at = torch.arange(9, dtype=torch.int32, device=dev) + 5
    got, _ = qk_norm_rope(q, None, at, Rope(rot, interleaved=interleaved, device=dev))
    torch.testing.assert_close(got[..., rot:], q[..., rot:], rtol=0, atol=0, equal_nan=True)
    assert torch.isfinite(got[..., :rot]).all()


def test_tokens_without_a_page_are_not_stored(cuda_device):
    from xcalibur_b200 import PagedKVCache, Rope, _lib

    dev = cuda_device
    cache = PagedKVCache(1, 4, 1, 16, 64, max_seqs=2, max_pages=2, device=dev)
    cache.kv.zero_()
    cache.page_table.copy_(torch.tensor([[0, -1], [4, 1]]))
    q, k, v = rows(dev, 6, 2, 1, 64, BF)
    pos = torch.tensor([15, 16, 3, -1, 32, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    seqs = torch.tensor([0, 0, 1, 0, 1, 1], dtype=torch.int32, device=dev)
    rope = Rope(64, device=dev)
    cache.append(0, q, k, v, pos, seqs, rope)
    assert cache.check_device_status() == _lib.XCB_STATUS_BAD_PAGE
    stored = cache.kv[0, 1, :, 0].float().abs().sum(-1) > 0
    assert stored.nonzero().tolist() == [[0, 15]]
    assert torch.equal(cache.kv[0, 1, 0, 0, 15], v[0, 0])
    cache.append(0, q[:1], k[:1], v[:1], pos[:1], torch.tensor([2], dtype=torch.int32, device=dev), rope)
    assert cache.check_device_status() == _lib.XCB_STATUS_BAD_SEQ


def test_store_past_32_bit_offsets(cuda_device):
    from xcalibur_b200 import PagedKVCache, Rope

    dev, ps, dim, heads = cuda_device, 64, 128, 2
    pages = (1 << 32) // (heads * ps * dim * 2) + 2
    cache = PagedKVCache(1, pages, heads, ps, dim, max_seqs=1, max_pages=1, device=dev)
    cache.page_table.fill_(pages - 1)
    q, k, v = rows(dev, 1, 4, heads, dim, BF)
    at = torch.full((1,), 63, dtype=torch.int32, device=dev)
    cache.append(0, q, k, v, at, torch.zeros_like(at), Rope(0, device=dev))
    assert torch.equal(cache.kv[0, 0, -1, :, 63], k[0]) and torch.equal(cache.kv[0, 1, -1, :, 63], v[0])


def test_refusals(cuda_device):
    from xcalibur_b200 import PagedKVCache, Rope, qk_norm_rope

    dev = cuda_device
    q, k, v = rows(dev, 4, 4, 2, 64, BF)
    pos = torch.arange(4, dtype=torch.int32, device=dev)
    rope = Rope(64, device=dev)
    w = torch.ones(64, dtype=BF, device=dev)
    ok = dict(q=q, k=k, positions=pos, rope=rope)
    for kw in [dict(q=q.cpu()), dict(q=q.float()), dict(k=k.half()), dict(k=k[:3]), dict(positions=pos[:3]),
               dict(positions=pos.long()), dict(rope=Rope(128, device=dev)), dict(rope=Rope(64, device="cpu")),
               dict(q_weight=w[:32]), dict(q_weight=w.double()), dict(q_weight=w, k_weight=w.float()),
               dict(q_out=torch.empty_like(q).half()), dict(q=q[0])]:
        args = {**ok, **kw}
        with pytest.raises(ValueError):
            qk_norm_rope(args.pop("q"), args.pop("k"), args.pop("positions"), args.pop("rope"), **args)
    with pytest.raises(_lib_error()):
        qk_norm_rope(torch.zeros(2, 1, 264, dtype=BF, device=dev), None, pos[:2], rope)
    cache = PagedKVCache(1, 4, 2, 16, 64, max_seqs=2, max_pages=2, device=dev)
    for kw in [dict(layer=1), dict(q=q.half(), k=k.half(), v=v.half()), dict(k=k[:, :1]), dict(seqs=pos[:2]), dict(v=None)]:
        a = {**dict(layer=0, q=q, k=k, v=v, positions=pos, seqs=pos, rope=rope), **kw}
        with pytest.raises(ValueError):
            cache.append(a["layer"], a["q"], a["k"], a["v"], a["positions"], a["seqs"], a["rope"])
    empty = qk_norm_rope(q[:0], k[:0], pos[:0], rope)
    assert empty[0].shape == (0, 4, 64)


def _lib_error():
    from xcalibur_b200._lib import XcbError

    return XcbError
