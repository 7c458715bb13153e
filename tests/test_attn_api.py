"""The attention side's C-ABI and host code without a GPU: the header is what the binding binds, argument errors are
found before any launch, rotation frequencies follow their formulas."""
import ctypes
import math
import os
import re

import pytest
import torch

from xcalibur_b200 import PagedKVCache, Rope, _lib, qk_norm_rope

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def header_symbols():
    src = open(os.path.join(ROOT, "include", "xcb_attn.h")).read()
    return sorted(set(re.findall(r"^\s*(?:const\s+)?\w[\w\s\*]*?\b(xcb_\w+)\s*\(", src, re.M)))


def test_header_declares_what_the_binding_binds_and_the_library_exports():
    assert header_symbols() == sorted(_lib.ATTN_EXPORTS)
    lib = _lib.load()
    for name in header_symbols():
        assert hasattr(lib, name), name


def _cache(**kw):
    # addresses that are never read: every call below is refused on the host
    c = _lib.XcbKvCache(2, 8, 2, 16, 64, _lib.XCB_DTYPE_BF16, 4, 4, 256, 256, 256, 256, None, None, 256)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def test_cache_shapes():
    lib = _lib.load()

    def size(**kw):
        c = _cache(**kw)
        return lib.xcb_kv_workspace_bytes(ctypes.addressof(c))

    assert size() > 0
    assert size(num_pages=16) > size()
    for bad in (dict(layers=0), dict(num_pages=-1), dict(kv_heads=0), dict(page_size=0), dict(head_dim=0),
                dict(max_seqs=0), dict(max_pages=0), dict(dtype=3), dict(dtype=-1), dict(head_dim=60),
                dict(head_dim=264), dict(head_dim=72, dtype=_lib.XCB_DTYPE_E4M3), dict(kv=None), dict(kv=264),
                dict(page_table=None), dict(seq_lens=None), dict(status=None), dict(page_table=258),
                dict(page_size=65536, max_pages=65536), dict(max_seqs=1 << 20, max_pages=1 << 12)):
        assert size(**bad) == 0, bad
    assert lib.xcb_kv_workspace_bytes(None) == 0


def test_page_calls_refuse_before_launch():
    lib = _lib.load()
    c = _cache()
    at, need = ctypes.addressof(c), lib.xcb_kv_workspace_bytes(ctypes.addressof(c))
    bad, small = _lib.XCB_ERR_INVALID_ARG, _lib.XCB_ERR_WORKSPACE
    assert lib.xcb_kv_extend(at, 256, 256, 5, 256, need, None) == bad          # more entries than sequences
    assert lib.xcb_kv_extend(at, 256, 256, -1, 256, need, None) == bad
    assert lib.xcb_kv_extend(at, None, 256, 1, 256, need, None) == bad
    assert lib.xcb_kv_extend(at, 256, None, 1, 256, need, None) == bad
    assert lib.xcb_kv_extend(at, 256, 256, 1, None, need, None) == bad
    assert lib.xcb_kv_extend(at, 256, 256, 1, 256, need - 1, None) == small
    assert lib.xcb_kv_extend(at, 256, 256, 0, 256, need, None) == _lib.XCB_OK
    assert lib.xcb_kv_fork(at, 256, None, 1, None) == bad
    assert lib.xcb_kv_fork(at, 257, 256, 1, None) == bad
    assert lib.xcb_kv_truncate(at, None, 256, 1, None) == bad
    assert lib.xcb_kv_compact(at, 256, 16, None) == small
    assert lib.xcb_kv_copy_pages(at, 256, 256, 9, None) == bad
    assert lib.xcb_kv_copy_pages(at, 256, 256, 0, None) == _lib.XCB_OK
    assert lib.xcb_kv_read_status(at, None, None) == bad
    c.refcounts = None
    assert lib.xcb_kv_truncate(at, 256, 256, 1, None) == bad
    assert lib.xcb_kv_fork(None, 256, 256, 1, None) == bad


def test_attention_refuses_before_launch():
    lib = _lib.load()
    c = _cache()

    def call(cache=c, ws=256, **kw):
        a = _lib.XcbAttnArgs(2, 1, 4, _lib.XCB_DTYPE_BF16, 0, 0, 0.1, 256, (256, 256, 64), 256, None, None)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.xcb_paged_attention(ctypes.addressof(cache), ctypes.addressof(a), ws, 1 << 40, None)

    bad, un = _lib.XCB_ERR_INVALID_ARG, _lib.XCB_ERR_UNSUPPORTED
    assert call(batch=0) == _lib.XCB_OK
    for kw in (dict(batch=-1), dict(batch=5), dict(new_tokens=0), dict(q_heads=0), dict(q_heads=3), dict(layer=2),
               dict(layer=-1), dict(window=-1), dict(q=None), dict(q=264), dict(out=None), dict(out=258),
               dict(q_stride=(256, 256, 60)), dict(dtype=_lib.XCB_DTYPE_E4M3), dict(lse=257), dict(seqs=254)):
        assert call(**kw) == bad, kw
    assert call(dtype=_lib.XCB_DTYPE_F16) == un                    # a bf16 cache
    assert call(new_tokens=65537) == un
    assert call(ws=None) == bad and call(ws=16) == bad
    assert lib.xcb_paged_attention(ctypes.addressof(c), None, 256, 1 << 40, None) == bad
    assert lib.xcb_paged_attention(None, None, 256, 1 << 40, None) == bad


def test_norm_rope_refuses_before_launch():
    lib = _lib.load()
    c = _cache()

    def call(cache=None, **kw):
        a = _lib.XcbRopeArgs(tokens=2, q_heads=4, kv_heads=2, head_dim=64, rotary_dim=64, dtype=_lib.XCB_DTYPE_BF16,
                             weight_dtype=_lib.XCB_DTYPE_BF16, q=256, k=256, v=256, q_out=256, k_out=256,
                             positions=256, seqs=256, turns=256)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.xcb_qk_norm_rope(None if cache is None else ctypes.addressof(cache), ctypes.addressof(a), None)

    bad, un = _lib.XCB_ERR_INVALID_ARG, _lib.XCB_ERR_UNSUPPORTED
    assert call(tokens=0) == _lib.XCB_OK
    for kw in (dict(tokens=-1), dict(q_heads=-1), dict(head_dim=0), dict(rotary_dim=-2), dict(rotary_dim=63),
               dict(rotary_dim=66), dict(eps=-1.0), dict(eps=math.nan), dict(dtype=_lib.XCB_DTYPE_F32),
               dict(weight_dtype=_lib.XCB_DTYPE_F16), dict(positions=None), dict(turns=None), dict(q_out=None),
               dict(k_out=None), dict(q=258), dict(q_stride=(4, 64)), dict(q_weight=264), dict(turns=260)):
        assert call(**kw) == bad, kw
    assert call(head_dim=68, rotary_dim=0) == un and call(head_dim=264) == un
    for kw in (dict(layer=2), dict(kv_heads=1), dict(head_dim=32, rotary_dim=32), dict(v=None), dict(k=None),
               dict(seqs=None)):
        assert call(cache=c, **kw) == bad, kw
    assert call(cache=c, dtype=_lib.XCB_DTYPE_F16, weight_dtype=_lib.XCB_DTYPE_F16) == un


def test_frequencies():
    plain = Rope(64, base=10000.0, device="cpu")
    assert plain.mscale == 1.0
    assert plain.frequencies == pytest.approx([10000.0 ** (-i / 32) for i in range(32)], rel=1e-14)
    turns = [int(t) % (1 << 64) / 2.0 ** 64 for t in plain.turns]
    assert turns == pytest.approx([f / (2 * math.pi) for f in plain.frequencies], rel=1e-14)
    linear = Rope(64, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert linear.frequencies == pytest.approx([f / 4 for f in plain.frequencies], rel=1e-14)
    ntk = Rope(64, scaling={"type": "ntk", "factor": 4.0}, device="cpu")
    # the fastest pair stays, the slowest turns `factor` times slower
    assert ntk.frequencies[0] == 1.0 and ntk.frequencies[-1] == pytest.approx(plain.frequencies[-1] / 4, rel=1e-12)
    yarn = Rope(64, scaling={"type": "yarn", "factor": 4.0, "original": 4096}, device="cpu")
    assert yarn.frequencies[0] == plain.frequencies[0]
    assert yarn.frequencies[-1] == pytest.approx(plain.frequencies[-1] / 4, rel=1e-12)
    assert all(p / 4 * (1 - 1e-12) <= y <= p for y, p in zip(yarn.frequencies, plain.frequencies))
    assert yarn.mscale == pytest.approx(0.1 * math.log(4.0) + 1.0)
    assert Rope(0, device="cpu").frequencies == []


def test_host_refusals():
    for kw in (dict(rotary_dim=3), dict(rotary_dim=-2), dict(rotary_dim=300), dict(rotary_dim=64, base=0.0),
               dict(rotary_dim=64, scaling={"type": "other"}), dict(rotary_dim=64, scaling={"type": "linear", "x": 1}),
               dict(rotary_dim=64, scaling={"type": "linear", "factor": 0.0}), dict(rotary_dim=64, base=1e-3)):
        with pytest.raises(ValueError):
            Rope(kw.pop("rotary_dim"), device="cpu", **kw)
    with pytest.raises(ValueError, match="no CPU path"):
        qk_norm_rope(torch.zeros(1, 1, 64, dtype=torch.bfloat16), None, torch.zeros(1, dtype=torch.int32),
                     Rope(64, device="cpu"))
    with pytest.raises(ValueError, match="no CPU path"):
        PagedKVCache(1, 1, 1, 16, 64, max_seqs=1, max_pages=1, device="cpu")


def test_scaling_without_its_entries_is_refused():
    """A factor alone was ignored: the rotation came out unscaled."""
    for bad in ({"factor": 8.0}, {"type": None, "factor": 8.0}, {"type": "yarn", "factor": 4.0},
                {"type": "linear", "factor": math.inf}, {"type": "linear", "factor": math.nan}):
        with pytest.raises(ValueError):
            Rope(64, scaling=bad, device="cpu")
    assert Rope(64, scaling={}, device="cpu").frequencies == Rope(64, device="cpu").frequencies
