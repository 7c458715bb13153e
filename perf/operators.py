"""Measured cases of the attention-side operators that stand next to the mixture-of-experts layer in a decoder.

Three operators share one paged key-value cache ``kv [layers, 2, pages, kv_heads, page_size, head_dim]``:

* ``append``: norms of queries and keys for each head, the position rotation, and the store of keys and values into
  the cache's pages, in one pass.
* ``attend``: attention of the newest token (or of a few draft tokens) of each sequence over its pages.
* ``pages``: growing, forking, rolling back and compacting sequences of the cache.

``own`` false: the plain form, elementary torch operations in 32 bits, rounded once.  ``own`` true: the calls a user
makes of the framework.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "f16": 2, "fp8": 1}
ROPE_BASE = 1.0e6
YARN = {"type": "yarn", "factor": 4.0, "original": 32768}
LINEAR = {"type": "linear", "factor": 8.0}
SCALING = {"none": None, "linear": LINEAR, "yarn": YARN}
EPS = 1e-6


def listed():
    append = dict(op="append", q_heads=32, kv_heads=4, head_dim=128, rotary=128, interleaved=False, scaling="none",
                  norm=True, dtype="bf16", cache="bf16", page=64)
    attend = dict(op="attend", q_heads=32, kv_heads=4, head_dim=128, new=1, window=0, dtype="bf16", cache="bf16",
                  page=64, lse=False)
    pages = dict(op="pages", kv_heads=4, head_dim=128, page=64, cache="bf16")
    return [
        # one decode step of a single user: latency only
        dict(append, name="append decode 1", tokens=1, seqs=1, max_pos=32768),
        # one decode step of a busy server whose cache is held in 8 bits; half of each head rotates, long context
        dict(append, name="append decode 64 fp8", tokens=64, seqs=64, max_pos=131072, rotary=64, interleaved=True,
             scaling="yarn", cache="fp8"),
        # prompts of four users in one pass
        dict(append, name="append prompt 8192", tokens=8192, seqs=4, max_pos=8192),
        # a ragged chunk of prompts, small odd heads, rotation alone (no norm), short pages
        dict(append, name="append ragged 1531", tokens=1531, seqs=7, max_pos=16384, q_heads=20, kv_heads=5,
             head_dim=80, rotary=32, interleaved=True, scaling="linear", norm=False, dtype="f16", cache="f16", page=16),
        # one user, a short chat: latency only
        dict(attend, name="attend 1 x 777", batch=1, max_len=777, spread=False),
        # one user, a very long document: the length has to be split over the whole GPU
        dict(attend, name="attend 1 x 131072", batch=1, max_len=131072, spread=False),
        # a server's batch, every length from a few tokens to thousands, short pages
        dict(attend, name="attend 64 ragged", batch=64, max_len=8192, spread=True, page=16),
        # a large batch over a cache in 8 bits; the log-sum-exp goes on to be joined with another device's part
        dict(attend, name="attend 128 fp8", batch=128, max_len=4000, spread=True, q_heads=64, kv_heads=8, cache="fp8",
             lse=True),
        # verification of four draft tokens per user under a sliding window, small heads
        dict(attend, name="verify 48 x 4 window", batch=48, max_len=9000, spread=True, new=4, q_heads=40, kv_heads=8,
             head_dim=64, window=4096, dtype="f16", cache="f16", page=32),
        # page bookkeeping of one verification step: room for four drafts each, the rejected ones rolled back
        dict(pages, name="pages step 256", mode="step", layers=1, parents=256, children=0, length=1000, num_pages=8192),
        # parallel sampling: three more samples from each of 64 prompts; their last pages part at the first new token
        dict(pages, name="pages fork 64 x 3", mode="fork", layers=16, parents=64, children=3, length=500,
             num_pages=1024),
        # a fragmented pool before it is made smaller
        dict(pages, name="pages compact 1024", mode="compact", layers=16, parents=96, children=0, length=640,
             num_pages=1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "pages"])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8, 16])
    head_dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    cache = rng.choice([dtype, dtype, "fp8"])
    page = rng.choice([16, 32, 64, 64, 128, 24])
    if op == "append":
        rotary = rng.choice([head_dim, head_dim, head_dim // 2, 16])
        row = (kv_heads * group + 2 * kv_heads) * head_dim
        tokens = _log(rng, 1, max(2, min(8192, 8192 * 40 * 128 // row)))
        return dict(op=op, q_heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, rotary=rotary,
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "yarn"]),
                    norm=rng.random() < 0.7, dtype=dtype, cache=cache, page=page, tokens=tokens,
                    seqs=min(tokens, _log(rng, 1, 64)), max_pos=max(tokens, _log(rng, 1024, 131072)))
    if op == "attend":
        new = rng.choice([1, 1, 1, 2, 3, 4, 8])
        batch = _log(rng, 1, 128)
        row = 2 * kv_heads * head_dim * BYTES[cache]
        # the largest listed call reads about 270 MB of keys and values, and computes no more than 32 rows per head
        most = 200e6 / (batch * row) * min(1.0, 32.0 / (new * group))
        return dict(op=op, q_heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, new=new,
                    window=rng.choice([0, 0, 0, 1000]), dtype=dtype, cache=cache, page=page, lse=rng.random() < 0.5,
                    batch=batch, max_len=_log(rng, 16, max(32, min(131072, most))), spread=rng.random() < 0.7)
    mode = rng.choice(["step", "fork", "compact"])
    layers = 1 if mode == "step" else _log(rng, 1, 24)
    length = _log(rng, 20, 1500)
    each = -(-(length + 4) // page)
    children = rng.choice([1, 2, 3, 7]) if mode == "fork" else 0
    # the pool holds at most about 1.5 GB
    room = int(1.5e9 / (layers * 2 * kv_heads * page * head_dim * BYTES[cache]))
    parents = max(1, min(_log(rng, 2, 256), room // (2 * each + 2 * children + 2)))
    return dict(op=op, kv_heads=kv_heads, head_dim=head_dim, page=page, cache=cache, mode=mode, layers=layers,
                parents=parents, children=children, length=length,
                num_pages=2 * parents * each + 2 * parents * (children + 1) + rng.randrange(64))


# ------------------------------------------------------------------------------------------------ inputs

def _spread(c):
    """Sequence lengths of an attend case: the same for all, or from a few tokens to max_len (the last is max_len)."""
    b, top = c["batch"], c["max_len"]
    if not c["spread"] or b == 1:
        return [top] * b
    low = max(1, top // 64)
    return [int(round(low * (top / low) ** (((i * 7919) % b) / (b - 1)))) for i in range(b)]


def _chunks(c):
    """(first position, tokens) of each sequence of an append case."""
    n, s = c["tokens"], c["seqs"]
    sizes = [n // s + (1 if i < n % s else 0) for i in range(s)]
    return [(int((c["max_pos"] - m) * (((i + 1) * 0.381966) % 1.0)), m) for i, m in enumerate(sizes)]


def _frequencies(c):
    """Rotation frequencies in 64 bits and the factor on cos and sin."""
    rot = c["rotary"]
    f = [ROPE_BASE ** (-2.0 * i / rot) for i in range(rot // 2)]
    if c["scaling"] == "linear":
        return [x / LINEAR["factor"] for x in f], 1.0
    if c["scaling"] == "yarn":
        at = lambda turns: rot * math.log(YARN["original"] / (turns * 2 * math.pi)) / (2 * math.log(ROPE_BASE))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(rot // 2)]
        return [x / YARN["factor"] * r + x * (1 - r) for x, r in zip(f, ramp)], 0.1 * math.log(YARN["factor"]) + 1.0
    return f, 1.0


def _pool(c, layers, pages, gen, dev):
    shape = (layers, 2, pages, c["kv_heads"], c["page"], c["head_dim"])
    kv = torch.empty(shape, dtype=DTYPES[c["cache"]], device=dev)
    for i in range(layers):
        x = torch.randn(shape[1:], device=dev, generator=gen, dtype=torch.float32)
        kv[i] = (x * 16.0 if c["cache"] == "fp8" else x).to(kv.dtype)
    return kv


def _scales(c, gen, dev):
    if c["cache"] != "fp8":
        return None, None
    n = c["kv_heads"]
    return tuple((torch.rand(n, device=dev, generator=gen) + 0.5) / 16.0 for _ in range(2))


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    s = {"case": c, "seed": seed}
    ps = c["page"]
    if c["op"] == "append":
        chunks = _chunks(c)
        width = -(-max(c["max_pos"], 1) // ps)
        spans = [(p // ps, -(-(p + m) // ps)) for p, m in chunks]
        used = sum(b - a for a, b in spans)
        pages = used + max(4, used // 8)
        ids = torch.randperm(pages, generator=host).tolist()
        table = torch.full((len(chunks), width), -1, dtype=torch.int32)
        for i, (a, b) in enumerate(spans):
            table[i, a:b] = torch.tensor([ids.pop() for _ in range(b - a)], dtype=torch.int32)
        dtype, n = DTYPES[c["dtype"]], c["tokens"]
        heads = c["q_heads"] + 2 * c["kv_heads"]
        # queries, keys and values come out of one projection, so each is a strided view of its rows
        qkv = torch.randn((n, heads, c["head_dim"]), device=dev, generator=gen).to(dtype)
        s["q"], s["k"], s["v"] = qkv.split([c["q_heads"], c["kv_heads"], c["kv_heads"]], dim=1)
        s["wq"], s["wk"] = ((1.0 + 0.1 * torch.randn(c["head_dim"], device=dev, generator=gen)).to(dtype)
                            if c["norm"] else None for _ in range(2))
        s["positions"] = _ints([p + j for p, m in chunks for j in range(m)], dev)
        s["token_seqs"] = _ints([i for i, (p, m) in enumerate(chunks) for _ in range(m)], dev)
        s["kv"] = _pool(c, 1, pages, gen, dev)
        s["table"] = table.to(dev)
        s["lens"] = _ints([p + m for p, m in chunks], dev)
        freqs, s["mscale"] = _frequencies(c)
        s["freqs"] = torch.tensor(freqs, dtype=torch.float32, device=dev)
    elif c["op"] == "attend":
        lens = _spread(c)
        each = [-(-n // ps) for n in lens]
        pages = sum(each) + max(4, sum(each) // 8)
        ids = torch.randperm(pages, generator=host)
        table = torch.full((len(lens), max(each)), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(each):
            table[i, :n] = ids[at:at + n].to(torch.int32)
            at += n
        s["q"] = torch.randn((len(lens), c["new"], c["q_heads"], c["head_dim"]), device=dev,
                             generator=gen).to(DTYPES[c["dtype"]])
        s["kv"] = _pool(c, 1, pages, gen, dev)
        s["table"], s["lens"] = table.to(dev), _ints(lens, dev)
    else:
        n, kids = c["parents"], c["children"]
        rows = n * (1 + kids)
        lens = [max(1, c["length"] - (i * 37) % max(1, c["length"] // 2)) for i in range(n)]
        each = [-(-x // ps) for x in lens]
        width = -(-(c["length"] + 4) // ps) + 1
        pages = c["num_pages"]
        if c["mode"] == "compact":  # sequences come and go: what is left is spread over the whole pool
            ids = torch.randperm(pages, generator=host)
        else:                       # the low pages are taken, a tenth of them have been given back
            ids = torch.randperm(min(pages, sum(each) + sum(each) // 10), generator=host)
        meta = torch.zeros(rows * width + rows + pages, dtype=torch.int32)
        table, length, refs = meta.split([rows * width, rows, pages])
        table = table.view(rows, width)
        table.fill_(-1)
        at = 0
        for i, m in enumerate(each):
            table[i, :m] = ids[at:at + m].to(torch.int32)
            at += m
        length[:n] = torch.tensor(lens, dtype=torch.int32)
        refs[ids[:at]] = 1
        # tables, lengths and counts lie in one block, so that one copy sets a pass's start again
        s["meta0"] = meta.to(dev)
        s["meta"] = s["meta0"].clone()
        table, s["lens"], s["refs"] = s["meta"].split([rows * width, rows, pages])
        s["table"] = table.view(rows, width)
        s["kv"] = _pool(c, c["layers"], pages, gen, dev)
        s["src"] = torch.arange(n, dtype=torch.int32, device=dev).repeat_interleave(kids)
        s["dst"] = torch.arange(n, rows, dtype=torch.int32, device=dev)
        s["all"] = torch.arange(rows, dtype=torch.int32, device=dev)
        s["grow"] = torch.full((rows,), 4 if c["mode"] == "step" else 1, dtype=torch.int32, device=dev)
        accept = [(i * 3) % 5 for i in range(n)]
        s["to"] = _ints([x + a for x, a in zip(lens, accept)], dev) if c["mode"] == "step" else None
    s["k_scale"], s["v_scale"] = _scales(c, gen, dev)
    if own:
        from xcalibur_b200 import PagedKVCache, Rope

        s["cache"] = PagedKVCache.from_tensors(s["kv"], s["table"], s["lens"], s.get("refs"), k_scale=s["k_scale"],
                                               v_scale=s["v_scale"])
        if c["op"] == "append":
            s["rope"] = Rope(c["rotary"], base=ROPE_BASE, interleaved=c["interleaved"],
                             scaling=SCALING[c["scaling"]], device=dev)
    return s


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    s, c = state, state["case"]
    if c["op"] == "append":
        q = _append_own(s) if own else _append_plain(s, c)
        return {"q": q, "kv": s["kv"]}
    if c["op"] == "attend":
        out = s["cache"].attend(0, s["q"], window=c["window"], return_lse=c["lse"]) if own else _attend_plain(s, c)
        return {"out": out[0], "lse": out[1]} if c["lse"] else {"out": out if own else out[0]}
    s["meta"].copy_(s["meta0"])
    if own:
        _pages_own(s, c)
    else:
        _pages_plain(s, c)
    out = {"table": s["table"], "lens": s["lens"], "refs": s["refs"]}
    if c["mode"] != "step":
        out["kv"] = s["kv"]
    return out


def _append_own(s):
    return s["cache"].append(0, s["q"], s["k"], s["v"], s["positions"], s["token_seqs"], s["rope"], q_weight=s["wq"],
                             k_weight=s["wk"], eps=EPS)


def _pages_own(s, c):
    cache = s["cache"]
    if c["mode"] == "step":
        cache.extend(s["all"], s["grow"])
        cache.truncate(s["all"], s["to"])
    elif c["mode"] == "fork":
        cache.fork(s["src"], s["dst"])
        cache.extend(s["all"], s["grow"])
    else:
        cache.compact()


def _rotate(x, cos, sin, rot, interleaved):
    head, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _append_plain(s, c):
    angle = s["positions"].float()[:, None] * s["freqs"]
    cos, sin = (angle.cos() * s["mscale"])[:, None], (angle.sin() * s["mscale"])[:, None]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["wq"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["wk"].float()
    q = _rotate(q, cos, sin, c["rotary"], c["interleaved"])
    k = _rotate(k, cos, sin, c["rotary"], c["interleaved"])
    kv, at = s["kv"][0], s["positions"].long()
    page = s["table"][s["token_seqs"].long(), at // c["page"]].long()
    if c["cache"] == "fp8":
        k = (k / s["k_scale"][:, None]).clamp(-448.0, 448.0)
        v = (v / s["v_scale"][:, None]).clamp(-448.0, 448.0)
    # 8-bit types have no indexed store: their bytes are stored
    raw = torch.uint8 if c["cache"] == "fp8" else torch.int16
    store = kv.view(raw)
    store[0, page, :, at % c["page"]] = k.to(kv.dtype).view(raw)
    store[1, page, :, at % c["page"]] = v.to(kv.dtype).view(raw)
    return q.to(s["q"].dtype)


def _attend_plain(s, c):
    b, new, hq, d = s["q"].shape
    hkv, ps = c["kv_heads"], c["page"]
    pages = s["table"].clamp(min=0).long()
    raw = s["kv"][0].view(torch.uint8 if c["cache"] == "fp8" else torch.int16)
    k, v = (raw[i][pages].view(s["kv"].dtype).float().transpose(1, 2).reshape(b, hkv, -1, d) for i in (0, 1))
    if c["cache"] == "fp8":
        k, v = k * s["k_scale"][:, None, None], v * s["v_scale"][:, None, None]
    q = s["q"].float().reshape(b, new, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    scores = (q @ k.transpose(-1, -2) * d ** -0.5).reshape(b, hkv, hq // hkv, new, -1)
    at = torch.arange(k.shape[2], device=k.device)
    last = s["lens"][:, None].long() - new + torch.arange(new, device=k.device)  # position of each new token
    seen = at <= last[..., None]
    if c["window"]:
        seen = seen & (at > last[..., None] - c["window"])
    seen = seen[:, None, None]
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = (scores - top.masked_fill(top == float("-inf"), 0.0)).exp()
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0, 1.0)
    out = (p.reshape(b, hkv, -1, p.shape[-1]) @ v).reshape(b, hkv, hq // hkv, new, d)
    lse = (top + total.log()).squeeze(-1)
    return out.permute(0, 3, 1, 2, 4).reshape(b, new, hq, d).to(s["q"].dtype), lse.permute(0, 3, 1, 2).reshape(b, new, hq)


def _pages_plain(s, c):
    if c["mode"] == "compact":
        _compact_plain(s)
        return
    if c["mode"] == "fork":
        row = s["table"][s["src"].long()]
        s["table"][s["dst"].long()] = row
        s["lens"][s["dst"].long()] = s["lens"][s["src"].long()]
        live = (row >= 0).to(torch.int32)
        s["refs"].index_add_(0, row.clamp(min=0).flatten().long(), live.flatten())
    _extend_plain(s, c)
    if c["mode"] == "step":
        ps, seqs = c["page"], s["all"].long()
        row = s["table"][seqs]
        gone = (torch.arange(row.shape[1], device=row.device) >= -(-s["to"] // ps)[:, None]) & (row >= 0)
        s["refs"].index_add_(0, row.clamp(min=0).flatten().long(), -gone.flatten().to(torch.int32))
        s["table"][seqs] = row.masked_fill(gone, -1)
        s["lens"][seqs] = s["to"]


def _extend_plain(s, c):
    """Room for ``grow`` more tokens in each sequence: the lowest free pages go to the sequences in their order.  A
    last page that is part full and shared is copied first; where all its holders grow, the first one keeps it."""
    refs, ps, seqs = s["refs"], c["page"], s["all"].long()
    n, pages, dev = seqs.numel(), refs.numel(), refs.device
    row, ln = s["table"][seqs].long(), s["lens"][seqs].long()
    have, want = -(-ln // ps), -(-(ln + s["grow"]) // ps)
    last = row.gather(1, (have - 1).clamp(min=0)[:, None])[:, 0].clamp(min=0)
    shared = (ln % ps != 0) & (refs[last] > 1)
    order = torch.arange(n, device=dev)
    holders = torch.zeros(pages, dtype=torch.int32, device=dev).index_add_(0, last, shared.to(torch.int32))
    first = torch.full((pages,), n, dtype=torch.long, device=dev)
    first.scatter_reduce_(0, last, torch.where(shared, order, n), "amin")
    copied = shared & ~((holders[last] == refs[last]) & (first[last] == order))
    need = want - have + copied
    start = (have - copied.long())[:, None]
    offset = (need.cumsum(0) - need)[:, None]
    free = refs == 0
    ids = torch.arange(pages, device=dev)
    free_list = torch.zeros(pages + 1, dtype=torch.long, device=dev)
    free_list.scatter_(0, torch.where(free, free.cumsum(0) - 1, pages), ids)
    j = torch.arange(row.shape[1], device=dev)
    fresh = (j >= start) & (j < want[:, None])
    grown = torch.where(fresh, free_list[(offset + j - start).clamp(0, pages - 1)], row)
    refs.index_add_(0, last, -copied.to(torch.int32))
    refs.index_add_(0, grown.clamp(min=0).flatten(), fresh.flatten().to(torch.int32))
    s["table"][seqs] = grown.to(torch.int32)
    s["lens"][seqs] = (ln + s["grow"]).to(torch.int32)
    if c["mode"] == "fork":  # only forked sequences share pages; how many are copied is known on the device alone
        at = copied.nonzero()[:, 0]
        raw = s["kv"].view(torch.uint8 if c["cache"] == "fp8" else torch.int16)
        to, frm = grown[at, have[at] - 1], last[at]
        kept = (torch.arange(ps, device=dev) < (ln % ps)[at][:, None])[:, None, :, None]
        raw[:, :, to] = torch.where(kept, raw[:, :, frm], raw[:, :, to])


def _compact_plain(s):
    """Live pages from the top of the pool fill the holes below, both in ascending order."""
    refs, raw = s["refs"], s["kv"].view(torch.uint8 if s["kv"].element_size() == 1 else torch.int16)
    live, ids = refs > 0, torch.arange(refs.numel(), device=refs.device)
    count = live.sum()
    frm, to = (live & (ids >= count)).nonzero()[:, 0], (~live & (ids < count)).nonzero()[:, 0]
    raw[:, :, to] = raw[:, :, frm]
    moved = ids.clone()
    moved[frm] = to
    refs[to] = refs[frm]
    refs[frm] = 0
    s["table"].copy_(torch.where(s["table"] >= 0, moved[s["table"].clamp(min=0).long()].to(torch.int32), s["table"]))


# ------------------------------------------------------------------------------------------------ what a pass needs

def work(case):
    c, d = case, case["head_dim"]
    es = BYTES[c["cache"]]
    if c["op"] == "append":
        n, hq, hkv = c["tokens"], c["q_heads"], c["kv_heads"]
        b = n * d * (2 * (2 * hq + 2 * hkv) + 2 * hkv * es) + n * 12
        return {"bytes": b, "flops": n * (hq + hkv) * d * (8 if c["norm"] else 4)}
    if c["op"] == "attend":
        new, hq, hkv = c["new"], c["q_heads"], c["kv_heads"]
        read = pairs = 0
        for n in _spread(c):
            span = c["window"] or n
            read += min(n, span + new - 1)
            pairs += sum(min(span, max(0, n - new + i + 1)) for i in range(new))
        b = read * hkv * 2 * d * es + c["batch"] * new * hq * d * 4 + read // c["page"] * 4
        return {"bytes": b, "flops": 4 * d * hq * pairs}
    plane = c["layers"] * 2 * c["kv_heads"] * d * es
    n, ps = c["parents"], c["page"]
    lens = [max(1, c["length"] - (i * 37) % max(1, c["length"] // 2)) for i in range(n)]
    rows = n * (1 + c["children"])
    meta = 4 * (c["num_pages"] + rows * 8)
    if c["mode"] == "step":
        return {"bytes": meta, "flops": 0}
    if c["mode"] == "fork":
        moved = sum(x % ps for x in lens) * c["children"]
    else:  # a live page lies above the live count with the chance that the count leaves free
        live = sum(-(-x // ps) for x in lens)
        moved = live * (1 - live / c["num_pages"]) * ps
    return {"bytes": meta + 2 * moved * plane, "flops": 0}


# ------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    """The definitions in 64 bits, one sequence at a time."""
    s, c = prepare(case, seed), case
    ps, hkv, d = c["page"], c["kv_heads"], c["head_dim"]
    if c["op"] == "append":
        return _append_exact(s, c)
    if c["op"] == "attend":
        lens, table = s["lens"].tolist(), s["table"].tolist()
        raw = s["kv"][0].view(torch.uint8 if c["cache"] == "fp8" else torch.int16)
        g = c["q_heads"] // hkv
        outs, lses = [], []
        for i, n in enumerate(lens):
            lo = max(0, n - c["new"] + 1 - c["window"]) // ps if c["window"] else 0
            ids = torch.tensor(table[i][lo:-(-n // ps)], dtype=torch.long, device=raw.device)
            k, v = (raw[j][ids].view(s["kv"].dtype).double().transpose(0, 1).reshape(hkv, -1, d) for j in (0, 1))
            if c["cache"] == "fp8":
                k, v = k * s["k_scale"].double()[:, None, None], v * s["v_scale"].double()[:, None, None]
            rows, sums = [], []
            for t in range(c["new"]):
                end = n - c["new"] + t + 1
                begin = max(0, end - c["window"]) if c["window"] else 0
                if end <= begin:
                    rows.append(torch.zeros(c["q_heads"], d, dtype=torch.float64, device=raw.device))
                    sums.append(torch.full((c["q_heads"],), -math.inf, dtype=torch.float64, device=raw.device))
                    continue
                q = s["q"][i, t].double().view(hkv, g, d)
                score = torch.einsum("hgd,htd->hgt", q, k[:, begin - lo * ps:end - lo * ps]) / math.sqrt(d)
                rows.append(torch.einsum("hgt,htd->hgd", score.softmax(-1), v[:, begin - lo * ps:end - lo * ps]).reshape(-1, d))
                sums.append(score.logsumexp(-1).reshape(-1))
            outs.append(torch.stack(rows))
            lses.append(torch.stack(sums))
        out = {"out": torch.stack(outs)}
        return dict(out, lse=torch.stack(lses)) if c["lse"] else out
    if c["mode"] == "step":
        return None
    table, lens, refs = s["table"].tolist(), s["lens"].tolist(), s["refs"].tolist()
    raw = s["kv"].view(torch.uint8 if c["cache"] == "fp8" else torch.int16)
    if c["mode"] == "compact":
        live = [i for i, r in enumerate(refs) if r]
        holes = [i for i, r in enumerate(refs) if not r and i < len(live)]
        for frm, to in zip([i for i in live if i >= len(live)], holes):
            raw[:, :, to] = raw[:, :, frm]
        return {"table": None, "lens": None, "refs": None, "kv": s["kv"]}
    n, kids = c["parents"], c["children"]
    for k in range(n * kids):  # every sample holds its prompt's pages
        table[n + k], lens[n + k] = list(table[k // kids]), lens[k // kids]
        for p in table[n + k]:
            if p >= 0:
                refs[p] += 1
    free = iter([i for i, r in enumerate(refs) if r == 0])
    for i in range(len(lens)):  # the prompts come first in the list, so each keeps its last page
        used = lens[i] % ps
        if used == 0:
            next(free)
        elif i >= n:
            to = next(free)
            raw[:, :, to, :, :used] = raw[:, :, table[i][lens[i] // ps], :, :used]
    return {"table": None, "lens": None, "refs": None, "kv": s["kv"]}


def _append_exact(s, c):
    freqs, mscale = _frequencies(c)
    freqs = torch.tensor(freqs, dtype=torch.float64, device=s["q"].device)
    where, owner, table = s["positions"].tolist(), s["token_seqs"].tolist(), s["table"].tolist()
    rot, ps = c["rotary"], c["page"]
    angle = torch.tensor(where, dtype=torch.float64, device=freqs.device)[:, None] * freqs
    turn = torch.polar(torch.full_like(angle, mscale), angle)[:, None]

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
        if c["interleaved"]:
            z = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) * turn
            return torch.cat([torch.view_as_real(z).flatten(-2), x[..., rot:]], -1)
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * turn
        return torch.cat([z.real, z.imag, x[..., rot:]], -1)

    kv = s["kv"].double()
    slot = torch.tensor([table[o][p // ps] * ps + p % ps for o, p in zip(owner, where)], device=freqs.device)
    for i, x in enumerate((turned(s["k"], s["wk"]), s["v"].double())):
        if c["cache"] == "fp8":
            x = (x / (s["k_scale"], s["v_scale"])[i].double()[:, None]).clamp(-448.0, 448.0)
        kv[0, i].transpose(1, 2)[slot // ps, slot % ps] = x
    return {"q": turned(s["q"], s["wq"]), "kv": kv}
