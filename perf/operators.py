"""Measured cases of the attention-sublayer operators: per-head norms with the
position rotation (norm_rope), appending keys and values to the paged 8-bit
cache (append), attention over that cache (attend), and the two in one call as
a decoder layer runs them (layer).

A cache holds blocks of 16 tokens: 8-bit values and one scale for each block
and head. Pages are [n_pages][kv_heads][blocks of the page], a key block
[D/64][16][64] and a value block [D][16]. Sequence b of a batch has past_b
cached tokens and new_b new rows; row i sits at position past_b + i.
"""
import functools
import math
import os
import sys

import torch

own = False

ACT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
THETA, EPS = 1.0e6, 1.0e-6


def listed():
    wide = {"q_heads": 32, "kv_heads": 4, "D": 128, "rope": 128, "interleaved": False, "page": 64, "window": 0}
    small = {"q_heads": 14, "kv_heads": 2, "D": 64, "rope": 32, "interleaved": True, "page": 16, "window": 0}
    return [
        # one token of a few chats: launch latency
        {"name": "norm_rope decode f32", "op": "norm_rope", "act": "f32", "B": 8, "past": 4000, "new": 1, "ragged": True, **wide},
        # ragged prompts, half of a head rotating in interleaved pairs, odd row count
        {"name": "norm_rope prompts bf16", "op": "norm_rope", "act": "bf16", "B": 9, "past": 70000, "new": 1801, "ragged": True, **small},
        # a decode step of a serving batch
        {"name": "append decode f32", "op": "append", "act": "f32", "B": 64, "past": 3000, "new": 1, "ragged": True, **wide},
        # prompts that start and end inside a block
        {"name": "append prompts bf16", "op": "append", "act": "bf16", "B": 5, "past": 1003, "new": 2500, "ragged": True, **wide},
        # one chat with a short history: latency
        {"name": "attend one short f32", "op": "attend", "act": "f32", "B": 1, "past": 700, "new": 1, "ragged": False, **wide},
        # a full serving batch of uneven histories
        {"name": "attend batch bf16", "op": "attend", "act": "bf16", "B": 64, "past": 8190, "new": 1, "ragged": True, **wide},
        # one very long history: work split over its length
        {"name": "attend one long f32", "op": "attend", "act": "f32", "B": 1, "past": 131000, "new": 1, "ragged": False, **wide},
        # a few drafted tokens at a time under a sliding window, seven query heads for each key head
        {"name": "attend drafts windowed f16", "op": "attend", "act": "f16", "B": 17, "past": 5001, "new": 5, "ragged": True, **{**small, "window": 1024}},
        # the second half of a long prompt
        {"name": "attend prompt bf16", "op": "attend", "act": "bf16", "B": 1, "past": 4096, "new": 4096, "ragged": False, **wide},
        # ragged prompt chunks with 32-bit activations
        {"name": "attend prompts f32", "op": "attend", "act": "f32", "B": 3, "past": 1500, "new": 1025, "ragged": True, **wide},
        # a decoder layer's attention for a batch of single tokens
        {"name": "layer decode f32", "op": "layer", "act": "f32", "B": 32, "past": 2040, "new": 1, "ragged": True, **wide},
        # and for ragged prompts, some of them new
        {"name": "layer prompts bf16", "op": "layer", "act": "bf16", "B": 4, "past": 300, "new": 1300, "ragged": True, **wide},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    D = rng.choice((64, 128))
    c = {"op": rng.choice(("norm_rope", "append", "attend", "attend", "attend", "layer", "layer")),
         "act": rng.choice(("f32", "f16", "bf16")), "q_heads": kv_heads * rng.choice((1, 2, 4, 5, 7, 8, 12, 16)),
         "kv_heads": kv_heads, "D": D, "rope": rng.choice((D, D, D // 2, 2)), "interleaved": rng.random() < 0.4,
         "page": rng.choice((16, 32, 64, 128, 256)), "window": rng.choice((0, 0, _log(rng, 1, 5000)))}
    if rng.random() < 0.55:   # single tokens or a few drafted ones
        new = rng.choice((1, 1, 1, 2, 3, 5, 8))
        B = _log(rng, 1, 96)
        past = _log(rng, 1, min(130000, 400000 // B))
    else:                     # prompts and their chunks
        B = _log(rng, 1, 6)
        new = _log(rng, 9, 4000 // B)
        past = rng.choice((0, _log(rng, 1, 5000)))
    return {**c, "B": B, "past": past, "new": new, "ragged": rng.random() < 0.7}


def _lengths(c):
    """Cached tokens and new rows of each sequence; ragged: uneven histories and prompts, one of them without new rows."""
    past, new = [], []
    for b in range(c["B"]):
        drop = c["ragged"] and b > 0
        past.append(c["past"] - (b * 7919 % (c["past"] // 2 + 1) if drop else 0))
        new.append(c["new"] - (b * 4099 % (c["new"] // 2 + 1) if drop else 0))
    if c["ragged"] and c["B"] > 3 and c["new"] > 1:
        new[2] = 0
    return past, new


def work(case):
    c, (past, new) = case, _lengths(case)
    T, D, hq, hk = sum(new), case["D"], case["q_heads"], case["kv_heads"]
    size = 4 if c["act"] == "f32" else 2
    w = {"bytes": 0.0, "flops": 0.0}
    if c["op"] == "norm_rope":
        w["bytes"] += 2.0 * T * (hq + hk) * D * size
        w["flops"] += 8.0 * T * (hq + hk) * D
    if c["op"] in ("append", "layer"):   # rows in, 8-bit blocks and scales out, the open block in and out
        w["bytes"] += 2.0 * T * hk * D * size
        w["bytes"] += sum(2.0 * hk * (-(-(p % 16 + n) // 16) * (16 * D + 4) + (p % 16 + (p + n) % 16) * D * 4)
                          for p, n in zip(past, new) if n)
        w["flops"] += 10.0 * T * hk * D
    if c["op"] in ("attend", "layer"):
        w["bytes"] += 2.0 * T * hq * D * size
        for p, n in zip(past, new):
            if n:
                first = max(0, p - c["window"] + 1) if c["window"] else 0
                w["bytes"] += 2.0 * (p + n - first) * hk * (D + 0.25)
                seen = sum(min(p + i + 1, c["window"]) for i in range(n)) if c["window"] else n * p + n * (n + 1) // 2
                w["flops"] += 4.0 * seen * hq * D
    return w


def prepare(case, seed):
    c, (past, new) = case, _lengths(case)
    dev, act = "cuda", ACT[case["act"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    B, hq, hk, D, page = c["B"], c["q_heads"], c["kv_heads"], c["D"], c["page"]
    T = sum(new)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    def offsets(v):
        return ints([sum(v[:b]) for b in range(B + 1)])

    s = {"case": dict(c), "past": ints(past), "new": ints(new), "row_start": offsets(new), "T": T, "max_new": max(new),
         "slot": torch.randperm(B, generator=g, device=dev).to(torch.int32)}
    # rows of one fused projection: queries, keys, values side by side
    width = (hq + 2 * hk) * D
    s["qkv"] = torch.randn(T, width, generator=g, device=dev).to(act)
    s["q"], s["k"], s["v"] = s["qkv"].split([hq * D, hk * D, hk * D], dim=1)
    s["q_norm"] = 1.0 + 0.2 * torch.randn(D, generator=g, device=dev)
    s["k_norm"] = 1.0 + 0.2 * torch.randn(D, generator=g, device=dev)
    if c["op"] == "norm_rope":
        return s
    pages = [-(-(p + n) // page) for p, n in zip(past, new)]
    n_pages, stride = sum(pages) + 2, max(pages) + 1
    ids = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((B, stride), -1, dtype=torch.int32, device=dev)
    slots, at = s["slot"].tolist(), 0
    for b in range(B):
        table[slots[b], : pages[b]] = ids[at: at + pages[b]]
        at += pages[b]
    s["table"] = table
    blocks = page // 16
    for name, inner in (("k", (D // 64, 16, 64)), ("v", (D, 16))):
        pool = torch.empty((n_pages, hk, blocks) + inner, dtype=torch.int8, device=dev)
        flat = pool.view(-1)
        for i in range(0, flat.numel(), 1 << 27):
            n = min(1 << 27, flat.numel() - i)
            flat[i: i + n] = torch.randn(n, generator=g, device=dev).mul_(36.0).round_().clamp_(-127, 127).to(torch.int8)
        s[name + "_pool"] = pool
        s[name + "_scale"] = 0.03 * torch.exp(0.3 * torch.randn(n_pages, hk, blocks, generator=g, device=dev))
        s[name + "_open"] = torch.randn(B, hk, 16, D, generator=g, device=dev)
    if c["op"] != "attend":   # the blocks an append touches, as rows to read back
        base = [p // 16 * 16 if n else p for p, n in zip(past, new)]
        s["base"] = ints(base)
        s["read_start"] = offsets([p + n - t for p, n, t in zip(past, new, base)])
        s["read_rows"] = sum(p + n - t for p, n, t in zip(past, new, base))
        s["most_read"] = max(p + n - t for p, n, t in zip(past, new, base))
    return s


# ---------------------------------------------------------------- plain form


def _rows(start, count, most):
    """Rows of each sequence as [B, most] with a mask of the real ones."""
    i = torch.arange(most, device=start.device)
    return start[:-1, None].long() + i, i < count[:, None]


def _positions(s):
    """Position of each row [T]."""
    row = torch.arange(s["T"], dtype=torch.int32, device="cuda")
    b = torch.searchsorted(s["row_start"][1:].contiguous(), row, right=True)
    return s["past"][b].long() + row - s["row_start"][b].long()


def _norm_rope(x, w, pos, c):
    """x [T, heads, D] normed per head and rotated, in x's type (32 or 64 bits); the angles in 64 bits."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.to(x.dtype)
    R = c["rope"]
    inv = THETA ** (-torch.arange(0, R, 2, dtype=torch.float64, device=x.device) / R)
    angle = pos[:, None].double() * inv
    cos, sin = angle.cos().to(x.dtype)[:, None], angle.sin().to(x.dtype)[:, None]
    turn, rest = x[..., :R], x[..., R:]
    if c["interleaved"]:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turn[..., : R // 2], turn[..., R // 2:]
        turn = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turn, rest), -1)


def _quantise(x):
    """Blocks x [..., 16, D] in 32 bits: 8-bit values and the scale of each block. In 64 bits, for values next to a border."""
    scale = (x.abs().amax((-1, -2)).double() / 127).float()
    q = (x.double() / scale.double().clamp(min=1e-30)[..., None, None]).round()
    return q.to(torch.int8), scale


def _append(s):
    c = s["case"]
    hk, D, page = c["kv_heads"], c["D"], c["page"]
    head = s["past"] % 16
    total = torch.where(s["new"] > 0, head + s["new"], 0)    # tokens from the first touched block on
    W = (s["max_new"] + 15 + 15) // 16 * 16
    rows, real = _rows(s["row_start"], s["new"], W)
    i = torch.arange(W, device="cuda")
    rows = (rows - head[:, None]).clamp(0, s["T"] - 1)       # row of each token from the block's start on
    fresh = (i >= head[:, None]) & (i < total[:, None])
    nb = W // 16
    block = torch.arange(nb, device="cuda")
    touched = block * 16 < total[:, None]
    at = s["past"][:, None] // 16 + block
    pages = s["table"][s["slot"].long()[:, None], (at * 16 // page).clamp(max=s["table"].shape[1] - 1)]
    k = _norm_rope(s["k"].view(-1, hk, D).double(), s["k_norm"], _positions(s), c).float()
    v = s["v"].reshape(-1, hk, D).float()
    last = total - (s["past"] + s["new"]) % 16               # first token of the block left open
    for name, x in (("k", k), ("v", v)):
        old = s[name + "_open"][s["slot"].long()].transpose(1, 2)                      # [B, 16, hk, D]
        old = torch.nn.functional.pad(old, (0, 0, 0, 0, 0, W - 16))
        x = torch.where(fresh[..., None, None], x[rows], torch.where((i < head[:, None])[..., None, None], old, 0.0))
        x = torch.where((i < total[:, None])[..., None, None], x, 0.0)
        # the open block's rows
        j = torch.arange(16, device="cuda")
        keep = (j < ((s["past"] + s["new"]) % 16)[:, None]) & (s["new"] > 0)[:, None]
        tail = torch.gather(x, 1, (last[:, None] + j).clamp(0, W - 1)[..., None, None].expand(-1, -1, hk, D))
        slots = s["slot"].long()
        cur = s[name + "_open"][slots]
        s[name + "_open"][slots] = torch.where(keep[:, None, :, None], tail.transpose(1, 2), cur)
        q, scale = _quantise(x.view(-1, nb, 16, hk, D).transpose(2, 3))                # [B, nb, hk, 16, D]
        q = q.unflatten(-1, (D // 64, 64)).transpose(3, 4) if name == "k" else q.transpose(3, 4)
        p, blk = pages[touched].long(), (at % (page // 16))[touched].long()
        s[name + "_pool"].transpose(1, 2)[p, blk] = q[touched]
        s[name + "_scale"].transpose(1, 2)[p, blk] = scale[touched]


def _cached(s, name, first_block, blocks):
    """Values of `blocks` blocks of each sequence from first_block [B] on: [B, hk, blocks * 16, D] in 32 bits."""
    c, page = s["case"], s["case"]["page"]
    at = first_block[:, None] + torch.arange(blocks, device="cuda")
    p = s["table"][s["slot"].long()[:, None], (at * 16 // page).clamp(max=s["table"].shape[1] - 1)].long().clamp(min=0)
    blk = at % (page // 16)
    x = s[name + "_pool"].transpose(1, 2)[p, blk]                                      # [B, blocks, hk, ...]
    x = x.transpose(3, 4).flatten(4) if name == "k" else x.transpose(3, 4)             # [B, blocks, hk, 16, D]
    x = x.float() * s[name + "_scale"].transpose(1, 2)[p, blk][..., None, None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _read(s):
    """The cache's rows from each sequence's first touched block on, in the rows' type."""
    c = s["case"]
    count = s["read_start"][1:] - s["read_start"][:-1]
    rows, real = _rows(s["read_start"], count, (s["most_read"] + 15) // 16 * 16)
    got = [_cached(s, n, torch.div(s["base"], 16, rounding_mode="floor"), rows.shape[1] // 16).transpose(1, 2)[real]
           for n in ("k", "v")]
    return [x.to(ACT[c["act"]]) for x in got]


def _attend(s, q):
    """q [T, hq, D] in 32 bits."""
    c = s["case"]
    B, hq, hk, D, n = c["B"], c["q_heads"], c["kv_heads"], c["D"], s["max_new"]
    L = (int(c["past"]) + int(c["new"]) + 15) // 16 * 16
    rows, real = _rows(s["row_start"], s["new"], n)
    x = q[rows.clamp(max=s["T"] - 1)].view(B, n, hk, hq // hk, D).permute(0, 2, 1, 3, 4).flatten(2, 3)
    zero = torch.zeros_like(s["past"])
    p = x @ _cached(s, "k", zero, L // 16).transpose(-1, -2) * (1.0 / math.sqrt(D))    # [B, hk, n * g, L]
    pos = (s["past"][:, None] + torch.arange(n, device="cuda")).repeat_interleave(hq // hk, 1)[:, None, :, None]
    j = torch.arange(L, device="cuda")
    seen = j <= pos
    if c["window"]:
        seen = seen & (j > pos - c["window"])
    p.masked_fill_(~seen, -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    v = _cached(s, "v", zero, L // 16)
    v.masked_fill_((j >= (s["past"] + s["new"])[:, None])[:, None, :, None], 0.0)
    o = (p @ v) / p.sum(-1, keepdim=True)
    o = o.view(B, hk, n, hq // hk, D).permute(0, 2, 1, 3, 4).flatten(2)
    return o[real].to(ACT[c["act"]])


def _plain(s):
    c = s["case"]
    hq, hk, D, act = c["q_heads"], c["kv_heads"], c["D"], ACT[c["act"]]
    if c["op"] == "norm_rope":
        pos = _positions(s)
        return {n: _norm_rope(s[n].reshape(-1, h, D).float(), s[n + "_norm"], pos, c).to(act) for n, h in (("q", hq), ("k", hk))}
    if c["op"] == "attend":
        return {"out": _attend(s, s["q"].reshape(-1, hq, D).float())}
    _append(s)
    out = {}
    if c["op"] == "layer":
        out["out"] = _attend(s, _norm_rope(s["q"].reshape(-1, hq, D).float(), s["q_norm"], _positions(s), c))
    out["k"], out["v"] = _read(s)
    return {**out, **{n: s[n] for n in ("k_scale", "v_scale", "k_open", "v_open")}}


# ------------------------------------------------------- the framework's calls


@functools.lru_cache(None)
def _context():
    """The library's context, as a program holds it: on torch's stream, the legacy default one."""
    sys.path.insert(0, os.path.join(os.getcwd(), "jero-engine_b200"))
    import jeromoe
    ctx = jeromoe.Context(0, max_tokens=1 << 16)
    ctx.set_stream(jeromoe.STREAM_LEGACY)
    return jeromoe, ctx


def _handles(s):
    """The descriptions of cache, batch and rows that a program keeps over its steps."""
    jm, ctx = _context()
    c = s["case"]
    act = {"f32": jm.F32, "f16": jm.F16, "bf16": jm.BF16}[c["act"]]
    hq, hk, D = c["q_heads"], c["kv_heads"], c["D"]
    h = {"batch": jm.KvBatch(n_seqs=c["B"], n_tokens=s["T"], past=s["past"].data_ptr(), row_start=s["row_start"].data_ptr(),
                             slot=s["slot"].data_ptr(), max_new=s["max_new"]),
         "rope": jm.Rope(rope_dim=c["rope"], interleaved=c["interleaved"], theta=THETA, eps=EPS,
                         q_norm=s["q_norm"].data_ptr(), k_norm=s["k_norm"].data_ptr()),
         "rows": jm.QkvRows(act=act, q_heads=hq, kv_heads=hk, head_dim=D, q=s["q"].data_ptr(), k=s["k"].data_ptr(),
                            v=s["v"].data_ptr(), q_stride=s["qkv"].stride(0), k_stride=s["qkv"].stride(0),
                            v_stride=s["qkv"].stride(0)),
         "opts": jm.AttnOpts(window=c["window"])}
    if c["op"] != "norm_rope":
        h["cache"] = jm.KvCache(head_dim=D, kv_heads=hk, page_tokens=c["page"], n_pages=s["k_pool"].shape[0],
                                n_slots=s["table"].shape[0], table_stride=s["table"].shape[1],
                                page_table=s["table"].data_ptr(), k=s["k_pool"].data_ptr(), v=s["v_pool"].data_ptr(),
                                k_scale=s["k_scale"].data_ptr(), v_scale=s["v_scale"].data_ptr(),
                                open_k=s["k_open"].data_ptr(), open_v=s["v_open"].data_ptr())
    if "base" in s:
        h["touched"] = jm.KvBatch(n_seqs=c["B"], n_tokens=s["read_rows"], past=s["base"].data_ptr(),
                                  row_start=s["read_start"].data_ptr(), slot=s["slot"].data_ptr(), max_new=s["most_read"])
    return h


def _own(s):
    jm, ctx = _context()
    if "handles" not in s:
        s["handles"] = _handles(s)
    h, c, act = s["handles"], s["case"], ACT[s["case"]["act"]]
    hq, hk, D, T = c["q_heads"], c["kv_heads"], c["D"], s["T"]

    def rows(n, heads):
        return torch.empty((n, heads, D), dtype=act, device="cuda")

    def into(q=None, k=None, v=None):
        r = h["rows"]
        return jm.QkvRows(act=r.act, q_heads=hq, kv_heads=hk, head_dim=D, q=q.data_ptr() if q is not None else 0,
                          k=k.data_ptr() if k is not None else 0, v=v.data_ptr() if v is not None else 0,
                          q_stride=hq * D, k_stride=hk * D, v_stride=hk * D)

    if c["op"] == "norm_rope":
        q, k = rows(T, hq), rows(T, hk)
        ctx.qk_norm_rope(h["batch"], h["rope"], h["rows"], into(q, k))
        return {"q": q, "k": k}
    if c["op"] == "attend":
        out = torch.empty((T, hq * D), dtype=act, device="cuda")
        ctx.kv_attention(h["cache"], h["batch"], h["opts"], h["rows"], out.data_ptr(), hq * D)
        return {"out": out}
    got = {}
    if c["op"] == "append":
        ctx.kv_append(h["cache"], h["batch"], h["rope"], h["rows"])
    else:
        got["out"] = torch.empty((T, hq * D), dtype=act, device="cuda")
        ctx.attention(h["cache"], h["batch"], h["rope"], h["opts"], h["rows"], got["out"].data_ptr(), hq * D)
    got["k"], got["v"] = rows(s["read_rows"], hk), rows(s["read_rows"], hk)
    ctx.kv_read(h["cache"], h["touched"], into(k=got["k"], v=got["v"]))
    return {**got, **{n: s[n] for n in ("k_scale", "v_scale", "k_open", "v_open")}}


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------- 64-bit definition


def _turned(x, w, first, c):
    """Rows x [n, heads, D] at positions first, first + 1, ...: the definition in 64 bits, by complex numbers."""
    x = x.double()
    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()
    R = c["rope"]
    i = torch.arange(R // 2, device=x.device, dtype=torch.float64)
    angle = (first + torch.arange(x.shape[0], device=x.device, dtype=torch.float64))[:, None] * torch.exp(-math.log(THETA) * 2.0 * i / R)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    y = x.clone()
    if c["interleaved"]:
        z = torch.view_as_complex(x[..., :R].reshape(*x.shape[:-1], R // 2, 2).contiguous()) * turn
        y[..., :R] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., : R // 2], x[..., R // 2: R]) * turn
        y[..., : R // 2], y[..., R // 2: R] = z.real, z.imag
    return y


def exact(case, seed):
    s, c, (past, new) = prepare(case, seed), case, _lengths(case)
    hq, hk, D, page = c["q_heads"], c["kv_heads"], c["D"], c["page"]
    q_in, k_in, v_in = (s[n].reshape(-1, h, D) for n, h in (("q", hq), ("k", hk), ("v", hk)))
    outs, ks, vs, at = [], [], [], 0
    for b, (p, n) in enumerate(zip(past, new)):
        rows = slice(at, at + n)
        at += n
        if not n:
            continue
        if c["op"] == "norm_rope":
            outs.append(_turned(q_in[rows], s["q_norm"], p, c))
            ks.append(_turned(k_in[rows], s["k_norm"], p, c))
            continue
        slot, total = int(s["slot"][b]), p + n
        page_ids = s["table"][slot, : -(-total // page)].long()
        full = {}
        for name in ("k", "v"):
            pool = s[name + "_pool"][page_ids].transpose(0, 1).flatten(1, 2)           # [hk, blocks, ...]
            scale = s[name + "_scale"][page_ids].transpose(0, 1).flatten(1, 2)
            if c["op"] != "attend":
                x = _turned(k_in[rows], s["k_norm"], p, c).float() if name == "k" else v_in[rows].float()
                x = torch.cat((s[name + "_open"][slot, :, : p % 16], x.transpose(0, 1)), 1)
                left = x.shape[1] % 16
                if left:
                    s[name + "_open"][slot, :, :left] = x[:, -left:]
                x = torch.nn.functional.pad(x, (0, 0, 0, -x.shape[1] % 16)).unflatten(1, (-1, 16))
                sc = (x.double().abs().flatten(2).max(-1).values / 127).float()
                qv = torch.round(x.double() / sc.double()[..., None, None])
                first = p // 16
                pool = pool.double()
                pool[:, first: first + x.shape[1]] = (qv.unflatten(-1, (D // 64, 64)).permute(0, 1, 3, 2, 4) if name == "k"
                                                      else qv.transpose(2, 3))
                scale = scale.clone()
                scale[:, first: first + x.shape[1]] = sc
                blocks = torch.arange(first, first + x.shape[1], device="cuda")
                s[name + "_scale"][page_ids[blocks * 16 // page], :, blocks % (page // 16)] = sc.transpose(0, 1)
            pool = pool.double() * scale.double().view(hk, -1, *[1] * (pool.dim() - 2))
            pool = pool.transpose(2, 3).flatten(3) if name == "k" else pool.transpose(2, 3)
            full[name] = pool.reshape(hk, -1, D)[:, :total]
        if c["op"] != "attend":
            ks.append(full["k"][:, p // 16 * 16:].transpose(0, 1))
            vs.append(full["v"][:, p // 16 * 16:].transpose(0, 1))
        if c["op"] == "append":
            continue
        q = q_in[rows].double() if c["op"] == "attend" else _turned(q_in[rows], s["q_norm"], p, c)
        where = p + torch.arange(n, device="cuda")[:, None]
        key = torch.arange(total, device="cuda")
        hide = key > where
        if c["window"]:
            hide |= key <= where - c["window"]
        o = torch.empty(n, hq, D, dtype=torch.float64, device="cuda")
        for h in range(hq):
            e = torch.einsum("id,jd->ij", q[:, h], full["k"][h * hk // hq]) / math.sqrt(D)
            o[:, h] = torch.softmax(e.masked_fill_(hide, -math.inf), -1) @ full["v"][h * hk // hq]
        outs.append(o)
    if c["op"] == "norm_rope":
        return {"q": torch.cat(outs), "k": torch.cat(ks)}
    got = {"out": torch.cat(outs).flatten(1)} if outs else {}
    if c["op"] == "attend":
        return got
    return {**got, "k": torch.cat(ks), "v": torch.cat(vs),
            **{n: s[n].double() for n in ("k_scale", "v_scale", "k_open", "v_open")}}
