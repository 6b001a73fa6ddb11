"""The operators around a cache held in 4 bits, case by case: the write that quantises, the read-back, attention of
new tokens over such a cache, and the copy of whole pages (of any cache type) that a fork of sequences makes.

``run`` computes a case either in its plain form (elementary torch operations in fp32) or, with ``own`` set, through
``ijb200.ops``.  Shapes follow the engine: 8 KV heads of 64 or 128 dims under 32 (or 24) query heads, pages of 8..32
tokens, fp32 activations (or fp16).

The cache is ``[pages][K, V][kv heads][page][head dim / 2]`` bytes, an e2m1 code each half (the even dim the low one),
and ``[pages][K, V][kv heads][page][head dim / 32]`` scale bytes: 32 dims of a row share the scale that has the bits
byte << 7 as an fp16 number.  It is the nearest such number to fp32's max|x| / 6 (10240 at most), and a code is the e2m1
value nearest to fp32's product of x and 1 / scale, ties to the even code.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 32  # dims that share a scale
TOP = 226   # the largest scale's byte, 10240: 6 times it is still an fp16 number


def _ops():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "inferencer-jetson_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from ijb200 import ops
    return ops


# ------------------------------------------------------------------ cases --

def listed():
    att = dict(op="attend", kv_heads=8, page=16)
    return [
        # one user, one new token: the smallest call of a decode loop, latency counts
        dict(att, name="attend one token", heads=32, batch=1, q_lo=1, q_hi=1, ctx_lo=2043, ctx_hi=2043, dim=64, q="f32"),
        # the engine's ragged batch: 64 sequences with prompts and outputs of mixed lengths
        dict(att, name="attend 64 ragged", heads=32, batch=64, q_lo=1, q_hi=1, ctx_lo=23, ctx_hi=1499, dim=64, q="f32"),
        # a batch of long documents being answered: the cache read decides
        dict(att, name="attend 16 long", heads=32, batch=16, q_lo=1, q_hi=1, ctx_lo=11003, ctx_hi=40111, dim=128,
             q="f16"),
        # drafted tokens being checked, three query heads to a KV head
        dict(att, name="attend drafts", heads=24, batch=24, q_lo=2, q_hi=5, ctx_lo=700, ctx_hi=9001, dim=128, q="f32"),
        # a few short prompts prefilled together, on the engine's fp32 activations
        dict(att, name="attend 5 prompts", heads=32, batch=5, q_lo=61, q_hi=777, ctx_lo=0, ctx_hi=0, dim=64, q="f32"),
        # a chunk of a long prompt: new tokens behind thousands of cached ones
        dict(att, name="attend chunk", heads=32, batch=1, q_lo=448, q_hi=448, ctx_lo=30001, ctx_hi=30001, dim=128,
             q="f16"),
        # a decode step's new rows, one for each of 64 sequences, as the next attention finds them
        dict(op="write", name="write 64 rows", n=64, batch=64, kv_heads=8, dim=64, page=16, type="f32"),
        # a prefill's rows, long sequences
        dict(op="write", name="write 12k rows", n=12289, batch=4, kv_heads=8, dim=128, page=16, type="f32"),
        # one sequence's rows read back (to look at it, or to move it to another pool)
        dict(op="read", name="read 1k rows", n=1021, batch=1, kv_heads=8, dim=64, page=16, type="f32"),
        # a batch of long sequences read back as fp16
        dict(op="read", name="read 32k rows", n=32749, batch=8, kv_heads=8, dim=128, page=16, type="f16"),
        # a sequence forked in the middle of a page: that page's copy in each of 16 layers
        dict(op="copy", name="copy 16 pages", n=16, kv_heads=8, dim=64, page=16, cache="f16"),
        # long sequences moved to other pages as a whole
        dict(op="copy", name="copy 6k pages", n=6007, kv_heads=8, dim=128, page=16, cache="e4m3"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "read", "copy"])
    kv_heads, dim, page = rng.choice([1, 2, 4, 8, 8, 8]), rng.choice([64, 128]), rng.choice([8, 16, 16, 32])
    if op == "copy":
        return dict(op=op, n=_log(rng, 1, 6000), kv_heads=kv_heads, dim=dim, page=page, cache=rng.choice(["f16", "e4m3"]))
    if op in ("write", "read"):
        n = _log(rng, 1, 12289 if op == "write" else 32749)
        return dict(op=op, n=n, batch=rng.randint(1, min(n, 64)), kv_heads=kv_heads, dim=dim, page=page,
                    type=rng.choice(["f32", "f16"]))
    c = dict(op=op, heads=kv_heads * rng.choice([1, 2, 3, 4, 4, 6, 8]), kv_heads=kv_heads, dim=dim, page=page,
             q=rng.choice(["f32", "f16"]))
    kind = rng.choice(["decode", "decode", "chunk", "prompts"])
    if kind == "decode":  # single tokens, sometimes a few at once (drafts to check)
        c["batch"] = _log(rng, 1, 96)
        c["q_lo"], c["q_hi"] = 1, rng.choice([1, 1, 1, 4])
        c["ctx_hi"] = _log(rng, 16, max(64, min(65536, 400000 // c["batch"])))
        c["ctx_lo"] = rng.randint(1, c["ctx_hi"])
    elif kind == "chunk":  # new tokens behind cached ones
        c["batch"] = rng.randint(1, 4)
        c["q_hi"] = _log(rng, 8, 440 // c["batch"])
        c["q_lo"] = rng.randint(1, c["q_hi"])
        c["ctx_hi"] = _log(rng, 64, 24000 // c["batch"])
        c["ctx_lo"] = rng.randint(0, c["ctx_hi"])
    else:
        c["batch"] = rng.randint(1, 8)
        c["q_hi"] = _log(rng, 16, 3000 // c["batch"])
        c["q_lo"] = rng.randint(1, c["q_hi"])
        c["ctx_lo"] = c["ctx_hi"] = 0
    return c


def _spread(lo, hi, n):
    """n lengths between lo and hi, in no order, hi among them."""
    return [hi - int((hi - lo + 0.999) * ((i * 0.6180339887) % 1.0)) if hi > lo else hi for i in range(n)]


def _lengths(case):
    """(new tokens, cached tokens before them) of each sequence."""
    b = case["batch"]
    return _spread(case["q_lo"], case["q_hi"], b), _spread(case["ctx_lo"], case["ctx_hi"], b)[::-1]


def _page_bytes(case):
    rows = 2 * case["kv_heads"] * case["page"]
    return rows * case["dim"] * 2 if case["cache"] == "f16" else rows * (case["dim"] + 1)


def work(case):
    if case["op"] == "copy":
        return {"bytes": case["n"] * (2 * _page_bytes(case) + 8), "flops": 0}
    rows, row = case["kv_heads"] * 2, case["dim"] // 2 + case["dim"] // BLOCK
    if case["op"] in ("write", "read"):
        io = case["dim"] * (4 if case["type"] == "f32" else 2)
        # written rows come in once, and their values go out once
        return {"bytes": case["n"] * (rows * (row + io * (2 if case["op"] == "write" else 1)) + 8),
                "flops": 2 * case["n"] * rows * case["dim"]}
    new, old = _lengths(case)
    io = 4 if case["q"] == "f32" else 2
    pairs = sum(l * o + l * (l + 1) // 2 for l, o in zip(new, old))
    return {"bytes": sum(new) * case["heads"] * case["dim"] * io * 2 + (sum(new) + sum(old)) * rows * row,
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ----------------------------------------------------------------- inputs --

_TYPES = {"f32": torch.float32, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _scale(byte):
    return (byte.int() << 7).to(torch.int16).view(torch.float16).float()


def _quantise(x):
    """Packed e2m1 codes and scale bytes of fp32 rows (last axis)."""
    x = x.reshape(x.shape[:-1] + (-1, BLOCK))
    r = x.abs().amax(-1) / 6
    e = (torch.frexp(r)[1] - 1).clamp(min=-14)
    byte = ((e + 14) * 8 + torch.round(torch.ldexp(r, 3 - e)).int()).clamp(max=TOP)
    scale = _scale(byte)
    inv = torch.where(scale > 0, 1.0 / torch.where(scale > 0, scale, 1.0), 0.0)
    y = x * inv.unsqueeze(-1)
    a = y.abs()
    code = (a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte()
    code = code + (a >= 3.5).byte() + (a > 5).byte() + (torch.signbit(y).byte() << 3)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.to(torch.uint8)


def _pool(case, pages, g):
    """A cache with every page filled, as a program that has been serving holds it: some K channels far larger than
    others."""
    shape = (pages, 2, case["kv_heads"], case["page"], case["dim"])
    data = torch.empty(shape[:-1] + (case["dim"] // 2,), device="cuda", dtype=torch.uint8)
    scale = torch.empty(shape[:-1] + (case["dim"] // BLOCK,), device="cuda", dtype=torch.uint8)
    wide = 1 + 3 * (torch.rand((2, case["kv_heads"], 1, case["dim"]), generator=g, device="cuda") > 0.97).float()
    wide[1] = 1
    for i in range(0, pages, 2048):  # in parts, for the fp32 rows' memory
        x = torch.randn((min(2048, pages - i),) + shape[1:], generator=g, device="cuda") * wide
        data[i:i + 2048], scale[i:i + 2048] = _quantise(x)
    return data.view(torch.float4_e2m1fn_x2), scale


def _table(lengths, page, g):
    """Page table of sequences of these lengths over a pool that has them in no order, and the pool's pages."""
    need = [-(-n // page) for n in lengths]
    total, width = sum(need) + 3, max(need)
    ids = torch.randperm(total, generator=g, device="cuda", dtype=torch.int32)
    start = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda").unsqueeze(1)
    at = torch.arange(width, device="cuda").unsqueeze(0)
    used = at < torch.tensor(need, device="cuda").unsqueeze(1)
    return torch.where(used, ids[(start + at).clamp(max=total - 1)], 0).int().contiguous(), total


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    dim, kvh, page = case["dim"], case["kv_heads"], case["page"]
    if case["op"] == "copy":
        pages = 2 * case["n"] + 5
        shape = (pages, 2, kvh, page, dim)
        if case["cache"] == "f16":
            s["data"], s["scale"] = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16), None
        else:
            s["data"] = torch.randint(0, 120, shape, generator=g, device="cuda", dtype=torch.uint8).view(_TYPES["e4m3"])
            s["scale"] = torch.randint(100, 130, shape[:-1], generator=g, device="cuda", dtype=torch.uint8)
        ids = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
        s["src"], s["dst"] = ids[:case["n"]].contiguous(), ids[case["n"]:2 * case["n"]].contiguous()
        s["page_table"] = s["dst"].view(1, -1)
    elif case["op"] in ("write", "read"):
        n, b = case["n"], case["batch"]
        counts = [n // b + (i < n % b) for i in range(b)]
        before = _spread(0, 40, b)
        s["page_table"], pages = _table([c + o for c, o in zip(counts, before)], page, g)
        s["data"], s["scale"] = _pool(case, pages, g)
        s["seq"] = torch.tensor([i for i, c in enumerate(counts) for _ in range(c)], device="cuda", dtype=torch.int32)
        s["pos"] = torch.tensor([o + j for c, o in zip(counts, before) for j in range(c)], device="cuda",
                                dtype=torch.int32)
        if case["op"] == "write":  # K rows as a projection leaves them, some heads far larger than others
            x = torch.randn((2, n, kvh, dim), generator=g, device="cuda")
            x *= torch.exp2(torch.randint(-6, 5, (2, n, kvh, 1), generator=g, device="cuda").float())
            s["k"], s["v"] = x[0].to(_TYPES[case["type"]]), x[1].to(_TYPES[case["type"]])
    else:
        new, old = _lengths(case)
        s["page_table"], pages = _table([a + b for a, b in zip(new, old)], page, g)
        s["data"], s["scale"] = _pool(case, pages, g)
        s["q"] = torch.randn((sum(new), case["heads"], dim), generator=g, device="cuda").to(_TYPES[case["q"]])
        s["q_start"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], device="cuda", dtype=torch.int32)
        s["kv_len"] = torch.tensor([a + b for a, b in zip(new, old)], device="cuda", dtype=torch.int32)
        s["max_q"], s["max_kv"] = max(new), max(a + b for a, b in zip(new, old))
    # the e2m1 values of the 16 codes
    s["value"] = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    if own:
        s["cache"] = _ops().PagedKV(s["data"], s["page_table"], s["scale"])
    return s


# ------------------------------------------------------------- plain forms --

def _decode(s, data, scale):
    """fp32 values of packed rows."""
    code = torch.stack([data & 15, data >> 4], -1).flatten(-2).int()
    x = s["value"][code]
    return (x.view(x.shape[:-1] + (-1, BLOCK)) * _scale(scale).unsqueeze(-1)).flatten(-2)


def _rows(s, which, seq, pos):
    """fp32 K (0) or V (1) rows of positions [...] of sequences [...]: [..., kv heads, dim]."""
    page = s["case"]["page"]
    at = s["page_table"][seq, torch.div(pos, page, rounding_mode="floor")].long()
    return _decode(s, s["data"].view(torch.uint8)[at, which, :, pos % page], s["scale"][at, which, :, pos % page])


def _plain_attend(s):
    q, start, kv_len = s["q"], s["q_start"].long(), s["kv_len"].long()
    heads, kvh, dim = s["case"]["heads"], s["case"]["kv_heads"], s["case"]["dim"]
    batch, dev = kv_len.numel(), q.device
    t = torch.arange(s["max_kv"], device=dev)
    held = t < kv_len.unsqueeze(1)  # [batch, t]
    seq = torch.arange(batch, device=dev).unsqueeze(1)
    pos = torch.where(held, t, 0)
    k, v = _rows(s, 0, seq, pos), _rows(s, 1, seq, pos)  # [batch, t, kv heads, dim]
    l = torch.arange(s["max_q"], device=dev)
    new = start[1:] - start[:-1]
    x = q[(start[:-1].unsqueeze(1) + l).clamp(max=q.shape[0] - 1)].float()  # [batch, l, heads, dim]
    x = x.view(batch, -1, kvh, heads // kvh, dim).permute(0, 2, 3, 1, 4).reshape(batch, kvh, -1, dim)
    score = torch.matmul(x, k.permute(0, 2, 3, 1)).view(batch, kvh, heads // kvh, -1, t.numel())
    score = score * (1.0 / math.sqrt(dim))
    seen = held.unsqueeze(1) & (t <= (kv_len - new).unsqueeze(1).unsqueeze(2) + l.unsqueeze(1))  # [batch, l, t]
    score = torch.where(seen.unsqueeze(1).unsqueeze(1), score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = torch.where(held.unsqueeze(-1).unsqueeze(-1), v, 0.0).permute(0, 2, 1, 3)
    o = torch.matmul(p.view(batch, kvh, -1, t.numel()), v).view(batch, kvh, heads // kvh, -1, dim)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(batch, -1, heads, dim)
    row = torch.arange(q.shape[0], device=dev)
    at = torch.searchsorted(start, row, right=True) - 1
    return o[at, row - start[at]].to(q.dtype)


def _plain_read(s):
    k, v = (_rows(s, which, s["seq"].long(), s["pos"].long()) for which in (0, 1))
    return [k.to(_TYPES[s["case"]["type"]]), v.to(_TYPES[s["case"]["type"]])]


def _plain_write(s):
    page, pos = s["case"]["page"], s["pos"].long()
    at = s["page_table"][s["seq"].long(), torch.div(pos, page, rounding_mode="floor")].long()
    codes, scale = _quantise(torch.stack([s["k"], s["v"]], 1).float())  # [n, K V, kv heads, dim]
    s["data"].view(torch.uint8)[at, :, :, pos % page] = codes
    s["scale"][at, :, :, pos % page] = scale
    return _plain_read(s)  # what the cache holds now, as values


def _copied(s):
    return s["data"] if s["scale"] is None else {"data": s["data"], "scale": s["scale"]}


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    data = s["data"] if s["scale"] is None else s["data"].view(torch.uint8)
    data[dst] = data[src]
    if s["scale"] is not None:
        s["scale"][dst] = s["scale"][src]
    return _copied(s)


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "attend":
            return s["cache"].attention(s["q"], s["q_start"], s["kv_len"], max_q=s["max_q"])
        if op == "copy":
            s["cache"].copy_pages(s["src"], s["dst"])
            return _copied(s)
        if op == "write":
            s["cache"].append(s["k"], s["v"], s["seq"], s["pos"])
        return list(s["cache"].gather(s["seq"], s["pos"], _TYPES[s["case"]["type"]]))
    return {"attend": _plain_attend, "read": _plain_read, "write": _plain_write, "copy": _plain_copy}[op](s)


# ------------------------------------------------------------------- exact --

def _values(data, scale):
    """The values of packed rows as 64-bit numbers."""
    b = data.view(torch.uint8)
    c = torch.empty(b.shape[:-1] + (2 * b.shape[-1],), device="cuda", dtype=torch.float64)
    for i, n in ((0, b & 15), (1, b >> 4)):
        m, e = (n & 1).double(), ((n >> 1) & 3).double()
        x = torch.where(e > 0, (1 + m / 2) * torch.pow(2.0, e - 1), m / 2)
        c[..., i::2] = torch.where(n > 7, -x, x)
    m, e = (scale & 7).double(), (scale >> 3).double()
    f = torch.where(e > 0, (1 + m / 8) * torch.pow(2.0, e - 15), m / 8 * 2.0 ** -14)
    return c * f.repeat_interleave(BLOCK, -1)


def _nearest(x, levels):
    """The values that a 4-bit cache holds for rows: both roundings by a search of all the numbers there are (the
    definition's quotient and product are fp32's)."""
    byte = torch.arange(TOP + 1, device="cuda").double()
    scales = torch.where(byte < 8, byte / 8 * 2.0 ** -14, (1 + byte % 8 / 8) * torch.pow(2.0, torch.floor(byte / 8) - 15))

    def search(table, v):  # index of the nearest, ties to the even one
        hi = torch.searchsorted(table, v).clamp(max=table.numel() - 1)
        lo = (hi - 1).clamp(min=0)
        up, down = table[hi] - v, v - table[lo]
        return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)

    y = x.double().unflatten(-1, (-1, BLOCK))
    scale = scales[search(scales, (y.abs().amax(-1, keepdim=True) / 6).float().double())]
    scaled = (y * (1 / scale.clamp(min=2.0 ** -17)).float().double()).float().double()
    value = levels[search(levels, scaled.abs().contiguous())] * scale
    return torch.where(y < 0, -value, value).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    page = case["page"]
    if case["op"] == "attend":
        new, old = _lengths(case)
        if sum(l * (l + o) for l, o in zip(new, old)) * case["heads"] > 3e9:
            return None
        out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
        group, first = case["heads"] // case["kv_heads"], 0
        for b, (l, o) in enumerate(zip(new, old)):
            pages = s["page_table"][b, :-(-(l + o) // page)].long()
            rows = _values(s["data"].view(torch.uint8)[pages], s["scale"][pages])  # [pages, K V, kv heads, page, dim]
            hidden = torch.ones((l, l + o), device="cuda", dtype=torch.bool).triu(o + 1)
            for h in range(case["heads"]):
                k, v = (rows[:, which, h // group].reshape(-1, case["dim"])[:l + o] for which in (0, 1))
                score = s["q"][first:first + l, h].double() @ k.T / math.sqrt(case["dim"])
                out[first:first + l, h] = torch.softmax(score.masked_fill_(hidden, -math.inf), -1) @ v
            first += l
        return out
    if case["op"] == "read":
        at, off = s["page_table"][s["seq"].long(), s["pos"].long() // page].long(), s["pos"].long() % page
        return [_values(s["data"].view(torch.uint8)[at, which, :, off], s["scale"][at, which, :, off]) for which in (0, 1)]
    if case["op"] == "write":
        return [_nearest(s["k"], s["value"][:8].double()), _nearest(s["v"], s["value"][:8].double())]
    data = s["data"].double()
    data[s["dst"].long()] = data[s["src"].long()]
    return data if s["scale"] is None else {"data": data, "scale": None}
