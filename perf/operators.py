"""The serving operators around the paged cache, case by case: the cache write that quantises, its read-back,
attention of new tokens over the cache, and sampling from the logits.

``run`` computes a case either in its plain form (elementary torch operations, fp32 throughout, 64-bit where sums are
compared with a border) or, with ``own`` set, through ``ijb200.ops``.  Shapes follow the engine: 32 query heads over 8
KV heads of 64 or 128 dims, vocabulary 128256, pages of 8..32 tokens, fp32 activations (or fp16).

The cache is one tensor ``[pages][K, V][kv heads][page][head dim]``, fp16 or e4m3; an e4m3 row (one token's K or V of
one head) has a power-of-two scale 2^(s - 127), the least with max|row| <= 448 * 2^(s - 127), kept as the byte s.
"""
import math
import os
import sys

import torch

own = False

VOCAB = 128256
FIXED = 1 << 44  # sampling weights are held as whole multiples of 2^-44, so that their sums have one value


def _ops():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "inferencer-jetson_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from ijb200 import ops
    return ops


# ------------------------------------------------------------------ cases --

def listed():
    att = dict(op="attend", heads=32, kv_heads=8, page=16)
    return [
        # one user, one new token: the smallest call of a decode loop, latency counts
        dict(att, name="attend one token", batch=1, q_lo=1, q_hi=1, ctx_lo=1957, ctx_hi=1957, dim=64, cache="f16",
             q="f32"),
        # the engine's ragged batch: 64 sequences with prompts and outputs of mixed lengths
        dict(att, name="attend 64 ragged", batch=64, q_lo=1, q_hi=1, ctx_lo=17, ctx_hi=1311, dim=64, cache="e4m3",
             q="f32"),
        # a batch of long documents being answered: the cache read decides
        dict(att, name="attend 16 long", batch=16, q_lo=1, q_hi=1, ctx_lo=9001, ctx_hi=32768, dim=128, cache="e4m3",
             q="f16"),
        # four short prompts prefilled together, on the engine's fp32 activations
        dict(att, name="attend 4 prompts", batch=4, q_lo=93, q_hi=700, ctx_lo=0, ctx_hi=0, dim=64, cache="f16",
             q="f32"),
        # a chunk of a long prompt: 512 new tokens behind 32 thousand cached ones
        dict(att, name="attend chunk", batch=1, q_lo=512, q_hi=512, ctx_lo=32011, ctx_hi=32011, dim=128,
             cache="e4m3", q="f16"),
        # one long prompt in a single call: the products decide
        dict(att, name="attend prompt", batch=1, q_lo=8192, q_hi=8192, ctx_lo=0, ctx_hi=0, dim=128, cache="f16",
             q="f16"),
        # a decode step's new rows, one for each of 64 sequences
        dict(op="write", name="write 64 rows", n=64, batch=64, kv_heads=8, dim=64, page=16, cache="e4m3", src="f32"),
        # a prefill's rows, long sequences
        dict(op="write", name="write 16k rows", n=16383, batch=4, kv_heads=8, dim=128, page=16, cache="e4m3",
             src="f32"),
        # one sequence's rows read back (to move it to another pool, or to look at it)
        dict(op="read", name="read 1k rows", n=1023, batch=1, kv_heads=8, dim=64, page=16, cache="e4m3", dst="f32"),
        # a batch of long sequences read back as fp16
        dict(op="read", name="read 32k rows", n=32768, batch=8, kv_heads=8, dim=128, page=16, cache="e4m3",
             dst="f16"),
        # one user's next token, with the usual settings
        dict(op="sample", name="sample one", n=1, vocab=VOCAB, mix="chat", spread=2.5),
        # a full batch whose rows have different settings: no filter, wide nuclei, greedy rows
        dict(op="sample", name="sample 256", n=256, vocab=VOCAB, mix="all", spread=2.5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "read", "sample"])
    kv_heads, dim = rng.choice([1, 2, 4, 8, 8, 8]), rng.choice([64, 128])
    page, cache = rng.choice([8, 16, 16, 32]), rng.choice(["f16", "e4m3"])
    if op == "sample":
        return dict(op=op, n=_log(rng, 1, 256), vocab=rng.choice([VOCAB, VOCAB, _log(rng, 300, 131072)]),
                    mix=rng.choice(["chat", "all"]), spread=round(rng.uniform(0.5, 6.0), 2))
    if op in ("write", "read"):
        n = _log(rng, 1, 16383)
        c = dict(op=op, n=n, batch=rng.randint(1, min(n, 64)), kv_heads=kv_heads, dim=dim, page=page, cache=cache)
        c["src" if op == "write" else "dst"] = rng.choice(["f32", "f16"])
        return c
    c = dict(op=op, heads=kv_heads * rng.choice([1, 2, 3, 4, 4, 6, 8]), kv_heads=kv_heads, dim=dim, page=page,
             cache=cache, q=rng.choice(["f32", "f16"]))
    kind = rng.choice(["decode", "decode", "chunk", "prompts"])
    if kind == "decode":  # single tokens, sometimes a few at once (drafts to check)
        c["batch"] = _log(rng, 1, 96)
        c["q_lo"], c["q_hi"] = 1, rng.choice([1, 1, 1, 4])
        c["ctx_hi"] = _log(rng, 16, max(64, min(65536, 400000 // c["batch"])))
        c["ctx_lo"] = rng.randint(1, c["ctx_hi"])
    elif kind == "chunk":  # new tokens behind cached ones
        c["batch"] = rng.randint(1, 4)
        c["q_hi"] = _log(rng, 8, 600 // c["batch"])
        c["q_lo"] = rng.randint(1, c["q_hi"])
        c["ctx_hi"] = _log(rng, 64, 24000 // c["batch"])
        c["ctx_lo"] = rng.randint(0, c["ctx_hi"])
    else:
        c["batch"] = rng.randint(1, 8)
        c["q_hi"] = _log(rng, 16, 3600 // c["batch"])
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


def work(case):
    if case["op"] == "sample":
        return {"bytes": case["n"] * (case["vocab"] * 4 + 28), "flops": 4 * case["n"] * case["vocab"]}
    rows, elem = case["kv_heads"] * 2, 2 if case["cache"] == "f16" else 1
    row = case["dim"] * elem + (1 if elem == 1 else 0)
    if case["op"] in ("write", "read"):
        other = 4 if case.get("src", case.get("dst")) == "f32" else 2
        return {"bytes": case["n"] * (rows * (row + case["dim"] * other) + 8),
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


def _quantise(x):
    """e4m3 values of fp32 rows (last axis) and their scale bytes."""
    frac, exp = torch.frexp(x.abs().amax(-1))
    e = torch.where(frac > 0, exp - 9 + (frac > 0.875).int(), -200).clamp(-126, 127)
    codes = torch.ldexp(x, -e.unsqueeze(-1)).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _pool(case, pages, g):
    """A cache with every page filled, as a program that has been serving holds it."""
    shape = (pages, 2, case["kv_heads"], case["page"], case["dim"])
    if case["cache"] == "f16":
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float16), None
    codes = torch.empty(shape, device="cuda", dtype=torch.float8_e4m3fn)
    scale = torch.empty(shape[:-1], device="cuda", dtype=torch.uint8)
    for i in range(0, pages, 4096):  # in parts, for the fp32 rows' memory
        x = torch.randn((min(4096, pages - i),) + shape[1:], generator=g, device="cuda")
        codes[i:i + 4096], scale[i:i + 4096] = _quantise(x)
    return codes, scale


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
    if case["op"] == "sample":
        n = case["n"]
        s["logits"] = torch.randn((n, case["vocab"]), generator=g, device="cuda") * case["spread"]
        s["u"] = torch.rand((n,), generator=g, device="cuda")
        i = torch.arange(n, device="cuda")
        if case["mix"] == "chat":
            s["temperature"] = torch.full((n,), 0.7, device="cuda")
            s["top_k"] = torch.full((n,), 40, device="cuda", dtype=torch.int32)
            s["top_p"] = torch.full((n,), 0.95, device="cuda")
            s["min_p"] = torch.full((n,), 0.02, device="cuda")
        else:
            s["temperature"] = torch.tensor([1.0, 0.6, 1.3, 0.0, 0.9], device="cuda")[i % 5]
            s["top_k"] = torch.tensor([0, 50, 0, 1000, 1, 20000, 0], device="cuda", dtype=torch.int32)[i % 7]
            s["top_p"] = torch.tensor([1.0, 0.9, 0.99, 1.0], device="cuda")[i % 4]
            s["min_p"] = torch.tensor([0.0, 0.0, 0.05], device="cuda")[i % 3]
        return s
    dim, kvh, page = case["dim"], case["kv_heads"], case["page"]
    if case["op"] in ("write", "read"):
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
            s["k"], s["v"] = x[0].to(_TYPES[case["src"]]), x[1].to(_TYPES[case["src"]])
    else:
        new, old = _lengths(case)
        s["page_table"], pages = _table([a + b for a, b in zip(new, old)], page, g)
        s["data"], s["scale"] = _pool(case, pages, g)
        s["q"] = (torch.randn((sum(new), case["heads"], dim), generator=g, device="cuda") * 1.5).to(_TYPES[case["q"]])
        s["q_start"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], device="cuda", dtype=torch.int32)
        s["kv_len"] = torch.tensor([a + b for a, b in zip(new, old)], device="cuda", dtype=torch.int32)
        s["max_q"], s["max_kv"] = max(new), max(a + b for a, b in zip(new, old))
    if own:
        s["cache"] = _ops().PagedKV(s["data"], s["page_table"], s["scale"])
    return s


# ------------------------------------------------------------- plain forms --

def _rows(s, which, seq, pos):
    """fp32 K (0) or V (1) rows of positions [...] of sequences [...]: [..., kv heads, dim]."""
    page = s["case"]["page"]
    at = s["page_table"][seq, torch.div(pos, page, rounding_mode="floor")].long()
    x = s["data"][at, which, :, pos % page].float()
    if s["scale"] is not None:
        x = x * torch.exp2(s["scale"][at, which, :, pos % page].float() - 127).unsqueeze(-1)
    return x


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


def _plain_write(s):
    page, pos = s["case"]["page"], s["pos"].long()
    at = s["page_table"][s["seq"].long(), torch.div(pos, page, rounding_mode="floor")].long()
    x = torch.stack([s["k"], s["v"]], 1).float()  # [n, K V, kv heads, dim]
    if s["scale"] is None:
        s["data"][at, :, :, pos % page] = x.half()
        return s["data"]
    codes, scale = _quantise(x)
    s["data"].view(torch.uint8)[at, :, :, pos % page] = codes.view(torch.uint8)
    s["scale"][at, :, :, pos % page] = scale
    return {"data": s["data"], "scale": s["scale"]}


def _plain_read(s):
    k, v = (_rows(s, which, s["seq"].long(), s["pos"].long()) for which in (0, 1))
    return [k.to(_TYPES[s["case"]["dst"]]), v.to(_TYPES[s["case"]["dst"]])]


def _plain_sample(s):
    x, n = s["logits"], s["logits"].shape[1]
    x = torch.where(x.isnan(), -math.inf, x)
    greedy, temp = s["temperature"] <= 0, torch.where(s["temperature"] > 0, s["temperature"], 1.0)
    top = x.amax(-1, keepdim=True)
    w = torch.exp(torch.where(x == top, 0.0, (x - top) / temp.unsqueeze(1)))
    fixed = torch.round(w.double() * FIXED).long()
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1]
    sorted_w = fixed.gather(1, order)
    mass = sorted_w.cumsum(-1)
    k = torch.where(s["top_k"] > 0, s["top_k"], n).clamp(max=n).long().unsqueeze(1)
    kept = mass.gather(1, k - 1)  # of the top k
    want = torch.ceil(s["top_p"].double().unsqueeze(1) * kept.double()).long()
    want = torch.where(s["top_p"].unsqueeze(1) < 1, torch.minimum(want, kept), kept).clamp(min=1)
    kept = mass.gather(1, torch.searchsorted(mass, want))  # the shortest prefix that reaches top_p of it
    above = torch.where((w >= s["min_p"].unsqueeze(1)) | (w == 1), fixed, 0).sum(-1, keepdim=True)
    kept = torch.minimum(kept, above)
    target = torch.floor(s["u"].double().unsqueeze(1) * kept.double()).long().clamp(min=0)
    at = torch.searchsorted(mass, torch.minimum(target, kept - 1), right=True)
    prob = (sorted_w.gather(1, at).double() / kept.double()).float().squeeze(1)
    token = torch.where(greedy, x.argmax(-1), order.gather(1, at).squeeze(1))
    return [token.int(), torch.where(greedy, 1.0, prob)]


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "sample":
            return list(_ops().sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"]))
        if op == "attend":
            return s["cache"].attention(s["q"], s["q_start"], s["kv_len"], max_q=s["max_q"])
        if op == "read":
            return list(s["cache"].gather(s["seq"], s["pos"], _TYPES[s["case"]["dst"]]))
        s["cache"].append(s["k"], s["v"], s["seq"], s["pos"])
        return s["data"] if s["scale"] is None else {"data": s["data"], "scale": s["scale"]}
    return {"sample": _plain_sample, "attend": _plain_attend, "read": _plain_read, "write": _plain_write}[op](s)


# ------------------------------------------------------------------- exact --

def _values(s):
    """The cache's rows as 64-bit numbers."""
    data = s["data"].double()
    return data if s["scale"] is None else data * torch.pow(2.0, s["scale"].double() - 127).unsqueeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    page = case["page"] if "page" in case else 1
    if case["op"] == "attend":
        new, old = _lengths(case)
        if sum(l * (l + o) for l, o in zip(new, old)) * case["heads"] > 3e9:
            return None
        out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
        group, first = case["heads"] // case["kv_heads"], 0
        for b, (l, o) in enumerate(zip(new, old)):
            pages = s["page_table"][b, :-(-(l + o) // page)].long()
            part = {"data": s["data"][pages], "scale": None if s["scale"] is None else s["scale"][pages]}
            rows = _values(part)  # [pages, K V, kv heads, page, dim]
            hidden = torch.ones((l, l + o), device="cuda", dtype=torch.bool).triu(o + 1)
            for h in range(case["heads"]):
                k, v = (rows[:, which, h // group].reshape(-1, case["dim"])[:l + o] for which in (0, 1))
                score = s["q"][first:first + l, h].double() @ k.T / math.sqrt(case["dim"])
                out[first:first + l, h] = torch.softmax(score.masked_fill_(hidden, -math.inf), -1) @ v
            first += l
        return out
    if case["op"] == "read":
        at, off = s["page_table"][s["seq"].long(), s["pos"].long() // page].long(), s["pos"].long() % page
        rows = _values(s)
        return [rows[at, which, :, off] for which in (0, 1)]
    if case["op"] == "write":
        rows = s["data"].double()
        at, off = s["page_table"][s["seq"].long(), s["pos"].long() // page].long(), s["pos"].long() % page
        for which, x in enumerate((s["k"].double(), s["v"].double())):
            if s["scale"] is not None:  # a value in units of its row's scale
                e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 448))
                x = x / torch.pow(2.0, e)
            rows[at, which, :, off] = x
        return rows if s["scale"] is None else {"data": rows, "scale": None}
    prob = torch.ones((case["n"],), device="cuda", dtype=torch.float64)
    for i in range(case["n"]):
        temp = float(s["temperature"][i])
        if temp <= 0:
            continue
        p = torch.softmax(s["logits"][i].double() / temp, -1).sort(descending=True)[0]
        if int(s["top_k"][i]) > 0:
            p = p[:int(s["top_k"][i])] / p[:int(s["top_k"][i])].sum()
        keep = p.numel()
        if float(s["top_p"][i]) < 1:
            keep = min(keep, int((p.cumsum(0) < float(s["top_p"][i])).sum()) + 1)
        keep = max(1, min(keep, int((p >= float(s["min_p"][i]) * p[0]).sum())))
        p = p[:keep] / p[:keep].sum()
        prob[i] = p[min(keep - 1, int((p.cumsum(0) <= float(s["u"][i])).sum()))]
    return [None, prob]
