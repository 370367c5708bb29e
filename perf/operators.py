"""Measured cases of the 4-bit KV cache, the attention that reads it, and beam search's step.

Each case is one pass through one operator as a serving program calls it: rows stored into a q4_0 cache and read
back (``store``), attention of a decode step or of a prompt over the cache (``attend``), the choice of a step's
best continuations (``beam``) and the reordering of the beams' caches (``reorder``). ``own`` selects the library's
kernels; otherwise ``run`` computes the same values with elementary torch operations in 32 bits.

A cache's content is known as ggml q4_0 rows: per 32 values {fp16 d; 16 bytes}, byte j holding the codes of
values j (low four bits) and j + 16 (high), each standing for d (code - 8).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_device = None


def _dev():
    """The library's device handle, opened once as a program does."""
    global _device
    if _device is None:
        path = os.path.join(os.getcwd(), "tesseract-npu_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import tsrc
        _device = tsrc.Device(0)
    return _device


# ---- cases -----------------------------------------------------------------------------------------------------

def listed():
    return [
        # a chat's next token over a long context (32 query heads on 8 KV heads of 128)
        dict(name="token 8192 f32", op="attend", dtype="f32", heads=32, kv_heads=8, dim=128, seqs=1, tokens=1, cap=8192,
             ragged=False, window=0, mask=False),
        # a small model's next token after a 512-token prompt: launch latency counts
        dict(name="token 640 f32 d64", op="attend", dtype="f32", heads=14, kv_heads=2, dim=64, seqs=1, tokens=1, cap=640,
             ragged=False, window=0, mask=False),
        # a server's decode step: 64 conversations of different lengths
        dict(name="64 ragged sequences bf16", op="attend", dtype="bf16", heads=32, kv_heads=8, dim=128, seqs=64, tokens=1,
             cap=4096, ragged=True, window=0, mask=False),
        # a tree of drafted tokens under a mask, checked in one pass
        dict(name="13 drafted tokens f16", op="attend", dtype="f16", heads=32, kv_heads=8, dim=128, seqs=1, tokens=13,
             cap=4113, ragged=False, window=0, mask=True),
        # a prompt's attention
        dict(name="prompt 2048 bf16", op="attend", dtype="bf16", heads=32, kv_heads=8, dim=128, seqs=1, tokens=2048,
             cap=2048, ragged=False, window=0, mask=False),
        # the last chunk of a long prompt, in full precision
        dict(name="prompt chunk 512 f32", op="attend", dtype="f32", heads=32, kv_heads=8, dim=128, seqs=1, tokens=512,
             cap=4096, ragged=False, window=0, mask=False),
        # the new rows of a decode step, one for each of 64 sequences
        dict(name="store 64 rows f32", op="store", dtype="f32", kv_heads=8, dim=128, rows=64, cells=65536, scattered=True),
        # a prompt's rows
        dict(name="store 8192 rows bf16", op="store", dtype="bf16", kv_heads=8, dim=128, rows=8192, cells=8192, scattered=False),
        # one request with 4 beams
        dict(name="4 beams f32", op="beam", dtype="f32", groups=1, beams=4, vocab=151936, out=8),
        # a batch of 32 requests with 8 beams each
        dict(name="32 x 8 beams bf16", op="beam", dtype="bf16", groups=32, beams=8, vocab=128256, out=16),
        # the caches of one request's beams
        dict(name="reorder 4 x 640", op="reorder", kv_heads=2, dim=64, groups=1, beams=4, cap=640, len=640),
        # the caches of a batch's beams
        dict(name="reorder 8 x 8 x 2048", op="reorder", kv_heads=8, dim=128, groups=8, beams=8, cap=2048, len=2040),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["attend", "attend", "attend", "store", "beam", "reorder"])
        if op == "attend":
            kv_heads, dim = rng.choice([(8, 128), (2, 64), (4, 128), (8, 64), (1, 128), (4, 256), (2, 512), (16, 64)])
            c = dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), heads=kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8]),
                     kv_heads=kv_heads, dim=dim)
            form = rng.choice(["token", "batch", "draft", "prompt"])
            if form == "token":
                c.update(seqs=1, tokens=1, cap=_log_int(rng, 1, 65536))
            elif form == "batch":
                c.update(seqs=_log_int(rng, 2, 96), tokens=rng.choice([1, 1, 1, 2, 4]), cap=_log_int(rng, 16, 8192))
            elif form == "draft":
                c.update(seqs=1, tokens=rng.randint(2, 40), cap=_log_int(rng, 64, 16384))
            else:
                tokens = _log_int(rng, 41, 2048)
                c.update(seqs=1, tokens=tokens, cap=tokens + rng.choice([0, 0, _log_int(rng, 1, 8192)]))
            c["tokens"] = min(c["tokens"], c["cap"])
            c.update(ragged=c["seqs"] > 1 and rng.random() < 0.7, window=rng.choice([0, 0, 0, _log_int(rng, 16, 1024)]),
                     mask=c["seqs"] == 1 and rng.random() < 0.3)
        elif op == "store":
            kv_heads, dim = rng.choice([(8, 128), (2, 64), (4, 128), (4, 256), (2, 512), (5, 64)])
            rows = _log_int(rng, 1, 8192)
            c = dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), kv_heads=kv_heads, dim=dim, rows=rows,
                     cells=rows + rng.randint(0, 4096), scattered=rng.random() < 0.5)
        elif op == "beam":
            beams = rng.randint(1, 12)
            c = dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), groups=_log_int(rng, 1, 32), beams=beams,
                     vocab=_log_int(rng, 1000, 152064), out=rng.choice([beams, 2 * beams]))
        else:
            kv_heads, dim = rng.choice([(8, 128), (2, 64), (4, 128), (4, 256), (2, 512)])
            cap = _log_int(rng, 8, 4096)
            c = dict(op=op, kv_heads=kv_heads, dim=dim, groups=_log_int(rng, 1, 8), beams=rng.randint(2, 12), cap=cap,
                     len=rng.randint(1, cap))
        w = work(c)
        if w["flops"] <= 7.0e10 and w["bytes"] <= 6.0e8 and _held(c) <= 3.0e8:
            return c


def _held(c):
    """Cache values that the case's program holds in one plane, or logits: a bound on a case's memory."""
    if c["op"] == "attend":
        return max(c["seqs"] * c["cap"] * c["kv_heads"] * c["dim"], c["tokens"] * c["seqs"] * c["heads"] * c["cap"])
    if c["op"] == "store":
        return c["cells"] * c["kv_heads"] * c["dim"]
    if c["op"] == "beam":
        return 4 * c["groups"] * c["beams"] * c["vocab"]
    return c["groups"] * c["beams"] * c["cap"] * c["kv_heads"] * c["dim"]


def _lens(c):
    """Cells each sequence holds: all of its room, or, ragged, from half of it up."""
    if not c["ragged"]:
        return [c["cap"]] * c["seqs"]
    least = max(c["tokens"], c["cap"] // 2)
    return [least + (7919 * (i + 1)) % (c["cap"] - least + 1) for i in range(c["seqs"])]


def _spans(c):
    """[lo, hi) of the cells each token sees, sequence i's cells starting at i * cap: causal, maybe in a window."""
    spans = []
    for i, n in enumerate(_lens(c)):
        for j in range(c["tokens"]):
            hi = n - c["tokens"] + j + 1
            spans.append((i * c["cap"] + (max(0, hi - c["window"]) if c["window"] else 0), i * c["cap"] + hi))
    return spans


def work(c):
    if c["op"] == "attend":
        size = DTYPES[c["dtype"]].itemsize
        spans = _spans(c)
        g, cells = c["tokens"], 0
        for i in range(c["seqs"]):
            part = spans[i * g:(i + 1) * g]
            cells += max(h for _, h in part) - min(l for l, _ in part)
        seen = sum(h - l for l, h in spans)
        return {"bytes": 2 * cells * c["kv_heads"] * c["dim"] // 32 * 18 + 2 * len(spans) * c["heads"] * c["dim"] * size
                + (2 * seen if c["mask"] else 0), "flops": 4 * c["dim"] * c["heads"] * seen}
    if c["op"] == "store":
        n = 2 * c["rows"] * c["kv_heads"] * c["dim"]
        # rows in, blocks out; blocks in, rows out
        return {"bytes": 2 * n * DTYPES[c["dtype"]].itemsize + 2 * n // 32 * 18, "flops": 4 * n}
    if c["op"] == "beam":
        n = c["groups"] * c["beams"] * c["vocab"]
        return {"bytes": n * DTYPES[c["dtype"]].itemsize + 12 * c["groups"] * c["out"], "flops": 3 * n}
    n = 2 * c["groups"] * c["len"] * c["kv_heads"] * c["dim"]        # values of one beam of every group
    return {"bytes": n // 32 * 18 * (_survivors(c) + c["beams"] - 1) + 2 * n * c["beams"], "flops": n * c["beams"]}


# ---- inputs ----------------------------------------------------------------------------------------------------

def _rows(gen, n, kv_heads, dim, dtype):
    """K or V rows: normal values, a few channels of each head several times larger, as keys have."""
    x = torch.randn(n, kv_heads, dim, device="cuda", generator=gen)
    big = 1.0 + 4.0 * (torch.rand(kv_heads, dim, device="cuda", generator=gen) > 0.97)
    return (x * big).to(dtype).reshape(n, kv_heads * dim)


def _survivors(c):
    return max(1, c["beams"] // 2)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    st = {"case": c}
    if c["op"] == "store":
        st["k"], st["v"] = (_rows(gen, c["rows"], c["kv_heads"], c["dim"], DTYPES[c["dtype"]]) for _ in range(2))
        order = torch.randperm(c["cells"], device="cuda", generator=gen)[:c["rows"]]
        st["cells"] = order if c["scattered"] else torch.arange(c["rows"], device="cuda")
        if own:
            st["cache"] = _dev().kv4_create(c["kv_heads"], c["dim"], c["cells"])
        else:
            st["kb"], st["vb"] = (torch.zeros(c["cells"], c["kv_heads"] * c["dim"] // 32, 18, dtype=torch.uint8,
                                              device="cuda") for _ in range(2))
        return st
    if c["op"] == "beam":
        n = c["groups"] * c["beams"]
        x = 2.5 * torch.randn(n, c["vocab"], device="cuda", generator=gen)
        likely = torch.randint(0, c["vocab"], (n, 20), device="cuda", generator=gen)
        x.scatter_add_(1, likely, 8.0 * torch.rand(n, 20, device="cuda", generator=gen))
        banned = torch.randint(0, c["vocab"], (n, 4), device="cuda", generator=gen)
        st["logits"] = x.scatter_(1, banned, -math.inf).to(DTYPES[c["dtype"]])
        st["scores"] = -20.0 * torch.rand(c["groups"], c["beams"], device="cuda", generator=gen)
        return st
    n = c["seqs"] * c["cap"] if c["op"] == "attend" else c["groups"] * c["beams"] * c["cap"]
    kb, vb = (_quantise(_rows(gen, n, c["kv_heads"], c["dim"], torch.float32)) for _ in range(2))
    if own:
        st["cache"] = _dev().kv4_create(c["kv_heads"], c["dim"], n)
        st["cache"].set_bytes(0, kb)
        st["cache"].set_bytes(1, vb)
    else:
        st["kb"], st["vb"] = kb, vb
    if c["op"] == "reorder":
        # about half of a group's beams live on, in any order
        dead = torch.rand(c["groups"], c["beams"], device="cuda", generator=gen).argsort(1)
        pick = torch.randint(0, _survivors(c), (c["groups"], c["beams"]), device="cuda", generator=gen)
        st["parent"] = dead.gather(1, pick).to(torch.int32).contiguous()
        seqs = torch.arange(c["groups"] * c["beams"], device="cuda")
        st["cells"] = (seqs[:, None] * c["cap"] + torch.arange(c["len"], device="cuda")).flatten()
        return st
    tokens = c["seqs"] * c["tokens"]
    st["q"] = torch.randn(tokens, c["heads"], c["dim"], device="cuda", generator=gen).to(DTYPES[c["dtype"]])
    st["spans"] = torch.tensor(_spans(c), dtype=torch.int32).cuda()
    st["longest"] = max(_lens(c))
    if c["mask"]:
        # drafted tokens see the whole context and about half of the drafted cells before them, with a slope by distance
        hide = torch.rand(tokens, n, device="cuda", generator=gen) > 0.5
        hide[:, :c["cap"] - c["tokens"]] = False
        hide |= torch.arange(n, device="cuda")[None, :] >= st["spans"][:, 1:]
        slope = -0.002 * (c["cap"] - 1 - torch.arange(n, device="cuda")).float()
        st["mask"] = torch.where(hide, -math.inf, slope).half()
    return st


# ---- plain forms -----------------------------------------------------------------------------------------------

def _quantise(x):
    """Rows of values -> q4_0 blocks [..., n / 32, 18], each step in 32 bits as the format defines it."""
    x = x.float().reshape(x.shape[0], -1, 32)
    top = x.gather(-1, x.abs().argmax(-1, keepdim=True))
    d = top / -8.0
    inv = torch.where(d == 0, 0.0, 1.0 / d)
    n = (x * inv + 8.5).nan_to_num(8.0).clamp(0, 15).to(torch.uint8)
    return torch.cat([d.half().view(torch.uint8), n[..., :16] | (n[..., 16:] << 4)], -1)


def _values(b):
    """q4_0 blocks -> the values they stand for, [rows, blocks * 32]."""
    d = b[..., :2].contiguous().view(torch.float16).float()
    n = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).float()
    return (d * (n - 8.0)).reshape(b.shape[0], -1)


def _plain_attend(st):
    c = st["case"]
    S, g, L, Hk, D = c["seqs"], c["tokens"], c["cap"], c["kv_heads"], c["dim"]
    G = c["heads"] // Hk
    k = _values(st["kb"]).view(S, L, Hk, D).permute(0, 2, 3, 1)
    v = _values(st["vb"]).view(S, L, Hk, D).permute(0, 2, 1, 3)
    q = st["q"].float().view(S, g, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(S, Hk, g * G, D)
    s = torch.matmul(q, k).mul_(1.0 / math.sqrt(D)).view(S, Hk, g, G, L)
    cell = torch.arange(S * L, device="cuda", dtype=torch.int32).view(S, 1, L)
    span = st["spans"].view(S, g, 2)
    seen = (cell >= span[..., :1]) & (cell < span[..., 1:])
    if c["mask"]:
        m = st["mask"].float().view(S, g, L)
        seen &= m > -math.inf
        m = m - torch.where(seen, m, -math.inf).amax(-1, keepdim=True).nan_to_num(neginf=0.0)
        s += torch.where(seen, m, 0.0).view(S, 1, g, 1, L)
    seen = seen.view(S, 1, g, 1, L)
    s = s.masked_fill_(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, Hk, g * G, L), v).view(S, Hk, g, G, D)
    o = torch.where(total == 0, 0.0, o / total)
    return o.permute(0, 2, 1, 3, 4).reshape(S * g, c["heads"], D).to(DTYPES[c["dtype"]])


def _plain_beam(st):
    c = st["case"]
    x = st["logits"].double().view(c["groups"], c["beams"], c["vocab"])
    top = x.amax(-1, keepdim=True)
    total = (x - top).exp().sum(-1, keepdim=True).log() + top
    s = (st["scores"].double()[..., None] + (x - total)).nan_to_num(-math.inf, neginf=-math.inf)
    best, at = s.view(c["groups"], -1).sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :c["out"]], at[:, :c["out"]]
    none = best == -math.inf
    return (best.float(), torch.where(none, -1, at // c["vocab"]).int(), torch.where(none, -1, at % c["vocab"]).int())


def _plain_reorder(st):
    c = st["case"]
    outs = []
    base = torch.arange(c["groups"], device="cuda")[:, None] * c["beams"]
    src = (base + st["parent"]).reshape(-1)
    for b in (st["kb"], st["vb"]):
        b = b.view(c["groups"] * c["beams"], c["cap"], -1, 18)
        b[:, :c["len"]] = b[src, :c["len"]]
        outs.append(_values(b[:, :c["len"]].reshape(len(src) * c["len"], -1, 18)).half())
    return outs


# ---- one pass --------------------------------------------------------------------------------------------------

def run(st):
    c = st["case"]
    if c["op"] == "attend":
        if not own:
            return _plain_attend(st)
        out = torch.empty_like(st["q"])
        _dev().flash_attn_q4(st["cache"], st["q"], out, T=len(st["q"]), n_head=c["heads"], n_kv=c["seqs"] * c["cap"],
                             scale=1.0 / math.sqrt(c["dim"]), ranges=st["spans"], group=c["tokens"], max_len=st["longest"],
                             mask=st.get("mask"))
        return out
    if c["op"] == "store":
        if not own:
            st["kb"][st["cells"]] = _quantise(st["k"])
            st["vb"][st["cells"]] = _quantise(st["v"])
            return [_values(st[b][st["cells"]]).to(DTYPES[c["dtype"]]) for b in ("kb", "vb")]
        k, v = torch.empty_like(st["k"]), torch.empty_like(st["v"])
        st["cache"].set_rows(st["k"], st["v"], cells=st["cells"])
        st["cache"].get_rows(k, v, cells=st["cells"])
        return [k, v]
    if c["op"] == "beam":
        if not own:
            return _plain_beam(st)
        score = torch.empty(c["groups"], c["out"], device="cuda")
        beam, token = (torch.empty(c["groups"], c["out"], dtype=torch.int32, device="cuda") for _ in range(2))
        _dev().beam_select(st["logits"], st["scores"], score, beam, token, n_group=c["groups"], n_beam=c["beams"],
                           n_vocab=c["vocab"], n_out=c["out"])
        return score, beam, token
    if not own:
        return _plain_reorder(st)
    st["cache"].reorder(st["parent"], n_group=c["groups"], n_beam=c["beams"], seq_stride=c["cap"], n=c["len"])
    k, v = (torch.empty(len(st["cells"]), c["kv_heads"] * c["dim"], dtype=torch.float16, device="cuda") for _ in range(2))
    st["cache"].get_rows(k, v, cells=st["cells"])
    return [k, v]


# ---- 64 bits ---------------------------------------------------------------------------------------------------

def _blocks64(x):
    """The format's own f32 steps in numpy on rows of values: codes (int64) and the stored scale (f64)."""
    x = np.asarray(x, np.float32).reshape(len(x), -1, 32)
    at = np.abs(x).argmax(-1)
    d = (np.take_along_axis(x, at[..., None], -1) / np.float32(-8)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(d == 0, np.float32(0), np.float32(1) / d).astype(np.float32)
    t = ((x * inv).astype(np.float32) + np.float32(8.5)).astype(np.float32)
    return np.clip(np.floor(t), 0, 15).astype(np.int64), d.astype(np.float16).astype(np.float64)


def exact(case, seed):
    """The outputs from the definitions, in 64 bits."""
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    c = case
    if c["op"] == "store":
        outs = []
        for x in (st["k"], st["v"]):
            n, d = _blocks64(x.float().cpu().numpy())
            outs.append((d * (n - 8)).reshape(len(x), -1))
        return outs
    if c["op"] == "reorder":
        outs = []
        parent = st["parent"].cpu().tolist()
        for b in (st["kb"], st["vb"]):
            d = b[..., :2].contiguous().view(torch.float16).double()
            w = d * torch.stack([b[..., 2:] % 16, b[..., 2:] // 16], -2).flatten(-2).double().sub(8)
            w = w.view(c["groups"], c["beams"], c["cap"], -1)
            got = [w[i, p, :c["len"]].half() for i, row in enumerate(parent) for p in row]   # held to what 16 bits keep
            outs.append(torch.cat(got))
        return outs
    if c["op"] == "beam":
        scores, beams, tokens = [], [], []
        for i in range(c["groups"]):
            x = st["logits"][i * c["beams"]:(i + 1) * c["beams"]].double()
            s = (torch.log_softmax(x, -1) + st["scores"][i].double()[:, None]).flatten()
            least = s.topk(min(c["out"], s.numel())).values[-1]
            few = (s >= least).nonzero().flatten().cpu().numpy()
            val = s[torch.from_numpy(few).cuda()].cpu().numpy()
            first = np.lexsort((few, -val))[:c["out"]]
            scores.append(val[first])
            beams.append(few[first] // c["vocab"])
            tokens.append(few[first] % c["vocab"])
        return np.stack(scores), np.stack(beams).astype(np.int32), np.stack(tokens).astype(np.int32)
    Hk, D = c["kv_heads"], c["dim"]
    G = c["heads"] // Hk
    out = torch.zeros(len(st["q"]), c["heads"], D, dtype=torch.float64, device="cuda")

    def plane(b, i, h):
        b = b[i * c["cap"]:(i + 1) * c["cap"], h * D // 32:(h + 1) * D // 32]
        d = b[..., :2].contiguous().view(torch.float16).double()
        return (d * (torch.stack([b[..., 2:] % 16, b[..., 2:] // 16], -2).flatten(-2).double() - 8)).flatten(1)

    for i in range(c["seqs"]):
        rows = slice(i * c["tokens"], (i + 1) * c["tokens"])
        cells = torch.arange(i * c["cap"], (i + 1) * c["cap"], device="cuda")
        bias = torch.zeros(c["tokens"], c["cap"], dtype=torch.float64, device="cuda")
        if c["mask"]:
            bias = st["mask"][rows].double()
        bias = bias.masked_fill((cells < st["spans"][rows, :1]) | (cells >= st["spans"][rows, 1:]), -math.inf)
        for h in range(Hk):
            k, v = plane(st["kb"], i, h), plane(st["vb"], i, h)
            for j in range(G):
                z = st["q"][rows, h * G + j].double() @ k.T / math.sqrt(D) + bias
                out[rows, h * G + j] = torch.softmax(z, -1).nan_to_num(0.0) @ v
    return out
