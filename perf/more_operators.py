"""The operators of beam search and of batches over one shared prefix as they are measured: attention whose sequences share
a prefix, the selection over beams and vocabulary, and the reordering of cache slots. `run` computes them in plain torch
operations, or (own = True) by the framework's own kernels.

Kinds of case (the "op" field):
  attend   n prefixes (p keys each), s sequences behind each with keys of their own: single tokens (tq = 1) and prompts
  select   the best k of the continuations of w beams over v tokens, for b searches at once
  reorder  slot i of a cache becomes a copy of slot parent[i], over the rows that it holds, in place

A sequence's query i sees the keys of its prefix and, of its own len keys, those up to its own: j <= len - tq + i. A row
without a key is 0. A continuation's value is the beam's score plus log softmax of its logits; a finished beam (done) has one
continuation, eos, at its score. Ties go to the lowest beam, then the lowest token. Where there are fewer than k finite
values, the places left hold score -inf, parent 0, token eos, done.
"""
import math
import random

import torch

own = False  # True: run calls the framework's kernels

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EOS = 2


def listed():
    return [
        # one decoded token of four beams of the text decoder behind an image and a prompt: latency
        dict(name="beam_token", op="attend", n=1, s=4, hkv=32, g=1, d=64, tq=1, plo=794, phi=794, lo=1, hi=64),
        # eight questions about one image, all rows of each: the image's keys, then the question's, causal
        dict(name="questions", op="attend", n=1, s=8, hkv=32, g=1, d=64, tq=32, plo=730, phi=730, lo=32, hi=32),
        # a serving batch of single tokens behind one long instruction; some sequences have no key of their own yet
        dict(name="serve_batch", op="attend", n=1, s=64, hkv=8, g=4, d=128, tq=1, plo=8001, phi=8001, lo=0, hi=2000),
        # six searches of eight beams, each behind its own prompt, lengths from one token to 16000
        dict(name="beam_groups", op="attend", n=6, s=8, hkv=8, g=4, d=128, tq=1, plo=1, phi=16000, lo=1, hi=200),
        # a very long shared document
        dict(name="long_prefix", op="attend", n=1, s=16, hkv=8, g=4, d=128, tq=1, plo=131071, phi=131071, lo=0, hi=512),
        # chunks of prompts behind two shared documents: where the matrix units bound it
        dict(name="prompt_shared", op="attend", n=2, s=2, hkv=8, g=4, d=128, tq=1024, plo=5000, phi=8001, lo=1024, hi=1500),
        # four beams over the text decoder's vocabulary: latency
        dict(name="select_token", op="select", b=1, w=4, v=51200, k=4, type="bf16", done=0.0, banned=0.0),
        # 32 searches of eight beams, some of them finished
        dict(name="select_batch", op="select", b=32, w=8, v=51200, k=8, type="bf16", done=0.2, banned=0.01),
        # wide beams over a large vocabulary of odd size, logits in fp32
        dict(name="select_wide", op="select", b=16, w=16, v=131071, k=16, type="fp32", done=0.05, banned=0.0),
        # the text decoder's 24 layers, four beams, 40 generated rows: every step
        dict(name="reorder_step", op="reorder", layers=24, b=1, w=4, h=32, d=64, ctx=64, lo=40, hi=40),
        # eight searches of eight beams with long continuations of their own
        dict(name="reorder_batch", op="reorder", layers=8, b=8, w=8, h=8, d=128, ctx=512, lo=1, hi=500),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(("attend", "attend", "attend", "select", "select", "reorder"))
    if op == "attend":
        d = rng.choice((64, 128))
        hkv, g = rng.choice(((32, 1), (12, 1), (8, 4), (4, 7), (2, 8), (1, 32), (3, 3)))
        tq = 1 if rng.random() < 0.6 else _log(rng, 2, 1000)
        n = rng.choice((1, 1, 1, 2, 5))
        s = _log(rng, 1, 64 if tq == 1 else 8)
        rows = n * s * hkv * g * tq
        # the keys: bounded by the caches' bytes, the scores of the plain form and the products
        phi = _log(rng, 1, min(131071, 10 ** 8 // (n * hkv * d), 10 ** 9 // rows, 10 ** 11 // (rows * d)))
        hi = _log(rng, 1, min(8000, 10 ** 8 // (n * s * hkv * d), 10 ** 9 // rows, 10 ** 11 // (rows * d)))
        return dict(op=op, n=n, s=s, hkv=hkv, g=g, d=d, tq=tq, plo=phi if rng.random() < 0.5 else rng.randint(0, phi),
                    phi=phi, lo=hi if rng.random() < 0.3 else rng.randint(0, hi), hi=hi)
    if op == "select":
        w = rng.choice((1, 2, 3, 4, 5, 8, 12, 16, 32))
        v = rng.choice((51200, 32000, 50257, 131071, rng.randint(40, 150000)))
        return dict(op=op, b=_log(rng, 1, max(1, min(64, 3 * 10 ** 7 // (w * v)))), w=w, v=v, k=rng.choice((w, w, min(32, 2 * w), 1)),
                    type=rng.choice(("bf16", "bf16", "fp32")), done=rng.choice((0.0, 0.2)), banned=rng.choice((0.0, 0.0, 0.5)))
    w, d, h = rng.choice((2, 3, 4, 8, 16, 32)), rng.choice((64, 128)), rng.choice((1, 4, 8, 12, 32))
    b, layers = _log(rng, 1, 8), _log(rng, 1, 32)
    ctx = _log(rng, 1, max(1, 15 * 10 ** 7 // (2 * layers * b * w * h * d)))
    hi = rng.randint(1, ctx)
    return dict(op=op, layers=layers, b=b, w=w, h=h, d=d, ctx=ctx, lo=rng.randint(0, hi), hi=hi)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(r, count, lo, hi):
    """count lengths of lo .. hi, both ends among them where there is room."""
    lens = [r.randint(lo, hi) for _ in range(count)]
    lens[r.randrange(count)] = lo
    lens[r.randrange(count)] = hi
    return torch.tensor(lens, device="cuda", dtype=torch.int32)


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=F32).to(BF)
    s = dict(c=c)
    if c["op"] == "attend":
        n, b = c["n"], c["n"] * c["s"]
        s["plens"], s["lens"] = _lengths(r, n, c["plo"], c["phi"]), _lengths(r, b, c["lo"], c["hi"])
        s["pk"], s["pv"] = normal(n, c["hkv"], c["phi"], c["d"]), normal(n, c["hkv"], c["phi"], c["d"])
        s["k"], s["v"] = normal(b, c["hkv"], c["hi"], c["d"]), normal(b, c["hkv"], c["hi"], c["d"])
        s["q"] = normal(b, c["hkv"] * c["g"], c["tq"], c["d"])
    elif c["op"] == "select":
        b, w, v = c["b"], c["w"], c["v"]
        # a model's logits: a broad bulk, and a few dozen tokens that it finds likely
        x = torch.randn(b, w, v, generator=gen, device="cuda") * 2
        x += 9 * torch.rand(b, w, v, generator=gen, device="cuda") * (torch.rand(b, w, v, generator=gen, device="cuda") < 32 / v)
        if c["banned"]:
            x.masked_fill_(torch.rand(v, generator=gen, device="cuda") < c["banned"], -math.inf)
        s["logits"] = x.to(BF) if c["type"] == "bf16" else x
        s["scores"] = -(torch.rand(b, w, generator=gen, device="cuda") * 20).sort(1)[0]
        s["done"] = torch.rand(b, w, generator=gen, device="cuda") < c["done"]
    else:
        slots = c["b"] * c["w"]
        s["x"] = torch.randn(2 * c["layers"], slots, c["h"], c["ctx"], c["d"], generator=gen, device="cuda", dtype=BF)
        s["lens"] = _lengths(r, c["b"], c["lo"], c["hi"]).repeat_interleave(c["w"])
        s["parent"] = torch.randint(0, c["w"], (c["b"], c["w"]), generator=gen, device="cuda", dtype=torch.int32).sort(1)[0]
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _attend(s):
    c = s["c"]
    n, hkv, g, d, tq = (c[x] for x in ("n", "hkv", "g", "d", "tq"))
    b, m = n * c["s"], g * tq
    q = s["q"].float().view(b, hkv, m, d)
    shared = q.view(n, c["s"], hkv, m, d).transpose(1, 2).reshape(n, hkv, c["s"] * m, d)
    sp = torch.matmul(shared, s["pk"].float().transpose(2, 3).contiguous())
    p = torch.arange(c["phi"], device="cuda")
    sp = sp.masked_fill(p >= s["plens"].view(n, 1, 1, 1), -math.inf)
    sp = sp.view(n, hkv, c["s"], m, -1).transpose(1, 2).reshape(b, hkv, m, -1)
    so = torch.matmul(q, s["k"].float().transpose(2, 3).contiguous())
    j, i = torch.arange(c["hi"], device="cuda"), torch.arange(tq, device="cuda").repeat(g)
    limit = s["lens"].view(b, 1, 1, 1) - tq + 1 + i.view(1, 1, m, 1)  # keys that a row sees of its own
    so = so.masked_fill(j >= limit, -math.inf)
    top = torch.maximum(sp.amax(3, keepdim=True), so.amax(3, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    sp, so = torch.exp((sp - top) * d ** -0.5), torch.exp((so - top) * d ** -0.5)
    den = sp.sum(3, keepdim=True) + so.sum(3, keepdim=True)
    sp = sp.view(n, c["s"], hkv, m, -1).transpose(1, 2).reshape(n, hkv, c["s"] * m, -1)
    o = torch.matmul(sp, s["pv"].float()).view(n, hkv, c["s"], m, d).transpose(1, 2).reshape(b, hkv, m, d)
    o = o + torch.matmul(so, s["v"].float())
    o = torch.where(den > 0, o / den, 0.0)
    return o.view(b, hkv * g, tq, d).transpose(1, 2).reshape(b, tq, hkv * g * d).to(BF)


def _select(s):
    c = s["c"]
    b, v, k = c["b"], c["v"], c["k"]
    x, score, done = s["logits"].double(), s["scores"].double(), s["done"]
    top = x.amax(2, keepdim=True)
    x = score[:, :, None] + (x - (top + torch.exp(x - top).sum(2, keepdim=True).log()))
    x = torch.where(done[:, :, None], -math.inf, x)
    x[:, :, EOS] = torch.where(done, score, x[:, :, EOS])
    x, at = x.view(b, -1).sort(dim=1, descending=True, stable=True)
    x, at = x[:, :k], at[:, :k]
    empty = x == -math.inf
    parent = torch.where(empty, 0, at // v).int()
    token = torch.where(empty, EOS, at % v).int()
    return [x.float(), parent, token, token == EOS]


def _reorder(s):
    c, x = s["c"], s["x"]
    first = torch.arange(c["b"], device="cuda")[:, None] * c["w"]
    src = (first + s["parent"]).view(-1)
    held = torch.arange(c["ctx"], device="cuda") < s["lens"][src][:, None]
    x.copy_(torch.where(held[None, :, None, :, None], x[:, src], x))
    return x


def _own(s):
    from strix_halo_maxx_amd import ops
    c = s["c"]
    if c["op"] == "attend":
        return ops.sdpa_prefix(s["q"], s["pk"], s["pv"], s["k"], s["v"], s["lens"], prefix_len=s["plens"])
    if c["op"] == "select":
        return ops.beam_select(s["logits"], s["scores"], c["k"], done=s["done"], eos=EOS)
    return ops.reorder_slots(s["x"], s["parent"], s["lens"])


def run(s):
    if own:
        return _own(s)
    return {"attend": _attend, "select": _select, "reorder": _reorder}[s["c"]["op"]](s)


def work(c):
    if c["op"] == "attend":
        p, t = (c["plo"] + c["phi"]) / 2, (c["lo"] + c["hi"]) / 2
        b, hq = c["n"] * c["s"], c["hkv"] * c["g"]
        seen = p + max(t - c["tq"] / 2 if t > c["tq"] else t / 2, 0)
        return {"bytes": int(4 * c["hkv"] * c["d"] * (c["n"] * p + b * t) + 4 * b * hq * c["tq"] * c["d"]),
                "flops": int(4 * b * hq * c["tq"] * seen * c["d"])}
    if c["op"] == "select":
        cells = c["b"] * c["w"] * c["v"]
        return {"bytes": cells * (2 if c["type"] == "bf16" else 4) + 9 * c["b"] * (c["w"] + c["k"]), "flops": 4 * cells}
    # a sorted draw of parents: the slots that are read, and those that change (all but about one of each search)
    rows = c["layers"] * 2 * c["b"] * c["h"] * (c["lo"] + c["hi"]) / 2
    used = c["w"] * (1 - (1 - 1 / c["w"]) ** c["w"])
    return {"bytes": int(2 * rows * c["d"] * (used + max(c["w"] - 1, 1))), "flops": 0}


# ------------------------------------------------------------------------------------------------ 64-bit results
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "reorder":
        out, lens, parent = s["x"].clone(), s["lens"].tolist(), s["parent"].flatten().tolist()
        for i, p in enumerate(parent):
            src = i // c["w"] * c["w"] + p
            out[:, i, :, :lens[src]] = s["x"][:, src, :, :lens[src]]
        return out
    if c["op"] == "select":
        rows = []
        for x, score, done in zip(s["logits"], s["scores"], s["done"]):
            live = [torch.log_softmax(x[i].double(), 0) + score[i].double() for i in range(c["w"]) if not done[i]]
            rows.append(torch.cat(live + [score[done].double(), torch.full((c["k"],), -math.inf, device="cuda", dtype=F64)])
                        .topk(c["k"])[0])
        return [torch.stack(rows), None, None, None]
    if c["n"] * c["s"] * c["hkv"] * c["g"] * c["tq"] * (c["phi"] + c["hi"]) * c["d"] > 4 * 10 ** 11:
        return None
    b, g, d, tq = c["n"] * c["s"], c["g"], c["d"], c["tq"]
    out = torch.zeros(b, tq, c["hkv"] * g, d, device="cuda", dtype=F64)
    for i, (t, p) in enumerate(zip(s["lens"].tolist(), s["plens"].repeat_interleave(c["s"]).tolist())):
        for h in range(c["hkv"]):
            k = torch.cat([s["pk"][i // c["s"], h, :p], s["k"][i, h, :t]]).double()
            v = torch.cat([s["pv"][i // c["s"], h, :p], s["v"][i, h, :t]]).double()
            sc = (s["q"][i, h * g:(h + 1) * g].double().reshape(g * tq, d) @ k.t() / math.sqrt(d)).view(g, tq, -1)
            last = p + t - tq + torch.arange(tq, device="cuda")[:, None]
            j = torch.arange(p + t, device="cuda")
            sc = sc.masked_fill((j >= p) & (j > last), -math.inf)
            w = torch.where((sc > -math.inf).any(2, keepdim=True), torch.softmax(sc, 2), 0.0) if p + t else sc
            out[i, :, h * g:(h + 1) * g] = (w.view(g * tq, -1) @ v).view(g, tq, d).transpose(0, 1)
    return out.flatten(2)
