"""The operators of `delayrepay_amd.nn` on representative work: what is run, what it has to move and
compute, and what it should give.

A case names an operator and its sizes.  `prepare` makes the inputs on the GPU, `run` makes one pass:
in elementary torch operations where `own` is false, with the framework's calls where it is true.
"""
import math

import torch

own = False

# ---- cases -----------------------------------------------------------------------------------
# op        attention (forward), train (forward with the statistics kept, then the gradients),
#           rotary, rotary_grad, sample
# b, hq, hkv, lq, lk, d      batch, query and key heads, query rows, key rows, head size
# lengths   "full": every key row is used; "ragged": sequence i uses a part of them (`lengths_of`)
# mask      none | causal | prefix (the first lk // 4 keys are seen by every row) |
#           documents (causal, and only inside the row's own document)
# cap       tanh cap of the scores, 0 for none; slopes: bias falling linearly with distance


def _attention(name, op="attention", b=1, hq=8, hkv=8, lq=1, lk=1, d=128, lengths="full", mask="causal", cap=0.0, slopes=False):
    return dict(name=name, op=op, b=b, hq=hq, hkv=hkv, lq=lq, lk=lk, d=d, lengths=lengths, mask=mask, cap=cap, slopes=slopes)


def _rotary(name, op="rotary", b=1, h=8, n=1, d=128, dims=128, interleaved=False, norm=True, far=0, stretch=1.0):
    return dict(name=name, op=op, b=b, h=h, n=n, d=d, dims=dims, interleaved=interleaved, norm=norm, far=far, stretch=stretch)


def _sample(name, b=1, v=32000, top_k=0, top_p=1.0, min_p=0.0, temperature=1.0):
    return dict(name=name, op="sample", b=b, v=v, top_k=top_k, top_p=top_p, min_p=min_p, temperature=temperature)


def listed():
    return [
        # a prompt of 4096 tokens, four query heads to a key head
        _attention("prompt", hq=32, hkv=8, lq=4096, lk=4096),
        # a long prompt whose scores are capped, every head its own keys
        _attention("prompt capped", hq=8, hkv=8, lq=8192, lk=8192, cap=30.0),
        # several documents packed into rows of odd length, bias by distance, a head size that is no power of two
        _attention("packed documents", b=3, hq=12, hkv=4, lq=1111, lk=1111, d=80, mask="documents", slopes=True),
        # a short prompt behind a cached prefix that all its rows see, sequences of several lengths
        _attention("prefix", b=4, hq=16, hkv=4, lq=333, lk=777, d=64, lengths="ragged", mask="prefix"),
        # one token for each of 64 sequences against a cache of 8192 rows: what serving does all day
        _attention("token, many sequences", b=64, hq=32, hkv=8, lq=1, lk=8192, lengths="ragged"),
        # one token of one sequence: latency, and few rows to share a long axis
        _attention("token, one sequence", b=1, hq=32, hkv=8, lq=1, lk=5000),
        # a training step of an attention layer
        _attention("train", op="train", b=2, hq=16, hkv=4, lq=2048, lk=2048),
        # the same, small and odd: packed documents with capped scores
        _attention("train documents", op="train", b=3, hq=6, hkv=2, lq=517, lk=517, d=64, mask="documents", cap=20.0, slopes=True),
        # queries and keys of a prompt side by side, normalised for each head and turned
        _rotary("rotary prompt", b=4, h=40, n=4096),
        # their gradient, with part of the head turned, neighbouring elements paired, far positions of a stretched context
        _rotary("rotary gradient", op="rotary_grad", b=2, h=20, n=1777, dims=64, interleaved=True, far=200000, stretch=4.0),
        # the answers of a large batch with a large vocabulary
        _sample("sample batch", b=256, v=128000, top_k=50, top_p=0.9, temperature=0.8),
        # the answer of one sequence
        _sample("sample one", b=1, v=32000, top_p=0.95, min_p=0.02),
    ]


def _between(rng, low, high):
    """A whole number in [low, high], spread evenly over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "token", "train", "rotary", "rotary_grad", "sample"])
    if op in ("attention", "train"):
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 3, 4])
        lk = _between(rng, 17, (4096 if hq <= 16 else 2800) if op == "attention" else 1500)
        lq = lk if rng.random() < 0.6 else _between(rng, max(1, lk // 16), lk)
        mask = rng.choice(["none", "causal", "prefix", "documents"])
        b = rng.randint(1, 3) if hq * lq * lk < 1 << 26 else 1
        c = _attention("", op=op, b=b, hq=hq, hkv=hkv, lq=lq, lk=lk, d=rng.choice([32, 48, 64, 80, 96, 128]),
                       lengths=rng.choice(["full", "ragged"]), mask=mask, cap=rng.choice([0.0, 0.0, 15.0, 50.0]), slopes=rng.random() < 0.3)
    elif op == "token":
        hkv = rng.choice([1, 2, 4, 8])
        c = _attention("", b=_between(rng, 1, 48), hq=hkv * rng.choice([1, 2, 4, 5, 8]), hkv=hkv, lq=rng.choice([1, 1, 1, 2, 3]), lk=_between(rng, 1, 8192),
                       d=rng.choice([64, 80, 96, 128]), lengths=rng.choice(["full", "ragged"]), mask="causal", cap=rng.choice([0.0, 0.0, 30.0]), slopes=rng.random() < 0.3)
    elif op in ("rotary", "rotary_grad"):
        d = rng.choice([32, 64, 80, 96, 128, 192, 256])
        c = _rotary("", op=op, b=rng.randint(1, 4), h=rng.randint(1, 40), n=_between(rng, 1, 2048), d=d, dims=d if rng.random() < 0.6 else 2 * rng.randint(1, d // 2),
                    interleaved=rng.random() < 0.5, norm=rng.random() < 0.6, far=_between(rng, 1, 1000000), stretch=rng.choice([1.0, 1.0, 2.0, 8.0]))
    else:
        c = _sample("", b=_between(rng, 1, 256), v=_between(rng, 50, 128000), top_k=rng.choice([0, 1, 20, 50, 1000]), top_p=rng.choice([1.0, 0.5, 0.9, 0.99]),
                    min_p=rng.choice([0.0, 0.0, 0.01, 0.1]), temperature=rng.choice([0.0, 0.5, 0.8, 1.0, 1.5]))
    del c["name"]
    return c


# ---- what a case's sizes say -----------------------------------------------------------------

def lengths_of(c):
    """Key rows in use, for each sequence: all, or between a fifth and all of them in an order without a trend; at least the rows asked about."""
    if c["lengths"] == "full":
        return [c["lk"]] * c["b"]
    low = min(c["lk"], max(c["lq"], c["lk"] // 5))
    return [low + ((i * 7919 + 4001) * 104729) % (c["lk"] - low + 1) for i in range(c["b"])]


def documents_of(c):
    """The document that each key row belongs to: documents of 1 to lk // 3 rows, one after the other."""
    rows = []
    for i in range(c["b"]):
        row, at = [], 0
        while len(row) < c["lk"]:
            at += 1
            row += [at] * (1 + ((at * 31 + i * 17) * 7907) % max(1, c["lk"] // 3))
        rows.append(row[:c["lk"]])
    return rows


def _pairs(c):
    """How many (query row, key row) pairs the masks leave, over all sequences."""
    total = 0
    for i, n in enumerate(lengths_of(c)):
        rows = torch.arange(n - c["lq"], n)
        cols = torch.arange(n)
        if c["mask"] == "none":
            total += c["lq"] * n
        elif c["mask"] == "documents":
            first = {}
            for j, x in enumerate(documents_of(dict(c, b=i + 1))[i]):
                first.setdefault(x, j)
            at = documents_of(dict(c, b=i + 1))[i]
            total += sum(int(p) - first[at[int(p)]] + 1 for p in rows)
        else:
            seen = rows + 1
            if c["mask"] == "prefix":
                seen = torch.clamp(seen, min=min(n, c["lk"] // 4))
            total += int(torch.clamp(seen, max=len(cols)).sum())
    return total


def work(c):
    if c["op"] in ("attention", "train"):
        q = c["b"] * c["hq"] * c["lq"] * c["d"] * 4
        kv = 2 * sum(lengths_of(c)) * c["hkv"] * c["d"] * 4
        whole = 2 * c["b"] * c["lk"] * c["hkv"] * c["d"] * 4
        pairs = _pairs(c) * c["hq"] * c["d"]
        if c["op"] == "attention":
            return {"bytes": 2 * q + kv, "flops": 4 * pairs}
        # q, k, v, dout are read; the output and the three gradients are written; two products forward, five backward
        return {"bytes": 4 * q + kv + whole, "flops": 14 * pairs}
    if c["op"] == "sample":
        return {"bytes": c["b"] * (c["v"] * 4 + 16), "flops": 4 * c["b"] * c["v"]}
    n = c["b"] * c["h"] * c["n"] * c["d"]
    reads = n * 4 * (2 if c["op"] == "rotary_grad" and c["norm"] else 1)
    return {"bytes": reads + n * 4, "flops": n * (10 if c["norm"] else 4)}


# ---- inputs ----------------------------------------------------------------------------------

def prepare(c, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    s = {"case": c}
    if c["op"] in ("attention", "train"):
        # tokens first in memory, as a projection leaves them; the operators see heads first
        s["q"] = normal(c["b"], c["lq"], c["hq"], c["d"]).transpose(1, 2)
        s["k"] = normal(c["b"], c["lk"], c["hkv"], c["d"]).transpose(1, 2)
        s["v"] = normal(c["b"], c["lk"], c["hkv"], c["d"]).transpose(1, 2)
        if c["op"] == "train":
            s["dout"] = normal(c["b"], c["lq"], c["hq"], c["d"]).transpose(1, 2)
        s["lengths"] = torch.tensor(lengths_of(c), dtype=torch.int32, device="cuda")
        if c["mask"] == "documents":
            s["documents"] = torch.tensor(documents_of(c), dtype=torch.int32, device="cuda")
        if c["slopes"]:
            s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / c["hq"]) for h in range(c["hq"])], device="cuda")
    elif c["op"] == "sample":
        s["logits"] = normal(c["b"], c["v"]) * 2.5
        s["u"] = torch.rand(c["b"], generator=g, device="cuda", dtype=torch.float64)
    else:
        s["x"] = normal(c["b"], c["n"], c["h"], c["d"]).transpose(1, 2) * 1.5
        start = torch.randint(0, c["far"] + 1, (c["b"], 1), generator=g, device="cuda")
        s["positions"] = (start + torch.arange(c["n"], device="cuda")).to(torch.int32)
        if c["norm"]:
            s["weight"] = 1.0 + 0.2 * normal(c["h"], c["d"])
        if c["op"] == "rotary_grad":
            s["dy"] = normal(c["b"], c["n"], c["h"], c["d"]).transpose(1, 2)
    return s


# ---- the plain forms -------------------------------------------------------------------------

def _scores(c, q, k, lengths, documents, slopes):
    """(scores, factor of their derivative, whether a pair counts); heads are (key heads, queries of one key head x rows)."""
    b, hq, lq, d = q.shape
    hkv, lk = k.shape[1:3]
    s = (q.reshape(b, hkv, hq // hkv * lq, d) @ k.transpose(2, 3)).view(b, hkv, hq // hkv, lq, lk) * (1.0 / math.sqrt(d))
    slope = None
    if c["cap"]:
        t = torch.tanh(s / c["cap"])
        s, slope = c["cap"] * t, 1.0 - t * t
    j = torch.arange(lk, device=q.device)
    p = lengths.long()[:, None] - lq + torch.arange(lq, device=q.device)  # positions of the rows: they are the last ones
    ok = (j < lengths[:, None])[:, None, :].expand(b, lq, lk)
    if c["mask"] != "none":
        seen = j <= p[:, :, None]
        if c["mask"] == "prefix":
            seen = seen | (j < c["lk"] // 4)
        ok = ok & seen
    if c["mask"] == "documents":
        here = torch.where((p >= 0) & (p < lk), torch.gather(documents, 1, p.clamp(0, lk - 1)), -1)
        ok = ok & (here[:, :, None] == documents[:, None, :])
    if slopes is not None:
        s = s - slopes.view(hkv, hq // hkv, 1, 1) * (p[:, :, None] - j).abs()[:, None, None].to(s.dtype)
    return s, slope, ok[:, None, None]


def _forward(c, q, k, v, lengths, documents, slopes):
    b, hq, lq, d = q.shape
    hkv, lk = k.shape[1:3]
    s, slope, ok = _scores(c, q, k, lengths, documents, slopes)
    s = torch.where(ok, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    o = p.view(b, hkv, hq // hkv * lq, lk) @ v
    return o.view(b, hq, lq, d), p, slope


def _backward(c, dout, q, k, v, o, p, slope):
    b, hq, lq, d = q.shape
    hkv, lk = k.shape[1:3]
    rows = (b, hkv, hq // hkv * lq)
    g, o, q, p = dout.reshape(*rows, d), o.reshape(*rows, d), q.reshape(*rows, d), p.reshape(*rows, lk)
    dv = p.transpose(2, 3) @ g
    ds = p * (g @ v.transpose(2, 3) - (g * o).sum(-1, keepdim=True))
    if slope is not None:
        ds = ds * slope.reshape(*rows, lk)
    ds = ds * (1.0 / math.sqrt(d))
    return (ds @ k).view(b, hq, lq, d), ds.transpose(2, 3) @ q, dv


def _turn(c, x, cos, sin):
    dims = c["dims"]
    head, rest = x[..., :dims], x[..., dims:]
    if c["interleaved"]:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., :dims // 2], head[..., dims // 2:]
        head = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([head, rest], -1)


def _angles(c, positions, dtype):
    """Cosines and sines of a row's angles; the angles themselves in 64 bits, since those of far positions need them."""
    i = torch.arange(c["dims"] // 2, device=positions.device, dtype=torch.float64)
    angle = positions.double()[:, None, :, None] * (10000.0 ** (-2.0 * i / c["dims"]) / c["stretch"])
    return torch.cos(angle).to(dtype), torch.sin(angle).to(dtype)


def _rotary_plain(c, x, positions, weight):
    cos, sin = _angles(c, positions, x.dtype)
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight[:, None, :]
    return _turn(c, x, cos, sin)


def _rotary_grad_plain(c, dy, x, positions, weight):
    cos, sin = _angles(c, positions, x.dtype)
    g = _turn(c, dy, cos, -sin)
    if weight is None:
        return (g,)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    hat = x * r
    dweight = (g * hat).double().sum((0, 2)).to(x.dtype)
    g = g * weight[:, None, :]
    return r * (g - hat * (g * hat).mean(-1, keepdim=True)), dweight


def _sample_plain(c, logits, u):
    if c["temperature"] == 0.0:
        return logits.argmax(-1)
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    w = torch.exp((order.values.double() - order.values[:, :1].double()) / c["temperature"])
    if c["top_k"]:
        w[:, c["top_k"]:] = 0.0
    before = torch.cumsum(w, -1) - w
    keep = (before < c["top_p"] * w.sum(-1, keepdim=True)) | (c["top_p"] >= 1.0)
    w = torch.where(keep & (w >= c["min_p"]), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order.indices, w)  # drawn in the order of the vocabulary
    at = torch.cumsum(w, -1)
    return ((at > (u[:, None] * at[:, -1:])) & (w > 0)).to(torch.uint8).argmax(-1)


# ---- one pass --------------------------------------------------------------------------------

def _arrays(s):
    """The framework's arrays over the state's memory.  A program that computes with the framework holds its data in
    them: they are made the first time that a state is run."""
    if "arrays" not in s:
        import delayrepay_amd as np
        c = s["case"]
        if c["op"] in ("attention", "train"):
            s["o"] = torch.empty_like(s["q"])
            if c["op"] == "train":
                s["lse"] = torch.empty(s["q"].shape[:3], device="cuda")
                s["dq"], s["dk"], s["dv"] = (torch.empty_like(s[x]) for x in "qkv")
        elif c["op"] == "sample":
            s["token"] = torch.empty(c["b"], device="cuda", dtype=torch.int64)
        else:
            s["y"] = torch.empty_like(s["x"])
            if c["op"] == "rotary_grad" and c["norm"]:
                s["dweight"] = torch.empty_like(s["weight"])
        s["arrays"] = {k: np.from_dlpack(t) for k, t in s.items() if isinstance(t, torch.Tensor)}
    return s["arrays"]


def _run_own(s):
    from delayrepay_amd import nn
    c, a = s["case"], _arrays(s)
    if c["op"] in ("attention", "train"):
        how = dict(causal=c["mask"] != "none", cap=c["cap"] or None, lengths=a["lengths"], prefix=c["lk"] // 4 if c["mask"] == "prefix" else None,
                   documents=a.get("documents"), slopes=a.get("slopes"))
        if c["op"] == "attention":
            nn.attention(a["q"], a["k"], a["v"], out=a["o"], **how)
            return [s["o"]]
        nn.attention(a["q"], a["k"], a["v"], with_lse=True, out=(a["o"], a["lse"]), **how)
        nn.attention_grad(a["dout"], a["q"], a["k"], a["v"], a["o"], a["lse"], out=(a["dq"], a["dk"], a["dv"]), **how)
        return [s["o"], s["dq"], s["dk"], s["dv"]]
    if c["op"] == "sample":
        nn.sample(a["logits"], a["u"], temperature=c["temperature"], top_k=c["top_k"] or None, top_p=c["top_p"], min_p=c["min_p"], out=a["token"])
        return [s["token"]]
    how = dict(dims=c["dims"], interleaved=c["interleaved"], stretch=c["stretch"], weight=a.get("weight"))
    if c["op"] == "rotary":
        nn.rotary(a["x"], a["positions"], out=a["y"], **how)
        return [s["y"]]
    if c["norm"]:
        nn.rotary_grad(a["dy"], a["x"], a["positions"], out=(a["y"], a["dweight"]), **how)
        return [s["y"], s["dweight"]]
    nn.rotary_grad(a["dy"], None, a["positions"], out=a["y"], **how)
    return [s["y"]]


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["op"] in ("attention", "train"):
        o, p, slope = _forward(c, s["q"], s["k"], s["v"], s["lengths"], s.get("documents"), s.get("slopes"))
        if c["op"] == "attention":
            return [o]
        return [o, *_backward(c, s["dout"], s["q"], s["k"], s["v"], o, p, slope)]
    if c["op"] == "sample":
        return [_sample_plain(c, s["logits"], s["u"])]
    if c["op"] == "rotary":
        return [_rotary_plain(c, s["x"], s["positions"], s.get("weight"))]
    return list(_rotary_grad_plain(c, s["dy"], s["x"], s["positions"], s.get("weight")))


# ---- the same in 64 bits ---------------------------------------------------------------------

def _exact_attention(c, s):
    """Row block by row block from the definition: softmax over the pairs that count, and its derivative."""
    b, hq, lq, d = s["q"].shape
    hkv, lk = s["k"].shape[1:3]
    o, dq = (torch.zeros(b, hq, lq, d, dtype=torch.float64, device="cuda") for _ in range(2))
    dk, dv = (torch.zeros(b, hkv, lk, d, dtype=torch.float64, device="cuda") for _ in range(2))
    step = max(1, (1 << 26) // lk)
    for i, n in enumerate(lengths_of(c)):
        docs = torch.tensor(documents_of(c)[i], device="cuda") if c["mask"] == "documents" else None
        for h in range(hq):
            k, v = s["k"][i, h * hkv // hq, :n].double(), s["v"][i, h * hkv // hq, :n].double()
            for r in range(0, lq, step):
                q = s["q"][i, h, r:r + step].double()
                at = (n - lq + r + torch.arange(len(q), device="cuda"))[:, None]
                col = torch.arange(n, device="cuda")[None, :]
                raw = q @ k.T / math.sqrt(d)
                z = c["cap"] * torch.tanh(raw / c["cap"]) if c["cap"] else raw
                if "slopes" in s:
                    z = z - s["slopes"][h].double() * (at - col).abs()
                hidden = torch.zeros_like(z, dtype=torch.bool)
                if c["mask"] in ("causal", "documents"):
                    hidden |= col > at
                if c["mask"] == "prefix":
                    hidden |= (col > at) & (col >= c["lk"] // 4)
                if docs is not None:
                    hidden |= docs[at.clamp(min=0)] != docs[:n][None, :]
                z = z.masked_fill(hidden, -math.inf)
                p = torch.softmax(z, -1).nan_to_num(0.0)
                o[i, h, r:r + step] = p @ v
                if c["op"] == "train":
                    g = s["dout"][i, h, r:r + step].double()
                    dv[i, h * hkv // hq, :n] += p.T @ g
                    dz = p * (g @ v.T - (g * (p @ v)).sum(-1, keepdim=True))
                    if c["cap"]:
                        dz = dz / torch.cosh(raw / c["cap"]) ** 2
                    dz = dz / math.sqrt(d)
                    dq[i, h, r:r + step] = dz @ k
                    dk[i, h * hkv // hq, :n] += dz.T @ q
    return [o] if c["op"] == "attention" else [o, dq, dk, dv]


def _exact_rotary(c, s):
    """As a product of complex numbers: a pair (a, b) is a + ib, and turning it multiplies it by exp(i angle)."""
    x, half = s["x"].double(), c["dims"] // 2
    rate = torch.tensor([10000.0 ** (-2.0 * i / c["dims"]) / c["stretch"] for i in range(half)], dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, None, :, None] * rate)

    def apply(t, by):
        head = t[..., :c["dims"]]
        pair = head.unflatten(-1, (half, 2)) if c["interleaved"] else head.unflatten(-1, (2, half)).transpose(-1, -2)
        new = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * by)
        new = new if c["interleaved"] else new.transpose(-1, -2)
        return torch.cat([new.flatten(-2), t[..., c["dims"]:]], -1)

    size = (x.square().sum(-1, keepdim=True) / c["d"] + 1e-6).sqrt()
    w = s["weight"].double()[:, None, :] if c["norm"] else None
    if c["op"] == "rotary":
        return [apply(x / size * w if c["norm"] else x, turn)]
    g = apply(s["dy"].double(), turn.conj())
    if not c["norm"]:
        return [g]
    dot = (g * w * x).sum(-1, keepdim=True)
    return [g * w / size - x * dot / (c["d"] * size ** 3), (g * x / size).sum((0, 2))]


def _exact_sample(c, s):
    """Sequence by sequence on the host, as a list of tokens sorted by probability would be cut and drawn from."""
    import numpy
    got = []
    for row, u in zip(s["logits"].double().cpu().numpy(), s["u"].cpu().numpy()):
        if c["temperature"] == 0.0:
            got.append(int(row.argmax()))
            continue
        order = numpy.lexsort((numpy.arange(len(row)), -row))
        p = numpy.exp((row[order] - row[order[0]]) / c["temperature"])
        if c["top_k"]:
            order, p = order[:c["top_k"]], p[:c["top_k"]]
        if c["top_p"] < 1.0:
            n = int((numpy.cumsum(p) < c["top_p"] * p.sum()).sum()) + 1
            order, p = order[:n], p[:n]
        order, p = order[p >= c["min_p"]], p[p >= c["min_p"]]
        back = numpy.argsort(order)
        at = numpy.cumsum(p[back])
        got.append(int(order[back][min(len(at) - 1, int(numpy.searchsorted(at, u * at[-1], side="right")))]))
    return [torch.tensor(got, device="cuda")]


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] in ("attention", "train"):
        return _exact_attention(c, s)
    return _exact_sample(c, s) if c["op"] == "sample" else _exact_rotary(c, s)
