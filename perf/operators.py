"""Work that the batched attention-cache operators and the token log probabilities are measured on.

Four operators, each in a plain form (elementary torch operations in 32 bits) and through the binding
(dflash-swift_b200/dflashcuda.py):

  append    q/k RMSNorm, rotary embedding and the write of k and v into a batch of attention caches held in
            16, 8 or 4 bits, then the rows read back
  attend    decode attention of a batch of sequences over their quantised caches, with the output gate
  shared    the same for sequences that share a prefix, whose cache is held (and read) once
  logprobs  log probabilities of given tokens, entropy and the most likely alternatives of rows of logits
"""
import math
import os
import sys

import torch

own = False


def _binding():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dflash-swift_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import dflashcuda
    return dflashcuda


# ----------------------------------------------------------------------------- cases

def _attn(op, name, S, T, hq, hkv, d, bits, group, lens, prefix=0, rot=64):
    """lens: the longest sequence's cached tokens; the others have between a half of it and all."""
    return {"name": name, "op": op, "S": S, "T": T, "hq": hq, "hkv": hkv, "d": d, "bits": bits, "group": group,
            "len": lens, "prefix": prefix, "rot": rot}


def _lp(name, R, V, pad, dtype, n, top):
    return {"name": name, "op": "logprobs", "R": R, "V": V, "pad": pad, "dtype": dtype, "n": n, "top": top}


def listed():
    return [
        _attn("append", "append-block-8bit", 1, 8, 24, 4, 256, 8, 64, 1024),
        _attn("append", "append-prompt-4bit", 2, 2051, 24, 4, 256, 4, 64, 300, prefix=70001),
        _attn("attend", "attend-block-8bit", 1, 8, 24, 4, 256, 8, 64, 1024),
        _attn("attend", "attend-batch-4bit", 33, 1, 24, 4, 256, 4, 64, 4096),
        _attn("attend", "attend-prompt-8bit", 2, 509, 16, 2, 128, 8, 32, 7000),
        _attn("attend", "attend-long-8bit", 1, 8, 24, 4, 256, 8, 64, 131071),
        _attn("shared", "shared-few-bf16", 4, 1, 8, 2, 64, 16, 0, 61, prefix=515),
        _attn("shared", "shared-batch-8bit", 32, 1, 20, 4, 128, 8, 64, 250, prefix=8190),
        _attn("shared", "shared-large-bf16", 64, 4, 24, 4, 256, 16, 0, 200, prefix=32768),
        _lp("logprobs-block-bf16", 8, 248320, 0, "bfloat16", 1, 20),
        _lp("logprobs-batch-fp32", 61, 50021, 3, "float32", 2, 5),
        _lp("logprobs-prompt-bf16", 509, 248320, 0, "bfloat16", 1, 8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "shared", "logprobs"])
    if op == "logprobs":
        V = _log(rng, 500, 248320)
        dtype = rng.choice(["bfloat16", "float32"])
        R = _log(rng, 1, max(1, min(600, (250 << 20) // (V * (4 if dtype == "float32" else 2)))))
        c = _lp("", R, V, rng.choice([0, 0, 1, 8, 13]), dtype, rng.randint(1, 4), rng.choice([0, 1, 5, 20, 32]))
    else:
        d = rng.choice([64, 128, 256])
        hkv = rng.choice([1, 2, 4, 8])
        G = rng.randint(1, 8)
        bits = rng.choice([16, 8, 4] if op != "attend" else [8, 4])
        group = 0 if bits == 16 else rng.choice([g for g in (32, 64, 128) if g <= d])
        rot = 64 * rng.randint(0, d // 64)
        if op == "append":
            S = _log(rng, 1, 64)
            c = _attn(op, "", S, _log(rng, 1, max(1, 4096 // S)), hkv * G, hkv, d, bits, group, _log(rng, 1, 500),
                      rng.choice([0, _log(rng, 1, 200000)]), rot)
        elif op == "attend":
            S, T = _log(rng, 1, 48), rng.choice([1, 1, rng.randint(1, 16), _log(rng, 16, 500)])
            if T > 16:
                S = min(S, 4)
            most = (128 << 20) // (S * hkv * d)
            c = _attn(op, "", S, T, hkv * G, hkv, d, bits, group, _log(rng, 1, min(131072, most, (1 << 22) // (S * T))),
                      0, rot)
        else:
            S, T = _log(rng, 2, 64), rng.choice([1, 1, rng.randint(1, 4)])
            c = _attn(op, "", S, T, hkv * G, hkv, d, bits, group, _log(rng, 1, 400),
                      _log(rng, 30, min(32768, (1 << 29) // (S * T * hkv * G))), rot)
    del c["name"]
    return c


def _row_lens(c):
    """Cached tokens of each sequence before the block (deterministic, ragged)."""
    return [c["len"] - (i * 7919) % (c["len"] // 2 + 1) for i in range(c["S"])]


def work(c):
    if c["op"] == "logprobs":
        n = c["R"] * c["V"]
        return {"bytes": n * (4 if c["dtype"] == "float32" else 2) + c["R"] * (8 * c["n"] + 4 + 8 * c["top"]),
                "flops": 5 * n}
    S, T, hq, hkv, d = (c[k] for k in ("S", "T", "hq", "hkv", "d"))
    row = 2 * d if c["bits"] == 16 else d * c["bits"] // 8 + 4 * (d // c["group"])  # bytes of one cached k or v
    rows = S * T
    if c["op"] == "append":
        return {"bytes": rows * (2 * hq * d * 2 + 2 * hkv * (2 * d + 2 * row + 2 * d)),
                "flops": rows * 10 * (hq + 2 * hkv) * d}
    lens = _row_lens(c)
    keys = c["prefix"] + sum(lens) + rows
    pairs = T * (S * c["prefix"] + sum(lens)) + S * T * (T + 1) // 2
    return {"bytes": keys * hkv * 2 * row + rows * hq * d * 6, "flops": 4 * d * hq * pairs}


# ----------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _stored(x, bits, group):
    """A cache tensor of the rows x (fp32 [..., d]): (rows, None, None) in bf16, or 8- / 4-bit affine codes packed
    in 32-bit words with a bf16 scale and bias per group."""
    if bits == 16:
        return x.to(torch.bfloat16), None, None
    top = 2 ** bits - 1
    xg = x.unflatten(-1, (-1, group))
    lo, hi = xg.amin(-1), xg.amax(-1)
    low, span = lo.abs() > hi.abs(), hi - lo
    edge, sign = torch.where(low, lo, hi), torch.where(low, 1.0, -1.0)
    # the code of zero as one division, so that a symmetric group (edge / span = 1/2) is a tie, which goes to even
    tiny = span / top < 1e-7
    zero = sign * torch.where(tiny, torch.round(edge / 1e-7), torch.round(edge * top / span))
    s = torch.where(zero != 0, edge / zero, sign * torch.clamp(span / top, min=1e-7)).to(torch.bfloat16)
    b = torch.where(zero != 0, edge, torch.zeros_like(edge)).to(torch.bfloat16)
    c = torch.round((xg - b.float()[..., None]) / s.float()[..., None]).clamp(0, top).to(torch.int32).flatten(-2)
    return _packed(c, bits), s, b


def _packed(c, bits):
    """int32 codes [..., d] -> 32-bit words [..., d bits / 32], lowest element in the lowest bits."""
    c = c.unflatten(-1, (-1, 32 // bits))
    shift = torch.arange(0, 32, bits, device=c.device, dtype=torch.int32)
    return torch.bitwise_left_shift(c, shift).sum(-1, dtype=torch.int32)


def _values(t, bits, group):
    """fp32 values of a stored cache tensor."""
    x, s, b = t
    if bits == 16:
        return x.float()
    shift = torch.arange(0, 32, bits, device=x.device, dtype=torch.int32)
    c = torch.bitwise_and(torch.bitwise_right_shift(x[..., None], shift), 2 ** bits - 1).flatten(-2)
    return (c.float().unflatten(-1, (-1, group)) * s.float()[..., None] + b.float()[..., None]).flatten(-2)


def prepare(c, seed):
    g = _gen(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if c["op"] == "logprobs":
        dt = getattr(torch, c["dtype"])
        R, V = c["R"], c["V"]
        buf = torch.empty(R, V + c["pad"], dtype=dt, device="cuda")
        for r0 in range(0, R, 64):  # rows of different sharpness, from nearly flat to nearly certain
            x = rnd(min(64, R - r0), V + c["pad"])
            buf[r0:r0 + 64] = (x * (0.5 + 4.0 * torch.rand(x.shape[0], 1, generator=g, device="cuda"))).to(dt)
        tokens = torch.randint(0, V, (R, c["n"]), generator=g, device="cuda", dtype=torch.int32)
        tokens[:, 0] = buf[:, :V].float().argmax(1).to(torch.int32)
        return {"c": c, "logits": buf[:, :V], "tokens": tokens}
    S, T, hq, hkv, d, bits, group = (c[k] for k in ("S", "T", "hq", "hkv", "d", "bits", "group"))
    lens = _row_lens(c)
    st = {"c": c, "lengths": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    rows, L = S * T, c["len"] + T
    spread = torch.ones(d, device="cuda")
    spread[:: max(1, d // 4)] = 3.0  # a few channels larger than the rest, as keys have
    if c["op"] == "append":
        st["qkv"] = rnd(rows, (2 * hq + 2 * hkv) * d).to(torch.bfloat16)
        st["q_norm"] = (1 + 0.1 * rnd(d)).to(torch.bfloat16)
        st["k_norm"] = ((1 + 0.1 * rnd(d)) * spread).to(torch.bfloat16)
        st["k"] = _stored(torch.zeros(S, hkv, L, d, device="cuda"), bits, group)
        st["v"] = _stored(torch.zeros(S, hkv, L, d, device="cuda"), bits, group)
    else:
        st["q"] = rnd(rows, hq * d).to(torch.bfloat16)
        st["gate"] = rnd(rows, hq * d).to(torch.bfloat16)
        st["k"] = _stored(rnd(S, hkv, L, d) * spread, bits, group)
        st["v"] = _stored(0.5 * rnd(S, hkv, L, d), bits, group)
        if c["op"] == "shared":
            st["pk"] = _stored(rnd(1, hkv, c["prefix"], d) * spread, bits, group)
            st["pv"] = _stored(0.5 * rnd(1, hkv, c["prefix"], d), bits, group)
    if own:  # the handles that a program keeps beside its caches
        dc = _binding()
        st["cache"] = dc.KVCache.of(st["k"], st["v"], bits, group)
        st["prefix"] = dc.KVCache.of(st["pk"], st["pv"], bits, group) if "pk" in st else None
    return st


# ----------------------------------------------------------------------------- one pass

_EPS, _THETA = 1e-6, 1e7


def run(st):
    c = st["c"]
    if own:
        dc = _binding()
        if c["op"] == "logprobs":
            return dc.logprobs(st["logits"], st["tokens"], top=c["top"])
        if c["op"] == "append":
            q = dc.stack_attn_prep_batch(st["qkv"], st["q_norm"], st["k_norm"], st["cache"], st["lengths"], c["hq"],
                                         c["rot"], _EPS, _THETA, position0=c["prefix"])
            k, v = dc.stack_kv_read(st["cache"], c["T"], starts=st["lengths"])
            return {"q": q, "k": k, "v": v}
        return dc.stack_attn_decode_batch(st["q"], st["cache"], st["lengths"], 1.0 / math.sqrt(c["d"]),
                                          gate=st["gate"], prefix=st["prefix"])
    return {"append": _append, "attend": _attend, "shared": _attend, "logprobs": _logprobs}[c["op"]](st)


def _append(st):
    c = st["c"]
    S, T, hq, hkv, d, rot = (c[k] for k in ("S", "T", "hq", "hkv", "d", "rot"))
    x = st["qkv"].view(S, T, 2 * hq + 2 * hkv, d).float()
    slots = st["lengths"].long()[:, None] + torch.arange(T, device="cuda")
    freq = _THETA ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / max(rot, 1))
    angle = (slots + c["prefix"]).double()[..., None] * freq
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]

    def normed(y, w):
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + _EPS) * w.float()
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., rot:]], -1)

    q = normed(x[:, :, :hq], st["q_norm"]).to(torch.bfloat16).reshape(S * T, hq * d)
    rows = torch.arange(S, device="cuda")[:, None]
    back = {}
    for name, y in (("k", normed(x[:, :, 2 * hq:2 * hq + hkv], st["k_norm"])), ("v", x[:, :, 2 * hq + hkv:])):
        cache, new = st[name], _stored(y, c["bits"], c["group"])
        for old, n in zip(cache, new):
            if old is not None:
                old[rows, :, slots] = n
        back[name] = _values(tuple(None if t is None else t[rows, :, slots] for t in cache), c["bits"], c["group"])
    return {"q": q, "k": back["k"].transpose(1, 2).to(torch.bfloat16).contiguous(),
            "v": back["v"].transpose(1, 2).to(torch.bfloat16).contiguous()}


def _attend(st):
    c = st["c"]
    S, T, hq, hkv, d = (c[k] for k in ("S", "T", "hq", "hkv", "d"))
    G, bits, group = hq // hkv, c["bits"], c["group"]
    q = st["q"].float().view(S, T, hkv, G, d).permute(0, 2, 1, 3, 4).reshape(S, hkv, T * G, d) / math.sqrt(d)
    k, v = _values(st["k"], bits, group), _values(st["v"], bits, group)
    L = k.shape[2]
    last = st["lengths"].long()[:, None] + torch.arange(T, device="cuda")
    seen = torch.arange(L, device="cuda") <= last[..., None]                       # [S, T, L]
    seen = seen[:, None, :, None, :].expand(S, hkv, T, G, L).reshape(S, hkv, T * G, L)
    s = (q @ k.transpose(-1, -2)).masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    if "pk" in st:
        pk, pv = _values(st["pk"], bits, group)[0], _values(st["pv"], bits, group)[0]   # [hkv, P, d]
        rows = q.transpose(0, 1).reshape(hkv, S * T * G, d)
        sp = rows @ pk.transpose(-1, -2)                                              # [hkv, S T G, P]
        m = torch.maximum(m, sp.amax(-1).view(hkv, S, T * G).transpose(0, 1)[..., None])
        ep = torch.exp(sp - m.transpose(0, 1).reshape(hkv, S * T * G, 1))
    e = torch.exp(s - m)
    den, num = e.sum(-1, keepdim=True), e @ v
    if "pk" in st:
        den = den + ep.sum(-1).view(hkv, S, T * G).transpose(0, 1)[..., None]
        num = num + (ep @ pv).view(hkv, S, T * G, d).transpose(0, 1)
    o = (num / den).view(S, hkv, T, G, d).permute(0, 2, 1, 3, 4).reshape(S * T, hq * d)
    return (o / (1 + torch.exp(-st["gate"].float()))).to(torch.bfloat16)


def _logprobs(st):
    c = st["c"]
    x = st["logits"].float()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["top"]]
    return {"logprobs": x.gather(1, st["tokens"].long()) - lse,
            "entropy": (torch.log(total) - (e * (x - m)).sum(1, keepdim=True) / total)[:, 0],
            "top_ids": ids.to(torch.int32), "top_logprobs": x.gather(1, ids) - lse}


# ----------------------------------------------------------------------------- the definition in 64 bits

def exact(c, seed):
    st = prepare(c, seed)
    if c["op"] == "logprobs":
        logp = torch.empty(c["R"], c["n"], dtype=torch.float64, device="cuda")
        ent = torch.empty(c["R"], dtype=torch.float64, device="cuda")
        best = torch.empty(c["R"], c["top"], dtype=torch.float64, device="cuda")
        for r in range(c["R"]):
            lp = torch.log_softmax(st["logits"][r].double(), 0)
            logp[r] = lp[st["tokens"][r].long()]
            ent[r] = -(lp.exp() * lp).sum()
            best[r] = lp.topk(c["top"]).values
        return {"logprobs": logp, "entropy": ent, "top_ids": None, "top_logprobs": best}

    def wide(t, i):  # rows of sequence i in 64 bits, [hkv, rows, d]
        w, s, b = (None if x is None else x[i] for x in t)
        if c["bits"] == 16:
            return w.double()
        w = w.long() & 0xFFFFFFFF
        code = torch.stack([(w >> k) & (2 ** c["bits"] - 1) for k in range(0, 32, c["bits"])], -1).flatten(-2)
        per = lambda x: x.double().repeat_interleave(c["group"], -1)  # noqa: E731
        return code.double() * per(s) + per(b)

    S, T, hq, hkv, d, rot = (c[k] for k in ("S", "T", "hq", "hkv", "d", "rot"))
    lens, G = st["lengths"].tolist(), hq // hkv
    if c["op"] == "append":
        x = st["qkv"].double().view(S, T, -1, d)
        pos = torch.tensor([[c["prefix"] + n + t for t in range(T)] for n in lens], dtype=torch.float64, device="cuda")

        def head(y, w):
            y = y / (y.pow(2).mean(-1, keepdim=True) + _EPS).sqrt() * w.double()
            if rot:
                i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
                turn = torch.polar(torch.ones_like(pos)[..., None], pos[..., None] * _THETA ** (-2 * i / rot))
                z = torch.complex(y[..., :rot // 2], y[..., rot // 2:rot]) * turn[:, :, None]
                y = torch.cat([z.real, z.imag, y[..., rot:]], -1)
            return y

        def held(y):  # what the cache's bits stand for
            y = y.transpose(1, 2)
            if c["bits"] == 16:
                return y.clone()
            top, y = 2 ** c["bits"] - 1, y.unflatten(-1, (-1, c["group"]))
            lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
            low = lo.abs() > hi.abs()
            step = ((hi - lo) / top).clamp(min=1e-7) * (2.0 * low - 1.0)
            edge = torch.where(low, lo, hi)
            zero = torch.where(step.abs() > 1e-7, edge * top / (hi - lo) * (2.0 * low - 1.0), edge / step).round()
            step = torch.where(zero == 0, step, edge / zero.where(zero != 0, torch.ones_like(zero)))
            bias = edge * (zero != 0)
            step, bias = step.bfloat16().double(), bias.bfloat16().double()
            return (((y - bias) / step).round().clamp(0, top) * step + bias).flatten(-2)

        return {"q": head(x[:, :, :hq], st["q_norm"]).reshape(S * T, hq * d),
                "k": held(head(x[:, :, 2 * hq:2 * hq + hkv], st["k_norm"])), "v": held(x[:, :, 2 * hq + hkv:])}
    out = torch.empty(S, T, hkv, G, d, dtype=torch.float64, device="cuda")
    gate = torch.sigmoid(st["gate"].double()).view(S, T, hkv, G, d)
    pk, pv = (wide(st["pk"], 0), wide(st["pv"], 0)) if "pk" in st else (None, None)
    for i, n in enumerate(lens):
        k, v = wide(st["k"], i)[:, :n + T], wide(st["v"], i)[:, :n + T]
        future = torch.arange(n + T, device="cuda")[None] > n + torch.arange(T, device="cuda")[:, None]
        for h in range(hkv):
            qh = st["q"].double().view(S, T, hkv, G, d)[i, :, h]
            a = torch.einsum("tgd,nd->tgn", qh, k[h]) * d ** -0.5
            a = a.masked_fill(future[:, None], -math.inf)
            vals = v[h]
            if pk is not None:
                a, vals = torch.cat([torch.einsum("tgd,nd->tgn", qh, pk[h]) * d ** -0.5, a], -1), torch.cat([pv[h], vals])
            out[i, :, h] = torch.softmax(a, -1) @ vals * gate[i, :, h]
    return out.reshape(S * T, hq * d)
