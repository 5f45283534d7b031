"""Cases of the attention operators around the paged KV cache: the cache held
in 4 bits (write, read back, attention over it) and attention with shaped
scores (tanh cap, distance bias, window, per-token intervals) over every
cache format.

``run`` is one call as a serving loop makes it; with ``own`` false it computes
the same thing from elementary torch operations.  Sequence lengths are spread
evenly over [lo, hi] of the case, so that they are ragged and known without
the seed.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"

# LT_KV_Q4_0: groups of 32 values share one scale d; a value reads back as
# (code - 8) * d.  d has 8 significant bits, is held as f16 and is at most D4MAX.
GROUP, D4MAX = 32, 2720.0


def _attend(name, fmt, batch, lo, hi, heads, kv_heads, dim, dtype, nq=1, fused=False, **shape):
    return {"name": name, "op": "shaped" if shape else "attend4", "fmt": fmt, "batch": batch, "lo": lo, "hi": hi,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "nq": nq, "fused": fused,
            "softcap": shape.get("softcap", 0.0), "window": shape.get("window", 0), "alibi": shape.get("alibi", False),
            "docs": shape.get("docs", 0), "prefix": shape.get("prefix", 0)}


def _write(name, tokens, kv_heads, dim, dtype):
    return {"name": name, "op": "write4", "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}


def listed():
    return [
        # the rows of one decode step of 16 sequences, one layer
        _write("write4 decode step", 16, 8, 128, "f32"),
        # a prefill chunk of an odd size at head_dim 64
        _write("write4 ragged chunk d64", 777, 4, 64, "f32"),
        # a large prefill batch of f16 rows
        _write("write4 prefill", 4096, 8, 128, "f16"),
        # one short chat turn on a small model: launch latency counts
        _attend("attend4 one short sequence", "q4_0", 1, 17, 17, 32, 4, 64, "f32"),
        # the decode microbenchmark: 64 sequences over U[512, 4096]
        _attend("attend4 decode 64 x 512..4096", "q4_0", 64, 512, 4096, 32, 8, 128, "f32"),
        # long contexts with the wide head group
        _attend("attend4 decode 16 x 32768", "q4_0", 16, 32768, 32768, 64, 8, 128, "f16"),
        # a decode step with its append fused in, ragged lengths down to one token
        _attend("attend4 append ragged", "q4_0", 33, 1, 2001, 32, 8, 128, "f32", fused=True),
        # chunked prefill: 4 chunks of 256 tokens behind 2048 cached ones
        _attend("attend4 prefill chunk", "q4_0", 4, 2304, 2304, 32, 8, 128, "f16", nq=256),
        # capped scores and a sliding window over the f16 cache
        _attend("shaped f16 cap window", "f16", 64, 512, 4096, 32, 8, 128, "f32", softcap=50.0, window=1024),
        # distance bias over long contexts
        _attend("shaped f16 distance bias", "f16", 8, 16384, 16384, 32, 8, 128, "f16", alibi=True),
        # a chunk of packed documents with a bidirectional prefix, int8 cache
        _attend("shaped q8_0 documents prefix", "q8_0", 3, 300, 1400, 32, 4, 64, "f32", nq=48, docs=200, prefix=64),
        # one sequence with every score term over the 4-bit cache
        _attend("shaped q4_0 all terms", "q4_0", 2, 100, 777, 64, 8, 128, "f32", nq=1, softcap=30.0, window=300,
                alibi=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.25:
        return {k: v for k, v in _write("", _log_int(rng, 1, 4096), rng.choice([1, 2, 4, 8]), rng.choice([64, 128]),
                                        rng.choice(["f32", "f16"])).items() if k != "name"}
    shaped = rng.random() < 0.45
    fmt = rng.choice(["f16", "q8_0", "q4_0"]) if shaped else "q4_0"
    kv_heads, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([64, 128])
    hi = _log_int(rng, 1, 32768)
    lo = max(1, int(hi * rng.random()))
    # positions of all sequences stay below half of the largest listed case's
    batch = min(_log_int(rng, 1, 96), max(1, 262144 // hi))
    nq, fused, shape = 1, False, {}
    if shaped:
        terms = rng.sample(["softcap", "window", "alibi", "docs", "prefix"], rng.randint(1, 3))
        if "softcap" in terms:
            shape["softcap"] = float(rng.choice([20.0, 30.0, 50.0]))
        if "window" in terms:
            shape["window"] = _log_int(rng, 1, 4096)
        if "alibi" in terms:
            shape["alibi"] = True
        if "docs" in terms:
            shape["docs"] = _log_int(rng, 16, 4096)
        if "prefix" in terms:
            shape["prefix"] = _log_int(rng, 1, 1024)
    if hi <= 4096 and rng.random() < 0.3:
        nq = min(lo, _log_int(rng, 2, 256))
        # the largest listed case does 3.6e10 operations
        batch = max(1, min(batch, 1024 // nq, int(3e10 / (4 * nq * hi * group * kv_heads * dim))))
    elif not shaped:
        fused = rng.random() < 0.4
    c = _attend("", fmt, batch, lo, hi, group * kv_heads, kv_heads, dim, rng.choice(["f32", "f16"]), nq, fused, **shape)
    return {k: v for k, v in c.items() if k != "name"}


# ------------------------------------------------------------------ inputs

def _lens(c):
    if c["batch"] == 1:
        return [c["hi"]]
    return [c["lo"] + (c["hi"] - c["lo"]) * i // (c["batch"] - 1) for i in range(c["batch"])]


def _dt(name):
    return torch.float32 if name == "f32" else torch.float16


def _rows(shape, gen, gains):
    """K or V rows: normal values with a gain of its own for each channel."""
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)
    return x * gains if gains is not None else x


def _quant4(x):
    """x [..., D] f32 -> codes uint8 [..., D], scales f16 [..., D / 32].  The
    code is decided in 64 bits: floor(x / d + 1/2) next to a border."""
    g = x.unflatten(-1, (-1, GROUP))
    top, low = g.amax(-1).clamp(min=0), (-g.amin(-1)).clamp(min=0)
    d = torch.where(top >= low, -top, low) / 8
    d = d.to(torch.bfloat16).float().clamp(-D4MAX, D4MAX).half()
    e = d.double().unsqueeze(-1)
    code = torch.where(e == 0, 8.0, torch.floor(g.double() / torch.where(e == 0, 1.0, e) + 8.5)).clamp(0, 15)
    return code.to(torch.uint8).flatten(-2), d


def _value4(codes, d):
    return ((codes.unflatten(-1, (-1, GROUP)).float() - 8) * d.float().unsqueeze(-1)).flatten(-2)


def _quant8(x):
    g = x.unflatten(-1, (-1, GROUP))
    d = (g.abs().amax(-1) / 127).half()
    e = d.float().unsqueeze(-1)
    q = torch.where(e == 0, 0.0, torch.round(g / torch.where(e == 0, 1.0, e))).clamp(-127, 127)
    return q.to(torch.int8).flatten(-2), d


def _inputs(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dim, hkv = c["dim"], c["kv_heads"]
    gains = torch.exp(0.4 * torch.randn((hkv, dim), generator=gen, device=DEV))
    if c["op"] == "write4":
        k = _rows((c["tokens"], hkv, dim), gen, gains).to(_dt(c["dtype"]))
        v = _rows((c["tokens"], hkv, dim), gen, None).to(_dt(c["dtype"]))
        return {"k": k.flatten(1), "v": v.flatten(1)}
    lens, top, nq = _lens(c), c["hi"], c["nq"]
    s = {"q": torch.randn((c["batch"], nq, c["heads"], dim), generator=gen, device=DEV).to(_dt(c["dtype"]))}
    # the cache, padded to the longest sequence: 4-bit codes two to a byte,
    # int8 codes or f16 values, and the scales
    shape = (c["batch"], top, hkv)
    if c["fmt"] == "f16":
        for n in "kv":
            s[n] = torch.zeros((*shape, dim), device=DEV, dtype=torch.float16)
    else:
        four = c["fmt"] == "q4_0"
        for n in "kv":
            s[n] = torch.zeros((*shape, dim // 2 if four else dim), device=DEV,
                               dtype=torch.uint8 if four else torch.int8)
            s[n + "d"] = torch.zeros((*shape, dim // GROUP), device=DEV, dtype=torch.float16)
    for b, n_tok in enumerate(lens):
        for n in "kv":
            x = _rows((n_tok, hkv, dim), gen, gains if n == "k" else None)
            if c["fmt"] == "f16":
                s[n][b, :n_tok] = x.half()
            elif c["fmt"] == "q8_0":
                s[n][b, :n_tok], s[n + "d"][b, :n_tok] = _quant8(x)
            else:
                codes, s[n + "d"][b, :n_tok] = _quant4(x)
                s[n][b, :n_tok] = codes[..., 0::2] | (codes[..., 1::2] << 4)
    s["lens"] = torch.tensor(lens, device=DEV)
    pos = np.array(lens)[:, None] - nq + np.arange(nq)[None, :]  # the last nq positions of each sequence
    first, end = np.zeros_like(pos), pos + 1
    if c["docs"]:
        first = pos // c["docs"] * c["docs"]  # documents packed end to end
    if c["prefix"]:  # a bidirectional prefix at the start of each document or sequence
        end = np.maximum(end, np.minimum(first + c["prefix"], np.array(lens)[:, None]))
    s["pos"], s["first"], s["end"] = (torch.tensor(a, device=DEV) for a in (pos, first, end))
    if c["alibi"]:
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, c["heads"] + 1, device=DEV) / c["heads"]).float()
    if c["fused"]:
        s["k_new"] = _rows((c["batch"], hkv, dim), gen, gains).to(_dt(c["dtype"]))
        s["v_new"] = _rows((c["batch"], hkv, dim), gen, None).to(_dt(c["dtype"]))
    return s


def _cache_values(s, c, n, b=None):
    """Cached values of K or V in 32 bits (one sequence, or all of them)."""
    x = s[n] if b is None else s[n][b]
    if c["fmt"] == "f16":
        return x.float()
    d = s[n + "d"] if b is None else s[n + "d"][b]
    if c["fmt"] == "q8_0":
        return (x.unflatten(-1, (-1, GROUP)).float() * d.float().unsqueeze(-1)).flatten(-2)
    return _value4(torch.stack((x & 15, x >> 4), -1).flatten(-2), d)


def prepare(case, seed):
    c = case
    s = _inputs(c, seed)
    s["case"] = c
    if not own:
        return s
    from langtrain_studio_b200.kv import KvCache

    if c["op"] == "write4":
        n = c["tokens"]
        kv = KvCache(1, c["kv_heads"], c["dim"], n, max_seqs=1, max_batch=n, kv_format="q4_0")
        s["blocks"], s["slots"] = kv.append_batch(np.zeros(n), np.arange(n))
        s["kv"] = kv
        return s
    lens, hkv, dim, step = _lens(c), c["kv_heads"], c["dim"], 4096
    blocks = sum((n + 15) // 16 for n in lens)
    kv = KvCache(1, hkv, dim, blocks * 16, n_heads=c["heads"], max_seqs=c["batch"],
                 max_batch=max(step, c["batch"] * c["nq"]), max_blocks_per_seq=(c["hi"] + 15) // 16,
                 kv_format=c["fmt"])
    for b, n in enumerate(lens):
        k, v = (_cache_values(s, c, x, b).reshape(-1, hkv * dim) for x in "kv")
        for t in range(0, n, step):
            m = min(step, n - t)
            cells = kv.append_batch(np.full(m, b), np.arange(t, t + m))
            kv.write(0, *cells, k[t:t + m], v[t:t + m])
            if c["fused"] and t + m == n:
                s.setdefault("cells", []).append((cells[0][-1], cells[1][-1]))
    s["kv"] = kv
    if c["fused"]:
        s["blocks"], s["slots"] = (np.array(a, np.int32) for a in zip(*s["cells"]))
    s["seqs"] = np.repeat(np.arange(c["batch"]), c["nq"]).astype(np.uint32)
    s["positions"], s["first_host"], s["end_host"] = (s[x].cpu().numpy().reshape(-1).astype(np.uint32)
                                                      for x in ("pos", "first", "end"))
    # the cache holds the same values as the plain form's arrays now
    for x in ("k", "v", "kd", "vd"):
        s.pop(x, None)
    torch.cuda.synchronize()
    return s


# --------------------------------------------------------------------- run

def _run_write(s):
    if own:
        kv = s["kv"]
        kv.write(0, s["blocks"], s["slots"], s["k"], s["v"])
        return kv.read(0, s["blocks"], s["slots"])
    dim = s["case"]["dim"]
    return tuple(_value4(*_quant4(x.unflatten(-1, (-1, dim)).float())).flatten(1).half() for x in (s["k"], s["v"]))


def _run_plain(s):
    c = s["case"]
    extra = ()
    if c["fused"]:
        at = (torch.arange(c["batch"], device=DEV), s["lens"] - 1)
        (kc, kd), (vc, vd) = _quant4(s["k_new"].float()), _quant4(s["v_new"].float())
        s["k"][at], s["kd"][at] = kc[..., 0::2] | (kc[..., 1::2] << 4), kd
        s["v"][at], s["vd"][at] = vc[..., 0::2] | (vc[..., 1::2] << 4), vd
        extra = (_value4(kc, kd).flatten(1).half(), _value4(vc, vd).flatten(1).half())
    k, v = _cache_values(s, c, "k"), _cache_values(s, c, "v")  # [B, L, Hkv, D]
    batch, top, hkv, dim = k.shape
    q = s["q"].float().reshape(batch, c["nq"], hkv, -1, dim)
    score = torch.einsum("bnhgd,blhd->bnhgl", q, k) * (1.0 / math.sqrt(dim))
    j = torch.arange(top, device=DEV)
    pos, first, end = s["pos"], s["first"], s["end"]
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    if c["alibi"]:
        score = score - s["slopes"].view(1, 1, hkv, -1, 1) * (pos[..., None] - j).abs()[:, :, None, None].float()
    if c["window"]:
        first = torch.maximum(first, pos + 1 - c["window"])
    seen = ((j >= first[..., None]) & (j < end[..., None]))[:, :, None, None]
    score = torch.where(seen, score, -math.inf)
    most = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(most), 0.0, most))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = torch.einsum("bnhgl,blhd->bnhgd", p, v)
    return (out.reshape(batch * c["nq"], -1).to(_dt(c["dtype"])), *extra)


def run(state):
    s = state
    c = s["case"]
    if c["op"] == "write4":
        return _run_write(s)
    if not own:
        return _run_plain(s)
    kv, q = s["kv"], s["q"].view(c["batch"] * c["nq"], -1)
    if c["fused"]:
        k, v = s["k_new"].flatten(1), s["v_new"].flatten(1)
        out = kv.write_attend(0, s["blocks"], s["slots"], k, v, q, s["seqs"], s["positions"], out_dtype=q.dtype)
        return (out, *kv.read(0, s["blocks"], s["slots"]))
    if c["op"] == "attend4":
        return (kv.attend(0, q, s["seqs"], s["positions"], out_dtype=q.dtype),)
    return (kv.attend_shaped(0, q, s["seqs"], s["positions"], softcap=c["softcap"], window=c["window"],
                             slopes=s.get("slopes"), first=s["first_host"] if c["docs"] else None,
                             end=s["end_host"] if c["prefix"] else None, out_dtype=q.dtype),)


# -------------------------------------------------------------------- work

def work(case):
    c = case
    size = 4 if c.get("dtype") == "f32" else 2
    if c["op"] == "write4":
        values = 2 * c["tokens"] * c["kv_heads"] * c["dim"]
        return {"bytes": values * (size + 2 + 18 / 32), "flops": 4.0 * values}
    per = {"f16": 2.0, "q8_0": 34 / 32, "q4_0": 18 / 32}[c["fmt"]]
    rows = flops = 0
    for n in _lens(c):
        pos = n - c["nq"] + np.arange(c["nq"])
        first = pos // c["docs"] * c["docs"] if c["docs"] else 0 * pos
        end = np.maximum(pos + 1, np.minimum(first + c["prefix"], n)) if c["prefix"] else pos + 1
        if c["window"]:
            first = np.maximum(first, pos + 1 - c["window"])
        seen = np.maximum(end - first, 0)
        rows += int(min(n, end.max() - first.min()))  # the positions that some token sees
        flops += float(seen.sum()) * c["heads"] * c["dim"] * 4
    io = 2 * c["batch"] * c["nq"] * c["heads"] * c["dim"] * size
    if c["fused"]:
        io += 2 * c["batch"] * c["kv_heads"] * c["dim"] * (size + 2)
    return {"bytes": 2.0 * rows * c["kv_heads"] * c["dim"] * per + io, "flops": flops}


# ------------------------------------------------------------------- exact

def _nearest4(x):
    """The 4-bit values of x in 64 bits, from the format's definition."""
    g = x.double().unflatten(-1, (-1, GROUP))
    at = g.abs().amax(-1, keepdim=True)
    # the scale carries the sign that puts the largest magnitude on code 0
    positive = (g == at).any(-1, keepdim=True)
    m, e = torch.frexp(at / 8)
    d = torch.ldexp(torch.round(m * 256), e - 8)  # 8 significant bits, nearest even
    d = torch.round(d * 2.0 ** 24) / 2.0 ** 24    # f16 holds multiples of 2^-24
    d = d.clamp(max=D4MAX) * torch.where(positive, -1.0, 1.0)
    steps = torch.where(d == 0, 0.0, torch.floor(g / torch.where(d == 0, 1.0, d) + 0.5)).clamp(-8, 7)
    return (steps * d).flatten(-2)


def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    dim = c["dim"]
    if c["op"] == "write4":
        return tuple(_nearest4(x.unflatten(-1, (-1, dim))).flatten(1) for x in (s["k"], s["v"]))
    group = c["heads"] // c["kv_heads"]
    outs, news = [], ([], [])
    for b, n in enumerate(_lens(c)):
        rows = []
        for x in "kv":
            if c["fmt"] == "f16":
                r = s[x][b, :n].double()
            else:
                code = s[x][b, :n]
                if c["fmt"] == "q4_0":
                    code = torch.stack((code % 16, code // 16), -1).flatten(-2).double() - 8
                r = code.double() * s[x + "d"][b, :n].double().repeat_interleave(GROUP, -1)
            if c["fused"]:
                r[n - 1] = _nearest4(s[x + "_new"][b])
                news["kv".index(x)].append(r[n - 1].flatten())
            rows.append(r)
        k, v = rows
        j = torch.arange(n, device=DEV).double()
        pos = s["pos"][b].double()[:, None]
        seen = (j >= s["first"][b][:, None]) & (j < s["end"][b][:, None])
        if c["window"]:
            seen &= j > pos - c["window"]
        out = torch.zeros((c["nq"], c["heads"], dim), device=DEV, dtype=torch.float64)
        for h in range(c["heads"]):
            t = s["q"][b, :, h].double() @ k[:, h // group].T / math.sqrt(dim)
            if c["softcap"]:
                t = torch.tanh(t / c["softcap"]) * c["softcap"]
            if c["alibi"]:
                t = t - s["slopes"][h].double() * (pos - j).abs()
            t = t.masked_fill(~seen, -math.inf)
            w = torch.softmax(t, -1).nan_to_num(0.0)  # a token that sees nothing answers zero
            out[:, h] = w @ v[:, h // group]
        outs.append(out.reshape(c["nq"], -1))
    done = torch.cat(outs)
    return (done, *(torch.stack(x) for x in news)) if c["fused"] else (done,)
