"""The window operators of ``kvm_paper_b200.window`` as a serving program calls them, for measurement.

  prompt   ``window_attention``: causal attention of a prompt (or of a chunk of one behind earlier tokens) in which a token
           sees the last ``window`` tokens, itself among them, and the first ``sinks`` tokens of its sequence
  store    ``WindowCache.write`` of a prompt's keys and values in 4 bits, and ``WindowCache.read`` of what the cache holds
  token    ``WindowCache.attend``: one query per sequence over the cached tokens; with ``step`` the query's own token is
           written on the way (``WindowCache.step``), over a cache in 4 or in 16 bits

A case is described by plain values: kind, batch, q_heads, kv_heads, head_dim, window, sinks, bits (of a cached value),
tokens (of a prompt; 1 for a token), context (tokens before them: for a chunk those given with it, for the others those the
cache has seen), low (ragged batches: the shortest sequence, its tokens and context taken together; 0 = all alike), step.

The 4-bit form of a row: groups of 32 values share a scale s, a sixth of the group's largest magnitude rounded to 6
significant bits (ties to even; below the smallest normal float: 0, and so is the group); a value is held as the nearest of
0, .5, 1, 1.5, 2, 3, 4, 6 (either sign) to x / s, ties to the candidate with the even code."""

import math

import torch

own = False  # True: ``run`` calls the package's operators; False: the same in elementary operations

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
GROUP = 32


def _case(name, kind, batch, q_heads, kv_heads, head_dim, window, sinks, tokens, context, *, low=0, bits=16, step=False):
    c = dict(kind=kind, batch=batch, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, window=window, sinks=sinks,
             tokens=tokens, context=context, low=low, bits=bits, step=step)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # a chat turn of less than one window: launches and host work
        _case("prompt_250", "prompt", 1, 16, 16, 128, 512, 4, 250, 0),
        # a batch of padded prompts of a small model, grouped queries
        _case("prompt_6x2011_ragged_d64", "prompt", 6, 16, 4, 64, 512, 1, 2011, 0, low=333),
        # a chunk of two long prompts behind the sinks and the window that came before it
        _case("prompt_chunk_2x1024", "prompt", 2, 16, 8, 128, 4096, 16, 1024, 4111),
        # one layer of a 2048-wide model reading two 32k documents
        _case("prompt_2x32768", "prompt", 2, 16, 16, 128, 4096, 4, 32768, 0),
        # the keys and values of four prompts go into a cache of 4 bits and come back for the next chunk
        _case("store_4x8192", "store", 4, 16, 16, 128, 8192, 4, 8192, 0, bits=4),
        # ragged chunks written behind earlier tokens, some of which they push out
        _case("store_5x333_ragged_d64", "store", 5, 8, 4, 64, 1000, 3, 333, 2500, low=700, bits=4),
        # one conversation within its first window: the latency of a token
        _case("token4_1x300", "token", 1, 16, 16, 128, 512, 4, 1, 299, bits=4, step=True),
        # 64 conversations of very unequal length, all of it visible
        _case("token4_64x32768_ragged", "token", 64, 16, 4, 128, 32768, 0, 1, 32767, low=1024, bits=4),
        # one very long document
        _case("token4_1x262144", "token", 1, 32, 8, 128, 262144, 4, 1, 262143, bits=4),
        # sixteen query heads of 64 to a key head, windows that have wrapped around
        _case("token4_24x6000_group16", "token", 24, 32, 2, 64, 4000, 5, 1, 6000, low=300, bits=4),
        # 64 conversations beyond their window, 16 bits, the token written on the way
        _case("token16_64x4096_step", "token", 64, 16, 4, 128, 4096, 4, 1, 20000, low=900, step=True),
        # a small model's short window, 16 bits
        _case("token16_8x256_d64", "token", 8, 8, 8, 64, 256, 4, 1, 1000),
    ]


def draw(rng):
    """One more case of the same ranges: sizes over their logarithm, odd ones among them."""
    def size(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["prompt", "prompt", "store", "token", "token", "token"])
    head_dim = rng.choice([128, 128, 64, 32])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    q_heads = kv_heads * rng.choice([g for g in (1, 1, 2, 4, 5, 8, 16) if kv_heads * g <= 32])
    sinks = rng.choice([0, 1, 4, size(2, 130)])
    if kind == "prompt":
        batch, tokens = size(1, 8), size(1, 16384)
        window = size(16, 8192)
        context = rng.choice([0, 0, size(1, 8192)])
        while 4 * head_dim * batch * q_heads * tokens * min(window + sinks, tokens + context) > 1.5e12:
            tokens = (tokens + 1) // 2
        low = rng.choice([0, size(1, tokens + context)]) if batch > 1 else 0
        return _case(None, kind, batch, q_heads, kv_heads, head_dim, window, sinks, tokens, context, low=low)
    if kind == "store":
        batch, tokens = size(1, 16), size(1, 8192)
        window = size(16, 16384)
        context = rng.choice([0, size(1, 20000)])
        while batch > 1 and batch * kv_heads * (window + tokens) * head_dim > 4e7:
            batch = (batch + 1) // 2
        low = rng.choice([0, size(1, tokens + context)]) if batch > 1 else 0
        return _case(None, kind, batch, q_heads, kv_heads, head_dim, window, sinks, tokens, context, low=low, bits=4)
    batch = size(1, 96)
    window = size(16, 131072)
    context = size(1, 150000) - 1
    bits = rng.choice([4, 4, 16])
    while batch > 1 and batch * kv_heads * (window + sinks) * head_dim * bits > 2.2e9:
        batch = (batch + 1) // 2
    low = rng.choice([0, size(1, context + 1)]) if batch > 1 else 0
    # (a step returns what the cache holds beside its output: kept to caches of which that is a small part or which are small)
    step = rng.random() < 0.5 if bits == 16 else (rng.random() < 0.5 and batch * kv_heads * (window + sinks) * head_dim < 2e6)
    return _case(None, kind, batch, q_heads, kv_heads, head_dim, window, sinks, 1, context, low=low, bits=bits, step=step)


def _ends(case):
    """Tokens of every sequence, context and new ones together: spread evenly between ``low`` and the longest."""
    n, b = case["context"] + case["tokens"], case["batch"]
    if not case["low"] or b == 1:
        return [n] * b
    lo = min(case["low"], n)
    e = [lo + (n - lo) * i // (b - 1) for i in range(b)]
    return e[::2] + e[1::2][::-1]  # (neither rising nor falling over the batch)


def _new(case, end):
    """New tokens of a sequence of ``end`` tokens."""
    return min(case["tokens"], end)


def _row_bytes(case):
    d = case["head_dim"]
    return d * case["bits"] // 8 + (d // GROUP * 2 if case["bits"] == 4 else 0)


def work(case):
    b, hq, hkv, d, w, s = (case[x] for x in ("batch", "q_heads", "kv_heads", "head_dim", "window", "sinks"))
    ends = _ends(case)
    if case["kind"] == "prompt":
        t, c = case["tokens"], case["context"]
        pairs = 0
        for e in ends:  # query index i sees min(i + 1, w) tokens, and the sinks in front of those
            n = max(min(e, c + t) - c, 0)
            m = max(min(c + n, w + s) - c, 0)  # queries that see everything before them
            pairs += m * (2 * c + m + 1) // 2 + (n - m) * (w + s)
        q_rows = sum(max(min(e, c + t) - c, 0) for e in ends)
        k_rows = sum(min(e, min(c, s + w) + t) for e in ends)
        return {"bytes": 2 * d * (hq * q_rows + 2 * hkv * k_rows + hq * b * t), "flops": 4 * d * hq * pairs}
    if case["kind"] == "store":
        kept = [min(e, w + s) for e in ends]
        new = [min(_new(case, e), n) for e, n in zip(ends, kept)]
        return {"bytes": 2 * hkv * (sum(new) * (2 * d + _row_bytes(case)) + sum(kept) * _row_bytes(case) + b * (w + s) * 2 * d),
                "flops": 4 * d * hkv * sum(new)}
    seen = sum(min(e, w + s) for e in ends)
    extra = 0
    if case["step"]:  # the tokens' keys and values, and their rows of the cache
        extra = b * hkv * 2 * (2 * d + _row_bytes(case))
        if case["bits"] == 4:  # the whole cache is read back
            extra += 2 * hkv * (seen * _row_bytes(case) + b * (w + s) * 2 * d)
    return {"bytes": 2 * hkv * seen * _row_bytes(case) + 4 * b * hq * d + extra, "flops": 4 * d * hq * seen}


# ------------------------------------------------------------------------------------------------ inputs

def _inputs(case, seed):
    """Keys and queries as a per-head LayerNorm leaves them (some channels weighted more than others), values of unequal size;
    strides of [batch, token, head, channel] storage, as projections write them."""
    b, hq, hkv, d, t = (case[x] for x in ("batch", "q_heads", "kv_heads", "head_dim", "tokens"))
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def normed(rows, heads, weight):
        x = normal(b, rows, heads, d)
        x = (x - x.mean(-1, keepdim=True)) * (x.var(-1, unbiased=False, keepdim=True) + 1e-5).rsqrt() * weight
        return x.bfloat16().transpose(1, 2)

    def values(rows):
        x = normal(b, rows, hkv, d)
        return (x * torch.exp(0.5 * normal(b, rows, hkv, 1))).bfloat16().transpose(1, 2)

    wq, wk = torch.exp(0.2 * normal(d)), torch.exp(0.4 * normal(d))
    x = {"q": normed(t, hq, wq)}
    if case["kind"] == "prompt":
        n = case["context"] + t
        x["k"], x["v"] = normed(n, hkv, wk), values(n)
    else:
        keep = case["window"] + case["sinks"]
        x["k"], x["v"] = normed(t, hkv, wk), values(t)            # the new tokens
        before = keep if case["context"] else 0
        x["old_k"], x["old_v"] = normed(before, hkv, wk), values(before)  # what the cache holds of the earlier ones, in order
    return x


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def prepare(case, seed):
    x = _inputs(case, seed)
    ends = _ends(case)
    st = {"case": case, "q": x["q"], "k": x["k"], "v": x["v"]}
    if own:
        from kvm_paper_b200 import window
        st["window"] = window
    if case["kind"] == "prompt":
        st["lengths"] = _ints(ends) if case["low"] else None
        return st
    w, s, d, hkv, b = (case[n] for n in ("window", "sinks", "head_dim", "kv_heads", "batch"))
    # a step writes token `end - 1`; without one the cache holds that token already
    if case["kind"] == "store":
        new = [_new(case, e) for e in ends]
    else:
        new = [1 if case["step"] else 0] * b
    old = [e - n for e, n in zip(ends, new)]
    held = [min(o, w + s) for o in old]
    st["ends"], st["old"], st["new"] = _ints(ends), _ints(old), _ints(new)
    old_k, old_v = x["old_k"], x["old_v"]
    if case["kind"] == "token" and not case["step"] and not case["context"]:
        old_k, old_v, held = x["k"], x["v"], [1] * b
    if own:
        cache = st["window"].WindowCache(b, hkv, d, window=w, sinks=s, bits=case["bits"], device="cuda")
        if max(held):
            first = _ints([min(s, h) for h in held])
            if s:
                cache.write(old_k[:, :, :s], old_v[:, :, :s], 0, lengths=first)
            if old_k.size(2) > s:
                cache.write(old_k[:, :, s:], old_v[:, :, s:], torch.maximum(st["old"] - w, first), lengths=_ints(held) - first)
        st["cache"] = cache
        return st
    if case["bits"] == 4:
        st["old_k"], st["old_v"], st["held"] = _pack(old_k), _pack(old_v), held
    else:  # rows of the 16-bit cache: sinks (a multiple of 16), then a ring of the window (a multiple of 16)
        sp, ring = -(-s // 16) * 16, -(-w // 16) * 16
        st["rows_k"], st["rows_v"] = (torch.zeros(b, hkv, sp + ring, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        for i, (o, h) in enumerate(zip(old, held)):
            at = torch.tensor([_row(j if j < s else o - h + j, s, sp, ring) for j in range(h)], device="cuda", dtype=torch.long)
            st["rows_k"][i, :, at], st["rows_v"][i, :, at] = old_k[i, :, :h], old_v[i, :, :h]
    return st


def _row(token, sinks, sp, ring):
    return token if token < sinks else sp + (token - sinks) % ring


# ------------------------------------------------------------------------------------------------ plain forms

def _pack(x):
    """bf16 rows -> (index into the signed levels, scale per group)."""
    g = x.float().unflatten(-1, (-1, GROUP))
    s = g.abs().amax(-1, keepdim=True) / 6.0
    bits = s.view(torch.int32)
    s = ((bits + 0x1FFFF + ((bits >> 18) & 1)) >> 18 << 18).view(torch.float32)  # 6 significant bits
    s = torch.where(s < torch.finfo(torch.float32).tiny, torch.zeros_like(s), s)
    r = torch.where(s > 0, g.abs() / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(g))
    code = torch.zeros_like(r, dtype=torch.uint8)
    for i in range(7):  # a value on the border between two levels goes to the one with the even index
        mid = (LEVELS[i] + LEVELS[i + 1]) / 2
        code += ((r > mid) | ((r == mid) & (i % 2 == 1))).to(torch.uint8)
    code = code + 8 * (g < 0).to(torch.uint8)
    return code.flatten(-2), s.squeeze(-1)


def _unpack(packed):
    code, s = packed
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=code.device)
    return (table[code.int()].unflatten(-1, (-1, GROUP)) * s.unsqueeze(-1)).flatten(-2)


def _softmax_rows(scores, values):
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - m)
    return p @ values / p.sum(-1, keepdim=True)


def _plain_prompt(st):
    case, q, k, v, lengths = st["case"], st["q"], st["k"], st["v"], st["lengths"]
    w, s = case["window"], case["sinks"]
    B, Hq, T, D = q.shape
    Hkv, S = k.size(1), k.size(2)
    at = S - T
    out = torch.zeros(B, T, Hq * D, device=q.device, dtype=q.dtype)
    for t0 in range(0, T, 512):
        t1 = min(T, t0 + 512)
        lo = max(0, at + t0 - w + 1)
        hi = at + t1
        keys = torch.arange(lo, hi, device=q.device)
        if s and lo:
            keys = torch.cat([torch.arange(min(s, lo), device=q.device), keys])
        rows = torch.arange(at + t0, hi, device=q.device)
        see = (keys <= rows[:, None]) & ((keys > rows[:, None] - w) | (keys < s))
        qs = q[:, :, t0:t1].float().unflatten(1, (Hkv, -1))                       # [B,Hkv,G,t,D]
        scores = qs @ k[:, :, keys].float().unsqueeze(2).transpose(-1, -2) / math.sqrt(D)
        o = _softmax_rows(scores.masked_fill(~see, float("-inf")), v[:, :, keys].float().unsqueeze(2))
        if lengths is not None:
            o = torch.where((rows < lengths[:, None])[:, None, None, :, None], o, torch.zeros_like(o))
        out[:, t0:t1] = o.flatten(1, 2).transpose(1, 2).flatten(2).to(q.dtype)
    return out


def _plain_rows(case, b, old, new_k, new_v, st):
    """Keys and values (32 bits, in order) that the cache of sequence b holds behind the new tokens."""
    w, s = case["window"], case["sinks"]
    end, n = st["ends_h"][b], st["new_h"][b]
    held = st["held"][b]
    rows = []
    for name, new in (("old_k", new_k), ("old_v", new_v)):
        have = _unpack(tuple(t[b, :, :held] for t in st[name]))
        fresh = _unpack(_pack(new[b, :, :n])) if n else have[:, :0]
        x = torch.cat([have, fresh], 1)
        if end > w + s:
            x = torch.cat([x[:, :s], x[:, x.size(1) - w:]], 1)
        rows.append(x)
    return rows


def _plain_read(st):
    case = st["case"]
    keep = case["window"] + case["sinks"]
    out = [torch.zeros(case["batch"], case["kv_heads"], keep, case["head_dim"], device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    for b in range(case["batch"]):
        for o, x in zip(out, _plain_rows(case, b, st["old_h"][b], st["k"], st["v"], st)):
            o[b, :, :x.size(1)] = x.to(torch.bfloat16)
    return out


def _plain_token(st):
    case, q = st["case"], st["q"]
    w, s, hkv, d = case["window"], case["sinks"], case["kv_heads"], case["head_dim"]
    out = torch.empty(case["batch"], 1, case["q_heads"] * d, device=q.device, dtype=q.dtype)
    if case["bits"] == 16:
        rows = torch.arange(st["rows_k"].size(2), device=q.device)
        sp, ring = -(-s // 16) * 16, -(-w // 16) * 16
    for b in range(case["batch"]):
        end = st["ends_h"][b]
        if case["bits"] == 4:
            k, v = _plain_rows(case, b, st["old_h"][b], st["k"], st["v"], st)
        else:
            if case["step"]:
                at = _row(end - 1, s, sp, ring)
                st["rows_k"][b, :, at], st["rows_v"][b, :, at] = st["k"][b, :, 0], st["v"][b, :, 0]
            age = (end - 1 - s - (rows - sp)) % ring       # of the newest token in a ring row, if it has been written
            see = torch.where(rows < sp, rows < min(s, end), age < min(w, end - s))
            k, v = st["rows_k"][b][:, see].float(), st["rows_v"][b][:, see].float()
        qs = q[b].float().unflatten(0, (hkv, -1)).squeeze(2)
        o = _softmax_rows(qs @ k.transpose(-1, -2) / math.sqrt(d), v)
        out[b, 0] = o.flatten().to(q.dtype)
    return out


def run(st):
    case = st["case"]
    w, s = case["window"], case["sinks"]
    if own:
        if case["kind"] == "prompt":
            return st["window"].window_attention(st["q"], st["k"], st["v"], window=w, sinks=s, lengths=st["lengths"])
        cache = st["cache"]
        if case["kind"] == "store":
            cache.write(st["k"], st["v"], st["old"], lengths=st["new"])
            return cache.read(st["ends"])
        if not case["step"]:
            return cache.attend(st["q"], st["ends"])
        out = cache.step(st["q"], st["k"], st["v"], st["old"])
        return (out, *cache.read(st["ends"])) if case["bits"] == 4 else (out, cache.k, cache.v)
    if case["kind"] == "prompt":
        return _plain_prompt(st)
    if "ends_h" not in st:
        st["ends_h"], st["old_h"], st["new_h"] = (st[n].tolist() for n in ("ends", "old", "new"))
    if case["kind"] == "store":
        return tuple(_plain_read(st))
    out = _plain_token(st)
    if not case["step"]:
        return out
    return (out, *_plain_read(st)) if case["bits"] == 4 else (out, st["rows_k"], st["rows_v"])


# ------------------------------------------------------------------------------------------------ in 64 bits

def _held(x):
    """What the 4-bit form of the rows stands for, from the definition: the nearest level by distance."""
    g = x.double().reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    mant, expo = torch.frexp(g.abs().amax(-1, keepdim=True) / 6)
    s = torch.ldexp(torch.round(mant * 64), expo - 6)
    s = s * (s >= 2.0 ** -126)
    best = torch.zeros_like(g)
    dist = g.abs()
    for level in (1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0):  # codes 2, 4, 6 before 1, 3, 5, 7: an even code keeps a tie
        d = (g.abs() - level * s).abs()
        nearer = d < dist
        best, dist = torch.where(nearer, level * s, best), torch.where(nearer, d, dist)
    return torch.where(g < 0, -best, best).reshape(x.shape)


def exact(case, seed):
    x = _inputs(case, seed)
    b, hq, hkv, d, w, s = (case[n] for n in ("batch", "q_heads", "kv_heads", "head_dim", "window", "sinks"))
    ends, group = _ends(case), hq // hkv

    def attend(q, k, v, see=None):
        z = torch.einsum("gtd,nd->gtn", q.double(), k.double()) * d ** -0.5
        if see is not None:
            z = torch.where(see, z, torch.full_like(z, -math.inf))
        return torch.einsum("gtn,nd->gtd", torch.softmax(z, -1), v.double())

    if case["kind"] == "prompt":
        t, c = case["tokens"], case["context"]
        out = torch.zeros(b, t, hq, d, device="cuda", dtype=torch.float64)
        for i in range(b):
            for t0 in range(0, max(min(ends[i] - c, t), 0), 1024):
                t1 = min(t0 + 1024, ends[i] - c, t)
                row = torch.arange(c + t0, c + t1, device="cuda").view(-1, 1)
                lo = max(c + t0 - w + 1, 0)
                col = torch.cat([torch.arange(min(s, lo), device="cuda"), torch.arange(lo, c + t1, device="cuda")])
                see = ((row - col >= 0) & (row - col < w)) | ((col < s) & (col <= row))
                for h in range(hkv):
                    o = attend(x["q"][i, h * group:(h + 1) * group, t0:t1], x["k"][i, h, col], x["v"][i, h, col], see)
                    out[i, t0:t1, h * group:(h + 1) * group] = o.transpose(0, 1)
        return out.flatten(2)

    keep = w + s
    if case["kind"] == "token" and not case["step"] and not case["context"]:
        old_k, old_v, new = x["k"], x["v"], 0
        old = [1] * b
    else:
        old_k, old_v = x["old_k"], x["old_v"]
        new = None if case["kind"] == "store" else int(case["step"])
        old = [e - (_new(case, e) if new is None else new) for e in ends]
    out = torch.zeros(b, 1, hq * d, device="cuda", dtype=torch.float64)
    whole = case["kind"] == "store" or (case["step"] and case["bits"] == 4)
    back = [torch.zeros(b, hkv, keep, d, device="cuda", dtype=torch.float64) for _ in range(2)] if whole else None
    rows = None
    if case["step"] and case["bits"] == 16:
        sp, ring = (s + 15) // 16 * 16, (w + 15) // 16 * 16
        rows = [torch.zeros(b, hkv, sp + ring, d, device="cuda", dtype=torch.float64) for _ in range(2)]
    for i in range(b):
        have = min(old[i], keep)
        # the token of each row that the cache holds in order, first of the earlier ones, then of the new ones
        tokens = list(range(min(s, old[i]))) + list(range(max(old[i] - w, min(s, old[i])), ends[i] if new != 0 else old[i]))
        assert len(tokens) == have + (ends[i] - old[i] if new != 0 else 0)
        kv = []
        for name, o in (("k", old_k), ("v", old_v)):
            y = torch.cat([o[i, :, :have], x[name][i, :, :len(tokens) - have]], 1)
            kv.append(_held(y) if case["bits"] == 4 else y.double())
        end = ends[i]
        pick = [j for j, p in enumerate(tokens) if p < s or p >= end - w]
        if rows is not None:
            kept = {(p if p < s else sp + (p - s) % ring): j for j, p in enumerate(tokens)}  # (a later token takes an earlier one's row)
            at, j = (torch.tensor(list(t), device="cuda", dtype=torch.long) for t in (kept.keys(), kept.values()))
            for r, y in zip(rows, kv):
                r[i, :, at] = y[:, j]
        if len(pick) != len(tokens):
            j = torch.tensor(pick, device="cuda")
            kv = [y[:, j] for y in kv]
        if back is not None:
            for r, y in zip(back, kv):
                r[i, :, :len(pick)] = y
        if case["kind"] == "token":
            for h in range(hkv):
                out[i, 0, h * group * d:(h + 1) * group * d] = attend(x["q"][i, h * group:(h + 1) * group], kv[0][h], kv[1][h]).flatten()
    if case["kind"] == "store":
        return tuple(back)
    if not case["step"]:
        return out
    return (out, *back) if case["bits"] == 4 else (out, *rows)
