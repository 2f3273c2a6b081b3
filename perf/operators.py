"""The serving operators' cases: the paged 8-bit K/V cache (append and
attention) and the sampler, each in its plain form (elementary torch
operations in 32 bits) and as calls of sepia_b200.

Cache: blocks of `block` tokens for each KV head as e4m3 codes with one
power-of-two scale for K and one for V; a sequence's unfinished last block is
kept in fp16 (its tail) and rounded to 8 bits once, when its last token
arrives.
"""
import math

import torch

own = False

DEV = "cuda"
E4M3_MAX = 448.0
F16_MAX = 65504.0
W_ONE = 2147483648.0            # sampler: the integer weight of the best token, 2^31


# ------------------------------------------------------------------ cases
def _append(name, seqs, kv, new, heads, kv_heads, dim, block, dtype, norm, rot, adjacent):
    c = dict(op="append", seqs=seqs, kv=kv, new=new, heads=heads, kv_heads=kv_heads, dim=dim, block=block,
             dtype=dtype, norm=norm, rot=rot, adjacent=adjacent)
    return dict(c, name=name) if name else c


def _attention(name, seqs, kv, new, heads, kv_heads, dim, block, dtype, window, extent):
    c = dict(op="attention", seqs=seqs, kv=kv, new=new, heads=heads, kv_heads=kv_heads, dim=dim, block=block,
             dtype=dtype, window=window, extent=extent)
    return dict(c, name=name) if name else c


def _sample(name, rows, vocab, dtype, mode):
    c = dict(op="sample", rows=rows, vocab=vocab, dtype=dtype, mode=mode)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of one sequence, the decode engine's head layout: latency
        _append("append_1_token", 1, 4095, 1, 64, 8, 128, 32, "f32", True, 0, False),
        # one token of each of 48 sequences, half precision, keys and queries rotated
        _append("append_48_tokens_f16", 48, 3000, 1, 64, 8, 128, 32, "f16", True, 128, False),
        # pieces of prompts of 7 sequences, ragged, odd head count, half of each head rotated
        _append("append_ragged_f16", 7, 333, 301, 24, 4, 96, 16, "f16", True, 48, True),
        # a prompt of 8192 tokens in one call
        _append("append_prompt_8192", 1, 0, 8192, 64, 8, 128, 64, "f32", True, 0, False),
        # one token against a sliding window in a long context, the band as wide as the window
        _attention("attn_window_4096", 1, 20000, 1, 64, 8, 128, 32, "f32", 4096, 4096),
        # one token against a full context of 32768
        _attention("attn_global_32768", 1, 32768, 1, 64, 8, 128, 32, "f32", 0, 256),
        # 5 short ragged sequences, small odd heads, 3 new tokens each
        _attention("attn_short_ragged", 5, 317, 3, 18, 3, 96, 16, "f32", 100, 40),
        # a serving batch: 64 ragged sequences in half precision
        _attention("attn_64_seqs_f16", 64, 4096, 1, 64, 8, 128, 64, "f16", 0, 256),
        # 4 new tokens of each of 12 sequences
        _attention("attn_12_seqs_4_new", 12, 6001, 4, 64, 8, 128, 32, "f32", 0, 256),
        # one row of a 200k vocabulary, all filters
        _sample("sample_1_all", 1, 200058, "f32", "all"),
        # 33 rows of an odd half-precision vocabulary, every row with its own settings
        _sample("sample_33_mixed_f16", 33, 50021, "f16", "mixed"),
        # a large serving batch, nucleus sampling
        _sample("sample_192_top_p", 192, 200058, "f32", "top_p"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads = rng.choice([(64, 8), (32, 4), (16, 8), (8, 1), (24, 4), (18, 3), (16, 1)])
    dim = rng.choice([64, 96, 128, 128])
    block = rng.choice([16, 32, 64])
    dtype = rng.choice(["f32", "f16"])
    op = rng.choice(["append", "attention", "attention", "sample"])
    if op == "append":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, 8192 // seqs))
        rot = rng.choice([0, dim, dim // 2])
        return _append(None, seqs, rng.randrange(0, 4096), new, heads, kv_heads, dim, block, dtype,
                       rng.random() < 0.75, rot, rng.random() < 0.5)
    if op == "attention":
        seqs = _log(rng, 1, 64)
        new = rng.choice([1, 1, 1, 2, 3, 5, 8])
        kv = min(_log(rng, new, 32768), max(64, 200000 // (seqs * new)))
        window = rng.choice([0, 0, 512, 4096])
        extent = rng.choice([0, 33, 256, window])
        return _attention(None, seqs, max(kv, new), new, heads, kv_heads, dim, block, dtype, window, extent)
    vocab = _log(rng, 1000, 262144)
    return _sample(None, min(_log(rng, 1, 192), 38000000 // vocab), vocab, dtype,
                   rng.choice(["temperature", "top_k", "top_p", "min_p", "all", "mixed"]))


def _lens(case):
    """Held tokens before the call and new tokens of each sequence: ragged, the same for every seed."""
    n, held, new = case["seqs"], [], []
    for i in range(n):
        if case["op"] == "append":
            held.append(case["kv"] if n == 1 else (case["kv"] * (2 * n - i) // (2 * n) + 7 * i) % (case["kv"] + 1))
            new.append(case["new"] - (i * case["new"] // (2 * n)))
        else:   # kv counts the tokens that the last new token sees
            total = max(case["new"], case["kv"] - i * case["kv"] // (2 * n))
            t = case["new"] - (i % 2 if case["new"] > 1 else 0)
            held.append(total - t)
            new.append(t)
    return held, new


# ------------------------------------------------------------------ inputs
def _pow2_scale(amax):
    """The smallest power of two s with amax / s <= 448 (1 for an empty block)."""
    f, x = torch.frexp(amax)
    s = torch.ldexp(torch.ones_like(amax), x - torch.where(f <= 0.875, 9, 8))
    return torch.where(amax > 0, s, torch.ones_like(amax))


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = torch.float16 if case["dtype"] == "f16" else torch.float32
    if case["op"] == "sample":
        return _prepare_sample(case, g, dt)
    held, new = _lens(case)
    n, hk, d, b, h = case["seqs"], case["kv_heads"], case["dim"], case["block"], case["heads"]
    cols = max((x + y) // b + 2 + max(new) // b for x, y in zip(held, new))
    s = dict(case=case, op=case["op"], max_new=max(new), n_tokens=sum(new),
             max_kv=max(x + y for x, y in zip(held, new)))
    s["table"] = torch.randperm(n * cols, generator=g, device=DEV).to(torch.int32).reshape(n, cols)
    s["kv_len"] = torch.tensor(held, dtype=torch.int32, device=DEV)
    starts = [0]
    for t in new:
        starts.append(starts[-1] + t)
    s["start"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    s["slot"] = torch.randperm(n, generator=g, device=DEV).to(torch.int32)
    # keys after their norm: unit rows with a few strong channels; values: heads of unlike sizes
    loud = 1.0 + 7.0 * (torch.rand(hk, 1, d, generator=g, device=DEV) < 0.05)
    size = 0.05 + 2.0 * torch.rand(n * cols, hk, 1, 1, generator=g, device=DEV)
    for name, mul in (("k", loud), ("v", size)):
        x = torch.randn(n * cols, hk, b, d, generator=g, device=DEV) * mul
        sc = _pow2_scale(x.abs().amax(dim=(2, 3)))
        s[name + "_codes"] = (x / sc[:, :, None, None]).to(torch.float8_e4m3fn)
        s[name + "_scale"] = sc
        s[name + "_tail"] = (torch.randn(n, hk, b, d, generator=g, device=DEV) * (loud if name == "k" else 1.0)).half()
        del x
    rows = sum(new)
    if case["op"] == "append":
        # one projection's output: q, k and v of a token are slices of one row
        qkv = torch.randn(rows, (h + 2 * hk) * d, generator=g, device=DEV) * 1.5
        qkv = qkv.to(dt)
        s["q"], s["k"], s["v"] = (t.unflatten(1, (-1, d)) for t in qkv.split([h * d, hk * d, hk * d], dim=1))
        s["q_norm"] = s["k_norm"] = s["rotation"] = None
        if case["norm"]:
            s["q_norm"] = 1.0 + 0.1 * torch.randn(d, generator=g, device=DEV)
            s["k_norm"] = 1.0 + 0.1 * torch.randn(d, generator=g, device=DEV)
        if case["rot"]:
            r = case["rot"]
            freq = 10000.0 ** (-torch.arange(0, r, 2, device=DEV, dtype=torch.float64) / r)
            ang = torch.arange(s["max_kv"], device=DEV, dtype=torch.float64)[:, None] * freq
            s["rotation"] = torch.stack([ang.cos(), ang.sin()], dim=-1).float()
        s["q_scale"] = 1.0 + 0.2 * torch.rand(rows, generator=g, device=DEV)
    else:
        s["q"] = (torch.randn(rows, h, d, generator=g, device=DEV) * 4.0).to(dt)
        s["scale"] = 1.0 / d
        e = case["extent"]
        s["rel"] = 0.5 * torch.randn(rows, h, e, generator=g, device=DEV) if e else None
        s["tau"] = 1.0 + 0.3 * torch.rand(rows, generator=g, device=DEV)
    if own:
        from sepia_b200.kv8 import Kv8Cache, Kv8Step
        s["cache"] = Kv8Cache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"], s["k_tail"], s["v_tail"])
        s["step"] = Kv8Step(s["table"], s["kv_len"], start=s["start"], slot=s["slot"], n_tokens=s["n_tokens"],
                            max_new=s["max_new"], max_kv=s["max_kv"])
    return s


def _prepare_sample(case, g, dt):
    n, v, mode = case["rows"], case["vocab"], case["mode"]
    # a broad bulk and some tens of plausible tokens above it
    x = torch.randn(n, v, generator=g, device=DEV) * 2.0
    at = torch.randint(0, v // 64, (n, 64), generator=g, device=DEV) + v // 64 * torch.arange(64, device=DEV)
    x.scatter_(1, at, 17.0 - 9.0 * torch.rand(n, 64, generator=g, device=DEV).sqrt())
    x[:, v // 3] = -math.inf                       # a banned token
    s = dict(case=case, op="sample", logits=x.to(dt), u=torch.rand(n, generator=g, device=DEV))
    # each row its own settings; a filter is off where the mode does not use it. "mixed" goes round the modes by row
    kinds = ("temperature", "top_k", "top_p", "min_p", "all", "greedy")
    kind = torch.arange(n, device=DEV) % 6 if mode == "mixed" else torch.full((n,), kinds.index(mode), device=DEV)

    def on(name):
        return (kind == kinds.index(name)) | (kind == kinds.index("all"))
    t = 0.7 + 0.6 * torch.rand(n, generator=g, device=DEV)
    s["temperature"] = torch.where(kind == kinds.index("greedy"), 0.0, t)
    k = torch.randint(20, 200, (n,), generator=g, device=DEV, dtype=torch.int32)
    s["top_k"] = torch.where(on("top_k"), k, 0)
    p = 0.8 + 0.19 * torch.rand(n, generator=g, device=DEV)
    s["top_p"] = torch.where(on("top_p"), p, 1.0)
    m = 0.01 + 0.05 * torch.rand(n, generator=g, device=DEV)
    s["min_p"] = torch.where(on("min_p"), m, 0.0)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if s["op"] == "sample":
        if own:
            from sepia_b200.sampling import sample
            ids, prob = sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        else:
            ids, prob = _plain_sample(s)
        return {"ids": ids, "prob": prob}
    if s["op"] == "attention":
        if own:
            return s["cache"].attention(s["step"], s["q"], s["scale"], window=s["case"]["window"],
                                        rel_logits=s["rel"], tau=s["tau"])
        return _plain_attention(s)
    if own:
        q = s["cache"].append(s["step"], s["k"], s["v"], q=s["q"], k_norm=s["k_norm"], q_norm=s["q_norm"], eps=1e-6,
                              q_scale=s["q_scale"], rotation=s["rotation"], adjacent=s["case"]["adjacent"])
    else:
        q = _plain_append(s)
    return {"q": q, "k_codes": s["k_codes"], "v_codes": s["v_codes"], "k_scale": s["k_scale"],
            "v_scale": s["v_scale"], "k_tail": s["k_tail"], "v_tail": s["v_tail"]}


def _rows(s):
    """(sequence, index in the call, position) of each new token."""
    n = torch.arange(s["n_tokens"], device=DEV)
    seq = torch.searchsorted(s["start"][1:].long(), n, right=True)
    i = n - s["start"].long()[seq]
    return seq, i, s["kv_len"].long()[seq] + i


def _norm_rotate(x, w, cs, adjacent):
    x = x.float()
    if w is not None:
        x = w * (x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)))
    if cs is not None:
        r = 2 * cs.shape[1]
        cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
        y, rest = x[..., :r], x[..., r:]
        if adjacent:
            a, c = y[..., 0::2], y[..., 1::2]
            y = torch.stack([a * cos - c * sin, c * cos + a * sin], dim=-1).flatten(-2)
        else:
            a, c = y[..., : r // 2], y[..., r // 2:]
            y = torch.cat([a * cos - c * sin, c * cos + a * sin], dim=-1)
        x = torch.cat([y, rest], dim=-1)
    return x


def _plain_append(s):
    b, n, adj = s["case"]["block"], s["kv_len"].numel(), s["case"]["adjacent"]
    seq, i, pos = _rows(s)
    cs = s["rotation"][pos] if s["rotation"] is not None else None
    q = (_norm_rotate(s["q"], s["q_norm"], cs, adj) * s["q_scale"][:, None, None]).to(s["q"].dtype)
    held = s["kv_len"].long()
    total = held + (s["start"][1:] - s["start"][:-1]).long()
    b0, r0 = held // b, held % b
    touched = (s["max_new"] + b - 1) // b + 1
    at = b0[:, None] + torch.arange(touched, device=DEV)                 # blocks that the call may touch
    done = (at + 1) * b <= total[:, None]
    blocks = s["table"].long().gather(1, at.clamp(max=s["table"].shape[1] - 1))
    slot, row = s["slot"].long(), torch.arange(b, device=DEV)
    last = total // b - b0
    seqs = torch.arange(n, device=DEV)
    for name in ("k", "v"):
        x = _norm_rotate(s["k"], s["k_norm"], cs, adj) if name == "k" else s["v"].float()
        x = x.clamp(-F16_MAX, F16_MAX).half()
        tail, codes, scale = s[name + "_tail"], s[name + "_codes"], s[name + "_scale"]
        dense = x.new_zeros(n, touched * b, *x.shape[1:])
        dense[:, :b] = torch.where((row < r0[:, None])[:, :, None, None], tail[slot].transpose(1, 2), 0)
        dense[seq, pos - b0[seq] * b] = x
        dense = dense.unflatten(1, (touched, b)).transpose(2, 3)         # [seq, block, head, row, dim]
        y = dense.float()
        sc = _pow2_scale(y.abs().amax(dim=(3, 4)))
        c8 = (y / sc[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        raw = codes.view(torch.uint8)
        raw[blocks] = torch.where(done[:, :, None, None, None], c8, raw[blocks])
        scale[blocks] = torch.where(done[:, :, None], sc, scale[blocks])
        keep = (row >= (total % b)[:, None])[:, None, :, None]
        tail[slot] = torch.where(keep, tail[slot], dense[seqs, last])
    return q


def _held(s, name, first, span):
    """Positions first .. first+span-1 of every sequence as [seq, head, position, dim] in 32 bits, tails in place."""
    b, n = s["case"]["block"], s["kv_len"].numel()
    total = s["kv_len"].long() + (s["start"][1:] - s["start"][:-1]).long()
    p = first[:, None] + torch.arange(span, device=DEV)
    blk = s["table"].long().gather(1, (p // b).clamp(max=s["table"].shape[1] - 1))
    x = s[name + "_codes"][blk, :, p % b].float() * s[name + "_scale"][blk][..., None]
    t = s[name + "_tail"][s["slot"].long()[:, None].expand(n, span), :, p % b].float()
    in_tail = (p >= (total // b * b)[:, None])[:, :, None, None]
    return torch.where(in_tail, t, x).transpose(1, 2), p


def _plain_attention(s):
    c = s["case"]
    n, m, h, hk, d, w, e = (s["kv_len"].numel(), s["max_new"], c["heads"], c["kv_heads"], c["dim"], c["window"],
                            c["extent"])
    first = (s["kv_len"].long() - w + 1).clamp(min=0) if w else torch.zeros(n, dtype=torch.long, device=DEV)
    span = min(s["max_kv"], w + m) if w else s["max_kv"]
    k, p = _held(s, "k", first, span)
    at = (s["start"][:-1, None].long() + torch.arange(m, device=DEV)).clamp(max=s["n_tokens"] - 1)
    pos = s["kv_len"].long()[:, None] + torch.arange(m, device=DEV)
    q = s["q"].float()[at].unflatten(2, (hk, h // hk)).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)
    sc = (q @ k.transpose(-1, -2)) * s["scale"]                         # [seq, KV head, (head, token), position]
    del k
    sc = sc.unflatten(2, (h // hk, m))
    far = pos[:, :, None] - p[:, None]                                  # [seq, token, position]
    if e:
        near = ((far >= 0) & (far < e))[:, None].expand(n, h, m, span)
        rel = (s["rel"][at] * s["tau"][at][..., None, None]).transpose(1, 2)
        bias = rel.gather(3, far.clamp(0, e - 1)[:, None].expand(n, h, m, span))
        sc += torch.where(near, bias, 0.0).unflatten(1, (hk, h // hk))
        del bias, near
    seen = (far >= 0) & ((far < w) if w else (far >= 0))
    sc.masked_fill_(~seen[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    sc = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
    total = sc.sum(-1, keepdim=True)
    v, _ = _held(s, "v", first, span)
    o = sc.flatten(2, 3) @ v
    o = o / torch.where(total > 0, total, 1.0).flatten(2, 3)
    o = o.unflatten(2, (h // hk, m)).permute(0, 3, 1, 2, 4).flatten(2, 3)   # [seq, token, head, dim]
    seq, i, _ = _rows(s)
    return o[seq, i].to(s["q"].dtype)


def _plain_sample(s):
    x, v = s["logits"].float(), s["case"]["vocab"]
    t = s["temperature"][:, None]
    best = x.amax(1, keepdim=True)
    e = torch.exp((x - best) * (1.0 / torch.where(t > 0, t, 1.0)))
    e = torch.where(x == best, 1.0, e)
    w = torch.round(e * W_ONE).long()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    k = torch.where(s["top_k"] > 0, s["top_k"], v)[:, None]
    rank = torch.arange(v, device=DEV)[None]
    ws = torch.where(rank < k, ws, 0)
    before = ws.cumsum(1) - ws
    mass = ws.sum(1, keepdim=True)
    p = s["top_p"][:, None]
    keep = (rank < k) & ((p >= 1) | (before.double() < p.double() * mass.double()) | (rank == 0))
    keep &= e.gather(1, order) >= s["min_p"][:, None].clamp(max=1.0)
    keep &= (t > 0) | (rank == 0)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w.gather(1, order), 0))
    run_ = kept.cumsum(1)
    total = run_[:, -1:]
    target = (s["u"][:, None].double() * total.double()).floor().long().minimum(total - 1)
    ids = torch.searchsorted(run_, target, right=True)
    prob = (kept.gather(1, ids).double() / total.double()).float()
    return ids[:, 0].to(torch.int32), prob[:, 0]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 2 if case["dtype"] == "f16" else 4
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * v * size + n * 28, "flops": 4 * n * v}
    held, new = _lens(case)
    h, hk, d, b = case["heads"], case["kv_heads"], case["dim"], case["block"]
    if case["op"] == "append":
        nbytes = sum(new) * (2 * h + 2 * hk) * d * size
        for x, t in zip(held, new):
            ended = (x + t) // b - x // b
            nbytes += 2 * hk * ended * (b * d + 4)                               # codes and scales written
            nbytes += 2 * hk * d * 2 * (x % b if ended else 0)                   # tail rows of an ended block read
            nbytes += 2 * hk * d * 2 * ((x + t) % b if ended else t)             # tail rows written
            nbytes += 4 * t * case["rot"]
        return {"bytes": nbytes, "flops": sum(new) * (h + hk) * d * 8}
    nbytes, flops, w = 0, 0, case["window"]
    for x, t in zip(held, new):
        first = max(0, x - w + 1) if w else 0
        total = x + t
        coded = max(0, total // b * b - first)
        nbytes += 2 * hk * d * (coded + 2 * (total - first - coded)) + 8 * hk * (coded // b)
        nbytes += 2 * t * h * d * size
        for i in range(t):
            seen = min(x + i + 1, w) if w else x + i + 1
            flops += 4 * h * d * seen
            nbytes += 4 * h * min(case["extent"], seen)
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------ the definition in 64 bits
def _e4m3(x):
    """x (|x| <= 448, 64 bits) to the nearest e4m3 value, ties to even."""
    _, ex = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (ex - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    held, new = _lens(case)
    h, hk, d, b = case["heads"], case["kv_heads"], case["dim"], case["block"]
    if case["op"] == "append":
        return _exact_append(s, held, new, h, hk, d, b)
    out, n0 = [], 0
    for i, (x, t) in enumerate(zip(held, new)):
        total = x + t
        first = max(0, x - case["window"] + 1) if case["window"] else 0
        kv = []
        for name in ("k", "v"):
            blocks = s["table"][i, first // b:(total + b - 1) // b].long()
            y = s[name + "_codes"][blocks].double() * s[name + "_scale"][blocks].double()[:, :, None, None]
            if total % b:
                y[-1] = s[name + "_tail"][s["slot"][i].long()].double()
            y = y.transpose(0, 1).reshape(hk, -1, d)
            kv.append(y[:, first % b:first % b + total - first].repeat_interleave(h // hk, dim=0))
        for j in range(t):
            pos = x + j
            lo = max(0, pos - case["window"] + 1) if case["window"] else 0
            y = torch.einsum("hd,hpd->hp", s["q"][n0 + j].double(), kv[0][:, lo - first:pos + 1 - first]) / d
            e = min(case["extent"], pos + 1 - lo)
            if e:
                y[:, -e:] += s["rel"][n0 + j].double()[:, :e].flip(1) * s["tau"][n0 + j].double()
            out.append(torch.einsum("hp,hpd->hd", torch.softmax(y, dim=1), kv[1][:, lo - first:pos + 1 - first]))
        n0 += t
    return torch.stack(out)


def _exact_append(s, held, new, h, hk, d, b):
    pos = torch.cat([torch.arange(x, x + t, device=DEV) for x, t in zip(held, new)])
    rows = {}
    for name in ("q", "k", "v"):
        y = s[name].double()
        if name != "v" and s[name + "_norm"] is not None:
            y = y / (y.square().sum(-1, keepdim=True) / d + 1e-6).sqrt() * s[name + "_norm"].double()
        if name != "v" and s["rotation"] is not None:
            cs = s["rotation"].double()[pos]
            turn = torch.complex(cs[..., 0], cs[..., 1])[:, None]
            r = 2 * turn.shape[-1]
            z = y[..., :r].unflatten(-1, (-1, 2) if s["case"]["adjacent"] else (2, -1))
            z = z if s["case"]["adjacent"] else z.transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
            z = z if s["case"]["adjacent"] else z.transpose(-1, -2)
            y = torch.cat([z.flatten(-2), y[..., r:]], dim=-1)
        rows[name] = y
    out = {"q": rows["q"] * s["q_scale"].double()[:, None, None]}
    for name in ("k", "v"):
        codes, scale = s[name + "_codes"].double(), s[name + "_scale"].double()
        tail, n0 = s[name + "_tail"].double(), 0
        for i, (x, t) in enumerate(zip(held, new)):
            sl = int(s["slot"][i])
            y = torch.cat([tail[sl, :, :x % b], rows[name][n0:n0 + t].half().double().transpose(0, 1)], dim=1)
            n0 += t
            ended = y.shape[1] // b
            if ended:
                z = y[:, :ended * b].unflatten(1, (ended, b)).transpose(0, 1)
                sc = torch.exp2(torch.ceil(torch.log2(z.abs().amax(dim=(2, 3)) / E4M3_MAX)))
                at = s["table"][i, x // b:x // b + ended].long()
                codes[at], scale[at] = _e4m3(z / sc[:, :, None, None]), sc
            rest = y.shape[1] - ended * b
            tail[sl, :, :rest] = y[:, ended * b:]
        out.update({name + "_codes": codes, name + "_scale": scale, name + "_tail": tail})
    return out


def _exact_sample(s):
    ids, prob = [], []
    for i in range(s["case"]["rows"]):
        x = s["logits"][i].double()
        order = torch.sort(x, descending=True, stable=True).indices
        if not s["temperature"][i] > 0:
            ids.append(int(order[0]))
            prob.append(1.0)
            continue
        e = torch.exp((x[order] - x[order[0]]) / s["temperature"][i].double())
        k = int(s["top_k"][i])
        e = e[:k] if k > 0 else e
        top_p = float(s["top_p"][i])
        if top_p < 1:
            before = e.cumsum(0) - e
            e = e[(before < top_p * e.sum()) | (before == 0)]
        e = e[e >= float(s["min_p"][i])]
        kept, at = torch.sort(order[:e.numel()])
        run_ = e[at].cumsum(0)
        j = int(torch.searchsorted(run_, s["u"][i].double() * run_[-1], right=True).clamp(max=kept.numel() - 1))
        ids.append(int(kept[j]))
        prob.append(float(e[at][j] / run_[-1]))
    return {"ids": torch.tensor(ids, dtype=torch.int32), "prob": torch.tensor(prob, dtype=torch.float64)}
