"""GPU: the paged 8-bit K/V cache (sepia_cuda_kv8_append, sepia_cuda_kv8_attn)
against plain implementations in 64 bits.

Tolerances, from the formats:
  tails     fp16: half a unit in the last place, 2^-11 relative (2^-25 below
            the normal numbers), and 2e-6 relative for the fp32 arithmetic
            before it (a norm, a rotation: some ten roundings of 2^-24)
  codes     e4m3: 2^-4 relative, or 2^-10 of the scale in its subnormal
            range, on top of the tail's
  attention a score's error is at most head_dim * 2^-24 * sum |q k| * scale
            (an fp32 sum of exact products); the output moves by at most
            twice that, and by 2^-19 for exponentials and sums, times the
            largest |v|; fp16 in and out: 2^-10 of it more (the weights and
            the result have 11 bits)"""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16


def norm_rotate64(x, w, table, pos, adjacent, eps):
    """x [n, heads, dim] in 64 bits, or fp32/fp16 values of it."""
    y = np.asarray(x, np.float64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * np.asarray(w, np.float64)
    if table is not None:
        cs = np.asarray(table, np.float64)[pos]                # [n, rot/2, 2]
        r, out = 2 * cs.shape[1], y.copy()
        a_at = np.arange(0, r, 2) if adjacent else np.arange(r // 2)
        b_at = a_at + (1 if adjacent else r // 2)
        c, s = cs[:, None, :, 0], cs[:, None, :, 1]
        out[..., a_at] = y[..., a_at] * c - y[..., b_at] * s
        out[..., b_at] = y[..., b_at] * c + y[..., a_at] * s
        y = out
    return y


class Batch:
    """A cache and its sequences, with the true rows of every sequence in 64 bits."""

    def __init__(self, held, hk, dim, block, extra_blocks=3, fill=0x7F, seed=0, room=0):
        from sepia_b200.kv8 import Kv8Cache
        self.rng = np.random.default_rng(seed)
        self.hk, self.dim, self.block, self.n = hk, dim, block, len(held)
        self.cols = max(8, (max(held) if held else 0) // block + 8, room // block + 2)
        nb = self.n * self.cols + extra_blocks
        self.cache = Kv8Cache.allocate(nb, self.n + 2, hk, dim, block)
        # whatever is not written is NaN: it must never reach a result
        for t in (self.cache.k, self.cache.v):
            t.view(torch.uint8).fill_(fill)
        for t in (self.cache.k_scale, self.cache.v_scale, self.cache.k_tail, self.cache.v_tail):
            t.fill_(float("nan"))
        perm = self.rng.permutation(nb)[: self.n * self.cols]
        self.table = torch.tensor(perm.reshape(self.n, self.cols), dtype=torch.int32, device="cuda")
        self.slot = torch.tensor(self.rng.permutation(self.n + 2)[: self.n], dtype=torch.int32, device="cuda")
        self.kv_len = torch.zeros(self.n, dtype=torch.int32, device="cuda")
        self.rows = [[np.zeros((0, hk, dim)), np.zeros((0, hk, dim))] for _ in range(self.n)]
        if held and max(held):
            self.append(held)

    def step(self, new, **kw):
        from sepia_b200.kv8 import Kv8Step
        start = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
        return Kv8Step(self.table, self.kv_len, start=start, slot=self.slot, n_tokens=int(sum(new)),
                       max_new=max(max(new), 1), **kw)

    def append(self, new, dtype=F32, k_mul=1.0, v_mul=1.0, advance=True, k=None, v=None, **kw):
        n = sum(new)
        if k is None:
            k = torch.tensor(self.rng.standard_normal((n, self.hk, self.dim)) * k_mul, dtype=dtype, device="cuda")
            v = torch.tensor(self.rng.standard_normal((n, self.hk, self.dim)) * v_mul, dtype=dtype, device="cuda")
        q = self.cache.append(self.step(new), k, v, **kw)
        table = kw["rotation"].cpu().numpy() if kw.get("rotation") is not None else None
        w = kw["k_norm"].cpu().numpy() if kw.get("k_norm") is not None else None
        held = self.kv_len.tolist()
        if advance:
            n0 = 0
            for s, t in enumerate(new):
                pos = held[s] + np.arange(t)
                kk = norm_rotate64(k[n0:n0 + t].cpu().double().numpy(), w, table, pos, kw.get("adjacent", False),
                                   kw.get("eps", 1e-6))
                self.rows[s][0] = np.concatenate([self.rows[s][0], kk])
                self.rows[s][1] = np.concatenate([self.rows[s][1], v[n0:n0 + t].cpu().double().numpy()])
                n0 += t
            self.kv_len += torch.tensor(new, dtype=torch.int32, device="cuda")
        return q

    def held(self, s, which):
        """What the cache holds of sequence s, [tokens, hk, dim] in 64 bits, and the scale of each token and head."""
        n, b = int(self.kv_len[s]), self.block
        codes, scale, tail = [(self.cache.k, self.cache.k_scale, self.cache.k_tail),
                              (self.cache.v, self.cache.v_scale, self.cache.v_tail)][which]
        ids = self.table[s, : n // b].long()
        sc = scale[ids].double()
        x = (codes[ids].double() * sc[:, :, None, None]).transpose(1, 2).reshape(-1, self.hk, self.dim)
        t = tail[self.slot[s].long(), :, : n % b].double().transpose(0, 1)
        return (torch.cat([x, t]).cpu().numpy(), sc.repeat_interleave(b, dim=0).cpu().numpy())


def check_rows(B):
    for s in range(B.n):
        for which in (0, 1):
            got, scale = B.held(s, which)
            want = np.clip(B.rows[s][which], -65504, 65504)
            full = len(scale)
            tol = np.abs(want) * (2.0 ** -11 + 2e-6) + 2.0 ** -24
            code = np.maximum(np.abs(want[:full]) * 2.0 ** -4, scale[:, :, None] * 2.0 ** -10) * 1.002
            tol[:full] += code
            assert got.shape == want.shape and np.all(np.abs(got - want) <= tol), (s, which)
            # the scale: a power of two, the smallest that holds the block's largest magnitude
            if full:
                assert np.all(np.frexp(scale)[0] == 0.5)
                top = np.abs(want[:full]).reshape(-1, B.block, B.hk, B.dim).max(axis=(1, 3)) / scale[:: B.block]
                assert np.all((top <= 448 * 1.001) & (top > 224 * 0.999))


@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("dim,hk", [(128, 2), (16, 1), (48, 3), (96, 2)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_append_rows(lib, block, dim, hk, dtype):
    """Ragged steps: from one token to several blocks, ends on and off a block."""
    B = Batch([0, 0, 0, 0], hk, dim, block)
    for new in ([1, 0, block, 2 * block + 1], [block - 1, 3, 1, 1], [1, 5 * block, 0, block - 2], [2, 1, 1, 1]):
        B.append(new, dtype=dtype, k_mul=3.0, v_mul=0.01)
    check_rows(B)


@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("dim,rot", [(128, 128), (64, 32), (96, 8), (16, 16)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_append_norm_rotation_queries(lib, adjacent, dim, rot, dtype):
    from sepia_b200.kv8 import rotation_table
    rng = np.random.default_rng(dim + rot)
    hk, h = 2, 6
    B = Batch([0, 0, 0], hk, dim, 16, seed=5)
    table = rotation_table(200, rot)
    kn = torch.tensor(1 + 0.2 * rng.standard_normal(dim), dtype=F32, device="cuda")
    qn = torch.tensor(1 + 0.2 * rng.standard_normal(dim), dtype=F32, device="cuda")
    for new in ([7, 0, 33], [1, 1, 1], [20, 50, 15]):
        n = sum(new)
        # q, k and v as slices of one row: strides longer than a token
        qkv = torch.tensor(rng.standard_normal((n, (h + 2 * hk) * dim + 8)) * 2, dtype=dtype, device="cuda")
        q, k, v, _ = (t.unflatten(1, (-1, dim)) if t.shape[1] % dim == 0 and t.shape[1] >= dim else t
                      for t in qkv.split([h * dim, hk * dim, hk * dim, 8], dim=1))
        tau = torch.tensor(1 + rng.random(n), dtype=F32, device="cuda")
        held = B.kv_len.tolist()
        pos = np.concatenate([held[s] + np.arange(t) for s, t in enumerate(new)])
        got = B.append(new, k=k, v=v, q=q, k_norm=kn, q_norm=qn, eps=1e-5, q_scale=tau, rotation=table,
                       adjacent=adjacent)
        want = norm_rotate64(q.cpu().double().numpy(), qn.cpu().numpy(), table.cpu().numpy(), pos, adjacent, 1e-5)
        want = want * tau.cpu().double().numpy()[:, None, None]
        # a rotation adds two products: 2e-6 of the pair's length, at most sqrt(2) of the row's largest
        top = np.abs(want).max(-1, keepdims=True)
        tol = 4e-6 * top + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if dtype == F16 else 0)
        assert np.all(np.abs(got.cpu().double().numpy() - want) <= tol)
    for s in range(B.n):          # rotated keys: the same allowance on top of the formats'
        got, scale = B.held(s, 0)
        want = B.rows[s][0]
        full = len(scale)
        tol = np.abs(want) * 2.0 ** -11 + 2.0 ** -24 + 4e-6 * np.abs(want).max(-1, keepdims=True)
        tol[:full] += np.maximum(np.abs(want[:full]) * 2.0 ** -4, scale[:, :, None] * 2.0 ** -10) * 1.01
        assert np.all(np.abs(got - want) <= tol)


def test_append_content_does_not_depend_on_the_calls(lib):
    """One token at a time, in pieces and at once give the same bytes."""
    rng = np.random.default_rng(3)
    hk, dim, b, n = 2, 64, 32, 117
    k = torch.tensor(rng.standard_normal((n, hk, dim)), dtype=F32, device="cuda")
    v = torch.tensor(rng.standard_normal((n, hk, dim)), dtype=F32, device="cuda")
    seen = []
    for cuts in ([n], [1] * n, [31, 1, 2, 40, 22, 21], [33, 65, 19]):
        B = Batch([0], hk, dim, b, seed=9)
        at = 0
        for t in cuts:
            B.append([t], k=k[at:at + t], v=v[at:at + t])
            at += t
        ids = B.table[0, : n // b].long()
        sl = B.slot[0].long()
        c = B.cache
        seen.append([c.k.view(torch.uint8)[ids], c.v.view(torch.uint8)[ids], c.k_scale[ids], c.v_scale[ids],
                     c.k_tail[sl, :, : n % b], c.v_tail[sl, :, : n % b]])
    for other in seen[1:]:
        assert all(torch.equal(a, x) for a, x in zip(seen[0], other))


def test_append_extreme_values(lib):
    """Zeros, subnormal fp16, values beyond fp16 (saturated) and NaN (kept, its neighbours untouched)."""
    B = Batch([0], 1, 16, 16)
    k = torch.zeros(16, 1, 16, device="cuda")
    v = torch.randn(16, 1, 16, device="cuda") * 1e-7
    B.append([16], k=k, v=v)
    assert B.cache.k_scale[B.table[0, 0].long(), 0] == 1 and torch.all(B.cache.k.view(torch.uint8)[B.table[0, 0].long()] == 0)
    got, scale = B.held(0, 1)
    assert np.all(np.abs(got - B.rows[0][1]) <= 2.0 ** -25 + np.abs(B.rows[0][1]) * 2.0 ** -4 + scale[:, :, None] * 2.0 ** -10)
    k = torch.full((16, 1, 16), 1e9, device="cuda")
    k[3, 0, 2], k[5, 0, 1], k[6, 0, 1] = -float("inf"), float("nan"), 1.0
    B.append([16], k=k, v=v)
    got, _ = B.held(0, 0)
    x = got[16:, 0]
    assert np.isnan(x[5, 1]) and np.isnan(x).sum() == 1
    assert x[3, 2] == -65536 and x[0, 0] == 65536        # 65504 to the nearest e4m3 multiple of 2^8
    assert x[6, 1] == 1.0


# ------------------------------------------------------------------ attention
def attention64(B, q, held, new, scale, window, rel, tau):
    """Reference and the bound's ingredients per (token, head): out, max sum |q k|, max |v|."""
    q = q.cpu().double().numpy()
    h = q.shape[1]
    out, top, vmax, n = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape[:2]), 0
    for s, t in enumerate(new):
        keys, vals = (np.repeat(B.held(s, w)[0], h // B.hk, axis=1) for w in (0, 1))
        for i in range(t):
            p = held[s] + i
            lo = max(0, p - window + 1) if window else 0
            kk, vv = keys[lo:p + 1], vals[lo:p + 1]
            sc = np.einsum("hd,jhd->hj", q[n], kk) * scale
            top[n] = np.einsum("hd,jhd->hj", np.abs(q[n]), np.abs(kk)).max(1)
            if rel is not None:
                e = min(rel.shape[2], p + 1 - lo)
                sc[:, len(kk) - e:] += rel[n, :, :e].double().cpu().numpy()[:, ::-1] * (float(tau[n]) if tau is not None else 1.0)
            m = sc.max(1, keepdims=True)
            w = np.exp(sc - np.where(np.isfinite(m), m, 0))
            z = w.sum(1, keepdims=True)
            w = np.where(z > 0, w / np.where(z > 0, z, 1), 0)
            out[n] = np.einsum("hj,jhd->hd", w, vv)
            vmax[n] = np.abs(vv).max(axis=(0, 2))
            n += 1
    return out, top, vmax


def check_attention(B, new, h, dtype=F32, window=0, extent=0, with_tau=True, q_mul=2.0, rel=None, stream=None, **kw):
    rng = B.rng
    n = sum(new)
    held = B.kv_len.tolist()
    B.append(new, **kw)
    q = torch.tensor(rng.standard_normal((n, h, B.dim)) * q_mul, dtype=dtype, device="cuda")
    scale = 1.0 / B.dim
    if extent and rel is None:
        rel = torch.tensor(rng.standard_normal((n, h, extent)), dtype=F32, device="cuda")
    tau = torch.tensor(1 + rng.random(n), dtype=F32, device="cuda") if with_tau and rel is not None else None
    B.kv_len -= torch.tensor(new, dtype=torch.int32, device="cuda")
    step = B.step(new)
    outs = [B.cache.attention(step, q, scale, window=window, rel_logits=rel, tau=tau) for _ in range(2)]
    B.kv_len += torch.tensor(new, dtype=torch.int32, device="cuda")
    assert torch.equal(outs[0], outs[1])                 # no order of work changes the result
    want, top, vmax = attention64(B, q, held, new, np.float64(np.float32(scale)), window, rel, tau)
    tol = (2 * B.dim * 2.0 ** -24 * top * scale + 2.0 ** -19 + (2.0 ** -10 if dtype == F16 else 0)) * vmax
    err = np.abs(outs[0].cpu().double().numpy() - want)
    assert np.all(err <= tol[:, :, None]), float((err / (tol[:, :, None] + 1e-300)).max())
    return outs[0]


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("hk,group,dim", [(2, 8, 128), (1, 1, 64), (3, 6, 96), (2, 16, 128), (1, 5, 16), (2, 24, 48)])
def test_attention_lengths(lib, dtype, block, hk, group, dim):
    """One new token; held: none, one, up to the end of a block, one over, several blocks."""
    held = [0, 1, block - 1, block, block + 1, 5 * block - 2, 333]
    check_attention(Batch(held, hk, dim, block), [1] * len(held), hk * group, dtype, extent=20)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("new", [[2, 2, 2], [3, 0, 1], [8, 7, 1], [17, 33, 5], [70, 1, 64]])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_attention_several_new_tokens(lib, dtype, new, dim):
    check_attention(Batch([40, 130, 0], 2, dim, 16), new, 6, dtype, extent=9)


@pytest.mark.parametrize("window", [1, 7, 16, 64, 100, 5000])
@pytest.mark.parametrize("extent", [0, 1, 50, 300])
def test_attention_window_and_band(lib, window, extent):
    check_attention(Batch([0, 20, 64, 700], 2, 128, 32), [3, 1, 2, 3], 16, window=window, extent=extent)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_attention_long_context(lib, dtype):
    """The split over a long context, ragged beside a short one; loud scores."""
    check_attention(Batch([20011, 33], 2, 128, 32, seed=2), [1, 1], 16, dtype, extent=256, q_mul=30.0, k_mul=3.0)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_attention_blocks_of_unlike_sizes(lib, dtype):
    """Values of a million times one block's size in the next, keys likewise small."""
    B = Batch([0], 1, 64, 16, seed=4)
    for mul in (1e-4, 1.0, 30.0, 1e-3, 1e-5):
        B.append([16], k_mul=0.3 / max(mul, 0.05), v_mul=mul)
    check_attention(B, [5], 4, dtype, v_mul=1e-4)


def test_attention_rows_that_masks_leave_empty(lib):
    """Bands of -infinity over everything a token sees: zeros; of the type's
    lowest value: the plain mean; one row's mask does not touch another's."""
    hk, h, dim = 1, 4, 32
    B = Batch([40, 40], hk, dim, 16)
    rel = torch.zeros(2, h, 64, device="cuda")
    rel[0, 1] = -float("inf")
    rel[0, 2, 5:] = -float("inf")
    rel[1, 0] = torch.finfo(F32).min
    out = check_attention(B, [1, 1], h, rel=rel, with_tau=False)
    assert torch.all(out[0, 1] == 0)
    vals = B.held(1, 1)[0][:, 0]
    assert np.allclose(out[1, 0].cpu().numpy(), vals.mean(0), atol=1e-5)


def test_idle_sequences(lib):
    """kv_len < 0: nothing appended, zeros out, the others as ever; `start` left out."""
    from sepia_b200.kv8 import Kv8Step
    B = Batch([20, 33, 5], 2, 64, 16)
    k = torch.randn(3, 2, 64, device="cuda")
    v = torch.randn(3, 2, 64, device="cuda")
    lens = B.kv_len.clone()
    lens[1] = -1
    before = B.cache.k_tail[B.slot[1].long()].clone()
    step = Kv8Step(B.table, lens, slot=B.slot)
    q = B.cache.append(step, k, v, q=torch.randn(3, 4, 64, device="cuda"))
    out = B.cache.attention(step, q, 0.125)
    assert torch.equal(B.cache.k_tail[B.slot[1].long()].view(torch.int16), before.view(torch.int16))
    assert torch.all(out[1] == 0) and torch.all(out[0] != 0) and torch.isfinite(out).all()
    assert lib.sepia_cuda_device_error(None) == 0


@pytest.mark.parametrize("bad", ["block", "slot", "start", "max_kv", "rotation"])
def test_device_bounds(lib, bad):
    """What only the device can see sets the error word, and touches nothing."""
    from sepia_b200.kv8 import Kv8Step, rotation_table
    B = Batch([31, 40], 1, 16, 16)
    torch.cuda.synchronize()
    lib.sepia_cuda_device_error(None)
    table, slot, start, kw, ap = B.table.clone(), B.slot.clone(), [0, 1, 2], {}, {}
    if bad == "block":
        table[0, 1] = B.cache.struct.n_blocks
    elif bad == "slot":
        slot[0] = -1
    elif bad == "start":
        start = [0, -1, 2]
    elif bad == "max_kv":
        kw["max_kv"] = 31
    else:
        ap["rotation"] = rotation_table(31, 8)
    step = Kv8Step(table, B.kv_len, start=torch.tensor(start, dtype=torch.int32, device="cuda"), slot=slot, n_tokens=2,
                   max_new=1, **kw)
    q = B.cache.append(step, torch.randn(2, 1, 16, device="cuda"), torch.randn(2, 1, 16, device="cuda"),
                       q=torch.randn(2, 2, 16, device="cuda"), **ap)
    assert lib.sepia_cuda_device_error(None) == 2
    if bad != "rotation":
        B.cache.attention(step, q, 1.0)
        assert lib.sepia_cuda_device_error(None) == 2
    assert lib.sepia_cuda_device_error(None) == 0


def test_a_block_out_of_range_is_not_seen(lib):
    """Positions 16-31 lie in no block: what is left is the sequence of 16. The same keys in the same places, so the
    same sums."""
    from sepia_b200.kv8 import Kv8Step
    B = Batch([31], 2, 64, 16)
    q = torch.randn(1, 4, 64, device="cuda")
    table = B.table.clone()
    table[0, 1] = -1
    kv_len = torch.tensor([15], dtype=torch.int32, device="cuda")
    want = B.cache.attention(Kv8Step(B.table, kv_len, slot=B.slot), q, 0.125)
    torch.cuda.synchronize()
    lib.sepia_cuda_device_error(None)
    got = B.cache.attention(Kv8Step(table, B.kv_len, slot=B.slot), q, 0.125)
    assert lib.sepia_cuda_device_error(None) == 2
    assert torch.allclose(got, want, rtol=0, atol=1e-6) and want.abs().max() > 0.01


def test_offsets_past_32_bits(lib):
    """A pool of more than 2^32 codes; the sequence lives in its last blocks."""
    from sepia_b200.kv8 import Kv8Cache
    B = Batch([0], 8, 128, 64, seed=1)
    nb = (1 << 32) // (8 * 64 * 128) + 40
    B.cache = Kv8Cache.allocate(nb, 3, 8, 128, 64)
    B.table = torch.arange(nb - 1, nb - 1 - B.cols, -1, dtype=torch.int32, device="cuda").reshape(1, -1)
    check_attention(B, [150], 16)
    check_rows(B)


def test_on_another_stream(lib):
    B = Batch([100, 7], 2, 64, 16)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        check_attention(B, [2, 1], 4, extent=5)
        check_rows(B)


def test_results_belong_to_their_stream(lib):
    """Memory that a call takes for another stream is not handed to this one when it is freed."""
    B = Batch([100, 7], 2, 64, 16)
    step = B.step([1, 1])
    k, v, q = (torch.ones(2, heads, 64, device="cuda") for heads in (2, 2, 4))
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    turned = B.cache.append(step, k, v, q, stream=st)
    out = B.cache.attention(step, q, 0.125, stream=st)
    st.synchronize()
    theirs = {turned.data_ptr(), out.data_ptr()} | {ws[0] for ws in step._ws.values()}
    assert len(theirs) == 3
    del turned, out, step
    mine = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in (2048, 2048, 16, 4096) for _ in range(64)]
    assert not theirs & {t.data_ptr() for t in mine}


def test_graph_replay(lib):
    """A captured step is replayed as the lengths on the device change."""
    hk, h, dim, b = 2, 8, 64, 16
    B = Batch([30, 3], hk, dim, b)
    k, v = (torch.empty(2, hk, dim, device="cuda") for _ in range(2))
    q = torch.empty(2, h, dim, device="cuda")
    out = torch.empty(2, h, dim, device="cuda")
    step = B.step([1, 1])
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    # a first eager call outside the capture sizes the workspace; it writes row kv_len, which the replay rewrites
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        for t in (k, v, q):
            t.normal_()
        B.cache.append(step, k, v)
        B.cache.attention(step, q, 1.0 / dim, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        B.cache.append(step, k, v)
        B.cache.attention(step, q, 1.0 / dim, out=out)
        B.kv_len.add_(one)
    for _ in range(40):
        for t in (k, v, q):
            t.normal_()
        held = B.kv_len.tolist()
        g.replay()
        torch.cuda.synchronize()
        for s in range(2):
            B.rows[s][0] = np.concatenate([B.rows[s][0], k[s:s + 1].cpu().double().numpy()])
            B.rows[s][1] = np.concatenate([B.rows[s][1], v[s:s + 1].cpu().double().numpy()])
        want, top, vmax = attention64(B, q, held, [1, 1], np.float64(np.float32(1.0 / dim)), 0, None, None)
        tol = (2 * dim * 2.0 ** -24 * top / dim + 2.0 ** -19) * vmax
        assert np.all(np.abs(out.cpu().double().numpy() - want) <= tol[:, :, None])
    check_rows(B)


def test_refusals(lib):
    from sepia_b200 import lib as L
    from sepia_b200.kv8 import Kv8Cache, Kv8Step
    c = Kv8Cache.allocate(4, 2, 2, 32, 16)
    step = Kv8Step(torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"))
    k = torch.zeros(1, 2, 32, device="cuda")
    q = torch.zeros(1, 4, 32, device="cuda")
    with pytest.raises(RuntimeError, match="block of 24"):
        Kv8Cache.allocate(4, 2, 2, 32, 24).append(step, k, k)
    with pytest.raises(RuntimeError, match="head_dim 40"):
        Kv8Cache.allocate(4, 2, 2, 40, 16).append(step, torch.zeros(1, 2, 40, device="cuda"),
                                                  torch.zeros(1, 2, 40, device="cuda"))
    with pytest.raises(RuntimeError, match="rot_dim 12"):
        c.append(step, k, k, rotation=torch.zeros(5, 6, 2, device="cuda"))
    with pytest.raises(RuntimeError, match="query heads"):
        c.attention(step, torch.zeros(1, 3, 32, device="cuda"), 1.0)
    with pytest.raises(RuntimeError, match="negative window"):
        c.attention(step, q, 1.0, window=-1)
    with pytest.raises(ValueError, match="shape"):
        c.append(step, torch.zeros(2, 2, 32, device="cuda"), k)
    with pytest.raises(ValueError, match="side by side"):
        c.append(step, torch.zeros(1, 2, 64, device="cuda")[:, :, ::2], k)
    with pytest.raises(ValueError, match="one type"):
        c.append(step, k, k.half())
    with pytest.raises(ValueError, match="int32"):
        Kv8Step(torch.zeros(1, 2, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"))
    # the C entries: null pointers, a workspace that is missing or short, strides
    a = L.SepiaKv8Attn()
    a.n_heads, a.q, a.q_stride, a.out = 4, q.data_ptr(), 128, q.data_ptr()
    ref = C.byref(a)
    cs, bs = C.byref(c.struct), step._for(c)
    assert lib.sepia_cuda_kv8_attn(cs, bs, ref, None, 0, None) == 0 and b"workspace" in lib.sepia_cuda_last_error()
    assert lib.sepia_cuda_kv8_attn(cs, bs, None, None, 0, None) == 0
    assert lib.sepia_cuda_kv8_attn(None, bs, ref, None, 0, None) == 0
    assert lib.sepia_cuda_kv8_attn_ws_bytes(cs, bs, None) == 0
    a.q_stride = 127
    assert lib.sepia_cuda_kv8_attn(cs, bs, ref, q.data_ptr(), 1 << 20, None) == 0
    p = L.SepiaKv8Append()
    assert lib.sepia_cuda_kv8_append(cs, bs, C.byref(p), None) == 0
    assert lib.sepia_cuda_kv8_append(cs, bs, None, None) == 0
    assert lib.sepia_cuda_device_error(None) == 0


def test_no_tokens(lib):
    from sepia_b200.kv8 import Kv8Cache, Kv8Step
    c = Kv8Cache.allocate(4, 2, 2, 32, 16)
    step = Kv8Step(torch.zeros(0, 2, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"))
    k = torch.zeros(0, 2, 32, device="cuda")
    q = c.append(step, k, k, q=torch.zeros(0, 4, 32, device="cuda"))
    assert c.attention(step, q, 1.0).shape == (0, 4, 32)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("held,window", [(53, 20), (41, 0)])
def test_attention_not_numbers_behind_a_mask(lib, dtype, held, window):
    """Keys and values that are NaN at positions that a token does not see
    (behind its window, or later new tokens) leave its output as it is; a
    token that sees one gets NaN."""
    hk, h, dim, new = 2, 6, 64, 4
    outs = []
    for spoil in (False, True):
        B = Batch([0], hk, dim, 16, seed=6)
        rng = np.random.default_rng(8)
        k = torch.tensor(rng.standard_normal((held + new, hk, dim)), dtype=F32, device="cuda")
        v = torch.tensor(rng.standard_normal((held + new, hk, dim)), dtype=F32, device="cuda")
        if spoil:
            v[held + new - 1, 1, 7] = k[held + new - 1, 0, 3] = float("nan")      # the last new token: seen by itself only
            if window:
                v[held + new - 1 - window - 3, 0, 5] = float("nan")              # behind every window, in a tile that is read
                k[held + new - 1 - window - 3, 1, 2] = float("nan")
        B.append([held], k=k[:held], v=v[:held])
        step = B.step([new])
        q = torch.tensor(rng.standard_normal((new, h, dim)), dtype=dtype, device="cuda")
        B.cache.append(step, k[held:].contiguous(), v[held:].contiguous())
        outs.append(B.cache.attention(step, q, 1.0 / dim, window=window))
    assert torch.equal(outs[0][: new - 1], outs[1][: new - 1])
    assert torch.isnan(outs[1][new - 1]).view(hk, -1).any(dim=1).all()


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("held", [3000, 3001, 3017])
def test_attention_a_sink_and_a_faint_rest(lib, dtype, held):
    """One key far above all others, which together still weigh something:
    thousands of weights of 2^-20 of the largest, values of unlike size beside
    an unscaled tail."""
    B = Batch([0], 1, 64, 32, seed=11, room=held + 1)
    rng = np.random.default_rng(12)
    k = rng.standard_normal((held, 1, 64)) * 0.05
    v = 0.01 + 0.002 * rng.standard_normal((held, 1, 64))
    direction = rng.standard_normal(64)
    k[5, 0] = 8.0 * direction / np.linalg.norm(direction)
    v[5] = 0.0
    v[32:64] *= 40.0
    B.append([held], k=torch.tensor(k, dtype=F32, device="cuda"), v=torch.tensor(v, dtype=F32, device="cuda"))
    rows = [torch.tensor(direction / np.linalg.norm(direction) * g, dtype=F32) for g in (60.0, 100.0, 110.0, 0.0)]
    q = torch.stack(rows)[None].to(dtype).cuda()
    kn, vn = torch.zeros(1, 1, 64, device="cuda"), torch.full((1, 1, 64), 0.01, device="cuda")
    step = B.step([1])
    B.cache.append(step, kn, vn)
    out = B.cache.attention(step, q, 1.0 / 64)
    B.kv_len += 1
    want, top, vmax = attention64(B, q, [held], [1], np.float64(np.float32(1.0 / 64)), 0, None, None)
    # every output is a share of faint weights: relative to itself, a score's error and the formats'
    # (fp16: weights of 11 bits, rounded both ways, and the result's 2^-11)
    tol = (2 * 64 * 2.0 ** -24 * top / 64 + 2.0 ** -13 * (1 if dtype == F32 else 8))[:, :, None] * np.abs(want) + 1e-12
    err = np.abs(out.cpu().double().numpy() - want)
    assert np.all(err <= tol + (2.0 ** -24 if dtype == F16 else 0)), float((err / tol).max())
