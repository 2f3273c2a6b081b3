"""GPU: the decode engine over the 8-bit cache against the whole model in 64
bits, whose K and V are held as the cache holds them (e4m3 codes of finished
blocks, fp16 tails). So the wiring of a layer (window, band, tau, norms, the
order of append and attention) shows past the first block too, where the
distance to an fp32 cache is dominated by the rounding of K and V.

Bounds, in the logits' spread: the engine's arithmetic is fp32, and the
fp32-cache engine is within 1e-4 of the reference; half the steps have to be.
Where a code rounds the other way, one dim of a key or value moves by 1/16 of
itself: of some 50,000 codes, at 1e-6 before the rounding, one or two do, and
the worst step is allowed 1e-2. The bounds do not hold for the same model with a
mistake in its wiring (window one longer, no tau, a band moved by one)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def as_cached(rows, block):
    """[tokens, heads, dim] of fp16 values as the cache returns them."""
    out = rows.astype(np.float64)
    full = len(rows) // block * block
    if full:
        x = out[:full].reshape(-1, block, *rows.shape[1:])
        top = np.abs(x).max(axis=(1, 3), keepdims=True)
        scale = np.exp2(np.ceil(np.log2(np.where(top > 0, top, 448.0) / 448.0)))
        codes = torch.tensor(x / scale, dtype=torch.float32).to(torch.float8_e4m3fn).double().numpy()
        out[:full] = (codes * scale).reshape(out[:full].shape)
    return out


class Plain64:
    """A dense model, one token at a time."""

    def __init__(self, m, oracle, block, mistake=None):
        self.cfg, self.block, self.mistake = m.cfg, block, mistake
        self.w = {}
        for name, (t, shape, buf) in m.t.items():
            raw = buf.cpu().numpy()
            n = int(np.prod(shape))
            y = raw.view(np.float32)[:n] if t == 0 else oracle.dequantize(t, raw, n)
            self.w[name] = y.astype(np.float64).reshape([int(x) for x in shape][::-1])
        self.pos = 0
        self.hist, self.k, self.v = {}, {}, {}

    def norm(self, x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.cfg.rms_norm_eps) * w.reshape(-1)

    def conv(self, key, x, w):
        h = self.hist.setdefault(key, [np.zeros_like(x) for _ in range(self.cfg.conv_kernel_size - 1)])
        h.append(x)
        w = w.reshape(len(x), -1)
        y = x + sum(w[:, j] * h[j] for j in range(len(h)))
        h.pop(0)
        return y

    def attention(self, l, x):
        c, b = self.cfg, f"blk.{l}."
        nh, nkv, dh = c.heads(l)
        e = c.layer_rel_extent(l)
        q, k, v, r = (self.w[b + f"attn_{n}.weight"] @ x for n in "qkvr")
        k, v = (self.conv((l, n), y, self.w[b + f"shortconv_{n}.weight"]).reshape(nkv, dh) for n, y in (("k", k), ("v", v)))
        k = self.norm(k, self.w[b + "attn_k_norm.weight"])
        q = self.norm(q.reshape(nh, dh), self.w[b + "attn_q_norm.weight"])
        for store, row in ((self.k, k), (self.v, v)):
            store.setdefault(l, []).append(row.astype(np.float16))
        keys, vals = (as_cached(np.stack(s[l]), self.block) for s in (self.k, self.v))
        sliding, p, tau = c.layer_is_sliding[l], self.pos, 1.0
        if not sliding and c.log_scaling_n_floor is not None and self.mistake != "tau":
            tau = 1.0 + c.log_scaling_alpha * np.log(max(1.0, (p + 1) / c.log_scaling_n_floor))
        lo = max(0, p - c.sliding_window_size + 1 - (self.mistake == "window")) if sliding else 0
        keys, vals = (np.repeat(y[lo:], nh // nkv, axis=1) for y in (keys, vals))
        band = r.reshape(nh, -1) @ self.w[b + "attn_rel_proj.weight"].reshape(-1, e) * tau
        far = p - np.arange(lo, p + 1) + (self.mistake == "band")
        s = np.einsum("hd,jhd->hj", q * tau, keys) / dh + np.where(far < e, band[:, np.minimum(far, e - 1)], 0.0)
        s = np.exp(s - s.max(1, keepdims=True))
        return self.w[b + "attn_output.weight"] @ np.einsum("hj,jhd->hd", s / s.sum(1, keepdims=True), vals).reshape(-1)

    def step(self, token):
        w, c = self.w, self.cfg
        x = self.norm(w["token_embd.weight"][token], w["token_embd_norm.weight"])
        for l in range(c.num_hidden_layers):
            b = f"blk.{l}."
            y = self.attention(l, self.norm(x, w[b + "attn_norm.weight"]))
            x = x + self.conv((l, "attn"), y, w[b + "shortconv_attn.weight"])
            y = self.norm(x, w[b + "ffn_norm.weight"])
            g, u = w[b + "ffn_gate.weight"] @ y, w[b + "ffn_up.weight"] @ y
            y = w[b + "ffn_down.weight"] @ (g / (1.0 + np.exp(np.minimum(-g, 700.0))) * u) * float(w[b + "ffn_gscale.weight"].reshape(-1)[0])
            x = x + self.conv((l, "mlp"), y, w[b + "shortconv_mlp.weight"])
        self.pos += 1
        return w["output.weight"][: c.unpadded_vocab_size] @ (self.norm(x, w["output_norm.weight"]) / c.logits_mup_width_multiplier)


@pytest.fixture(scope="module")
def built(lib, tmp_path_factory):
    from sepia_b200 import container as CT
    from sepia_b200 import quants as Q
    tc = CT.synth_text_config(n_layers=3, n_dense=3, global_every=2, window=21, rel_extent=30)
    types = CT.ModelTypes(embed=Q.Q8_0, unembed=Q.Q6_K, attn=Q.Q4_K, dense=Q.Q5_K)
    return CT.synth_container(tmp_path_factory.mktemp("layers") / "m", tc, types=types, seed=5)


@pytest.mark.parametrize("block", [16, 32, 64])
def test_layers_past_window_and_block(built, oracle, block):
    from sepia_b200.model import DeviceModel
    m = DeviceModel.from_container(built, max_positions=160, kv_block=block)
    ids = np.random.default_rng(block).integers(0, m.cfg.unpadded_vocab_size, 150).astype(np.int32)
    dev = torch.as_tensor(ids, device="cuda")
    m.reset()
    models = {name: Plain64(m, oracle, block, name) for name in (None, "window", "tau", "band")}
    err = {name: [] for name in models}
    for i, token in enumerate(ids):
        m.prefill(dev[i:i + 1], True)
        got = m.logits().double().cpu().numpy()
        for name, plain in models.items():
            want = plain.step(int(token))
            err[name].append(np.abs(got - want).max() / (want.max() - want.min()))
    def holds(e):
        return np.median(e[70:]) <= 1e-4 and max(e) <= 1e-2
    assert holds(err[None]), (np.median(err[None][70:]), max(err[None]))
    for name in ("window", "tau", "band"):            # the bounds see these
        assert not holds(err[name]), name
