"""GPU: sepia_cuda_sample up to its largest vocabulary of 2^19, where fp32 rows
no longer fit the cluster's shared memory and a CTA's sums of 16-bit halves
are as full as they can be."""
import numpy as np
import pytest
import torch

from test_gpu_sample import draw, kept64, pick_u
from test_gpu_sample_cuts import last_in, ranked

pytestmark = pytest.mark.gpu
MOST = 1 << 19


@pytest.mark.parametrize("vocab", [262147, 400003, MOST - 1, MOST])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("kw", [{}, dict(top_k=50), dict(top_p=0.9), dict(temperature=0.7, top_k=3000, top_p=0.95, min_p=0.001),
                                dict(temperature=40.0, top_p=0.5), dict(temperature=0.0)], ids=lambda kw: "-".join(kw) or "plain")
def test_large_vocabularies(lib, vocab, dtype, kw):
    rng = np.random.default_rng(vocab % 1000)
    wide = torch.tensor(rng.standard_normal((3, vocab + 5)) * 2, dtype=dtype, device="cuda")
    wide[:, rng.integers(0, vocab, 30)] += 8
    dev = wide[:, 1:vocab + 1]                       # rows off the vector boundary, each at its own place
    x = dev.float().cpu().numpy()
    u, want, prob = [], [], []
    for r in range(3):
        at, share = kept64(x[r], kw.get("temperature", 1.0), kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0))
        j, uu = pick_u(share, rng)
        u.append(uu)
        want.append(at[j])
        prob.append(share[j])
    got, p = draw(dev, u, **kw)
    assert np.array_equal(got, want)
    assert np.allclose(p, prob, rtol=4e-6, atol=2e-9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_full_counters(lib, dtype):
    """All tokens but the best in one bin, with weights whose low 16 bits are nearly all ones: 65536 of them
    in a CTA come within a hundredth of 2^32."""
    low = torch.arange(-4.0, -0.5, 2.0 ** -9, dtype=torch.float64).to(dtype)
    w = torch.round(torch.exp(low.double()) * 2.0 ** 31).long() % 65536
    best = int(torch.where(w < 65500, w, 0).argmax())   # (a few ulps of fp32 exp below the end)
    assert w[best] > 64900
    x = torch.full((4, MOST), float(low[best]), dtype=dtype)
    x[:, 12345] = 0.0
    cut, u, want, share = [], [], [], []
    for m in (2, 70001, 300000, MOST - 1):
        order, e = ranked(x[0].float().numpy(), 1.0)
        i, s, uu = last_in(order, e, m)
        cut.append((e[:m].sum() - 0.5 * e[m - 1]) / e.sum())
        u.append(uu)
        want.append(i)
        share.append(s)
    got, p = draw(x.cuda(), u, top_p=np.asarray(cut))
    # a token's share of 2e-6 is met by u and top_p of 24 bits in its inner part only up to a third of the row
    assert np.array_equal(got[:2], want[:2]) and np.all(np.abs(got - want) <= 1) and np.allclose(p, share, rtol=1e-5)
