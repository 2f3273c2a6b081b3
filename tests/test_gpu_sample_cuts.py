"""GPU: sepia_cuda_sample at its cuts. A cut is worked out in several passes
(bins, their parts, lists) that have to agree on every token's place; a cut
that is off by one token shows here: the last token in is drawn by a u in the
middle of its interval, and its share is that of a set of exactly this size.

The cuts are put where the definition leaves no doubt: top-k is a count, and
top_p lies in the middle of the last token's mass. A share of 1e-5 moves by a
set's further token by as much as that token's share, far above the 4e-6 that
fp32 exponentials and their rounding leave (test_gpu_sample.py); tokens of
less than 3e-6 are passed over."""
import numpy as np
import pytest
import torch

from test_gpu_sample import draw

pytestmark = pytest.mark.gpu


def ranked(x, t):
    """Token order, and in it the weights relative to the best in 64 bits."""
    x = x.astype(np.float64)
    order = np.lexsort((np.arange(len(x)), -x))
    return order, np.exp((x[order] - x[order[0]]) / np.float64(np.float32(t)))


def last_in(order, e, m):
    """(id of the m-th token, its share, a u inside its interval) of the set of the first m."""
    share = e[:m] / e[:m].sum()
    before = share[order[:m] < order[m - 1]].sum()
    return int(order[m - 1]), share[m - 1], before + 0.5 * share[m - 1]


@pytest.mark.parametrize("vocab,t,spread", [(1000, 1.0, 2.0), (50021, 0.8, 3.0), (200058, 1.0, 2.0), (200058, 40.0, 2.0),
                                            (131072, 3.0, 1.0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("base", [0.0, 3000.0])
def test_the_last_token_in(lib, vocab, t, spread, dtype, base):
    rng = np.random.default_rng(vocab + int(t))
    n = 24
    dev = torch.tensor(rng.standard_normal((n, vocab)) * spread + base, dtype=dtype, device="cuda")
    x = dev.float().cpu().numpy()
    for by in ("top_k", "top_p"):
        cut, u, want, share = [], [], [], []
        for r in range(n):
            order, e = ranked(x[r], t)
            total, most = e.sum(), vocab - 1
            while True:
                m = int(np.exp(rng.uniform(0, np.log(most))))
                i, s, uu = last_in(order, e, m)
                if s > 3e-6 and (by == "top_k" or e[m - 1] / total > 3e-6):
                    break
                most = max(2, m)
            cut.append(m if by == "top_k" else (e[:m].sum() - 0.5 * e[m - 1]) / total)
            u.append(uu)
            want.append(i)
            share.append(s)
        got, p = draw(dev, u, temperature=t, **{by: np.asarray(cut)})
        assert np.array_equal(got, want), (by, np.flatnonzero(got != want), cut)
        assert np.allclose(p, share, rtol=4e-6, atol=2e-9), (by, np.max(np.abs(p / share - 1)))
