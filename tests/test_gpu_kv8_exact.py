"""GPU: the attention over the paged 8-bit cache where the coarse bounds of
test_gpu_kv8.py would not see a loss: results in half precision are the exact
ones rounded once.

Tolerance: half the spacing of fp16 at the result, and what the fp32 path has
(test_gpu_kv8.py: an fp32 sum's error of each score, twice, and 2^-19 for
exponentials and sums, times the largest |v|). Scores are small here, so the
second part is a hundredth of the first; weights of 11 bits would move one
result in five by more than both."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import F16, Batch, attention64

pytestmark = pytest.mark.gpu


def half_spacing(x):
    """Half the distance of fp16 numbers around x."""
    _, e = np.frexp(np.abs(x))
    return np.ldexp(0.5, np.maximum(e - 1, -14) - 10)


@pytest.mark.parametrize("block,hk,group,dim,new", [(16, 2, 8, 128, 1), (32, 1, 5, 64, 1), (64, 3, 6, 96, 1), (16, 2, 3, 16, 5),
                                                    (32, 2, 8, 128, 9), (16, 1, 24, 48, 4)])
def test_half_results_are_rounded_once(lib, block, hk, group, dim, new):
    held = [0, 3, block, 5 * block - 2, 333]
    B = Batch(held, hk, dim, block, seed=dim + new)
    news, h = [new] * len(held), hk * group
    B.append(news, advance=False)
    q = torch.tensor(B.rng.standard_normal((new * len(held), h, dim)) * 0.1, dtype=F16, device="cuda")
    out = B.cache.attention(B.step(news), q, 1.0 / dim)
    B.kv_len += new
    want, top, vmax = attention64(B, q, held, news, np.float64(np.float32(1.0 / dim)), 0, None, None)
    tol = half_spacing(want) + ((2 * dim * 2.0 ** -24 * top / dim + 2.0 ** -19) * vmax)[:, :, None]
    err = np.abs(out.cpu().double().numpy() - want)
    assert np.all(err <= tol), (float((err / tol).max()), float((err > tol).mean()))
