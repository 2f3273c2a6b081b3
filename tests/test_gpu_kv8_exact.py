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


def check_faint_rest(block, held, seqs, hk, zero, sink, dtype, window=0):
    """One key (sink) far above the others, its value zero as those of the
    keys in `zero`: the result is a share of faint weights alone, so it must be
    right relative to itself. Values of about 0.01, beside blocks of zeros whose
    scale is 1 by definition. Tolerance: test_gpu_kv8.py, a sink and a faint rest."""
    dim, g = 64, (60.0, 100.0, 110.0, 0.0)
    B = Batch([0] * seqs, hk, dim, block, seed=11, room=held + 1)
    rng = np.random.default_rng(12)
    k = rng.standard_normal((held, hk, dim)) * 0.05
    v = 0.01 + 0.002 * rng.standard_normal((held, hk, dim))
    direction = rng.standard_normal(dim)
    direction /= np.linalg.norm(direction)
    k[sink] = 8.0 * direction
    v[zero] = 0.0
    v[sink] = 0.0
    both = [torch.tensor(np.concatenate([x] * seqs), dtype=torch.float32, device="cuda") for x in (k, v)]
    B.append([held] * seqs, k=both[0], v=both[1])
    q = torch.stack([torch.tensor(direction * x, dtype=torch.float32) for x in g]).repeat(seqs, hk, 1).to(dtype).cuda()
    zeros = torch.zeros(seqs, hk, dim, device="cuda")
    step = B.step([1] * seqs)
    B.cache.append(step, zeros, zeros)
    out = B.cache.attention(step, q, 1.0 / dim, window=window)
    B.kv_len += 1
    want, top, _ = attention64(B, q, [held] * seqs, [1] * seqs, np.float64(np.float32(1.0 / dim)), window, None, None)
    tol = (2 * dim * 2.0 ** -24 * top / dim + 2.0 ** -13 * (8 if dtype == F16 else 1))[:, :, None] * np.abs(want) + 1e-12
    err = np.abs(out.cpu().double().numpy() - want)
    assert np.abs(want).min() > 1e-11 and np.all(err <= tol + (2.0 ** -24 if dtype == F16 else 0)), float((err / tol).max())


@pytest.mark.parametrize("dtype", [torch.float32, F16])
@pytest.mark.parametrize("block", [16, 32, 64])
def test_zero_blocks_beside_faint_weights(lib, dtype, block):
    """Every third 128 positions (blocks of 16: every second block) hold zeros:
    a warp of keys meets them before the rest."""
    held = 1100
    at = np.arange(held)
    zero = at // 16 % 2 == 0 if block == 16 else at // 128 % 3 == 0
    check_faint_rest(block, held, 24, 8, zero, 5, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, F16])
@pytest.mark.parametrize("block,held,window,sink", [(16, 16, 0, 5), (16, 80, 0, 70), (32, 96, 17, 85), (64, 192, 40, 188)])
def test_odd_tiles_beside_faint_weights(lib, dtype, block, held, window, sink):
    """An odd number of 16-key tiles, so that the last step has one that is not there."""
    check_faint_rest(block, held, 2, 2, np.zeros(held, bool), sink, dtype, window)
