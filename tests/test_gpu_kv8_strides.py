"""GPU: rows that start off the vector boundary (odd token strides, a first
element of any alignment) give what the same rows give side by side."""
import pytest
import torch

from test_gpu_kv8 import F16, F32, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("first,pad", [(0, 1), (1, 0), (3, 2), (2, 6)])
@pytest.mark.parametrize("dim,new", [(128, [1, 1]), (96, [20, 3]), (48, [70, 33])])
def test_rows_off_the_vector_boundary(lib, dtype, first, pad, dim, new):
    from sepia_b200.kv8 import rotation_table
    hk, h, n = 2, 6, sum(new)
    width = first + (h + 2 * hk) * dim + pad
    buffer = torch.randn(n, width, generator=torch.Generator("cuda").manual_seed(dim), device="cuda").to(dtype)
    parts = buffer[:, first:first + (h + 2 * hk) * dim].split([h * dim, hk * dim, hk * dim], dim=1)
    seen = []
    for whole in (False, True):
        q, k, v = ((t.contiguous() if whole else t).unflatten(1, (-1, dim)) for t in parts)
        B = Batch([31, 130], hk, dim, 16, seed=4)
        kw = dict(k_norm=torch.full((dim,), 1.1, device="cuda"), q_norm=torch.full((dim,), 0.9, device="cuda"),
                  rotation=rotation_table(300, 16))
        step = B.step(new)
        turned = B.cache.append(step, k, v, q=q, **kw)
        out = B.cache.attention(step, q, 1.0 / dim)                # the strided rows themselves
        c = B.cache
        seen.append([turned, out, c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale.view(torch.uint8),
                     c.v_scale.view(torch.uint8), c.k_tail.view(torch.uint8), c.v_tail.view(torch.uint8)])
    assert all(torch.equal(a, b) for a, b in zip(*seen))
    assert torch.isfinite(seen[0][1]).all() and seen[0][1].abs().max() > 0.01
