"""GPU: a sequence that breaks a bound of its step (include/sepia_cuda.h,
SepiaKv8Step) is skipped: its rows of the results are zeros, whatever the
buffers held before, nothing of the cache changes for it, the error word is
set, and its neighbours get what they get beside a sequence of no tokens."""
import pytest
import torch

from test_gpu_kv8 import F16, F32, Batch

pytestmark = pytest.mark.gpu
HK, H, DIM = 2, 6, 48


def kept(B):
    c = B.cache
    return [c.k.view(torch.uint8).clone(), c.v.view(torch.uint8).clone(), c.k_scale.clone(), c.v_scale.clone(),
            c.k_tail.clone(), c.v_tail.clone()]


def same(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


@pytest.mark.parametrize("bad", ["max_new", "many_more_than_max_new", "n_tokens", "slot", "max_kv", "idle"])
@pytest.mark.parametrize("max_kv", [100, 4000], ids=["one_chunk", "chunks"])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_a_broken_bound_gives_zeros(lib, bad, max_kv, dtype):
    from sepia_b200.kv8 import Kv8Step
    torch.cuda.synchronize()
    lib.sepia_cuda_device_error(None)
    runs = []
    for broken in (True, False):
        B = Batch([31, 40, 9], HK, DIM, 16, seed=3, room=4000)
        lens, slot = B.kv_len.clone(), B.slot.clone()
        new = [2, 3 if bad == "max_new" else 40 if bad.startswith("many") else 2, 1]
        bound = 2
        if bad == "n_tokens":                       # the last sequence, so that its rows end past n_tokens
            new = [2, 1, 2]
        at = 2 if bad == "n_tokens" else 1
        total = sum(new)
        n_tokens = total - 1 if bad == "n_tokens" else total
        g = torch.Generator(device="cuda").manual_seed(5)
        k, v, q = (torch.randn(total, heads, DIM, generator=g, device="cuda").to(dtype) for heads in (HK, HK, H))
        ends = [new[0], new[0] + new[1], total]
        start = [0, *ends]
        if not broken:                              # the same rows, with a sequence of no tokens in its place
            start[at + 1] = start[at]
            lens[at] = 5
            if at == 1:                             # (the last one's row is the end of the list)
                keep = list(range(new[0])) + list(range(ends[1], total))
                k, v, q, start, total, n_tokens = k[keep], v[keep], q[keep], [0, new[0], new[0], len(keep)], len(keep), len(keep)
            else:
                total = n_tokens = ends[1]
        elif bad == "slot":
            slot[at] = B.cache.struct.n_slots
        elif bad == "max_kv":
            lens[at] = max_kv - 1
        elif bad == "idle":
            lens[at] = -1
        step = Kv8Step(B.table, lens, start=torch.tensor(start, dtype=torch.int32, device="cuda"), slot=slot,
                       n_tokens=n_tokens, max_new=bound, max_kv=max_kv)
        q_out, out = (torch.full((n_tokens, H, DIM), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        before = kept(B)
        B.cache.append(step, k[:n_tokens], v[:n_tokens], q=q[:n_tokens], q_out=q_out)
        torch.cuda.synchronize()
        assert lib.sepia_cuda_device_error(None) == (2 if broken and bad != "idle" else 0)
        B.cache.attention(step, q_out, 0.125, out=out)
        torch.cuda.synchronize()
        assert lib.sepia_cuda_device_error(None) == (2 if broken and bad != "idle" else 0)
        after = kept(B)
        if broken:
            rows = slice(ends[at - 1], min(ends[at], n_tokens))
            assert torch.all(q_out[rows] == 0) and torch.all(out[rows] == 0)
            mask = torch.ones(n_tokens, dtype=torch.bool)
            mask[rows] = False
            q_out, out = q_out[mask.cuda()], out[mask.cuda()]
            if bad in ("idle", "slot"):             # its tail, and its blocks
                ids = B.table[at].long()
                assert all(torch.equal(x[ids], y[ids]) for x, y in zip(before[:2], after[:2]))
        runs.append((q_out, out, after))
    assert torch.all(runs[1][0] != 7) and torch.all(runs[1][1] != 7)
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    assert same(runs[0][2], runs[1][2])             # the cache: only the neighbours' tokens went in


def test_steps_with_start_need_no_max_new(lib):
    """Left out, the bound is all the step's tokens: no sequence is skipped."""
    from sepia_b200.kv8 import Kv8Step
    new = [2, 0, 5]
    start = torch.tensor([0, 2, 2, 7], dtype=torch.int32, device="cuda")
    k, v, q = (torch.randn(7, heads, DIM, device="cuda") for heads in (HK, HK, H))
    torch.cuda.synchronize()
    lib.sepia_cuda_device_error(None)
    results = []
    for kw in (dict(max_new=max(new)), dict()):
        B = Batch([31, 40, 9], HK, DIM, 16, seed=3)
        step = Kv8Step(B.table, B.kv_len, start=start, slot=B.slot, n_tokens=7, **kw)
        turned = B.cache.append(step, k, v, q=q)
        results.append((turned, B.cache.attention(step, turned, 0.125)))
    assert lib.sepia_cuda_device_error(None) == 0
    assert torch.equal(results[0][0], results[1][0]) and torch.allclose(results[0][1], results[1][1], rtol=0, atol=1e-5)
    assert torch.all(results[1][1] != 0)
    assert Kv8Step(B.table, B.kv_len).struct.max_new == 1


def test_a_prompt_of_many_row_tiles(lib):
    """16384 new tokens of 64 heads at once: what the append takes, the attention takes."""
    hk, h, dim, n, window = 8, 64, 16, 16384, 24
    B = Batch([0], hk, dim, 64, seed=13, room=n)
    B.append([n], advance=False)
    q = torch.randn(n, h, dim, device="cuda")
    out = B.cache.attention(B.step([n]), q, 1.0 / dim, window=window)
    B.kv_len += n
    keys, vals = (torch.tensor(B.held(0, w)[0]).repeat_interleave(h // hk, dim=1) for w in (0, 1))
    for t in [0, 1, 23, 24, n // 2, n - 1, *B.rng.integers(0, n, 200).tolist()]:
        at = slice(max(0, t - window + 1), t + 1)
        w = torch.softmax(torch.einsum("hd,jhd->hj", q[t].cpu().double(), keys[at]) / dim, dim=1)
        want = torch.einsum("hj,jhd->hd", w, vals[at])
        # an fp32 sum of exact products, twice, and 2^-19 for exponentials and sums (test_gpu_kv8.py)
        top = torch.einsum("hd,jhd->hj", q[t].abs().cpu().double(), keys[at].abs()).max() / dim
        tol = (2 * dim * 2.0 ** -24 * float(top) + 2.0 ** -19) * float(vals[at].abs().max())
        assert float((out[t].cpu().double() - want).abs().max()) <= tol, t
