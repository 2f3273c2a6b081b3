"""GPU: sepia_cuda_sample against the definition in 64 bits. The drawn token
depends on u only through which token's interval it falls into, so a row's
u is put well inside an interval (1e-4 of it from its ends, and intervals
shorter than 1e-6 are passed over: fp32 exponentials move an end by 1e-7);
then the ids are equal, not near."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def kept64(x, t=1.0, k=0, p=1.0, mp=0.0):
    """(kept indices ascending, their shares) of one row."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.lexsort((np.arange(len(x)), -x))
    if not t > 0:
        return order[:1], np.ones(1)
    with np.errstate(invalid="ignore"):
        e = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / np.float64(np.float32(t))))[order]
    if 0 < k < len(e):
        e = e[:k]
    if p < 1:
        before = np.cumsum(e) - e
        e = e[(before < np.float64(np.float32(p)) * e.sum()) | (np.arange(len(e)) == 0)]
    e = e[e >= min(np.float64(np.float32(mp)), 1.0)]
    at = order[: len(e)]
    by = np.argsort(at)
    return at[by], e[by] / e.sum()


def draw(x, u, **kw):
    from sepia_b200.sampling import sample
    n = x.shape[0]
    dev = {}
    for name, dt in (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32),
                     ("min_p", torch.float32)):
        if kw.get(name) is not None:
            dev[name] = torch.tensor(np.broadcast_to(kw[name], (n,)).copy(), dtype=dt, device="cuda")
    ids, prob = sample(x, torch.tensor(np.asarray(u), dtype=torch.float32, device="cuda"), **dev)
    return ids.cpu().numpy(), prob.cpu().numpy()


def pick_u(share, rng):
    """(position in the kept list, u inside its interval)."""
    ends = np.cumsum(share)
    ok = np.flatnonzero(share > 1e-6)
    j = int(rng.choice(ok))
    f = rng.uniform(0.1, 0.9)
    return j, float(ends[j] - share[j] * f)


SETTINGS = {
    "temperature": dict(temperature=0.8), "top_k": dict(top_k=40), "top_k_1": dict(top_k=1),
    "top_p": dict(temperature=1.3, top_p=0.9), "top_p_small": dict(top_p=1e-4), "top_p_0": dict(top_p=0.0),
    "min_p": dict(min_p=0.02), "min_p_1": dict(min_p=1.0), "min_p_2": dict(min_p=2.0),
    "all": dict(temperature=0.7, top_k=50, top_p=0.95, min_p=0.01), "greedy": dict(temperature=0.0, top_k=5),
    "top_k_past_vocab": dict(top_k=1 << 30, top_p=0.8), "hot": dict(temperature=50.0),
    "cold": dict(temperature=1e-3, top_p=0.5), "nothing": {},
}


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4099, 50021, 200058])
@pytest.mark.parametrize("name", list(SETTINGS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_settings(lib, vocab, name, dtype):
    rng = np.random.default_rng(vocab + len(name))
    n, kw = 5, SETTINGS[name]
    x = (rng.standard_normal((n, vocab)) * 2).astype(np.float32)
    x[:, rng.integers(0, vocab, 20)] += 8
    if vocab > 2:
        x[:, vocab // 2] = -np.inf
    dev = torch.tensor(x, dtype=dtype, device="cuda")
    x = dev.float().cpu().numpy()
    u, want, prob = [], [], []
    for r in range(n):
        at, share = kept64(x[r], kw.get("temperature", 1.0), kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0))
        j, uu = pick_u(share, rng)
        u.append(uu)
        want.append(at[j])
        prob.append(share[j])
    got, p = draw(dev, u, **kw)
    assert np.array_equal(got, want)
    # a share above 1e-6 has an exponent below 14 with three roundings of 2^-24; a weight is rounded to 2^-32 of the best
    assert np.allclose(p, prob, rtol=4e-6, atol=2e-9)


def test_ends_of_the_draw(lib):
    """u = 0 gives the first index in; the largest u below 1 the last whose share it reaches."""
    x = torch.tensor([[0.0, 1.0, -50.0, 1.0, 0.0, -np.inf]] * 3, device="cuda")
    ids, _ = draw(x, [0.0, 1 - 2.0 ** -24, 1.0])
    assert ids.tolist() == [0, 4, 4]
    ids, _ = draw(x, [0.0, 1 - 2.0 ** -24, 0.5], top_k=2)
    assert ids.tolist() == [1, 3, 3]
    ids, _ = draw(x, [0.0, 1 - 2.0 ** -24, 0.7], top_k=3)     # the tie of the two zeros goes to the lower index
    assert ids.tolist() == [0, 3, 3]


@pytest.mark.parametrize("vocab", [7, 3000, 200058])
def test_ties_go_to_the_lowest_index(lib, vocab):
    """All logits alike: a filter that keeps m tokens keeps the first m."""
    x = torch.full((4, vocab), 3.25, device="cuda")
    last = 1 - 2.0 ** -24
    k = vocab // 2 + 1
    ids, p = draw(x, [0.0, last, 0.0, last], top_k=k)
    assert ids.tolist() == [0, k - 1, 0, k - 1] and np.allclose(p, 1.0 / k, rtol=1e-6)
    ids, p = draw(x, [0.0, last, 0.0, last], top_p=0.5)
    m = -(-vocab // 2)
    assert ids.tolist() == [0, m - 1, 0, m - 1] and np.allclose(p, 1.0 / m, rtol=1e-6)
    ids, p = draw(x, [0.0, last, 0.5, 0.5], min_p=1.0)
    assert ids[0] == 0 and ids[1] == vocab - 1
    ids, p = draw(x, [last] * 4, temperature=0.0)
    assert ids.tolist() == [0] * 4 and p.tolist() == [1.0] * 4


@pytest.mark.parametrize("vocab", [5, 40000])
def test_few_distinct_values(lib, vocab):
    """Logits of three values only: cuts fall inside runs of ties."""
    rng = np.random.default_rng(1)
    x = rng.choice([0.0, 1.0, 1.5], (6, vocab)).astype(np.float32)
    dev = torch.tensor(x, device="cuda")
    for kw in (dict(top_k=vocab // 2), dict(top_p=0.61), dict(top_k=vocab * 3 // 4 + 1, top_p=0.9), dict(min_p=0.5, top_p=0.77)):
        u, want = [], []
        for r in range(6):
            at, share = kept64(x[r], 1.0, kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0))
            j, uu = pick_u(share, rng)
            u.append(uu)
            want.append(at[j])
        assert np.array_equal(draw(dev, u, **kw)[0], want), kw


def test_not_numbers_and_infinities(lib):
    nan, inf = float("nan"), float("inf")
    x = torch.tensor([[nan, nan, nan, nan], [-inf, -inf, -inf, -inf], [nan, 1.0, -inf, nan], [1.0, inf, 0.0, inf],
                      [-3e38, 3e38, nan, -inf]], device="cuda")
    for kw in ({}, dict(top_k=2), dict(top_p=0.9), dict(top_k=3, top_p=0.99, min_p=0.1)):
        ids, p = draw(x, [0.9] * 5, **kw)
        assert ids.tolist() == [-1, -1, 1, 3, 1], kw
        assert p.tolist() == [0.0, 0.0, 1.0, 0.5, 1.0], kw
    ids, p = draw(x, [0.9] * 5, temperature=0.0)
    assert ids.tolist() == [-1, -1, 1, 1, 1]


@pytest.mark.parametrize("vocab", [9, 5000, 60000])
def test_extreme_temperatures(lib, vocab):
    """Infinite and huge: all finite logits alike, -infinity still out; tiny: the best alone, ties and all."""
    x = torch.linspace(-5.0, 5.0, vocab, device="cuda").repeat(4, 1)
    x[:, 0] = x[:, vocab - 1] = -float("inf")
    x[:, 3] = x[:, 5] = 7.0
    m = vocab - 2
    for t in (float("inf"), 3e38):
        ids, p = draw(x, [0.0, 1 - 2.0 ** -24, 0.5, 0.25], temperature=t)
        assert ids[0] == 1 and ids[1] == vocab - 2 and np.allclose(p, 1.0 / m, rtol=1e-6)
        ids, p = draw(x, [0.0, 1 - 2.0 ** -24, 0.0, 0.9], temperature=t, top_k=2)
        assert ids.tolist() == [3, 5, 3, 5] and p.tolist() == [0.5] * 4
    for t in (1e-38, 1e-45):
        ids, p = draw(x, [0.0, 1 - 2.0 ** -24, 0.3, 0.6], temperature=t, top_p=0.9)
        assert ids.tolist() == [3, 5, 3, 5] and p.tolist() == [0.5] * 4


def test_row_stride_and_stream(lib):
    from sepia_b200.sampling import sample
    rng = np.random.default_rng(2)
    wide = torch.tensor(rng.standard_normal((9, 1037)), dtype=torch.float32, device="cuda")
    wide[:, 1000:] = 100.0                                  # padding that must not be drawn
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        u = torch.full((9,), 0.37, device="cuda")
        a = sample(wide[:, :1000], u, top_p=torch.full((9,), 0.9, device="cuda"))
        b = sample(wide[:, :1000].contiguous(), u, top_p=torch.full((9,), 0.9, device="cuda"))
        c = sample(wide[:, 1:1000], u)                      # rows off the vector boundary
        d = sample(wide[:, 1:1000].contiguous(), u)
    st.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(c[0], d[0]) and int(a[0].max()) < 1000


def test_results_belong_to_their_stream(lib):
    """Memory that a call takes for another stream is not handed to this one when it is freed."""
    from sepia_b200.sampling import sample
    x, u = torch.zeros(9, 1000, device="cuda"), torch.full((9,), 0.37, device="cuda")
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    ids, p = sample(x, u, stream=st)
    st.synchronize()
    theirs = {ids.data_ptr(), p.data_ptr()}
    assert ids.tolist() == [370] * 9
    del ids, p
    mine = [torch.empty(9, dtype=torch.int32, device="cuda") for _ in range(64)]
    assert not theirs & {t.data_ptr() for t in mine}


def test_frequencies(lib):
    """Evenly spread u meet each token as often as its share says, to one count."""
    rng = np.random.default_rng(3)
    n, v = 8192, 40
    x = (rng.standard_normal(v) * 1.5).astype(np.float32)
    at, share = kept64(x, 0.9, 30, 0.97, 0.0)
    ids, _ = draw(torch.tensor(x, device="cuda").expand(n, v).contiguous(), (np.arange(n) + 0.5) / n, temperature=0.9,
                  top_k=30, top_p=0.97)
    count = np.bincount(ids, minlength=v)
    assert np.all(np.abs(count[at] - share * n) <= 1.001) and count.sum() == count[at].sum()


def test_many_rows_with_their_own_settings(lib):
    rng = np.random.default_rng(4)
    n, v = 150, 20011
    x = (rng.standard_normal((n, v)) * 3).astype(np.float32)
    kw = dict(temperature=rng.choice([0.0, 0.7, 1.2], n), top_k=rng.choice([0, 1, 17, 5000], n),
              top_p=rng.choice([1.0, 0.5, 0.95], n), min_p=rng.choice([0.0, 0.03], n))
    u, want = [], []
    for r in range(n):
        at, share = kept64(x[r], kw["temperature"][r], kw["top_k"][r], kw["top_p"][r], kw["min_p"][r])
        j, uu = pick_u(share, rng)
        u.append(uu)
        want.append(at[j])
    assert np.array_equal(draw(torch.tensor(x, device="cuda"), u, **kw)[0], want)


@pytest.mark.parametrize("base", [0.0, 1e4, -3e6, 1e8])
def test_logits_far_from_zero(lib, base):
    """A common offset leaves few distinct logits (the spacing of fp32 grows): the cuts are those of the values as they are."""
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((6, 30011)) * 4 + base).astype(np.float32)
    for kw in (dict(top_p=0.7), dict(top_k=2000), dict(temperature=8.0, top_k=90, top_p=0.8), dict(min_p=0.3)):
        u, want = [], []
        for r in range(6):
            at, share = kept64(x[r], kw.get("temperature", 1.0), kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0))
            j, uu = pick_u(share, rng)
            u.append(uu)
            want.append(at[j])
        assert np.array_equal(draw(torch.tensor(x, device="cuda"), u, **kw)[0], want), kw


@pytest.mark.parametrize("k", [900, 1023, 1024, 1025, 1100])
def test_around_the_lists_capacity(lib, k):
    """Sets of about 1024 tokens, where the work changes hands; with and without top-p on top."""
    rng = np.random.default_rng(k)
    x = (rng.standard_normal((4, 60013)) * 2).astype(np.float32)
    for kw in (dict(top_k=k), dict(top_k=k, top_p=0.9), dict(top_k=k, min_p=0.1)):
        u, want = [], []
        for r in range(4):
            at, share = kept64(x[r], 1.0, k, kw.get("top_p", 1.0), kw.get("min_p", 0.0))
            j, uu = pick_u(share, rng)
            u.append(uu)
            want.append(at[j])
        assert np.array_equal(draw(torch.tensor(x, device="cuda"), u, **kw)[0], want), kw


@pytest.mark.parametrize("kw", [dict(top_p=0.9995), dict(top_k=20000), dict(top_k=30000, top_p=0.8),
                                dict(temperature=40.0, top_p=0.5), dict(temperature=40.0, top_k=70000)],
                         ids=lambda kw: "-".join(kw) + str(list(kw.values())[-1]))
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_cuts_in_the_crowd(lib, kw, dtype):
    """Thresholds among tens of thousands of near logits: bins far past the list's capacity."""
    rng = np.random.default_rng(6)
    dev = torch.tensor(rng.standard_normal((3, 200058)) * 2, dtype=dtype, device="cuda")
    x = dev.float().cpu().numpy()
    u, want = [], []
    for r in range(3):
        at, share = kept64(x[r], kw.get("temperature", 1.0), kw.get("top_k", 0), kw.get("top_p", 1.0), 0.0)
        j, uu = pick_u(share, rng)
        u.append(uu)
        want.append(at[j])
    assert np.array_equal(draw(dev, u, **kw)[0], want)


def test_refusals(lib):
    from sepia_b200.sampling import sample
    x, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    with pytest.raises(ValueError, match="float32 or float16"):
        sample(x.double(), u)
    with pytest.raises(ValueError, match="side by side"):
        sample(torch.zeros(2, 16, device="cuda")[:, ::2], u)
    with pytest.raises(ValueError, match="top_k"):
        sample(x, u, top_k=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError, match="u must"):
        sample(x, u[:1])
    with pytest.raises(RuntimeError, match="rows of"):
        sample(torch.zeros(1, (1 << 22) + 1, device="cuda"), u[:1])
    args = [None] * 4
    ids = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert lib.sepia_cuda_sample(0, x.data_ptr(), 7, 2, 8, u.data_ptr(), *args, ids.data_ptr(), None, None) == 0
    assert b"stride" in lib.sepia_cuda_last_error()
    assert lib.sepia_cuda_sample(0, None, 8, 2, 8, u.data_ptr(), *args, ids.data_ptr(), None, None) == 0
    assert lib.sepia_cuda_sample(0, x.data_ptr(), 8, -1, 8, u.data_ptr(), *args, ids.data_ptr(), None, None) == 0
    assert lib.sepia_cuda_sample(0, x.data_ptr(), 8, 0, 8, u.data_ptr(), *args, ids.data_ptr(), None, None) == 1
    empty, p = sample(torch.zeros(0, 8, device="cuda"), u[:0])
    assert empty.numel() == 0 and p.numel() == 0
