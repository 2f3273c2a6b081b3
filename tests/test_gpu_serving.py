"""GPU: the decode engine over the paged 8-bit cache and with drawn tokens
(sepia_model_create_kv8, sepia_model_decode_sampled, include/sepia_model.h).

What can be asked of an 8-bit cache beside the fp32 one: while a sequence is
shorter than a block nothing has been rounded to 8 bits (tails are fp16:
2^-11 relative), past it keys and values move by up to 2^-4. Errors are
measured in the logits' spread. A moved score may exchange two experts of
nearly equal score at some steps, which moves logits by more than the cache
does, so the bounds hold for the median step: 2^-6 with tails only (2^-11 in
each of 5 layers, grown by the norms), a quarter with codes.
Drawn ids are checked against a draw from the engine's own logits."""
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent / "golden"))
import make_model_golden as G  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def built(lib, tmp_path_factory):
    from sepia_b200.model import DeviceModel
    d, prompt, _ = G.build("baseline_types", tmp_path_factory.mktemp("serving") / "m")
    return d, prompt, DeviceModel.from_container(d, max_positions=300)


def steps(m, ids, n_prompt):
    """Logits after the prompt and after each further token, teacher-forced."""
    t = torch.as_tensor(np.asarray(ids, np.int32), device="cuda")
    m.reset()
    m.prefill(t[:n_prompt], True)
    out = [m.logits().double().cpu().numpy()]
    for i in range(n_prompt, len(ids)):
        m.prefill(t[i:i + 1], True)
        out.append(m.logits().double().cpu().numpy())
    return out


@pytest.mark.parametrize("block", [16, 32, 64])
def test_engine_over_the_8_bit_cache(built, block):
    from sepia_b200.model import DeviceModel
    d, prompt, ref = built
    ids = list(prompt) + list(ref.generate(prompt, 60))
    m = DeviceModel.from_container(d, max_positions=300, kv_block=block)
    short = min(block - 1, len(prompt))
    err = np.array([np.abs(a - b).max() / (a.max() - a.min())
                    for a, b in zip(steps(ref, ids, short), steps(m, ids, short))])
    held = short + np.arange(len(err))
    assert np.median(err[held < block]) <= 2.0 ** -6 and np.median(err[held >= block]) <= 0.25, err
    assert m.position() == len(ids)
    from sepia_b200 import ops
    assert ops.device_error() == 0


def test_graph_replay_equals_single_steps(built):
    """decode (graph) gives the ids of one eager step at a time, over the 8-bit cache."""
    from sepia_b200.model import DeviceModel
    d, prompt, _ = built
    m = DeviceModel.from_container(d, max_positions=300, kv_block=16)
    ids = m.generate(prompt, 70)
    t = torch.as_tensor(np.asarray(prompt, np.int32), device="cuda")
    m.reset()
    m.prefill(t, True)
    for i in range(70):
        assert int(m.logits().argmax()) == ids[i], i
        m.prefill(torch.as_tensor(ids[i:i + 1], device="cuda"), True)
    assert np.array_equal(m.generate(prompt, 70), ids)


@pytest.mark.parametrize("kv_block", [0, 32])
def test_drawn_tokens(built, kv_block):
    """Each id is the one that sampling.sample draws from the logits before it."""
    from sepia_b200.model import DeviceModel, Sampling
    from sepia_b200.sampling import sample
    d, prompt, ref = built
    m = DeviceModel.from_container(d, max_positions=300, kv_block=kv_block) if kv_block else ref
    n = 40
    u = torch.rand(n + 1, generator=torch.Generator().manual_seed(3)).cuda()
    for cfg in (Sampling(temperature=1.5, top_k=50, top_p=0.9, min_p=0.01), Sampling(temperature=0.7), Sampling(temperature=0.0)):
        ids = m.generate(prompt, n, sampling=cfg, u=u)
        again = m.generate(prompt, n, sampling=cfg, u=u)
        assert np.array_equal(ids, again)
        t = torch.as_tensor(np.asarray(prompt, np.int32), device="cuda")
        m.reset()
        m.prefill(t, True)

        def one(x, dt):
            return torch.tensor([x], dtype=dt, device="cuda")
        for i in range(n):
            want, _ = sample(m.logits()[None], u[i:i + 1], one(cfg.temperature, torch.float32), one(cfg.top_k, torch.int32),
                             one(cfg.top_p, torch.float32), one(cfg.min_p, torch.float32))
            assert int(want[0]) == ids[i], (cfg, i)
            m.prefill(torch.as_tensor(ids[i:i + 1], device="cuda"), True)
    greedy = m.generate(prompt, n)
    assert np.array_equal(m.generate(prompt, n, sampling=Sampling(temperature=0.0), u=u), greedy)


def test_generate_on_a_stream(built):
    from sepia_b200.model import Sampling
    _, prompt, m = built
    u = np.linspace(0.05, 0.95, 25).astype(np.float32)
    st = torch.cuda.Stream()
    for kw in (dict(), dict(sampling=Sampling(temperature=0.9, top_p=0.95), u=u)):
        want = m.generate(prompt, 24, **kw)
        torch.cuda.synchronize()
        assert (m.generate(prompt, 24, stream=st, **kw) == want).all()


def test_refusals(built, lib):
    from sepia_b200.model import DeviceModel, Sampling
    d, prompt, _ = built
    with pytest.raises(RuntimeError, match="blocks of 24"):
        DeviceModel.from_container(d, max_positions=64, kv_block=24)
    m = DeviceModel.from_container(d, max_positions=64, kv_block=16)
    u = torch.zeros(2, device="cuda")
    with pytest.raises(RuntimeError, match="before sepia_model_set_sampling"):
        m.draw(u)
    m.set_sampling(Sampling())
    assert lib.sepia_model_draw(m._h, None, None) == 0
    assert lib.sepia_model_decode_sampled(m._h, 1, None, u.data_ptr(), None) == 0
    assert lib.sepia_model_set_sampling(None, 1.0, 0, 1.0, 0.0, None) == 0
