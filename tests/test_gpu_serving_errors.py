"""GPU: the decode engine after a call that failed on the host."""
import ctypes as C
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent / "golden"))
import make_model_golden as G  # noqa: E402

pytestmark = pytest.mark.gpu


class InvalidatedCapture:
    """A stream whose capture has been invalidated (a synchronisation inside
    it): every launch there is refused on the host, and nothing reaches the GPU."""

    def __enter__(self):
        self.rt = C.CDLL(next(line.split()[-1] for line in open("/proc/self/maps") if "libcudart" in line))
        self.stream = torch.cuda.Stream()
        st = C.c_void_p(self.stream.cuda_stream)
        assert self.rt.cudaStreamBeginCapture(st, 2) == 0      # relaxed: other streams are not concerned
        assert self.rt.cudaStreamSynchronize(st) != 0
        return self.stream

    def __exit__(self, *exc):
        graph = C.c_void_p()
        assert self.rt.cudaStreamEndCapture(C.c_void_p(self.stream.cuda_stream), C.byref(graph)) != 0
        self.rt.cudaGetLastError()


@pytest.fixture(scope="module")
def model(lib, tmp_path_factory):
    from sepia_b200.model import DeviceModel, Sampling
    d, prompt, _ = G.build("baseline_types", tmp_path_factory.mktemp("errors") / "m")
    m = DeviceModel.from_container(d, max_positions=200)
    m.set_sampling(Sampling(temperature=0.9))
    return m, torch.as_tensor(np.asarray(prompt, np.int32), device="cuda")


@pytest.mark.parametrize("sampled", [False, True])
def test_a_call_after_a_failed_one_writes_its_own_arrays(model, sampled):
    """Ids go to the array of this call (and its numbers are read), not to
    those of the graph that was kept before the failed call."""
    m, prompt = model
    u_old, u_new = torch.full((6,), 0.1, device="cuda"), torch.full((6,), 0.9, device="cuda")

    def run(out, u, stream=None):
        if sampled:
            m.decode_sampled(out, u, stream=stream)
        else:
            m.decode(out, stream=stream)

    def fresh(u):
        m.reset()
        m.prefill(prompt, True)
        out = torch.full((6,), -7, dtype=torch.int32, device="cuda")
        run(out, u)
        return out
    want = fresh(u_new)
    old = fresh(u_old)
    kept = old.clone()
    m.reset()
    m.prefill(prompt, True)
    new = torch.full((6,), -7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with InvalidatedCapture() as bad:
        with pytest.raises(RuntimeError, match="decode"):
            run(new, u_new, stream=bad)
    run(new, u_new)
    torch.cuda.synchronize()
    assert torch.equal(new, want) and torch.equal(old, kept)


@pytest.mark.parametrize("kv_block", [0, 16])
def test_tokens_past_the_capacity(model, lib, tmp_path, kv_block):
    """They set the error word and touch nothing outside the caches: the tokens
    before them and a sequence after a reset are as ever."""
    from sepia_b200.model import DeviceModel
    d, _, _ = G.build("baseline_types", tmp_path / "m")
    ids = torch.as_tensor(np.random.default_rng(1).integers(0, 400, 48).astype(np.int32), device="cuda")
    m = DeviceModel.from_container(d, max_positions=40, kv_block=kv_block)
    torch.cuda.synchronize()
    lib.sepia_cuda_device_error(None)

    def upto(n):
        m.reset()
        m.prefill(ids[:n], True)
        return m.logits()
    want = upto(40)
    out = torch.empty(6, dtype=torch.int32, device="cuda")
    assert lib.sepia_cuda_device_error(None) == 0
    upto(48)
    assert lib.sepia_cuda_device_error(None) == 2
    upto(37)
    m.decode(out)                                       # three of the six fit
    assert lib.sepia_cuda_device_error(None) == 2
    assert torch.equal(upto(40), want) and lib.sepia_cuda_device_error(None) == 0
