"""GPU: host threads that share one Kv8Step on one stream. The attention of a
long context is two launches over one workspace, and the interpreter's lock is
released inside the call: two calls must not be in it at the same time."""
import threading
import time

import pytest
import torch

from test_gpu_kv8 import Batch

pytestmark = pytest.mark.gpu


def together(calls):
    errors = []

    def guarded(f):
        try:
            f()
        except BaseException as e:                  # noqa: BLE001 (handed to the test's own thread)
            errors.append(e)
    threads = [threading.Thread(target=guarded, args=(f,)) for f in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_calls_with_one_workspace_take_turns(lib):
    """The C entry is a stand-in that only records who is inside with which workspace (no kernel runs)."""
    B = Batch([3000], 2, 64, 16)
    step, q = B.step([1]), torch.zeros(1, 4, 64, device="cuda")
    inside, met, guard = {}, [], threading.Lock()

    def entry(cache, bound, args, ws, nbytes, stream):
        with guard:
            inside[ws] = inside.get(ws, 0) + 1
            met.append(inside[ws])
        time.sleep(0.05)
        with guard:
            inside[ws] -= 1
        return 1
    B.cache._attn = entry
    together([lambda: B.cache.attention(step, q, 0.125)] * 4)
    assert met == [1, 1, 1, 1]


def test_threads_get_their_own_results(lib):
    B = Batch([3000, 700], 2, 64, 16)
    step = B.step([1, 1])
    k = torch.randn(2, 2, 64, device="cuda")
    B.cache.append(step, k, k)
    queries = [torch.randn(2, 4, 64, device="cuda") for _ in range(4)]
    want = [B.cache.attention(step, q, 0.125) for q in queries]
    torch.cuda.synchronize()
    got = [[] for _ in queries]
    together([lambda i=i: got[i].extend(B.cache.attention(step, queries[i], 0.125) for _ in range(200)) for i in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(4) for x in got[i])
