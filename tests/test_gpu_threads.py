"""Calls of two host threads on one stream, each of several kernels that hand data over in a
workspace: every call has the bits that it has alone."""
import threading

import pytest
import torch

from specdec.attention import shared_prefix_attention_paged
from specdec.sampling import token_logprobs
from test_gpu_prefix_attention import make

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _turns(calls, times=200):
    """Each of `calls` by a thread of its own, `times` times; the results that differ from those of
    the call alone."""
    want = [[t.clone() for t in f()] for f in calls]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(len(calls))

    def run(f, w):
        start.wait()
        got = [f() for _ in range(times)]
        torch.cuda.synchronize()
        wrong.extend(1 for g in got if not all(torch.equal(a, b) for a, b in zip(g, w)))

    ts = [threading.Thread(target=run, args=(f, w)) for f, w in zip(calls, want)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    return len(wrong)


def test_shared_attention_of_two_threads():
    a = make(1, [4], [900], [40, 3, 0, 70], [1, 2, 1, 3], 8, 2, 128)
    b = make(2, [3, 2], [100, 700], [5, 70, 1, 2, 3], [1, 4, 2, 1, 1], 8, 2, 128)
    assert _turns([lambda: (shared_prefix_attention_paged(**a),),
                   lambda: (shared_prefix_attention_paged(**b),)]) == 0


def test_log_probabilities_of_two_threads():
    g = torch.Generator(device=DEV).manual_seed(4)
    x = [torch.randn((n, 50257), generator=g, device=DEV) for n in (3, 5)]
    ids = [torch.randint(0, 50257, (n, 2), generator=g, device=DEV) for n in (3, 5)]
    assert _turns([lambda: token_logprobs(x[0], ids[0], top_n=5),
                   lambda: token_logprobs(x[1], ids[1], top_n=20)]) == 0
