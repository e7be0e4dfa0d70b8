"""GPU parity of token_logprobs with the float64 oracle (oracle/logprobs.py).

Tolerance. With d = (x - m) / T, every fp32 exponential of the sums is off by at most
(2 |d| + 4) half steps relative (the shift, the product with log2(e) / T, the exponential,
the shifts to a larger maximum), the summation of z and w adds one half step per addend of a
thread's chain and per level of the joins, and z is over the chain's terms. So ln z is off
by at most u (n + 2 D + 24) with u = 2^-24, n = V / 256 + 32 the longest chain and D the
mean of |d| under p (at most the entropy plus ln V); log p adds 3 u |d|, and the entropy
w / z doubles its own part.
"""
import numpy as np
import pytest
import torch

from oracle import logprobs as OL
from specdec.sampling import gather_prob, to_probs, token_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _logits(rows, V, seed, dtype, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn((rows, V), generator=g, device=DEV) * spread).to(dtype)


def _check(x, ids, T, top_n, got=None):
    """x [rows, V], ids [rows, n] on the device."""
    logp, ent, tl, ti = token_logprobs(x, ids, temperature=T, top_n=top_n) if got is None else got
    V = x.shape[1]
    rl, re, rt, ri = OL.token_logprobs(x.double().cpu().numpy(), ids.cpu().numpy(), T, top_n)
    rows = ~np.isnan(re)
    base = U * (V / 256 + 32 + 24 + 2 * (np.where(rows, re, 0) + np.log(V)))

    def near(a, b, tol):
        a, b = a.double().cpu().numpy(), np.asarray(b)
        assert np.array_equal(np.isnan(a), np.isnan(b))
        fin = np.isfinite(b)
        assert np.array_equal(a[~fin & ~np.isnan(b)], b[~fin & ~np.isnan(b)])
        off = np.abs(a - b)[fin] - np.broadcast_to(tol, b.shape)[fin]
        assert off.size == 0 or off.max() <= 0, off.max()

    near(logp, rl, base[:, None] + 3 * U * np.abs(np.where(np.isfinite(rl), rl, 0)))
    near(ent, re, 2 * base * (1 + np.abs(np.where(rows, re, 0))))
    if top_n == 0:
        assert tl is None and ti is None
        return
    assert np.array_equal(ti.cpu().numpy()[rows], ri[rows])
    near(tl, rt, base[:, None] + 3 * U * np.abs(np.where(np.isfinite(rt), rt, 0)))
    assert ((ti >= -1) & (ti < V)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,V,n,top_n,T", [
    (1, 1, 1, 1, 1.0), (3, 2, 2, 2, 0.5), (2, 7, 1, 5, 1.0), (5, 63, 1, 63, 1.0),
    (4, 100, 3, 64, 0.7), (1, 2048, 1, 20, 1.0), (7, 2049, 1, 20, 1.3), (3, 4096, 4, 0, 1.0),
    (2, 8191, 1, 1, 1.0), (1, 32000, 1, 64, 0.6), (3, 50257, 2, 20, 1.0), (1, 151936, 1, 20, 1.0),
    (2, 262143, 1, 5, 0.8),
])
def test_matches_oracle(dtype, rows, V, n, top_n, T):
    x = _logits(rows, V, rows * 31 + V, dtype)
    ids = torch.randint(0, V, (rows, n), device=DEV)
    _check(x, ids, T, top_n)


def test_row_offsets_past_32_bits():
    """Rows further apart than 2^32 elements, split over workgroups and whole."""
    V, ld = 20000, (1 << 32) + 24
    buf = torch.empty(ld + V, dtype=torch.bfloat16, device=DEV)
    x = buf.as_strided((2, V), (ld, 1))
    x.copy_(_logits(2, V, 77, torch.bfloat16))
    _check(x, torch.randint(0, V, (2, 2), device=DEV), 0.9, 20)
    short = x[:, :300]
    _check(short, torch.randint(0, 300, (2, 2), device=DEV), 0.9, 20)


def test_many_rows_run_whole():
    """Rows enough that each is one workgroup's, beside the split of few rows above."""
    x = _logits(2300, 1000, 4, torch.bfloat16)
    _check(x, torch.randint(0, 1000, (2300, 1), device=DEV), 1.0, 20)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_row_strides_and_alignment(dtype):
    """Rows inside a wider buffer, at every offset from a 16-byte boundary; a row read twice."""
    buf = _logits(5, 1300, 8, dtype)
    for at in range(9):
        x = buf[:, at:at + 1111]
        _check(x, torch.randint(0, 1111, (5, 2), device=DEV), 1.0, 7)
    one = buf[2:3, 3:700].expand(4, -1)
    _check(one, torch.randint(0, 697, (4, 1), device=DEV), 1.0, 3)
    odd = buf.t()[:64].contiguous().t()  # a column stride of its own
    _check(odd, torch.randint(0, 64, (5, 1), device=DEV), 1.0, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [40, 3000, 40000])
def test_ties_go_to_the_lowest_id(dtype, V):
    """Few values, constant rows, zeros of both signs."""
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randint(-2, 3, (6, V), generator=g, device=DEV).float()
    x[1] = 0.25
    x[2] = torch.where(torch.rand(V, generator=g, device=DEV) < 0.5, 0.0, -0.0)
    x[3, :] = torch.arange(V, device=DEV) // 40      # ascending in steps
    x[4, :] = -(torch.arange(V, device=DEV) // 40)   # descending
    _check(x.to(dtype), torch.randint(0, V, (6, 1), device=DEV), 1.0, 33)


def test_best_tokens_of_one_thread():
    """More large values in the vectors of one thread than the collected list holds (a
    period of 256 vectors), for each type's vector and both sides of the split."""
    for dtype, vec in ((torch.float32, 4), (torch.bfloat16, 8)):
        for rows, V in ((1, 160000), (2100, 9000)):
            x = torch.zeros((rows, V), device=DEV) - 3.0
            col = torch.arange(V, device=DEV)
            hot = (col // vec) % 256 < 24
            x[:, hot] = (col[hot] * 7919 % 1013).float() / 8
            x = x.to(dtype)
            if rows > 1:
                x[1:] = x[0]
            logp, ent, tl, ti = token_logprobs(x, torch.zeros((rows, 1), dtype=torch.long, device=DEV),
                                               top_n=20)
            _check(x[:2], torch.zeros((min(rows, 2), 1), dtype=torch.long, device=DEV), 1.0, 20,
                   got=(logp[:2], ent[:2], tl[:2], ti[:2]))
            assert (ti == ti[0]).all() and torch.equal(tl, tl[:1].expand_as(tl))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [50, 5000, 70001])
def test_masked_and_nonfinite_rows(dtype, V):
    """-inf and the type's lowest value as masks, rows that they leave empty, +inf and NaN."""
    x = _logits(9, V, V, torch.float32)
    lowest = torch.finfo(dtype).min
    x[0, V // 2:] = -np.inf
    x[1, 1:] = -np.inf           # one token left: log p 0, entropy 0
    x[2] = -np.inf               # none left
    x[3] = lowest                # all masked alike: uniform
    x[4, V // 3:] = lowest
    x = x.to(dtype)
    x[5, V - 1] = np.inf
    x[6, V // 2] = np.nan
    x[7] = np.nan
    x[8, :3] = -np.inf
    ids = torch.tensor([[0, V - 1, -1, V]] * 9, device=DEV)
    _check(x, ids, 1.0, 5)
    logp, ent, tl, ti = token_logprobs(x, ids, top_n=5)
    assert logp[1, 0] == 0 and ent[1] == 0 and ti[1].tolist() == [0, 1, 2, 3, 4]
    assert ti[2].tolist() == [0, 1, 2, 3, 4]
    assert abs(ent[3].item() - np.log(V)) < 1e-4


def test_large_and_small_temperatures():
    x = _logits(3, 3001, 2, torch.float32, spread=30.0)
    ids = torch.randint(0, 3001, (3, 2), device=DEV)
    for T in (1e-3, 0.05, 50.0, 1e6):
        _check(x, ids, T, 4)


def test_shapes_and_agreement_with_to_probs():
    x = _logits(12, 5000, 6, torch.bfloat16).view(3, 4, 5000)
    ids = torch.randint(0, 5000, (3, 4), device=DEV)
    logp, ent, tl, ti = token_logprobs(x, ids, temperature=0.7, top_n=3)
    assert logp.shape == (3, 4) and ent.shape == (3, 4) and tl.shape == ti.shape == (3, 4, 3)
    p = gather_prob(to_probs(x, 0.7), ids)
    assert torch.allclose(logp.exp(), p, rtol=1e-4, atol=0)
    assert token_logprobs(x[:0], ids[:0])[0].shape == (0, 4)
    one = token_logprobs(x[0, 0], ids[0, 0])
    assert one[0].shape == () and abs((one[0] - token_logprobs(x, ids)[0][0, 0]).item()) < 1e-5
    assert token_logprobs(x, ids.to(torch.int32).unsqueeze(-1))[0].shape == (3, 4, 1)


def test_refusals():
    x = _logits(2, 30, 1, torch.float32)
    ids = torch.zeros(2, dtype=torch.long, device=DEV)
    for bad in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
                dict(temperature=float("inf")), dict(top_n=31), dict(top_n=-1)):
        with pytest.raises(ValueError):
            token_logprobs(x, ids, **bad)
    with pytest.raises(ValueError, match="top_n"):
        token_logprobs(_logits(1, 100, 1, torch.float32), ids[:1], top_n=65)
    with pytest.raises(ValueError, match="ids must be"):
        token_logprobs(x, ids[:1])
    with pytest.raises(TypeError, match="whole numbers"):
        token_logprobs(x, ids.float())
    with pytest.raises(RuntimeError, match="ROCm device"):
        token_logprobs(x.cpu(), ids)


def test_graph_replays_and_streams():
    """Captured calls of two graphs replayed in turn with eager calls between, and a call on
    a side stream, give the eager results bit for bit."""
    xs = [_logits(4, 50257, s, torch.bfloat16) for s in (1, 2)]
    ids = torch.randint(0, 50257, (4, 1), device=DEV)
    want = [[t.clone() for t in token_logprobs(x, ids, top_n=5)] for x in xs]
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            outs.append(token_logprobs(x, ids, top_n=5))
        graphs.append(g)
    for turn in range(4):
        for g in graphs:
            g.replay()
        eager = token_logprobs(xs[turn % 2], ids, top_n=5)
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[turn % 2]))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = token_logprobs(xs[0], ids, top_n=5)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(side, want[0]))
