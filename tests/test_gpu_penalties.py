"""GPU parity of penalize_logits with the float64 oracle.

Tolerance, elementwise: at most 4 + n fp32 roundings of values that M bounds (the product or
quotient by the repetition, frequency times count and its subtraction, the presence, n bias
entries), 2^-24 M each with one more for the oracle's own float64, and the rounding to the type, u
= half a step: u |y| + (1 + u) (5 + n) 2^-24 M, and half of the smallest fp16 below its normal
range. Logits that nothing concerns are equal bit for bit.
"""
import numpy as np
import pytest
import torch

from oracle import penalties as OP
from specdec.sampling import penalize_logits
from specdec.tree import tree_layout

pytestmark = pytest.mark.gpu
DEV = "cuda"
BITS = {torch.float32: torch.int32, torch.bfloat16: torch.int16, torch.float16: torch.int16}


def dev(x, dtype=None):
    return None if x is None else torch.as_tensor(np.asarray(x), device=DEV, dtype=dtype)


def make(seed, ns, V, dtype, H=40, biases=0, grammar=False, tree=False, path=True, prompt=True, ids=None,
         chain_cu=True):
    """Arguments of a call on the host; ids: how many different tokens come up."""
    rng = np.random.default_rng(seed)
    B, R = len(ns), sum(ns)
    ids = rng.integers(0, V, ids or min(V, 50))
    pick = lambda *s: rng.choice(ids, s)  # noqa: E731
    c = dict(history=pick(B, H), history_len=rng.integers(0, H + 1, B),
             cu_rows=np.concatenate([[0], np.cumsum(ns)]))
    if B:
        c["history_len"][0] = H
    c["prompt_len"] = (rng.random(B) * (c["history_len"] + 1)).astype(np.int64) if prompt else None
    f32 = lambda x: x.astype(np.float32)  # noqa: E731
    c["repetition"], c["frequency"], c["presence"] = (f32(rng.uniform(*x, B)) for x in
                                                      ((0.8, 1.5), (-0.5, 1.0), (-0.5, 2.0)))
    if biases:
        c["bias_ids"], c["bias"] = pick(B, biases), f32(rng.normal(0, 3, (B, biases)))
    if grammar:
        w = rng.integers(-2 ** 31, 2 ** 31, (R, (V + 31) // 32 + 2))
        w[rng.random(w.shape) < 0.3] = 0
        w[rng.random(w.shape) < 0.3] = -1
        if R > 1:
            w[1] = 0                                      # nothing may follow
        c["allowed"] = w.astype(np.int32)
    sees = None
    if path:
        c["node_tokens"] = pick(R)
        if tree:
            parents = [int(rng.integers(0, i)) if i else -1 for n in ns for i in range(n)]
            c["tree_mask"] = tree_layout(dev(parents, torch.int32), dev(c["cu_rows"]), dev(ns),
                                         max_nodes=max(ns))[0]
            m = c["tree_mask"].cpu().numpy().view(np.uint64)
            sees = [{64 * w + j for w in range(m.shape[1]) for j in range(64) if int(x[w]) >> j & 1} for x in m]
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn((R, V), generator=g, device=DEV) * 4).to(dtype)
    return x, c, sees


def call(x, c, **more):
    return penalize_logits(x, **{k: v if isinstance(v, torch.Tensor) else dev(v) for k, v in c.items()}, **more)


def check(x, c, sees, got, rows=None):
    want, size, touched = OP.penalize(x.double().cpu().numpy(), **{k: v for k, v in c.items() if k != "tree_mask"},
                                      sees=sees)
    n = c["bias"].shape[1] if "bias" in c else 0
    u = torch.finfo(x.dtype).eps / 2
    tol = u * np.abs(want) + (1 + u) * (5 + n) * 2.0 ** -24 * size + 2.0 ** -25
    g = got.double().cpu().numpy()
    assert got.dtype == x.dtype and got.shape == x.shape
    at = np.ones(len(want), dtype=bool) if rows is None else rows
    same = torch.as_tensor(~touched, device=DEV)
    b = BITS[x.dtype]
    assert torch.equal(got.contiguous().view(b)[same], x.contiguous().view(b)[same])
    inf = np.isinf(want)
    assert np.array_equal(g[inf], want[inf])
    off = (np.abs(np.where(inf, 0, g) - np.where(inf, 0, want)) - np.where(inf, 0, tol))[at]
    assert off.size == 0 or not (off > 0).any(), off.max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ns,V,kw", [
    ([1], 1, dict()),
    ([1], 7, dict(biases=3, grammar=True)),
    ([1, 1, 1], 1000, dict()),
    ([5, 0, 1, 3], 4099, dict(biases=2, grammar=True)),
    ([5, 0, 1, 3], 8192, dict(tree=True, grammar=True)),
    ([26, 64, 2], 8200, dict(tree=True)),
    ([2, 3], 50257, dict(biases=70, H=700)),
    ([1] * 40, 20000, dict(path=False, biases=1)),
    ([3] * 9, 16385, dict(prompt=False, tree=True)),
    ([200, 65], 1001, dict(tree=True, H=3)),
    ([4, 4], 300, dict(H=5000, ids=3, tree=True, biases=1024)),
])
def test_matches_float64(dtype, ns, V, kw):
    x, c, sees = make(len(ns) + V, ns, V, dtype, **kw)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    before = x.clone()
    check(x, c, sees, call(x, c, error=err))
    assert err.item() == 0 and torch.equal(x, before)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,ns,kw", [
    (24579, [3] * 30, dict(tree=True, grammar=True, biases=3, H=300)),     # slices of many rows
    (2048, [1] * 300, dict(path=False, H=90)), (2041, [2] * 130, dict(biases=2)), (2040, [2] * 130, dict()),
    (8192, [4, 0, 251], dict(tree=True, H=2500, ids=3000)), (8193, [1] * 127, dict(grammar=True)),
])
def test_many_rows(dtype, V, ns, kw):
    x, c, sees = make(V, ns, V, dtype, **kw)
    check(x, c, sees, call(x, c))
    wide = torch.full((sum(ns), V + 13), 7.0, device=DEV, dtype=dtype)     # odd strides, rows off alignment
    view = wide[:, 5:5 + V]
    view.copy_(x)
    check(x, c, sees, call(view, c, out=view))
    assert (wide[:, :5] == 7).all() and (wide[:, 5 + V:] == 7).all()


def test_ids_alike_in_their_low_bits():
    x, c, sees = make(5, [2, 1], 5000, torch.float32, H=64, biases=4)
    for k in ("history", "node_tokens", "bias_ids"):
        flat = c[k].reshape(-1)
        flat[1::3] += np.int64(1) << 32
        flat[2::7] -= np.int64(1) << 32
        flat[::5] = -1 - flat[::5] % 9
    check(x, c, sees, call(x, c))


def test_large_vocabulary_and_long_history():
    x, c, sees = make(3, [9, 4], 262144, torch.bfloat16, H=40000, ids=9000, tree=True, grammar=True, biases=5)
    check(x, c, sees, call(x, c))


@pytest.mark.parametrize("leave", ["history", "prompt_len", "repetition", "frequency", "presence", "bias",
                                   "allowed", "node_tokens", "tree_mask", "all"])
def test_arguments_that_are_left_out(leave):
    x, c, sees = make(4, [4, 7], 3000, torch.bfloat16, biases=4, grammar=True, tree=True)
    for k in {"history": ["history", "history_len", "prompt_len"], "bias": ["bias", "bias_ids"],
              "node_tokens": ["node_tokens", "tree_mask"],
              "all": [k for k in c if k != "cu_rows"]}.get(leave, [leave]):
        del c[k]
    want = dict(c)
    if "history" not in c:
        want.update(history=None, history_len=None)
    got = call(x, c)
    check(x, want, sees if "tree_mask" in c else None, got)
    if leave == "all":
        assert torch.equal(got, x)


def test_one_position_a_row_without_offsets():
    x, c, sees = make(5, [1] * 6, 5000, torch.float16, biases=2)
    want = call(x, c)
    check(x, c, sees, want)
    del c["cu_rows"]
    assert torch.equal(call(x, c), want)


def test_in_place_strides_and_alignment():
    x, c, sees = make(6, [3, 5], 4500, torch.bfloat16, biases=3, grammar=True, tree=True)
    want = call(x, c)
    y = x.clone()
    assert call(y, c, out=y) is y and torch.equal(y, want)
    for off, ld in ((0, 4504), (1, 4501), (3, 5000), (8, 4503), (2, 4502)):   # rows of a wider buffer
        buf = torch.full((8 * ld + 16,), 7.0, dtype=x.dtype, device=DEV)
        v = buf[off:off + 8 * ld].view(8, ld)[:, :4500]
        v.copy_(x)
        rest = buf.clone()
        assert torch.equal(call(v, c), want)
        assert call(v, c, out=v) is v and torch.equal(v, want)
        rest[off:off + 8 * ld].view(8, ld)[:, :4500].copy_(want)
        assert torch.equal(buf, rest)                     # nothing beside the rows
    out = torch.empty((8, 4601), dtype=x.dtype, device=DEV)[:, 1:4501]
    assert torch.equal(call(x, c, out=out), want)
    assert torch.equal(call(x.t().contiguous().t(), c), want)
    h = torch.zeros((2, 90), dtype=torch.int64, device=DEV)
    h[:, 3:43] = dev(c["history"])                        # the columns of a longer buffer
    assert torch.equal(call(x, {**c, "history": h[:, 3:43]}), want)
    assert torch.equal(call(x, {**c, "history": dev(c["history"]).to(torch.int32)}), want)
    with pytest.raises(RuntimeError, match="apart"):
        wide = torch.zeros((8, 5000), dtype=x.dtype, device=DEV)
        call(wide[:, :4500], c, out=wide[:, 1:4501])


def test_rows_out_of_range_and_behind_the_last_are_copied():
    for key, value in (("history_len", 41), ("history_len", -1), ("prompt_len", 99), ("prompt_len", -1)):
        x, c, sees = make(7, [3, 4, 2], 2000, torch.float32, grammar=True)
        c["history_len"][1], c["prompt_len"][1] = 20, 10
        c[key][1] = value
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = call(x, c, error=err)
        assert err.item() == 1 and torch.equal(got[3:7], x[3:7])
        c["history_len"][1], c["prompt_len"][1] = 20, 10
        check(torch.cat([x[:3], x[7:]]), {**{k: np.delete(v, 1, 0) for k, v in c.items() if k not in (
            "cu_rows", "allowed", "node_tokens")}, "cu_rows": [0, 3, 5], "allowed": np.delete(
                c["allowed"], range(3, 7), 0), "node_tokens": np.delete(c["node_tokens"], range(3, 7))},
            sees, torch.cat([got[:3], got[7:]]))
    x, c, sees = make(8, [3, 4], 2000, torch.bfloat16, grammar=True)
    pad = torch.randn((2, 2000), device=DEV).to(x.dtype)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = call(torch.cat([x, pad]), {**c, "allowed": np.concatenate([c["allowed"], np.zeros_like(c["allowed"][:2])]),
                                     "node_tokens": np.concatenate([c["node_tokens"], [1, 2]])}, error=err)
    assert torch.equal(got[7:], pad) and torch.equal(got[:7], call(x, c)) and err.item() == 0
    c["cu_rows"] = np.array([0, 3, 9])                     # past the rows
    got = call(x, c, error=err)
    assert err.item() == 1 and torch.equal(got[3:], x[3:])


def test_ids_outside_the_vocabulary_count_nowhere():
    x, c, sees = make(9, [3, 4], 2000, torch.float32, biases=6, tree=True)
    for k in ("history", "bias_ids", "node_tokens"):
        v = c[k].reshape(-1)
        v[::3] = [(-1, 2000, 2 ** 40, -2 ** 40)[i % 4] for i in range(len(v[::3]))]
    check(x, c, sees, call(x, c))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_infinities_and_nan(dtype):
    """They go through the formula as they are; refused ones become -inf."""
    V = 64
    x = torch.zeros((2, V), dtype=dtype, device=DEV)
    x[:, 0::4], x[:, 1::4], x[:, 2::4], x[:, 3::4] = float("inf"), float("-inf"), float("nan"), -0.0
    ids = np.arange(32)[None].repeat(2, 0)
    allowed = np.array([[-1, -1], [0x0F0F0F0F, 0]], dtype=np.int32)
    c = dict(history=ids, history_len=[32, 32], cu_rows=[0, 1, 2], repetition=np.float32([2, 2]),
             presence=np.float32([1, 1]), allowed=allowed)
    got = call(x, c).float()
    assert torch.equal(got[0, 0:32:4], x[0, 0:32:4].float()) and torch.equal(got[0, 1::4], x[0, 1::4].float())
    assert got[0, 2::4].isnan().all() and (got[0, 3:32:4] == -1).all()
    b = BITS[dtype]
    assert torch.equal(call(x, c)[0, 32:].view(b), x[0, 32:].view(b))
    v = np.arange(V)
    no = dev((allowed[1][v // 32] >> (v % 32)) & 1 == 0)
    assert (got[1][no] == -float("inf")).all() and not (got[1][~no] == -float("inf"))[0::4].any()


def test_two_streams_and_a_graph():
    x, c, sees = make(10, [3, 26, 1], 30000, torch.bfloat16, biases=4, grammar=True, tree=True)
    want = call(x, c)
    d = {k: v if isinstance(v, torch.Tensor) else dev(v) for k, v in c.items()}
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = penalize_logits(x, **d)
    assert torch.equal(penalize_logits(x, **d), want)
    s.synchronize()
    assert torch.equal(other, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = penalize_logits(x, **d)
    for seed in range(3):
        y, e, _ = make(10 + seed, [3, 26, 1], 30000, torch.bfloat16, biases=4, grammar=True, tree=True)
        x.copy_(y)
        for k in d:
            d[k].copy_(e[k] if isinstance(e[k], torch.Tensor) else dev(e[k]))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, penalize_logits(x, **d))
