"""GPU parity of the trees' layout and of the walk of accepted nodes with the row-by-row oracle:
whole numbers, equal."""
import numpy as np
import pytest
import torch

from oracle import tree as OT
from specdec.tree import tree_accept, tree_layout

pytestmark = pytest.mark.gpu
DEV = "cuda"


def dev(x, dtype=None):
    return torch.as_tensor(np.asarray(x), device=DEV, dtype=dtype)


def random_tree(rng, n, kind):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return ([-1] + [0] * n)[:n]
    if kind == "forest":
        return [-1 if i == 0 or rng.random() < 0.3 else int(rng.integers(0, i)) for i in range(n)]
    if kind == "binary":
        return [(i - 1) // 2 if i else -1 for i in range(n)]
    return [int(rng.integers(max(0, i - 6), i)) if i else -1 for i in range(n)]


def batch(seed, ns, kind, start, bs, pad=0):
    rng = np.random.default_rng(seed)
    parents = sum((random_tree(rng, n, kind) for n in ns), [])
    cu = np.concatenate([[0], np.cumsum(ns)])
    kv = np.asarray(ns) + np.asarray(start)
    mb = max(1, int(max(-(-kv // bs))))
    table = rng.permutation(len(ns) * mb).reshape(len(ns), mb)
    T = int(cu[-1]) + pad
    parents = np.asarray(parents + [5] * pad, dtype=np.int32)
    return parents, cu, kv, table, T


def sets(mask):
    m = mask.cpu().numpy().view(np.uint64)
    return [{64 * w + j for w in range(m.shape[1]) for j in range(64) if int(row[w]) >> j & 1}
            for row in m]


def check_layout(parents, cu, kv, table, bs, T, max_nodes, ok=True):
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    mask, pos, slots = tree_layout(dev(parents), dev(cu), dev(kv), None if table is None else
                                   dev(table, torch.int32), None if table is None else bs,
                                   max_nodes=max_nodes, error=err)
    words = -(-max_nodes // 64)
    sees, wpos, wslots, wok = OT.tree_layout(parents, cu, kv, table, bs, words, T)
    assert wok == ok and err.item() == (0 if ok else 1)
    assert mask.shape == (T, words) and sets(mask) == sees
    assert pos.tolist() == wpos.tolist()
    if table is None:
        assert slots is None
    else:
        assert slots.tolist() == wslots.tolist()


@pytest.mark.parametrize("kind", ["random", "chain", "star", "forest", "binary"])
@pytest.mark.parametrize("ns,max_nodes", [
    ([1], 1), ([26], 26), ([64], 64), ([63, 1, 0, 64, 2], 64), ([0, 0, 5], 7),
    ([65], 65), ([128, 1, 77], 128), ([512, 3], 512), ([300, 0, 64, 65], 301),
])
def test_layout(kind, ns, max_nodes):
    start = [7 * i for i in range(len(ns))]
    p, cu, kv, table, T = batch(len(ns) + max_nodes, ns, kind, start, 16)
    check_layout(p, cu, kv, table, 16, T, max_nodes)


def test_layout_of_many_rows_with_padding_and_without_pages():
    ns = [1 + i % 64 for i in range(300)]
    p, cu, kv, table, T = batch(3, ns, "random", [i * 13 % 4000 for i in range(300)], 8, pad=77)
    check_layout(p, cu, kv, table, 8, T, 64)
    check_layout(p, cu, kv, None, 8, T, 64)


@pytest.mark.parametrize("max_nodes", [64, 100])
def test_layout_refuses_rows(max_nodes):
    ns = [5, 9, 4, 6, 3]
    def fresh():
        return batch(1, ns, "random", [10, 20, 30, 40, 50], 16, pad=3)
    p, cu, kv, table, T = fresh()
    p[cu[1] + 2] = 2                       # its own parent
    check_layout(p, cu, kv, table, 16, T, max_nodes, ok=False)
    p, cu, kv, table, T = fresh()
    p[cu[2] + 1] = -2
    check_layout(p, cu, kv, table, 16, T, max_nodes, ok=False)
    p, cu, kv, table, T = fresh()
    p[cu[3] + 1] = 1 << 20
    check_layout(p, cu, kv, table, 16, T, max_nodes, ok=False)
    p, cu, kv, table, T = fresh()
    kv[0] = 3                              # fewer keys than nodes
    check_layout(p, cu, kv, table, 16, T, max_nodes, ok=False)
    p, cu, kv, table, T = fresh()
    kv[4] = table.shape[1] * 16 + 1
    check_layout(p, cu, kv, table, 16, T, max_nodes, ok=False)
    p, cu, kv, table, T = fresh()
    table[1, 1] = -1                       # a page that the row has not got
    check_layout(p, cu, kv, table, 16, T, max_nodes, ok=False)
    p, cu, kv, table, T = fresh()
    cu[-1] = T + 2                         # offsets past the nodes
    check_layout(p, cu, kv, table, 16, T, max_nodes, ok=False)


def test_layout_of_a_row_of_more_nodes_than_words():
    p, cu, kv, table, T = batch(2, [65, 4], "random", [0, 0], 16)
    check_layout(p, cu, kv, table, 16, T, 64, ok=False)
    p, cu, kv, table, T = batch(2, [129, 4], "random", [0, 0], 16)
    check_layout(p, cu, kv, table, 16, T, 128, ok=False)


def test_positions_past_32_bits():
    p, cu, kv, _, T = batch(2, [9, 4], "random", [0, 0], 16)
    check_layout(p, cu, kv + (1 << 40), None, 16, T, 64)


@pytest.mark.parametrize("kind", ["random", "chain", "star", "forest", "binary"])
@pytest.mark.parametrize("ns,max_path,vocab", [
    ([1], 1, 5), ([26], 16, 3), ([64, 0, 1, 63], 64, 2), ([7] * 200, 4, 4), ([512, 65, 64], 512, 2),
    ([100, 3], 1, 3), ([300], 7, 2),
])
def test_accept(kind, ns, max_path, vocab):
    rng = np.random.default_rng(sum(ns) + max_path)
    p, cu, kv, table, T = batch(5, ns, kind, [0] * len(ns), 16)
    tokens = rng.integers(0, vocab, T)
    choice = rng.integers(-1 if kind == "star" else 0, vocab, T)
    if kind == "chain":                     # the whole chain is accepted
        choice[:-1] = tokens[1:]
    active = rng.random(len(ns)) < 0.8
    for act in (None, active):
        path, keep, y = tree_accept(dev(tokens), dev(p), dev(choice), dev(cu), max_path,
                                    active=None if act is None else dev(act))
        wpath, wkeep, wy = OT.tree_accept(tokens, p, choice, cu, max_path, act)
        assert path.tolist() == wpath.tolist()
        assert keep.tolist() == wkeep.tolist() and y.tolist() == wy.tolist()


def test_accept_ends_on_any_parents():
    """Parents that point forward or at themselves are no children; rows out of range are refused."""
    tokens, choice = dev([1, 1, 1, 1]), dev([1, 1, 1, 1])
    path, keep, y = tree_accept(tokens, dev([3, 1, 1, -5], torch.int32), choice, dev([0, 4]), 4)
    assert path.tolist() == [[0, -1, -1, -1]] and keep.tolist() == [1] and y.tolist() == [1]
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    path, keep, y = tree_accept(tokens, dev([-1, 0, 1, 2], torch.int32), choice, dev([0, 3, 9]), 4,
                                error=err)
    assert keep.tolist() == [3, 0] and y.tolist() == [1, -1] and err.item() == 1
    assert path.tolist() == [[0, 1, 2, -1], [-1] * 4]


def test_a_graph_of_both_is_replayed():
    ns = [26, 3, 64]
    p, cu, kv, table, T = batch(8, ns, "random", [5, 60, 7], 16)
    rng = np.random.default_rng(0)
    tokens, choice = dev(rng.integers(0, 3, T)), dev(rng.integers(0, 3, T))
    args = [dev(p), dev(cu), dev(kv), dev(table, torch.int32)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lay = tree_layout(*args, 16)
        acc = tree_accept(tokens, args[0], choice, args[1], 8)
    for seed in range(3):
        p2, cu2, kv2, t2, _ = batch(seed, ns, "forest", [9, 1, 30 + seed], 16)
        args[0].copy_(dev(p2)); args[2].copy_(dev(kv2))
        tokens.copy_(dev(np.random.default_rng(seed).integers(0, 3, T)))
        g.replay()
        torch.cuda.synchronize()
        for got, want in zip((*lay, *acc), (*tree_layout(*args, 16),
                                            *tree_accept(tokens, args[0], choice, args[1], 8))):
            assert torch.equal(got, want)
