"""The float64 restatement of verification on trees: what is kept is distributed
as the target's own tokens, and one number per node stands for its refusals."""
import itertools

import numpy as np
import pytest

from oracle import tree as ref


def rows(rng, n, v):
    x = rng.random((n, v)) ** 3
    return x / x.sum(-1, keepdims=True)


@pytest.mark.parametrize("drafts", ["drawn", "distinct", "chosen"])
@pytest.mark.parametrize("children", [1, 2, 3])
def test_first_token_is_the_targets(drafts, children):
    """A root with some children: the probability of each first token, summed exactly over all
    drafts, acceptances and what is left, is the target's."""
    rng = np.random.default_rng(children)
    v = 5
    p, q = rows(rng, 1, v)[0], rows(rng, 1, v)[0]
    got = np.zeros(v)
    for xs in itertools.product(range(v), repeat=children):
        if drafts != "drawn" and len(set(xs)) < children:
            continue
        if drafts == "chosen":
            weight = 1.0
            if xs != tuple(range(children)):
                continue
        else:
            weight, left = 1.0, 1.0
            for x in xs:
                weight *= q[x] / left
                left -= q[x] if drafts == "distinct" else 0.0
        A, S, Q, alive = 0.0, 1.0, 1.0, weight
        out = np.ones(v)
        for x in xs:
            if drafts == "chosen":
                yes = p[x] * out[x] / S
                got[x] += alive * yes
                alive *= 1 - yes
                S -= p[x]
                out[x] = 0.0
                continue
            yes = min(1.0, max(p[x] - A * q[x], 0.0) * Q / (q[x] * S))
            got[x] += alive * yes
            alive *= 1 - yes
            A += S / Q
            S = np.maximum(p - A * q, 0.0).sum()
            if drafts == "distinct":
                Q = max(Q - q[x], 2.0 ** -24)
        r = p * out if drafts == "chosen" else np.maximum(p - A * q, 0.0)
        if alive > 0:
            got += alive * (r / r.sum() if r.sum() > 0 else p)
    assert np.abs(got - p).max() < 1e-12


@pytest.mark.parametrize("drafts", ["drawn", "distinct", "chosen"])
def test_oracle_follows_the_formula(drafts):
    """The oracle's normalised residual against A, S and Q, over random trees."""
    rng = np.random.default_rng(5)
    for trial in range(60):
        n, v = int(rng.integers(1, 12)), int(rng.integers(3, 40))
        parent = np.array([-1] + [int(rng.integers(-1, i)) for i in range(1, n)])
        p, q = rows(rng, n, v), rows(rng, n, v)
        tokens = np.zeros(n, int)
        for cur in range(-1, n):
            kids = [i for i in range(1, n) if parent[i] == cur]
            for i, x in zip(kids, rng.permutation(v)[:len(kids)]):
                tokens[i] = x
        u, last = rng.random(n), rng.random(1)
        d = None if drafts == "chosen" else q
        path, count, nxt = ref.verify(p, d, tokens, parent, u, last, [0, n], n, drafts == "distinct")
        cur, way = 0, [0]
        while True:
            A, S, Q, out, got = 0.0, 1.0, 1.0, np.ones(v), None
            for i in [i for i in range(1, n) if parent[i] == cur]:
                x = tokens[i]
                qx = 1.0 if d is None else q[cur, x]
                r = p[cur, x] * out[x] if d is None else max(p[cur, x] - A * q[cur, x], 0.0)
                if u[i] * qx * S < r * Q:
                    got = i
                    break
                if d is None:
                    S -= r
                    out[x] = 0.0
                else:
                    A += S / Q
                    S = np.maximum(p[cur] - A * q[cur], 0.0).sum()
                    Q = max(Q - qx, 2.0 ** -24) if drafts == "distinct" else Q
            if got is None:
                break
            cur = got
            way.append(cur)
        r = p[cur] * out if d is None else np.maximum(p[cur] - A * q[cur], 0.0)
        c = np.cumsum(r if r.sum() > 0 else p[cur])
        assert list(path[0, :count[0]]) == way and nxt[0] == np.flatnonzero(c > last[0] * c[-1])[0]


def test_ways_and_places():
    parent = np.array([-1, 0, 0, 2, 9, -5, 5, 7])  # 9 and 7 are no nodes before theirs
    assert [len(ref.way(parent, 0, i)) - 1 for i in range(8)] == [0, 1, 1, 2, 0, 0, 1, 0]
    pl = ref.places([0, 8], [20], parent, np.array([[0, 1]]), 8, 16, 2)
    assert [x[1] for x in pl] == [12, 13, 13, 14, 12, 12, 13, 12] and [x[3] for x in pl] == [12, 13, 14, 15, 0, 1, 2, 3]
    at = ref.seen([0, 8], np.array([20]), parent, np.array([[0, 1]]), 8, 16, 2, 1, 8, 0)
    assert at[3] == [(0, 15), (0, 14)] and at[4] == [(0, 11), (1, 0)]
