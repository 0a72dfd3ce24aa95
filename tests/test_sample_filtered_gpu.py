"""The draw behind top-k, top-p and min-p against its definition in 64 bits, id for id: a draw differs from the definition's
only where u * K falls within the errors of the sums (below 1e-11 of the whole) of a candidate's edge, which for these some
thousand draws has a chance of less than one in a thousand; the inputs are seeded, so it happens always or never."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def plain_draw(logits, temperature, top_k, top_p, min_p, u):
    """One row, from the definition."""
    l = np.asarray(logits, dtype=np.float64)
    usable = [i for i in range(len(l)) if not math.isnan(l[i]) and l[i] > -math.inf]
    if not usable:
        return 0
    best = max(usable, key=lambda i: (l[i], -i))
    if not temperature > 0 or np.isnan(l).any() or l[best] == math.inf:
        return best
    order = np.lexsort((np.arange(len(l)), -l))
    with np.errstate(over="ignore"):
        w = np.exp((l[order] - l[best]) / float(temperature))
    k = len(l) if top_k <= 0 else min(int(top_k), len(l))
    w[k:] = 0.0
    sums = np.cumsum(w)
    kept = k
    if top_p < 1:
        kept = min(kept, int(np.argmax(sums >= max(float(top_p), 0.0) * sums[-1])) + 1)
    if min_p > 0:
        kept = min(kept, max(1, int((w >= min(float(min_p), 1.0)).sum())))
    at = int(np.searchsorted(sums[:kept], float(u) * sums[kept - 1], side="right"))
    return int(order[min(at, kept - 1)])


def run(logits, temperature, top_k, top_p, min_p, u):
    from tokenizer_b200.kernels import ops
    out = torch.full((logits.shape[0],), -7, dtype=torch.int32, device="cuda")
    to = lambda v, t: None if v is None else torch.tensor(np.asarray(v), dtype=t, device="cuda")  # noqa: E731
    ops.sample_filtered(torch.tensor(logits, dtype=torch.float32, device="cuda"), to(temperature, torch.float32), to(top_k, torch.int32),
                        to(top_p, torch.float32), to(min_p, torch.float32), to(u, torch.float32), out)
    return out.cpu().tolist()


def compare(logits, temperature, top_k, top_p, min_p, u):
    n = len(logits)
    with np.errstate(over="ignore"):
        logits = np.asarray(logits, dtype=np.float32)
    f = lambda v: np.asarray(v, dtype=np.float32)  # noqa: E731
    want = [plain_draw(logits[r], f(temperature)[r], top_k[r], f(top_p)[r], f(min_p)[r], f(u)[r]) for r in range(n)]
    assert run(logits, temperature, top_k, top_p, min_p, u) == want


def settings(rng, n, vocab):
    temperature = np.where(rng.random(n) < 0.15, 0.0, rng.uniform(0.2, 3.0, n))
    top_k = np.where(rng.random(n) < 0.5, 0, np.exp(rng.uniform(0, math.log(vocab + 1), n)).astype(int))
    top_p = np.where(rng.random(n) < 0.4, 1.0, rng.uniform(0.0, 1.0, n))
    min_p = np.where(rng.random(n) < 0.6, 0.0, 10 ** rng.uniform(-4, 0, n))
    return temperature, top_k, top_p, min_p, rng.random(n).astype(np.float32)


@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 511, 513, 2047, 2049, 3001, 8193, 24577, 50001, 151936, 420001])
def test_sizes(vocab):
    rng = np.random.default_rng(vocab)
    n = 24 if vocab < 100000 else 6
    compare(rng.normal(size=(n, vocab)) * rng.uniform(0.3, 4.0, (n, 1)), *settings(rng, n, vocab))


@pytest.mark.parametrize("step", [0.0, 4.0, 0.25, 0.01])
@pytest.mark.parametrize("vocab", [700, 9000, 70001])
def test_equal_logits_go_by_id(vocab, step):
    rng = np.random.default_rng(5)
    logits = rng.normal(size=(12, vocab))
    logits = np.zeros_like(logits) if step == 0 else np.round(logits / step) * step
    compare(logits, *settings(rng, 12, vocab))


@pytest.mark.parametrize("vocab", [1500, 30000])
@pytest.mark.parametrize("what", ["outlier", "far below", "mostly -inf", "huge range", "hot", "cold", "signed zeros"])
def test_unusual_rows(what, vocab):
    rng = np.random.default_rng(9)
    logits = rng.normal(size=(10, vocab))
    temperature, top_k, top_p, min_p, u = settings(rng, 10, vocab)
    if what == "outlier":
        logits[:, 3] += 60
    elif what == "far below":
        logits[:, 3] = -1e30
        logits[:, 8] = -np.inf
    elif what == "mostly -inf":
        logits[:, 7:] = -np.inf
    elif what == "huge range":
        logits *= 1e38
    elif what == "hot":
        temperature = np.full(10, 1e6)
    elif what == "cold":
        temperature = np.full(10, 1e-30)
    else:
        logits = np.where(logits > 0, 0.0, -0.0)
    compare(logits, temperature, top_k, top_p, min_p, u)


@pytest.mark.parametrize("top_k", [0, 3000])
@pytest.mark.parametrize("vocab", [2500, 9000, 40001])
def test_a_nucleus_that_ends_behind_what_min_p_keeps(vocab, top_k):
    """min-p keeps some hundred to two thousand candidates, the nucleus would keep more."""
    rng = np.random.default_rng(vocab)
    n = 24
    logits = rng.normal(size=(n, vocab))
    compare(logits, np.full(n, 1.3), np.full(n, top_k), rng.uniform(0.8, 0.9999, n), 10 ** rng.uniform(-2.0, -0.7, n), rng.random(n).astype(np.float32))


def test_edges_of_the_settings():
    logits = np.tile(np.log(np.array([4.0, 2.0, 1.0, 1.0])), (12, 1))
    one, half = 1.0, 0.5
    rows = [(1, 0, one, 0, 0.0), (1, 0, one, 0, 0.9999999), (1, 1, one, 0, 0.99), (1, 4, one, 0, 0.99), (1, 99, one, 0, 0.99),
            (1, -3, one, 0, 0.99), (1, 0, 0.0, 0, 0.99), (1, 0, -1.0, 0, 0.99), (1, 0, half, 0, 0.99), (1, 0, one, 1.0, 0.99),
            (1, 0, one, 5.0, 0.99), (float("nan"), 0, one, 0, 0.99)]
    got = run(logits, *[[r[i] for r in rows] for i in range(5)])
    assert got == [0, 3, 0, 3, 3, 3, 0, 0, 0, 0, 0, 0]
    # nothing but a temperature; NaN filters filter nothing; a number outside [0, 1) is brought inside
    assert run(logits[:2], [1, 1], None, None, None, [0.4, 0.6]) == [0, 1]
    nan = float("nan")
    assert run(logits[:4], [1] * 4, [0] * 4, [nan, 1, 2, 1], [0, nan, 0, 0], [0.99, 0.99, 1.0, -1.0]) == [3, 3, 3, 0]


def test_rows_without_a_finite_sum_are_greedy():
    nan, inf = float("nan"), float("inf")
    logits = [[1.0, nan, 3.0, 2.0], [nan] * 4, [-inf] * 4, [0.0, inf, 1.0, inf], [-inf, nan, -inf, -inf]]
    assert run(np.array(logits), [1.0] * 5, [0] * 5, [1.0] * 5, [0.0] * 5, [0.99] * 5) == [2, 0, 0, 1, 0]


def test_a_row_does_not_depend_on_its_batch_and_repeats():
    rng = np.random.default_rng(2)
    logits = (2 * rng.normal(size=(300, 5003))).astype(np.float32)
    s = settings(rng, 300, 5003)
    whole = run(logits, *s)
    assert whole == run(logits, *s)
    for r in (0, 7, 299):
        assert run(logits[r:r + 1], *[v[r:r + 1] for v in s]) == [whole[r]]


def test_share_of_each_id():
    """Over a grid of u every kept id gets its share of the draws, to one place of the grid."""
    logits = np.array([0.3, 2.0, -1.0, 1.0, 0.3, -4.0])
    n = 4096
    got = run(np.tile(logits, (n, 1)), [0.7] * n, [5] * n, [0.95] * n, [0.001] * n, (np.arange(n) / n))
    order = [1, 3, 0, 4, 2]
    w = np.exp((logits[order] - 2.0) / 0.7)
    kept = int(np.argmax(np.cumsum(w) >= 0.95 * w.sum())) + 1
    share = w[:kept] / w[:kept].sum()
    for i, s in zip(order[:kept], share):
        assert abs(got.count(i) - n * s) <= 1.001


def test_captured_and_on_another_stream():
    from tokenizer_b200.kernels import ops
    torch.manual_seed(1)
    logits = torch.randn(5, 30011, device="cuda")
    t, p = torch.full((5,), 0.9, device="cuda"), torch.full((5,), 0.9, device="cuda")
    u, out = torch.rand(5, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    ops.sample_filtered(logits, t, None, p, None, u, out)
    first = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.sample_filtered(logits, t, None, p, None, u, out)
        out.zero_()
        graph.replay()
    side.synchronize()
    assert torch.equal(out, first)
    logits.neg_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    again = out.clone()
    ops.sample_filtered(logits, t, None, p, None, u, out)
    assert torch.equal(out, again)


def test_no_rows_and_refusals():
    from tokenizer_b200.kernels import ops
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    ids = z(2, dtype=torch.int32)
    ops.sample_filtered(z(0, 10), z(0), None, None, None, z(0), z(0, dtype=torch.int32))
    for bad in [(z(2, 0), z(2), None, None, None, z(2), ids), (z(2, 4).half(), z(2), None, None, None, z(2), ids),
                (z(2, 4), z(3), None, None, None, z(2), ids), (z(2, 4), None, None, None, None, z(2), ids),
                (z(2, 4), z(2), z(2), None, None, z(2), ids), (z(2, 4), z(2), None, z(1), None, z(2), ids),
                (z(2, 4), z(2), None, None, None, z(2), z(2)), (z(8), z(2), None, None, None, z(2), ids),
                (z(4, 2).t(), z(2), None, None, None, z(2), ids)]:
        with pytest.raises(ValueError):
            ops.sample_filtered(*bad)
