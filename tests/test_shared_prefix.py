"""Sets of rows with common beginnings (host), and attention that reads them once against the definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

from tokenizer_b200.cache import sharing
from tokenizer_b200.kernels import ops


# ---- the sets --------------------------------------------------------------------------------------------------------
def table_of(rows, width=None):
    width = width or max([len(r) for r in rows] + [1])
    return np.array([list(r) + [-1] * (width - len(r)) for r in rows], dtype=np.int32).reshape(len(rows), width)


def test_sets_of_common_beginnings():
    found = lambda rows, usable=None, **kw: sorted(  # noqa: E731
        (sorted(r), n) for r, n in sharing.common_beginnings(table_of(rows), usable or [len(r) for r in rows], **kw))
    assert found([]) == [] and found([[]]) == [] and found([[1, 2]]) == []
    assert found([[1, 2], [3, 4]]) == []
    assert found([[1, 2, 3], [1, 2, 4], [5, 6], [1, 2]]) == [([0, 1, 3], 2)]
    # pages a row does not hold whole are not its to share
    assert found([[1, 2, 3], [1, 2, 3]], [1, 3]) == [([0, 1], 1)] and found([[1], [1]], [0, 1]) == []
    # a short beginning for all against long ones for pairs: 3 * 1 < 2 * 1 * 4; at two pages for all 3 * 4 > 2 * 5
    assert found([[1, 2, 3, 4], [1, 2, 3, 4], [1, 6, 7, 8], [1, 6, 7, 8]]) == [([0, 1], 4), ([2, 3], 4)]
    rows = [[9, 9, 9, 9, 1], [9, 9, 9, 9, 1], [9, 9, 9, 9, 2], [9, 9, 9, 9, 2]]
    assert found(rows) == [([0, 1, 2, 3], 4)]
    assert found([[1, 2], [1, 3]], least=2) == [] and found([[1, 2], [1, 2]], least=2) == [([0, 1], 2)]
    # nothing behind a hole or behind the table is shared
    assert found([[1, -1, 3], [1, -1, 3]]) == [([0, 1], 1)] and found([[-1], [-1]]) == []
    assert found([[1, 2], [1, 2]], [9, 9]) == [([0, 1], 2)]
    # beginnings too short to count do not hide longer ones of parts
    assert found([[1, 2, 3], [1, 2, 3], [1, 4, 5]], least=3) == [([0, 1], 3)]


def test_the_plan_cuts_sets_into_tiles():
    rows = [[1, 2]] * 5 + [[7]] + [[3]] * 2
    shared, members, tiles = sharing.plan(table_of(rows), [len(r) for r in rows], 16, 2)
    assert shared.tolist() == [32] * 5 + [0] + [16] * 2
    assert members.tolist() == [0, 1, 2, 3, 4, 6, 7]
    assert tiles.tolist() == [[0, 2, 32, 0], [2, 2, 32, 0], [4, 1, 32, 0], [5, 2, 16, 0]]
    shared, members, tiles = sharing.plan(table_of([[1], [2]]), [1, 1], 16, 2)
    assert tiles.shape == (0, 4) and members.size == 0 and not shared.any()
    with pytest.raises(ValueError):
        sharing.plan(table_of(rows), [1] * 8, 16, 0)


@pytest.fixture(params=["apart", "by size"])
def form(request, monkeypatch):
    """Common keys read apart however little there is to read, and as the rule on sizes has it."""
    if request.param == "apart":
        monkeypatch.setattr(ops, "SHARED_PREFIX_LITTLE", 0)


# ---- the attention -----------------------------------------------------------------------------------------------------
def make(nh, nkv, d, page, sets, alone, own, dtype, seed=0, sink=False, idle=()):
    """A batch in shuffled order: `sets` of (rows, pages in common), `alone` rows that share nothing, own[i % len] keys each."""
    g = torch.Generator().manual_seed(seed)
    rows = [(s, pages) for s, (n, pages) in enumerate(sets) for _ in range(n)] + [(-1, 0)] * alone
    own = [own[i % len(own)] for i in range(len(rows))]
    n_pages = sum(p for _, p in sets) + sum(-(-k // page) for k in own) + 3
    free = iter(torch.randperm(n_pages, generator=g).tolist())
    begins = [[next(free) for _ in range(p)] for _, p in sets]
    lists = [(begins[s] if s >= 0 else []) + [next(free) for _ in range(-(-k // page))] for (s, _), k in zip(rows, own)]
    order = torch.randperm(len(rows), generator=g).tolist()
    lists, own, rows = [lists[i] for i in order], [own[i] for i in order], [rows[i] for i in order]
    width = max(len(p) for p in lists) + 1
    table = table_of(lists, width)
    keys = [p * page for _, p in rows]
    pos = [k + n - 1 for k, n in zip(keys, own)]
    row_req = [-1 if r in idle else r for r in range(len(rows))]
    most = ops.shared_prefix_tile_members(nh, nkv)
    members, tiles = [], []
    for s in range(len(sets)):
        of = [r for r in range(len(rows)) if rows[r][0] == s]
        for at in range(0, len(of), most):
            tiles.append([len(members), len(of[at:at + most]), sets[s][1] * page, 0])
            members += of[at:at + most]
    draw = lambda *shape: torch.randn(*shape, generator=g).to(dtype)  # noqa: E731
    return dict(q=1.5 * draw(len(rows), nh * d), k=draw(n_pages * page, nkv, d), v=draw(n_pages * page, nkv, d), table=torch.tensor(table),
                row_req=row_req, pos=pos, shared=keys, members=members, tiles=tiles, nh=nh, nkv=nkv, d=d, page=page,
                sink=torch.randn(nh, generator=g) if sink else None)


def plain(b, scale, softcap=None):
    """[rows, heads, size] in 64 bits, a row and a head at a time."""
    out = torch.zeros(len(b["pos"]), b["nh"], b["d"], dtype=torch.float64)
    q = b["q"].double().view(-1, b["nh"], b["d"])
    for r, p in enumerate(b["pos"]):
        if b["row_req"][r] < 0:
            continue
        slots = [int(b["table"][b["row_req"][r], i // b["page"]]) * b["page"] + i % b["page"] for i in range(p + 1)]
        k, v = b["k"][slots].double(), b["v"][slots].double()
        for h in range(b["nh"]):
            g = h // (b["nh"] // b["nkv"])
            x = k[:, g] @ q[r, h] * scale
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            if b["sink"] is not None:
                x = torch.cat([x, b["sink"][h:h + 1].double()])
            out[r, h] = torch.softmax(x, 0)[:p + 1] @ v[:, g]
    return out


def run(b, scale, softcap=None, n_pad_tiles=0):
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.full_like(b["q"], 7.0).cuda()
    tiles = ints(b["tiles"] + [[0, 0, 0, 0]] * n_pad_tiles).view(-1, 4)
    ops.shared_prefix_attention(b["q"].cuda(), b["k"].cuda(), b["v"].cuda(), out, b["table"].cuda(), ints(b["row_req"]), ints(b["pos"]),
                                ints(b["shared"]), ints(b["members"]), tiles, b["nh"], b["nkv"], b["d"], b["page"], scale,
                                sink=None if b["sink"] is None else b["sink"].cuda(), softcap=softcap)
    return out.view(-1, b["nh"], b["d"]).double().cpu()


# What an output element may be off.  32-bit: q.k has d products of 2^-24 each relative to sum |q k| <= |q| |k|; an error e of a
# score changes a weight by e; |score * scale| errors stay below 2^-24 * (d / 2 + 4) * sum|qk| * scale, here sum|qk| * scale < 40
# for all tests: 40 * 2^-24 * 132 < 3.2e-4 as a bound, and outputs are averages of |v| < 5.5: the bound is loose by the
# square root of d (random signs), 2^-24 * 40 * 12 * 5.5 = 1.6e-4 stays one.  bfloat16: probabilities are rounded,
# at most half a step 2^-8 relative, the sum of p |v| / sum p <= 5.5 at worst, on the average below 1; output rounded by 2^-8 |out|.
def near(got, want, b):
    seen = [r for r in range(len(b["pos"])) if b["row_req"][r] >= 0]
    if b["q"].dtype == torch.float32:
        assert (got[seen] - want[seen]).abs().max() <= 1.6e-4
    else:
        # |v| of the weighted average: at most sum p |v| / sum p, bounded by the largest |v| of the pool
        assert ((got[seen] - want[seen]).abs() <= 2 ** -8 * want[seen].abs() + 2 ** -8 * float(b["v"].abs().max())).all()
        # random signs: the relative 2-norm error is that of two roundings
        assert (got[seen] - want[seen]).norm() <= 2 * 2 ** -8 * want[seen].norm()
    assert torch.equal(got[[r for r in range(len(got)) if r not in seen]], torch.full_like(got[:len(got) - len(seen)], 7.0))


HEADS = [(14, 2, 64, 16), (12, 2, 128, 16), (28, 4, 128, 8), (8, 8, 64, 32), (16, 1, 128, 16), (4, 2, 48, 5), (6, 1, 20, 3), (2, 2, 256, 16), (3, 3, 1, 4),
         (14, 2, 64, 24), (40, 2, 64, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nh, nkv, d, page", HEADS)
@pytest.mark.parametrize("sets, alone, own", [([(4, 3)], 0, [5, 1, 40]), ([(2, 1), (3, 20), (5, 9)], 3, [1, 33, 130, 64]), ([(41, 6)], 1, [17, 3]),
                                              ([], 3, [1, 70])])
def test_against_the_definition(nh, nkv, d, page, sets, alone, own, dtype, form):
    b = make(nh, nkv, d, page, sets, alone, own, dtype, seed=d + page, sink=alone == 1)
    near(run(b, 1 / math.sqrt(d)), plain(b, 1 / math.sqrt(d)), b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("keys_pages, own", [(64, [1]), (130, [200, 7]), (1, [1500]), (257, [300])])
@pytest.mark.parametrize("softcap", [None, 2.5])
def test_long_beginnings(keys_pages, own, softcap, dtype, form):
    b = make(14, 2, 64, 16, [(9, keys_pages)], 2, own, dtype, seed=keys_pages, sink=softcap is not None)
    near(run(b, 0.125, softcap), plain(b, 0.125, softcap), b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("listed", [False, True])
def test_idle_rows_padded_tiles_and_garbage_behind_the_last_key(listed, dtype, form):
    """Idle rows among the members (the first one too), as -1, or not at all."""
    b = make(14, 2, 64, 16, [(600, 5)] if listed else [(6, 5)], 2, [3, 20], dtype, idle=(0, 1, 4))
    if listed:
        first = b["tiles"][0][0]
        b["row_req"][b["members"][first]] = -1
        b["members"][first + 1] = -1 if b["row_req"][b["members"][first + 1]] < 0 else b["members"][first + 1]
    else:
        b["members"] = [r for r in b["members"] if b["row_req"][r] >= 0]
        b["tiles"][0][1] = len(b["members"])
    want = plain(b, 0.125)
    # everything that no row sees: NaN in keys, infinities in values
    seen = torch.zeros(b["k"].shape[0], dtype=torch.bool)
    for r, p in enumerate(b["pos"]):
        if b["row_req"][r] >= 0:
            seen[[int(b["table"][r, i // 16]) * 16 + i % 16 for i in range(p + 1)]] = True
    b["k"][~seen] = float("nan")
    b["v"][~seen] = float("inf")
    near(run(b, 0.125, n_pad_tiles=0 if listed else 5), want, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_whose_own_keys_are_none(dtype, form):
    """A position at the end of the common keys: the row sees the tile's keys alone; a row that sees nothing is zero."""
    b = make(14, 2, 64, 16, [(5, 4)], 1, [16], dtype)
    for r in range(6):
        b["pos"][r] = b["shared"][r] - 1
    b["pos"] = [max(p, -1) for p in b["pos"]]
    got = run(b, 0.125)
    alone = b["shared"].index(0)
    assert not got[alone].any()
    b["row_req"] = [-1 if r == alone else r for r in range(6)]
    got[alone] = 7.0
    near(got, plain(b, 0.125), b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_scores_and_repeats(dtype, form):
    """Scores far apart (one key holds all the weight), and the same bits every time, alone and in a graph beside another stream."""
    b = make(12, 2, 128, 16, [(20, 40)], 3, [90, 5], dtype)
    b["q"] *= 6
    got, want = run(b, 0.3), plain(b, 0.3)
    # errors of scores of up to 400 grow with them: |dp| <= ds, ds <= 400 * 2^-24 * 12
    assert (got - want).norm() <= (2 * 2 ** -8 if dtype == torch.bfloat16 else 400 * 12 * 2 ** -24 * 4) * want.norm()
    for _ in range(5):
        assert torch.equal(run(b, 0.3), got)


@pytest.mark.gpu
def test_captured_graphs_on_two_streams(form):
    b = make(14, 2, 64, 16, [(9, 33)], 2, [40, 300], torch.bfloat16)
    c = make(14, 2, 64, 16, [(9, 30)], 2, [70, 20], torch.bfloat16, seed=3)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    want, graphs, outs, streams, keep = [run(x, 0.125) for x in (b, c)], [], [], [], []
    for x in (b, c):
        t = [x[n].cuda() for n in "qkv"] + [torch.zeros_like(x["q"]).cuda(), x["table"].cuda()] + \
            [ints(x[n]) for n in ("row_req", "pos", "shared", "members", "tiles")]
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            ops.shared_prefix_attention(*t, 14, 2, 64, 16, 0.125)
        graphs.append(graph), outs.append(t[3]), streams.append(stream), keep.append(t)
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert torch.equal(out.view(-1, 14, 64).double().cpu(), w)


@pytest.mark.gpu
def test_refusals_and_nothing_to_do():
    b = make(14, 2, 64, 16, [(4, 3)], 0, [5], torch.bfloat16)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q, k, v = (b[n].cuda() for n in "qkv")
    good = dict(q=q, k_pool=k, v_pool=v, out=torch.full_like(q, 7), block_table=b["table"].cuda(), row_req=ints(b["row_req"]),
                pos=ints(b["pos"]), shared=ints(b["shared"]), members=ints(b["members"]), tiles=ints(b["tiles"]), nh=14, nkv=2, d=64, page=16,
                scale=0.125)
    for change in [dict(q=q.half()), dict(q=q.float()), dict(k_pool=k[:-1]), dict(nh=7), dict(nkv=4), dict(d=300), dict(page=0),
                   dict(pos=ints(b["pos"]).long()), dict(pos=ints(b["pos"])[:2]), dict(tiles=ints(b["tiles"])[:, :3]), dict(shared=ints([0])),
                   dict(sink=torch.zeros(3, device="cuda")), dict(sink=torch.zeros(14, device="cuda").half()), dict(softcap=-1.0),
                   dict(softcap=0.0), dict(block_table=good["block_table"][0]), dict(k_pool=k.transpose(0, 1)), dict(out=q[:, ::2])]:
        with pytest.raises((ValueError, TypeError)):
            ops.shared_prefix_attention(**{**good, **change})
    none = {n: good[n][:0] for n in ("q", "out", "row_req", "pos", "shared", "members", "tiles")}
    ops.shared_prefix_attention(**{**good, **none})
    assert (good["out"] == 7).all()
    with pytest.raises(ops.KernelError):
        ops.shared_prefix_attention(**{**good, "q": q.cpu()})
