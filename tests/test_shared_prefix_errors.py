"""What the attention behind a shared prefix says when something is wrong that only the device can see."""
import ctypes

import pytest
import torch

from tokenizer_b200.kernels import ops


def test_an_unaligned_base_is_called_that(monkeypatch):
    """Reason 2 of a kernel whose blocks do not wait on one another."""
    value = ctypes.c_int(7 * 16 + 2)
    monkeypatch.setattr(ops, "_error_word", (value, 0))
    monkeypatch.setattr(ops, "_registered", {})
    with pytest.raises(ops.KernelError, match="shared_prefix_tcgen05: .*not aligned"):
        ops.raise_if_error()
    assert value.value == 0


def call(b, members=None, tiles=None):
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.zeros_like(b["q"]).cuda()
    ops.shared_prefix_attention(b["q"].cuda(), b["k"].cuda(), b["v"].cuda(), out, b["table"].cuda(), ints(b["row_req"]), ints(b["pos"]),
                                ints(b["shared"]), ints(b["members"] if members is None else members),
                                ints(b["tiles"] if tiles is None else tiles).view(-1, 4), b["nh"], b["nkv"], b["d"], b["page"], 0.125)
    torch.cuda.synchronize()
    return out.view(-1, b["nh"], b["d"]).double().cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nh, nkv, d", [(14, 2, 64), (12, 2, 128), (6, 1, 20)])
def test_tiles_that_are_none_raise(nh, nkv, d, dtype, monkeypatch):
    """Too many members, members behind the list's end or in front of its beginning, rows that the batch does not have."""
    from test_shared_prefix import make, near, plain
    monkeypatch.setattr(ops, "SHARED_PREFIX_LITTLE", 0)
    most = ops.shared_prefix_tile_members(nh, nkv)
    b = make(nh, nkv, d, 16, [(most + 1, 3)], 1, [9, 20], dtype)
    rows, keys, want = b["members"], 48, plain(b, 0.125)
    assert len(b["tiles"]) == 2
    ops.raise_if_error()
    near(call(b), want, b)
    ops.raise_if_error()
    for members, tiles in [(rows, [[0, most + 1, keys, 0]]), (rows, [[0, most, keys, 0], [most, 2, keys, 0]]),
                           (rows, [[-1, 2, keys, 0]]), (rows, [[2 ** 31 - 1, 2, keys, 0]]), ([], [[0, 1, keys, 0]]),
                           (rows[:-1] + [most + 2], b["tiles"]), ([2 ** 31 - 1] + rows[1:], b["tiles"])]:
        call(b, members, tiles)
        with pytest.raises(ops.KernelError, match="shared_prefix.*tile"):
            ops.raise_if_error()
    near(call(b), want, b)
    ops.raise_if_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nh, nkv, d", [(14, 2, 64), (6, 1, 20)])
def test_a_tile_may_list_more_places_than_the_batch_has_rows(nh, nkv, d, dtype, monkeypatch):
    """Members that are none (-1) take places too: five rows at the end of 24."""
    from test_shared_prefix import make, near, plain
    monkeypatch.setattr(ops, "SHARED_PREFIX_LITTLE", 0)
    b = make(nh, nkv, d, 16, [(5, 3)], 1, [9, 20], dtype)
    members = [-1] * 19 + b["members"]
    near(call(b, members, [[0, 24, 48, 0]]), plain(b, 0.125), b)
    ops.raise_if_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale, softcap", [(-0.3, None), (-0.3, 20.0), (0.0, None), (0.0, 20.0), (1e-38, 20.0)])
def test_scales_of_any_sign(scale, softcap, d, dtype, monkeypatch):
    """A factor that turns the order of the scores around, or makes them all alike."""
    from test_shared_prefix import make, near, plain, run
    monkeypatch.setattr(ops, "SHARED_PREFIX_LITTLE", 0)
    b = make(12, 2, d, 16, [(20, 40)], 3, [90, 5], dtype)
    b["q"] *= 6
    got, want = run(b, scale, softcap), plain(b, scale, softcap)
    assert torch.isfinite(got).all()
    if dtype == torch.bfloat16:
        near(got, want, b)
    else:
        # scores of up to 400, each off by 12 steps of 2^-24 of that; outputs move by as much of what they weigh
        assert (got - want).norm() <= 400 * 12 * 2 ** -24 * 4 * max(want.norm(), 1.0)
