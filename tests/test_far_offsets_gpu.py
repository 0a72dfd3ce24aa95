"""Elements that lie 2^31 and more behind the beginning of a tensor, in the words that the kernels count in."""
import pytest
import torch

from tokenizer_b200.kernels import ops

pytestmark = pytest.mark.gpu


def test_copies_of_single_bytes_far_behind():
    """Rows of an odd number of bytes are copied a byte at a time: offsets in bytes, 2.5e9 of them a plane."""
    page, pages, row = 64, 9600, 4093
    pool = torch.zeros(3, 1, pages * page, 1, row, dtype=torch.uint8, device="cuda")
    assert pool.stride(0) > 1 << 31 and pool.numel() > 1 << 32
    pool[:, :, -page:] = torch.randint(0, 256, (3, 1, page, 1, row), dtype=torch.uint8).cuda()
    far = pool[:, :, -page:].clone()
    ops.copy_pages(pool, page, [(pages - 1, pages - 2, 63), (pages - 1, 0, 5)])
    assert torch.equal(pool[:, :, -page:], far)
    assert torch.equal(pool[:, :, -2 * page:-page - 1], far[:, :, :63]) and torch.equal(pool[:, :, :5], far[:, :, :5])
    assert not pool[:, :, -page - 1:-page].any() and not pool[:, :, 5:page].any() and not pool[:, :, -3 * page:-2 * page].any()
    # and from the front to the far end
    ops.copy_pages(pool, page, [(0, pages - 1, 5)])
    assert torch.equal(pool[:, :, -page:], far)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("little", [False, True])
def test_keys_far_behind(dtype, little, monkeypatch):
    """A cache of more than 2^31 elements, its last pages in use: common keys apart, and read by every row."""
    from test_shared_prefix import make, near, plain, run
    if not little:
        monkeypatch.setattr(ops, "SHARED_PREFIX_LITTLE", 0)
    b = make(16, 8, 128, 16, [(5, 9)], 2, [40, 3], dtype, seed=4)
    want = plain(b, 0.088)
    used = b["k"].shape[0] // 16
    pages = (1 << 31) // (16 * 8 * 128) + 2 * used
    for name in "kv":
        far = torch.zeros(pages * 16, 8, 128, dtype=dtype, device="cuda")
        far[-used * 16:] = b[name].cuda()
        assert far.numel() - used * 16 * 8 * 128 > 1 << 31
        b[name] = far
    b["table"] = torch.where(b["table"] >= 0, b["table"] + (pages - used), b["table"])
    got = run(b, 0.088)
    b["v"] = b["v"][-used * 16:].cpu()
    near(got, want, b)


def test_draws_from_rows_far_behind():
    rows, vocab = 15000, 150001
    logits = torch.empty(rows, vocab, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    assert logits.numel() > 1 << 31
    logits[-3:] *= 3
    settings = [torch.full((rows,), v, device="cuda") for v in (0.8, 0.9, 0.02)]
    k, u = torch.full((rows,), 300, dtype=torch.int32, device="cuda"), torch.rand(rows, device="cuda")
    out = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    ops.sample_filtered(logits, settings[0], k, settings[1], settings[2], u, out)
    for at in (0, 14316, 14317, rows - 4):              # 2^31 lies in row 14,316
        few = torch.empty(4, dtype=torch.int32, device="cuda")
        part = slice(at, at + 4)
        ops.sample_filtered(logits[part].clone(), settings[0][part], k[part], settings[1][part], settings[2][part], u[part], few)
        assert torch.equal(out[part], few)
    assert (out >= 0).all() and (out < vocab).all()
