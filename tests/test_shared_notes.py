"""Which models have their steps' common beginnings looked for: those whose attention reads them."""
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")

from tokenizer_b200.cache import CachePlan
from tokenizer_b200.engine.step import Engine
from tokenizer_b200.parts.attention import GQAttention, SharedBeginnings
from tokenizer_b200.parts.base import CacheNeed, KVNeed


def notes(dtype, page, layers):
    """`Engine._shared_notes` for layers of (heads, key/value heads, lanes, window)."""
    blocks = []
    for nh, nkv, d, window in layers:
        mixer = GQAttention.__new__(GQAttention)
        mixer.nh, mixer.nkv, mixer.d, mixer.window = nh, nkv, d, window
        blocks.append(SimpleNamespace(mixer=mixer))
    plan = CachePlan([CacheNeed(kv=KVNeed(nkv, d, window)) for _, nkv, d, window in layers], 8, page, 2)
    bindings = [SimpleNamespace(group=plan.group_of_call[i]) for i in range(len(layers))]
    order = [SimpleNamespace(layer=i) for i in range(len(layers))]
    return Engine._shared_notes(SimpleNamespace(runtime=SimpleNamespace(dtype=dtype), cache=plan, bindings=bindings,
                                                model=SimpleNamespace(blocks=blocks, order=order)))


@pytest.mark.parametrize("dtype, page, layers, groups", [
    (torch.bfloat16, 16, [(14, 2, 64, None)], [0]),
    (torch.bfloat16, 16, [(4, 2, 96, None)], []),                # lanes of a head, heads of a group, keys of a page that the
    (torch.bfloat16, 16, [(40, 2, 64, None)], []),               # tensor-core kernels do not take
    (torch.bfloat16, 12, [(14, 2, 64, None)], []),
    (torch.float32, 12, [(40, 2, 96, None)], [0]),
    (torch.float32, 16, [(2, 1, 300, None)], []),
    (torch.bfloat16, 16, [(14, 2, 64, 32), (14, 2, 64, None), (4, 4, 128, None)], [1, 2]),
    (torch.bfloat16, 16, [(14, 2, 64, 32), (6, 6, 80, None)], []),
])
def test_notes_are_made_for_what_reads_them(dtype, page, layers, groups):
    made = notes(dtype, page, layers)
    assert [n.group for n in made] == groups
    for n in made:
        assert isinstance(n, SharedBeginnings) and n.page_size == page


def test_a_group_of_several_kinds_of_readers_has_tiles_that_all_of_them_take():
    made = notes(torch.bfloat16, 16, [(14, 2, 64, None), (4, 2, 64, None), (40, 2, 64, None)])
    assert [n.tile_members for n in made] == [2 * (128 // 7)]
