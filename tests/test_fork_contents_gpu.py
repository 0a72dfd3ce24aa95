"""What a fork holds, bit for bit: the rows of its begun page in every plane of every group, and its state."""
import pytest
import torch

from test_samples_gpu import DESIGNS, folder_of, run
from tiny import random_ids

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("module, name", DESIGNS)
def test_forks_hold_the_same_bits(module, name, dtype, tmp_path_factory):
    from tokenizer_b200.engine import Engine
    folder, vocab, page = folder_of(module, name, tmp_path_factory)
    engine = Engine.from_folder(folder, dtype=dtype, num_pages=40, page_size=page, max_requests=8)
    cache = engine.cache
    for pool in cache.pools:                     # what nobody has written is not zero
        pool.fill_(3.0)
    for at, length in enumerate((2 * page + 3, 2 * page, page - 1)):
        parent = cache.open(("p", at))
        run(engine, [parent], [random_ids(length, vocab, at)])
        before = [pool.clone() for pool in cache.pools]
        full, begun = divmod(length, page)
        children = cache.fork(parent, [("a", at), ("b", at)])
        for g, (pool, old) in enumerate(zip(cache.pools, before)):
            written = torch.zeros(pool.shape[2], dtype=torch.bool)
            for child in children:
                assert child.tables[g][:full] == parent.tables[g][:full]
                if begun:
                    source, target = parent.tables[g][full] * page, child.tables[g][full] * page
                    assert torch.equal(pool[:, :, target:target + begun], old[:, :, source:source + begun])
                    written[target:target + begun] = True
            assert torch.equal(pool[:, :, ~written], old[:, :, ~written])
        for arena in cache._arenas():
            for child in children:
                assert torch.equal(arena[child.state_slot], arena[parent.state_slot])
        for c in [parent] + children:
            cache.close(c)
