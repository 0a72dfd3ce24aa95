"""Several answers to one prompt where slots or pages run short, on the host: who is served first, what waits and what is computed again."""
import random

import pytest

from test_fork import ForkingEngine, alone, answers, finish
from tiny import random_ids
from tokenizer_b200.engine.generate import GenerateParams
from tokenizer_b200.engine.scheduler import Scheduler


class Engine(ForkingEngine):
    """A fake that forgets what a cache held when its object's address is used again."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.cache.on_open = lambda cache: self.history.pop(id(cache), None)


# ---- the line ------------------------------------------------------------------------------------------------------------
def check_line(s):
    """Run to the end; after every step the line is in order of arrival, and nobody started in front of an older one that waits."""
    while s.has_work():
        waited, ran = {r.id for r in s.waiting}, {r.id for r in s.running}
        s.step()
        line = [r.id for r in s.waiting]
        assert line == sorted(line)
        started = {r.id for r in s.running} - ran
        still = waited & set(line)
        assert not started or not still or max(started) < min(still)
        s.cache.check()
    for a in s.cache.allocators:
        assert a.all_released()


@pytest.mark.parametrize("share", [False, True])
@pytest.mark.parametrize("pages", [20, 24, 28, 32])
@pytest.mark.parametrize("seed", range(6))
def test_the_line_stays_in_order_of_arrival(pages, share, seed):
    rng = random.Random(100 * pages + seed)
    s = Scheduler(Engine(num_pages=pages, share_prefixes=share), max_batch_size=rng.randint(2, 8), token_budget=rng.choice([8, 64]))
    asked = []
    for at in range(4):
        prompt = random_ids(rng.randint(1, 24), 50, 7 * seed + at)
        params = [GenerateParams(max_tokens=rng.randint(1, 24), temperature=0.8, seed=at + i) for i in range(rng.choice([1, 1, 3, 5]))]
        asked += [(i, prompt, p) for i, p in zip(s.add_samples(prompt, params), params)]
    check_line(s)
    for i, prompt, p in asked:
        assert s.finished[i].tokens == alone(prompt, p)


def test_a_preempted_request_does_not_pass_older_forks():
    s = Scheduler(Engine(num_pages=20), max_batch_size=4, token_budget=64)
    s.add_samples(random_ids(9, 50, 1), answers(5))
    for at in range(3):
        s.add_request(random_ids(6, 50, 20 + at), GenerateParams(max_tokens=20))
    check_line(s)
    assert s.stats.preemptions > 0
