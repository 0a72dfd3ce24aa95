"""Several answers to one prompt where slots or pages run short, on the host: who is served first, what waits and what is computed again."""
import random

import pytest

from test_fork import CHUNK, FULL, STATE, WINDOW, ForkingEngine, alone, answers, finish, hold
from tiny import random_ids
from tokenizer_b200.cache import CachePlan, OutOfPages
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


# ---- room for what follows a fork ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("needs", [[FULL], [FULL, WINDOW], [WINDOW, CHUNK, STATE]])
@pytest.mark.parametrize("length", [3, 4, 8, 11, 24])
@pytest.mark.parametrize("n_new", [0, 1, 5, 9])
def test_as_many_forks_as_can_take_their_next_tokens(needs, length, n_new):
    for pages in range(8, 24):
        plan = CachePlan(needs, pages, 4, 12)
        parent = hold(plan, "p", length)
        n = plan.can_fork(parent, n_new)
        children = plan.fork(parent, list(range(n)))
        for child in children:
            plan.reserve(child, n_new)
        plan.check()
        if n < 11:                               # pages are what is short: one more would not do
            try:
                more, = plan.fork(parent, ["more"])
            except OutOfPages:
                continue
            assert not plan.can_reserve(more, n_new)


def test_forks_leave_the_pages_that_others_need_next():
    """A prompt that ends on a page's end, a younger request in the middle of its answer, few pages left."""
    for pages in range(5, 14):
        s = Scheduler(Engine(num_pages=pages), max_batch_size=8, token_budget=64)
        ids = s.add_samples(random_ids(8, 50, 1), answers(6))
        young = s.add_request(random_ids(3, 50, 2), GenerateParams(max_tokens=5))
        s.step()
        needed = sum(s.cache.pages_missing(r.cache, 1)[0] for r in s.running)
        assert len(s.running) >= 2 and needed <= s.cache.allocators[0].available, pages
        out = finish(s)
        assert [out[i].tokens for i in ids] == [alone(random_ids(8, 50, 1), p) for p in answers(6)]
        assert out[young].tokens == alone(random_ids(3, 50, 2), GenerateParams(max_tokens=5))
