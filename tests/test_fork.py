"""Forks of a request's cache and several answers to one prompt, on the host: who holds which page, what is copied, and that
answers are those that each request would get alone."""
import random

import pytest

from fake_engine import FakeEngine
from tiny import random_ids
from tokenizer_b200.cache import CachePlan, OutOfPages
from tokenizer_b200.engine.generate import GenerateParams, StopReason
from tokenizer_b200.engine.scheduler import Scheduler
from tokenizer_b200.parts.base import CacheNeed, KVNeed, StateNeed

FULL, WINDOW = CacheNeed(kv=KVNeed(1, 8, None)), CacheNeed(kv=KVNeed(2, 8, 9))
CHUNK, STATE = CacheNeed(kv=KVNeed(2, 8, None, chunk=12)), CacheNeed(state=StateNeed((4,)))


class Watched(CachePlan):
    """Remembers what the device side would be told to copy."""

    def on_fork(self, parent, children, copies):
        self.forked = getattr(self, "forked", []) + [(parent.state_slot, [c.state_slot for c in children], copies)]


def hold(plan, name, n):
    cache = plan.open(name)
    for _ in range(n):
        plan.reserve(cache, 1)
        plan.commit(cache, 1)
    return cache


@pytest.mark.parametrize("needs", [[FULL], [FULL, WINDOW], [WINDOW, CHUNK, STATE], [STATE]])
@pytest.mark.parametrize("length", [0, 1, 3, 4, 23, 24, 25, 47])
def test_a_fork_shares_full_pages_and_copies_the_begun_one(needs, length):
    plan = Watched(needs, 40, 4, 6)
    parent = hold(plan, "p", length)
    plan.reserve(parent, 3)                      # pages for a step that has not run are the parent's alone
    before = [a.available for a in plan.allocators]
    children = plan.fork(parent, ["a", "b"])
    plan.check()
    full, begun = divmod(length, 4)
    for child in children:
        assert child.length == length and not child.closed
        for g in range(len(plan.groups)):
            assert child.tables[g][:full] == parent.tables[g][:full]
            assert len(child.tables[g]) == full + (1 if begun else 0)
            if begun:
                assert child.tables[g][full] >= 0 and child.tables[g][full] != parent.tables[g][full]
    slot, slots, copies = plan.forked[-1]
    assert slot == parent.state_slot and slots == [c.state_slot for c in children] and len(set(slots + [slot])) == 3
    for g, pairs in enumerate(copies):
        assert pairs == ([(parent.tables[g][full], c.tables[g][full], begun) for c in children] if begun else [])
        assert before[g] - plan.allocators[g].available == len(pairs)
    # they go on apart, and every page comes back whoever ends first
    for n, cache in enumerate([children[0], parent, children[1]]):
        for _ in range(5 + n):
            plan.reserve(cache, 1)
            plan.commit(cache, 1)
        plan.check()
    order = [parent] + children
    random.Random(length).shuffle(order)
    for cache in order:
        plan.close(cache)
        plan.check()
    assert all(a.all_released() and a.available == a.capacity for a in plan.allocators)


def test_forks_are_all_or_nothing():
    plan = Watched([FULL], 4, 4, 3)
    parent = hold(plan, "p", 6)                 # two pages, two left
    assert plan.can_fork(parent) == 2
    with pytest.raises(OutOfPages):
        plan.fork(parent, ["a", "b", "c"])       # slots
    other = plan.open("x")
    assert plan.can_fork(parent) == 1
    plan.reserve(other, 8)
    assert plan.can_fork(parent) == 0
    with pytest.raises(OutOfPages):
        plan.fork(parent, ["a"])                 # pages
    assert not hasattr(plan, "forked") and set(plan.requests) == {"p", "x"}
    plan.check()
    plan.close(other)
    for bad in (["p"], ["a", "a"]):
        with pytest.raises(ValueError):
            plan.fork(parent, bad)
    assert plan.fork(parent, []) == []
    plan.close(parent)
    with pytest.raises(ValueError):
        plan.fork(parent, ["a"])


def test_forks_of_a_prompt_that_was_published_stay_findable():
    plan = CachePlan([FULL], 12, 4, 4, share_prefixes=True)
    tokens = list(range(10))
    parent = hold(plan, "p", 10)
    plan.publish_prompt(parent, tokens)
    child, = plan.fork(parent, ["a"])
    assert child.published == parent.published
    plan.close(parent)
    late = plan.open("late")
    assert plan.adopt_prefix(late, tokens[:9]) == 8 and late.tables[0] == child.tables[0][:2]
    plan.check()


# ---- answers -----------------------------------------------------------------------------------------------------------
class ForkingEngine(FakeEngine):
    """A fake whose pages hold what a copy brings, and whose draws know the filters."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.cache.on_fork = self._on_fork
        self.draws = []

    def _on_fork(self, parent, children, copies):
        for source, target, rows in copies[0]:
            for at in range(rows):
                self.page_contents[(target, at)] = self.page_contents[(source, at)]

    def sample(self, logits, temperature, top_p, uniform, top_k=None, min_p=None):
        self.draws.append((len(temperature), top_k, min_p))
        return super().sample(logits, temperature, top_p, uniform)


def alone(prompt, params):
    s = Scheduler(ForkingEngine(num_pages=256), max_batch_size=1, token_budget=1 << 20)
    rid = s.add_request(prompt, params)
    return s.run()[rid].tokens


def finish(s):
    while s.has_work():
        s.step()
        s.cache.check()
    for a in s.cache.allocators:
        assert a.all_released() and a.available == a.capacity
    return s.finished


def answers(n, **kw):
    return [GenerateParams(max_tokens=4 + i, temperature=0.9, seed=50 + i, **kw) for i in range(n)]


@pytest.mark.parametrize("length", [1, 3, 4, 8, 21])
@pytest.mark.parametrize("ahead", [None, False, True])
def test_every_answer_is_the_one_it_gets_alone(length, ahead):
    engine = ForkingEngine(num_pages=256, share_prefixes=True)
    if ahead is not None:
        engine.enable_ahead(launch=ahead)
    prompt = random_ids(length, 50, length)
    s = Scheduler(engine, max_batch_size=8, token_budget=16)
    other = s.add_request(random_ids(5, 50, 99), GenerateParams(max_tokens=9))
    ids = s.add_samples(prompt, answers(5))
    out = finish(s)
    assert [out[i].tokens for i in ids] == [alone(prompt, p) for p in answers(5)]
    assert out[other].tokens == alone(random_ids(5, 50, 99), GenerateParams(max_tokens=9))
    assert s.stats.forked == 4 and len(set(ids)) == 5
    # the prompt is run once
    assert sum(n for step in engine.steps for rid, n in step if rid in ids) == length + sum(len(out[i].tokens) - 1 for i in ids)


@pytest.mark.parametrize("batch, pages", [(2, 256), (1, 256), (8, 9), (3, 12)])
def test_answers_without_a_slot_or_pages_wait(batch, pages):
    engine = ForkingEngine(num_pages=pages, share_prefixes=True)
    prompt = random_ids(14, 50, 3)
    s = Scheduler(engine, max_batch_size=batch, token_budget=64)
    ids = s.add_samples(prompt, answers(6))
    late = s.add_request(random_ids(3, 50, 4), GenerateParams(max_tokens=3))
    out = finish(s)
    assert [out[i].tokens for i in ids] == [alone(prompt, p) for p in answers(6)]
    assert out[late].reason == StopReason.MAX_TOKENS and s.stats.forked < 5


def test_an_answer_that_cannot_run_does_not_take_the_others_with_it():
    s = Scheduler(ForkingEngine(num_pages=5), max_batch_size=4, token_budget=64)
    ids = s.add_samples(random_ids(30, 50, 1), answers(3))
    out = finish(s)
    assert [out[i].reason for i in ids] == [StopReason.FAILED] * 3
    # an answer of no tokens ends when the prompt is computed, its forks go on
    s = Scheduler(ForkingEngine(num_pages=64), max_batch_size=4, token_budget=64)
    prompt = random_ids(6, 50, 2)
    ids = s.add_samples(prompt, [GenerateParams(max_tokens=0)] + answers(2))
    out = finish(s)
    assert out[ids[0]].tokens == [] and [out[i].tokens for i in ids[1:]] == [alone(prompt, p) for p in answers(2)]


def test_bursts_wait_for_the_forks():
    engine = ForkingEngine(num_pages=64)
    s = Scheduler(engine, max_batch_size=4, token_budget=64, decode_burst=3)
    ids = s.add_samples([7], [GenerateParams(max_tokens=5) for _ in range(3)])
    out = finish(s)
    assert s.stats.forked == 2 and [out[i].tokens for i in ids] == [alone([7], GenerateParams(max_tokens=5))] * 3


def test_filters_are_passed_on_only_when_somebody_asks():
    engine = ForkingEngine(num_pages=64)
    s = Scheduler(engine, max_batch_size=4, token_budget=64)
    s.add_request([1, 2], GenerateParams(max_tokens=2, temperature=1.0))
    finish(s)
    assert all(k is None and m is None for _, k, m in engine.draws)
    s.add_samples([1, 2], [GenerateParams(max_tokens=1, temperature=1.0, top_k=3), GenerateParams(max_tokens=1, temperature=1.0, min_p=0.1)])
    finish(s)
    assert engine.draws[-1] == (2, [3, 0], [0.0, 0.1])


def test_refusals():
    s = Scheduler(ForkingEngine(num_pages=8, max_positions=10), max_batch_size=2)
    for prompt, params in ([[], answers(1)], [[1], []], [[1] * 8, answers(2)], [[1], [GenerateParams(top_k=-1)]],
                           [[1], [GenerateParams(top_k=2.5)]], [[1], [GenerateParams(top_k=1 << 31)]], [[1], [GenerateParams(min_p=1.5)]],
                           [[1], [GenerateParams(min_p=float("nan"))]], [[1], [GenerateParams(min_p=-0.1)]]):
        with pytest.raises(ValueError):
            s.add_samples(prompt, params)
    assert not s.has_work()


def test_streams_of_answers():
    seen = {}
    s = Scheduler(ForkingEngine(num_pages=64), max_batch_size=4)
    ids = s.add_samples([1, 2, 3], answers(3), token_bytes=lambda t: b"x", on_chunk=lambda i, text: seen.setdefault(i, []).append(text))
    out = finish(s)
    assert [len("".join(seen[i])) for i in range(3)] == [len(out[r].tokens) for r in ids]
