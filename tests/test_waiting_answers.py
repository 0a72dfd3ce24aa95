"""Several answers to one prompt where slots or pages run short, on the host: who is served first, what waits and what is computed again."""
import random

import pytest

from test_fork import CHUNK, FULL, STATE, WINDOW, ForkingEngine, alone, answers, finish, hold
from tiny import random_ids
from tokenizer_b200.cache import CachePlan, OutOfPages
from tokenizer_b200.engine.generate import Control, GenerateParams, StopReason
from tokenizer_b200.engine.scheduler import Scheduler


class Engine(ForkingEngine):
    """A fake that forgets what a cache held when its object's address is used again, and whose state slots remember every
    token that they have seen."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.state = {}
        self.cache.on_open = self._on_open
        self.cache.on_fork = self._on_fork

    def _on_open(self, cache):
        self.history.pop(id(cache), None)
        self.state[cache.state_slot] = []

    def _on_fork(self, parent, children, copies):
        super()._on_fork(parent, children, copies)
        for child in children:
            self.state[child.state_slot] = list(self.state[parent.state_slot])

    def step(self, entries):
        for e in entries:
            if self.cache.state_calls:
                assert len(self.state[e.cache.state_slot]) == e.cache.length
            self.state[e.cache.state_slot] = self.state[e.cache.state_slot] + [int(t) for t in e.tokens]
        logits = super().step(entries)
        for e in entries:
            if self.cache.state_calls:
                assert self.state[e.cache.state_slot] == [int(t) for t in self.history[id(e.cache)]]
        return logits


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


# ---- answers that wait -----------------------------------------------------------------------------------------------------
APART = [[FULL, STATE], [FULL, WINDOW], [FULL, CHUNK, STATE]]        # designs whose prefixes are not shared by hash


def tokens_run(engine):
    return sum(n for step in engine.steps for _, n in step)


@pytest.mark.parametrize("needs", APART)
@pytest.mark.parametrize("length", [40, 43])
@pytest.mark.parametrize("n, batch", [(24, 8), (9, 8), (3, 1), (8, 8)])
def test_a_prompt_is_computed_once_however_many_answers_wait(needs, length, n, batch, monkeypatch):
    """Through `generate_samples`, in the pool that it sizes."""
    from tokenizer_b200 import api
    made = []

    def engine_for(model, tokens, page_size, max_requests, shared_attention):
        made.append(Engine(num_pages=tokens // page_size, page_size=page_size, max_requests=max_requests, needs=needs, share_prefixes=True))
        return made[-1]

    monkeypatch.setattr(api, "engine_for", engine_for)
    prompt = random_ids(length, 50, length)
    params = [GenerateParams(max_tokens=12 + i % 3, temperature=0.9, seed=i) for i in range(n)]
    out = api.generate_samples(object(), prompt, n, params, max_batch_size=batch, page_size=4)
    assert [a.tokens for a in out] == [alone(prompt, p) for p in params]
    # nothing is preempted, nobody runs the prompt again
    assert tokens_run(made[0]) == length + sum(len(a.tokens) - 1 for a in out)
    rows = max(len(step) for step in made[0].steps)
    assert rows == min(n, batch)
    assert made[0].cache.allocators[0].all_released() and not made[0].cache.requests


def test_an_engine_without_a_slot_to_spare_gives_one_of_the_batch():
    engine = Engine(num_pages=256, max_requests=4, needs=[FULL, STATE])
    s = Scheduler(engine, max_batch_size=4, token_budget=64)
    prompt = random_ids(30, 50, 1)
    ids = s.add_samples(prompt, answers(9))
    check_line(s)
    assert [s.finished[i].tokens for i in ids] == [alone(prompt, p) for p in answers(9)]
    assert tokens_run(engine) == 30 + sum(len(s.finished[i].tokens) - 1 for i in ids) and s.stats.forked == 8


@pytest.mark.parametrize("slots", [1, 2, 3])
def test_few_slots(slots):
    s = Scheduler(Engine(num_pages=256, max_requests=slots, needs=[FULL, STATE]), max_batch_size=slots, token_budget=64)
    prompt = random_ids(9, 50, 1)
    ids = s.add_samples(prompt, answers(5))
    check_line(s)
    assert [s.finished[i].tokens for i in ids] == [alone(prompt, p) for p in answers(5)]


@pytest.mark.parametrize("needs", APART)
@pytest.mark.parametrize("pages", [9, 10, 12, 16, 24])
@pytest.mark.parametrize("seed", range(8))
def test_prompts_that_are_kept_give_way(needs, pages, seed):
    """Little room: a kept prompt is given up where nothing else can go on, and answers stay what they are."""
    rng = random.Random(10 * pages + seed)
    slots = rng.randint(2, 9)
    s = Scheduler(Engine(num_pages=pages, max_requests=slots, needs=needs), max_batch_size=rng.randint(1, slots),
                  token_budget=rng.choice([5, 64]))
    asked = []
    for at in range(3):
        prompt = random_ids(rng.randint(1, 20), 50, 7 * seed + at)
        params = [GenerateParams(max_tokens=rng.randint(0, 14), temperature=0.8, seed=at + i) for i in range(rng.choice([1, 4, 7]))]
        asked += [(i, prompt, p) for i, p in zip(s.add_samples(prompt, params), params)]
    check_line(s)
    assert not s.cache.requests
    for i, prompt, p in asked:
        assert s.finished[i].tokens == alone(prompt, p)


def test_an_answer_that_ends_with_its_first_id_takes_no_slot():
    engine = Engine(num_pages=64, max_requests=3, needs=[FULL, STATE])
    s = Scheduler(engine, max_batch_size=2, token_budget=64)
    prompt = random_ids(7, 50, 5)
    seen = []
    stop = lambda i, text: (seen.append(i), Control.STOP if i == 3 else Control.CONTINUE)[1]  # noqa: E731
    params = [GenerateParams(max_tokens=1 if i == 2 else 6, temperature=0.9, seed=i) for i in range(6)]
    ids = s.add_samples(prompt, params, token_bytes=lambda t: b"x", on_chunk=stop)
    check_line(s)
    assert len(s.finished[ids[2]].tokens) == 1 and s.finished[ids[3]].reason == StopReason.CANCELLED
    for i in (0, 1, 4, 5):
        assert s.finished[ids[i]].tokens == alone(prompt, params[i])
    assert engine.steps[0] == [(ids[0], 7)] and tokens_run(engine) == 7 + 4 * 5


@pytest.mark.gpu
@pytest.mark.parametrize("module, name", [("tiny", "a"), ("tiny", "c"), ("tiny_katopel", "a"), ("tiny_vizonex", "b"), ("tiny_kerudra", "a"),
                                          ("tiny_zobelorn", "b")])
def test_waiting_answers_of_every_kind_of_cache(module, name, tmp_path_factory):
    """On the device: two at a time, the others forked from the prompt that the last one keeps; the ids are those of all at once."""
    import tokenizer_b200 as tb
    from test_samples_gpu import folder_of
    folder, vocab, page = folder_of(module, name, tmp_path_factory)
    model = tb.load_model(folder, dtype="float32")
    prompt = random_ids(2 * page + 3, vocab, 5)
    params = [tb.GenerateParams(max_tokens=8 + i, temperature=0.8, top_k=30, seed=i) for i in range(7)]
    want = tb.generate_samples(model, prompt, 7, params, page_size=page)
    engine = tb.Engine(model, num_pages=60, page_size=page, max_requests=3, shared_attention=True)
    s = tb.Scheduler(engine, max_batch_size=2)
    ids = s.add_samples(prompt, params)
    out = s.run()
    assert [out[i].tokens for i in ids] == [a.tokens for a in want]
    assert s.stats.preemptions == 0 and s.stats.forked == 6
    assert s.stats.tokens_run == len(prompt) + sum(len(a.tokens) - 1 for a in want)
    engine.cache.check()
    assert not engine.cache.requests


@pytest.mark.parametrize("needs, share", [([FULL], True), ([FULL, STATE], False), ([FULL, WINDOW], False)])
@pytest.mark.parametrize("lengths, samples, batch", [([41], 64, 8), ([40, 17, 3], 5, 4), ([9] * 6, 3, 2), ([5], 2, 8)])
def test_the_command_line_sizes_its_pool_for_what_runs_together(needs, share, lengths, samples, batch, monkeypatch, tmp_path, capsys):
    import tokenizer_b200 as tb
    from tokenizer_b200 import cli
    made = []

    def engine(model, num_pages, page_size, max_requests, share_prefixes, shared_attention):
        made.append(Engine(num_pages=num_pages, page_size=page_size, max_requests=max_requests, needs=needs, share_prefixes=share_prefixes))
        return made[-1]

    monkeypatch.setattr(tb, "Engine", engine)
    monkeypatch.setattr(tb, "load_model", lambda *a, **kw: object())
    monkeypatch.setattr(tb, "load_eos_token_ids", lambda folder: [])
    prompts = [random_ids(n, 50, i) for i, n in enumerate(lengths)]
    args = [a for p in prompts for a in ("--ids", ",".join(map(str, p)))]
    assert cli.main(["--model", str(tmp_path), "--max-tokens", "9", "--temperature", "0.9", "--samples", str(samples), "--page-size", "4",
                     "--max-batch-size", str(batch)] + args) == 0
    lines = capsys.readouterr().out.strip().splitlines()
    want = [alone(p, GenerateParams(max_tokens=9, temperature=0.9, seed=i)) for p in prompts for i in range(samples)]
    assert lines == [" ".join(map(str, w)) for w in want]
    # a prompt's full pages once, and tails of at most 3 + 9 tokens (a page more for the next one) for those that run or are kept
    together = min(batch, len(prompts) * samples)
    assert made[0].cache.num_pages <= sum(n // 4 for n in lengths) + together * 4 + len(prompts)
    if not share:
        assert tokens_run(made[0]) == sum(lengths) + len(want) * 8
