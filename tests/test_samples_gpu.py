"""Several answers to one prompt on the GPU: the filters among other requests' draws, forks of every design's cache (pages,
windows, chunks, states) against requests of their own, steps that read common keys once, and the whole path from a prompt to
its answers."""
import importlib
import os
import subprocess
import sys

import pytest
import torch

from tiny import random_ids

pytestmark = pytest.mark.gpu

DESIGNS = [(m, n) for m, names in [("tiny", "abc"), ("tiny_pufuzen", "pqrst"), ("tiny_katopel", "abcd"), ("tiny_vizonex", "abcd"),
                                   ("tiny_zobelorn", "abcd"), ("tiny_kazepel", "abcd"), ("tiny_kerudra", "abcd")] for n in names]


@pytest.fixture
def every_set(monkeypatch):
    """Common keys are read apart however little that saves."""
    from tokenizer_b200.kernels import ops
    from tokenizer_b200.parts.attention import SharedBeginnings
    monkeypatch.setattr(SharedBeginnings, "LEAST_BYTES", 0)
    monkeypatch.setattr(ops, "SHARED_PREFIX_LITTLE", 0)


@pytest.fixture
def shared_calls(monkeypatch):
    from tokenizer_b200.kernels import ops
    calls, real = [], ops.shared_prefix_attention
    monkeypatch.setattr(ops, "shared_prefix_attention", lambda *a, **kw: (calls.append(a[9].shape[0]), real(*a, **kw))[1])
    return calls


# ---- the draws -----------------------------------------------------------------------------------------------------------
def test_rows_with_and_without_filters_are_drawn_as_each_is_alone():
    from tokenizer_b200.sampling import Sampler
    from test_sample_filtered_gpu import plain_draw
    torch.manual_seed(3)
    logits = (2 * torch.randn(12, 4001)).cuda()
    temperature = [0.0, 0.7, 1.3, 0.9] * 3
    top_p = [1.0, 0.8, 1.0, 0.95] * 3
    top_k = [5, 0, 40, 0] * 3
    min_p = [0.1, 0.0, 0.0, 0.02] * 3
    u = torch.rand(12).tolist()
    sampler = Sampler("cuda")
    got = sampler.sample(logits, temperature, top_p, u, top_k, min_p)
    for r in range(12):
        one = [logits[r:r + 1].contiguous()] + [[v[r]] for v in (temperature, top_p, u, top_k, min_p)]
        assert sampler.sample(*one) == [got[r]]
        if temperature[r] == 0 or (top_k[r] == 0 and min_p[r] == 0):
            assert sampler.sample(*one[:4]) == [got[r]]          # the kernel that it had without filters
        else:
            f = lambda x: float(torch.tensor(x, dtype=torch.float32))  # noqa: E731
            assert got[r] == plain_draw(logits[r].cpu().numpy(), f(temperature[r]), top_k[r], f(top_p[r]), f(min_p[r]), f(u[r]))


# ---- forks -----------------------------------------------------------------------------------------------------------------
def folder_of(module, name, tmp_path_factory):
    m = importlib.import_module(module)
    folder, config, page = m.make_folder(tmp_path_factory, name)
    return folder, getattr(config, "vocab_size", None) or config.vocab, page


def run(engine, caches, tokens):
    from tokenizer_b200.engine import StepEntry
    for c, t in zip(caches, tokens):
        engine.cache.reserve(c, len(t))
    return engine.step([StepEntry(c, t, [len(t) - 1]) for c, t in zip(caches, tokens)]).float().cpu().clone()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("module, name", DESIGNS)
def test_forks_go_on_as_requests_of_their_own(module, name, dtype, tmp_path_factory, every_set, shared_calls):
    from tokenizer_b200.engine import Engine
    folder, vocab, page = folder_of(module, name, tmp_path_factory)
    for length in (2 * page + 3, 2 * page):
        engine = Engine.from_folder(folder, dtype=dtype, num_pages=64, page_size=page, max_requests=8, shared_attention=True)
        other = Engine.from_folder(folder, dtype=dtype, num_pages=64, page_size=page, max_requests=8)
        prompt = random_ids(length, vocab, 7 + length)
        parent = engine.cache.open("p")
        run(engine, [parent], [prompt])
        caches = [parent] + engine.cache.fork(parent, ["a", "b", "c"])
        engine.cache.check()
        alone = [other.cache.open(i) for i in range(4)]
        run(other, alone, [prompt] * 4)
        for step in range(6):                    # plainly, captured, and over a page's end
            tokens = [random_ids(1, vocab, 100 * step + i) for i in range(4)]
            got, want = run(engine, caches, tokens), run(other, alone, tokens)
            if dtype == "float32":
                # both are within 1e-4 of the plain implementation (the bound that their replays are held to)
                assert (got - want).abs().max() <= 2e-4 * max(1.0, float(want.abs().max())), (module, name, length, step)
            else:
                rel = (got - want).pow(2).mean().sqrt() / (want - want.mean(dim=1, keepdim=True)).pow(2).mean().sqrt()
                assert torch.isfinite(got).all() and rel <= 0.2, (module, name, length, step, float(rel))
        assert engine.shared_notes or not shared_calls
        if module == "tiny" and dtype == "float32":
            assert shared_calls and all(n == 1 for n in shared_calls)
        for c in caches:
            engine.cache.close(c)
        engine.cache.check()
        assert all(a.all_released() for a in engine.cache.allocators)


def test_steps_with_sets_that_come_and_go(tmp_path_factory, every_set, shared_calls):
    """One engine: a batch with two sets and a lone request, then fewer of them, prompts between, a request that starts anew
    under its old cache; always against an engine that never reads common keys apart."""
    from tokenizer_b200.engine import Engine
    folder, vocab, page = folder_of("tiny", "b", tmp_path_factory)
    make = lambda **kw: Engine.from_folder(folder, dtype="float32", num_pages=160, page_size=page, max_requests=12, **kw)  # noqa: E731
    engine, other = make(shared_attention=True), make()
    caches, mirror = {}, {}

    def both(names, tokens):
        got, want = run(engine, [caches[n] for n in names], tokens), run(other, [mirror[n] for n in names], tokens)
        assert (got - want).abs().max() <= 2e-4 * max(1.0, float(want.abs().max()))

    for name, n in (("p", 30), ("q", 17), ("r", 5)):
        caches[name], mirror[name] = engine.cache.open(name), other.cache.open(name)
        both([name], [random_ids(n, vocab, n)])
    for name, forks in (("p", ["p1", "p2", "p3"]), ("q", ["q1"])):
        for source, target in ((engine, caches), (other, mirror)):
            target.update(zip(forks, source.cache.fork(target[name], forks)))
    one = lambda names, seed: [random_ids(1, vocab, seed + i) for i in range(len(names))]  # noqa: E731
    everybody = list(caches)
    for step in range(4):
        both(everybody, one(everybody, 10 * step))
    before = len(shared_calls)
    assert before >= 3 * 2                       # every layer, plainly and as captured; replays do not come by
    both(["r", "q"], one("rq", 50))              # nobody shares
    both(["p2", "r", "p1"], one("abc", 60))
    both(["p2", "r", "p1"], one("abc", 64))
    assert len(shared_calls) > before
    both(["p", "q1"], [random_ids(9, vocab, 70), random_ids(1, vocab, 71)])      # a portion beside a token
    for source, target in ((engine, caches), (other, mirror)):
        source.cache.release_pages(target["p1"])
    both(["p1"], [random_ids(20, vocab, 72)])
    both(["p2", "r", "p1"], one("abc", 80))      # the same requests, and other pages
    both(everybody, one(everybody, 90))
    engine.cache.check()


def test_bursts_and_prepared_steps_on_common_keys(tmp_path_factory, every_set):
    from tokenizer_b200.engine import Engine, StepEntry
    folder, vocab, page = folder_of("tiny", "a", tmp_path_factory)
    outs = []
    for shared in (True, False):
        engine = Engine.from_folder(folder, dtype="float32", num_pages=64, page_size=page, max_requests=8, shared_attention=shared)
        parent = engine.cache.open("p")
        run(engine, [parent], [random_ids(2 * page + 1, vocab, 5)])
        caches = [parent] + engine.cache.fork(parent, ["a", "b"])
        ids = engine.decode_steps([StepEntry(c, [3 + i]) for i, c in enumerate(caches)], 9)
        ids += engine.decode_steps([StepEntry(c, [ids[-1][i]]) for i, c in enumerate(caches)], 5)
        for step in range(3):
            run(engine, caches, [[7], [8], [9]])
        for c in caches:
            engine.cache.reserve(c, 1)
        prepared = engine.prepare_decode(caches)
        logits = engine.step_prepared(prepared, [1, 2, 3])
        outs.append((ids, logits.float().cpu().clone()))
    assert outs[0][0] == outs[1][0]
    assert (outs[0][1] - outs[1][1]).abs().max() <= 2e-4 * float(outs[1][1].abs().max())


@pytest.mark.parametrize("heads, kv, d", [(4, 2, 64), (7, 1, 128)])
def test_common_keys_on_the_tensor_cores_inside_a_model(heads, kv, d, every_set, shared_calls):
    """bfloat16, heads that the tensor-core kernels take: logits beside those of an engine that reads every row's keys."""
    import tokenizer_b200 as tb
    config = tb.Qwen2Config.from_dict({
        "architectures": ["Qwen2ForCausalLM"], "vocab_size": 512, "hidden_size": heads * d, "intermediate_size": 256,
        "num_hidden_layers": 3, "num_attention_heads": heads, "num_key_value_heads": kv, "max_position_embeddings": 2048,
        "sliding_window": 64, "max_window_layers": 3, "use_sliding_window": False, "tie_word_embeddings": True, "rope_theta": 10000.0,
        "rms_norm_eps": 1e-6, "hidden_act": "silu"})
    model = tb.random_model(config, 4)
    prompt = random_ids(700, 512, 1)
    engines = [tb.Engine(model, num_pages=200, page_size=16, max_requests=24, shared_attention=shared) for shared in (True, False)]
    caches = []
    for engine in engines:
        parent = engine.cache.open("p")
        run(engine, [parent], [prompt])
        caches.append([parent] + engine.cache.fork(parent, list(range(19))))
    for step in range(5):
        tokens = [random_ids(1, 512, 50 * step + i) for i in range(20)]
        got, want = (run(engine, c, tokens) for engine, c in zip(engines, caches))
        # two bfloat16 models whose attention rounds apart: an eighth of what a wrong key would move
        rel = (got - want).pow(2).mean().sqrt() / (want - want.mean(dim=1, keepdim=True)).pow(2).mean().sqrt()
        assert torch.isfinite(got).all() and rel <= 0.05, (step, float(rel))
    assert shared_calls


# ---- from a prompt to its answers --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_answers_to_one_prompt(dtype, tmp_path_factory, every_set, shared_calls):
    import tokenizer_b200 as tb
    folder, vocab, page = folder_of("tiny", "a", tmp_path_factory)
    model = tb.load_model(folder, dtype=dtype)
    prompt = random_ids(2 * page + 5, vocab, 11)
    params = tb.GenerateParams(max_tokens=20, temperature=0.9, top_k=40, top_p=0.95, min_p=0.01, seed=3)
    answers = tb.generate_samples(model, prompt, 6, params, page_size=page)
    assert [len(a.tokens) for a in answers] == [20] * 6 and all(a.reason == tb.StopReason.MAX_TOKENS for a in answers)
    assert len({tuple(a.tokens) for a in answers}) > 1
    assert bool(shared_calls) == (dtype == "float32")        # heads of 16 lanes stay on the decoding kernel in bfloat16
    again = tb.generate_samples(model, prompt, 6, params, page_size=page)
    assert [a.tokens for a in again] == [a.tokens for a in answers]
    if dtype == "float32":
        from dataclasses import replace
        for i, a in enumerate(answers):
            assert tb.generate(model, prompt, replace(params, seed=3 + i)).tokens == a.tokens
    greedy = tb.generate_samples(model, prompt, 3, tb.GenerateParams.greedy(8), page_size=page)
    assert greedy[0].tokens == greedy[1].tokens == greedy[2].tokens
    # more answers than slots: the others wait and find the prompt's pages
    few = tb.generate_samples(model, prompt, 6, params, page_size=page, max_batch_size=2)
    if dtype == "float32":
        assert [a.tokens for a in few] == [a.tokens for a in answers]
    with pytest.raises(ValueError):
        tb.generate_samples(model, prompt, 0, params)
    with pytest.raises(ValueError):
        tb.generate_samples(model, prompt, 2, [params])


def test_command_line_samples(tmp_path_factory):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    folder, vocab, page = folder_of("tiny", "a", tmp_path_factory)
    cli = lambda *a: subprocess.run([sys.executable, os.path.join(root, "bin", "qwen-infer"), "--model", folder, "--dtype", "float32",  # noqa: E731
                                     "--page-size", str(page), *a], capture_output=True, text=True, timeout=600)
    args = ["--max-tokens", "6", "--temperature", "0.8", "--top-k", "30", "--min-p", "0.02"]
    ids = ",".join(map(str, random_ids(20, vocab, 1)))
    several = cli(*args, "--samples", "3", "--seed", "4", "--ids", ids)
    assert several.returncode == 0, several.stderr
    lines = several.stdout.strip().splitlines()
    assert len(lines) == 3 and "top_k 30 min_p 0.02" in several.stderr
    alone = cli(*args, "--seed", "6", "--ids", ids)
    assert alone.stdout.strip() == lines[2]
    assert cli("--samples", "0", "--ids", "1").returncode == 2
    assert cli("--min-p", "2", "--ids", "1").returncode == 1
