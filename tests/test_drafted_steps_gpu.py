"""Steps over shared prompts and steps of drafted tokens through the runner and the scheduler: plans of shared pages, verification and the
cache together, against the plain implementation."""
import numpy as np
import pytest
import torch

import helpers
import plain_qwen2 as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model_dirs(tmp_path_factory):
    base = tmp_path_factory.mktemp("models")
    # head size 64 and 28 query rows a token: what the streaming and the tcgen05 kernels take
    wide = dict(hidden_size=448, intermediate_size=256, num_attention_heads=7, num_key_value_heads=1)
    dirs = {name: helpers.make_model_dir(base, name) for name in helpers.TINY}
    dirs["wide"] = helpers.make_model_dir(base / "wide", "A", **wide)
    return dirs


def started(model, prefix, tails, page, shared_prefix=True, pages=600):
    """A runner and one request per tail behind a common prompt, its pages shared."""
    from sprout_lm_b200 import ModelRunner
    from sprout_lm_b200.engine.batch import StepEntry
    runner = ModelRunner(model, num_pages=pages, page_tokens=page, max_requests=len(tails), shared_prefix=shared_prefix)
    if shared_prefix:
        runner.shared_prefix.always = True
    seqs = []
    for tail in tails:
        prompt = prefix + tail
        seq = runner.new_sequence(prompt)
        assert runner.reserve(seq, len(prompt) + 40)
        rest = prompt[seq.length:]
        runner.step([StepEntry(seq, rest, [])])
        runner.manager.publish(prompt, seq)
        seqs.append(seq)
    shared = len(prefix) // page
    assert all(seq.blocks[:shared] == seqs[0].blocks[:shared] for seq in seqs)
    return runner, seqs


def tolerance(model, dtype):
    """The tiny models' bar for their width of 64 and 96.  A logit is a sum over the width of normed activations (of order 1) times weights of
    0.02, and so is its error, the activations' own relative to them: both grow with the root of the width."""
    return helpers.TOL[dtype] * max(1.0, (model.config.hidden_size / 64) ** 0.5)


def nearly_greedy(model, directory, prompt, output, dtype):
    """Every token is an argmax of logits that are off by no more than the tolerance: within twice that of the plain implementation's largest."""
    rows = helpers.plain_logits(directory, prompt + output)[len(prompt) - 1:-1]
    return all(row.max() - row[token] <= 2 * tolerance(model, dtype) for row, token in zip(rows, output))


@pytest.mark.parametrize("name", ["A", "B", "wide"])
@pytest.mark.parametrize("tokens", [1, 4])
def test_logits_of_steps_over_a_shared_prompt(model_dirs, name, tokens):
    from sprout_lm_b200 import load_model
    from sprout_lm_b200.engine.batch import StepEntry
    directory = model_dirs[name]
    model = load_model(directory, dtype="bfloat16")
    sizes, _, page = helpers.TINY["A" if name == "wide" else name]
    vocab = sizes["vocab_size"]
    rng = np.random.default_rng(17)
    prefix = helpers.random_tokens(rng, 11 * page + 3, vocab)
    tails = [helpers.random_tokens(rng, n, vocab) for n in (1, 9, 30, 5, 2, 14)]
    runner, seqs = started(model, prefix, tails, page)
    histories = [prefix + tail for tail in tails]
    for step in range(3):
        new = [helpers.random_tokens(rng, 1 + (i + step) % tokens, vocab) for i in range(len(seqs))]
        logits = runner.step([StepEntry(seq, t, list(range(len(t)))) for seq, t in zip(seqs, new)])
        row = 0
        for history, t in zip(histories, new):
            history += t
            want = helpers.plain_logits(directory, history)[-len(t):]
            error = float(np.abs(logits[row:row + len(t)].float().cpu().numpy() - want).max())
            assert error <= tolerance(model, "bfloat16")
            row += len(t)
    assert runner.shared_prefix.steps == 3
    runner.check_status()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["B", "wide"])
def test_drafted_tokens_give_the_greedy_continuation(model_dirs, name, dtype):
    """Right, wrong and no drafts: the tokens that come out are the model's own greedy ones, several a step where drafts are right."""
    from sprout_lm_b200 import load_model
    from sprout_lm_b200.engine.batch import StepEntry
    from sprout_lm_b200.sampling import verify_uniforms
    directory = model_dirs[name]
    model = load_model(directory, dtype=dtype)
    cfg, weights = plain.read_model_folder(directory)
    page = 8
    vocab = model.spec.vocab_size
    rng = np.random.default_rng(23)
    prefix = helpers.random_tokens(rng, 9 * page, vocab)
    tails = [helpers.random_tokens(rng, n, vocab) for n in (3, 2, 12)]      # a request recomputes its last token: never all pages
    count = 14
    wanted = []
    for tail in tails:
        history = prefix + tail
        for _ in range(count + 6):
            history = history + [int(np.argmax(plain.logits(cfg, weights, history)[-1]))]
        wanted.append(history[len(prefix) + len(tail):])
    # the prompt's last token is the first step's input
    runner, seqs = started(model, prefix, [tail[:-1] for tail in tails], page)
    outputs, last = [[] for _ in tails], [tail[-1] for tail in tails]
    steps = 0
    while min(map(len, outputs)) < count:
        entries, accept, draw = [], [], []
        for r, seq in enumerate(seqs):
            at, drafts = len(outputs[r]), []
            for i in range((steps + r) % 5):
                right = wanted[r][at + i] if at + i < len(wanted[r]) else 0
                drafts.append(right if rng.random() < 0.8 else (right + 1) % vocab)
            assert runner.reserve(seq, seq.length + 1 + len(drafts))
            entries.append(StepEntry(seq, [last[r], *drafts], []))
            a, d = verify_uniforms(7, f"r{r}", at, 1 + len(drafts))
            accept += a
            draw += d
        before = [seq.length for seq in seqs]
        for r, new in enumerate(runner.step_and_verify(entries, [0.0] * len(seqs), accept, draw)):
            outputs[r] += new
            last[r] = new[-1]
            assert seqs[r].length == before[r] + len(new)
        steps += 1
    for tail, output, want in zip(tails, outputs, wanted):
        if dtype == "float32":
            assert output[:count] == want[:count]
        assert nearly_greedy(model, directory, prefix + tail, output[:count], dtype)
    assert steps < count                                   # some steps gave several tokens
    assert runner.shared_prefix.steps == (steps if dtype == "bfloat16" else 0)      # the 32-bit path keeps its own kernels
    runner.check_status()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_draft_model_of_the_same_logits_always_stands(model_dirs, dtype):
    """Drafts whose distribution is the target's own stand whatever the numbers, and the token behind them is the draw that plain sampling
    makes at the same number.  The 32-bit path gives the same bits in both runs; in bfloat16 two runs add split sums in any order, each
    within the tolerance t = 0.006 * sqrt(448 / 64) = 0.0159 of the exact logits, so they differ by at most 2 t, and p / q >=
    exp(-2 * 2 t / 0.7) = 0.913: drafts stand at numbers below that, and draws next to a border may differ."""
    from sprout_lm_b200 import load_model
    from sprout_lm_b200.engine.batch import StepEntry
    from sprout_lm_b200.sampling import verify_uniforms
    directory = model_dirs["wide"]
    model = load_model(directory, dtype=dtype)
    vocab, page = model.spec.vocab_size, 16
    rng = np.random.default_rng(29)
    prefix = helpers.random_tokens(rng, 6 * page, vocab)
    tails = [helpers.random_tokens(rng, n, vocab) for n in (3, 2, 12, 7)]
    runner, seqs = started(model, prefix, [tail[:-1] for tail in tails], page)
    temperatures = [0.9, 0.7, 1.3, 1.0]
    tokens = [[tail[-1], *helpers.random_tokens(rng, n, vocab)] for tail, n in zip(tails, (3, 0, 4, 1))]
    # the target's logits at every place, by a step whose tokens are taken back
    lengths = [seq.length for seq in seqs]
    logits = runner.step([StepEntry(seq, t, list(range(len(t)))) for seq, t in zip(seqs, tokens)])
    for seq, n in zip(seqs, lengths):
        seq.length = n
    counts = [len(t) for t in tokens]
    start = np.concatenate([[0], np.cumsum(counts)])
    drafted = torch.tensor([start[r] + i for r, n in enumerate(counts) for i in range(n - 1)], device=logits.device)
    accept, draw = [], []
    for r, n in enumerate(counts):
        a, d = verify_uniforms(3, f"r{r}", 5, n)
        accept += [1 - 2.0 ** -24 if dtype == "float32" else 0.91] * n
        draw += d
    results = runner.step_and_verify([StepEntry(seq, t, []) for seq, t in zip(seqs, tokens)], temperatures, accept, draw, draft_logits=logits[drafted])
    for r, (new, t) in enumerate(zip(results, tokens)):
        assert new[:-1] == t[1:]
        row = start[r + 1] - 1
        p = np.exp(logits[row].double().cpu().numpy() / temperatures[r])
        if dtype == "float32":
            assert new[-1] == int(np.searchsorted(np.cumsum(p), draw[row] * p.sum(), side="right"))
        assert seqs[r].length == lengths[r] + counts[r]
    runner.check_status()


def test_without_drafts_a_step_draws_what_plain_sampling_draws(model_dirs):
    from sprout_lm_b200 import ModelRunner, load_model
    from sprout_lm_b200.engine.batch import StepEntry
    from sprout_lm_b200.sampling import verify_uniforms
    model = load_model(model_dirs["B"], dtype="float32")
    rng = np.random.default_rng(31)
    runner = ModelRunner(model, num_pages=60, page_tokens=8, max_requests=4)
    entries = []
    for n in (5, 17, 2):
        seq = runner.new_sequence()
        assert runner.reserve(seq, 40)
        prompt = helpers.random_tokens(rng, n, model.spec.vocab_size)
        if n > 2:
            runner.step([StepEntry(seq, prompt[:-1], [])])
        entries.append(StepEntry(seq, prompt[-1:] if n > 2 else prompt[:1], []))
    temperatures, draw = [0.8, 0.0, 1.2], []
    for r in range(3):
        draw += verify_uniforms(1, f"r{r}", 0, 1)[1]
    lengths = [e.seq.length for e in entries]
    new = runner.step_and_verify(entries, temperatures, [0.5] * 3, draw)
    assert [e.seq.length for e in entries] == [n + 1 for n in lengths]
    for e, n in zip(entries, lengths):
        e.seq.length = n
    assert [t[0] for t in new] == runner.step_and_sample([StepEntry(e.seq, e.tokens, [0]) for e in entries], temperatures, draw)


def test_generation_with_shared_prompts(model_dirs):
    """The scheduler with the option on: plans are taken, and tokens are greedy ones."""
    from sprout_lm_b200 import EngineOptions, generate, load_model, make_engine
    model = load_model(model_dirs["B"], dtype="bfloat16")
    rng = np.random.default_rng(41)
    prefix = helpers.random_tokens(rng, 80, 509)
    prompts = [prefix + helpers.random_tokens(rng, n, 509) for n in (1, 20, 9, 33)]
    engine = make_engine(model, EngineOptions(block_size=8, num_blocks=120, max_sequences=4, max_batch_tokens=64, prefill_chunk_size=48, shared_prefix=True))
    engine.runner.shared_prefix.always = True
    generate(model, prompts[:1], max_new_tokens=1, ignore_eos=True, engine=engine)      # publishes the prefix
    results = generate(model, prompts, max_new_tokens=10, ignore_eos=True, engine=engine)
    assert engine.runner.shared_prefix.steps > 0 and all(r["prefix_hits"] > 0 for r in results)
    for prompt, result in zip(prompts, results):
        assert len(result["output"]) == 10 and nearly_greedy(model, model_dirs["B"], prompt, result["output"], "bfloat16")


@pytest.mark.parametrize("name", ["A", "B", "wide"])
def test_captured_steps_over_a_shared_prompt(model_dirs, name, monkeypatch):
    """Decode steps of the same requests: one captured over their pages serves as many as its plan does, the next is made behind it, and
    another request among them ends it."""
    from sprout_lm_b200 import load_model
    from sprout_lm_b200.engine import shared
    from sprout_lm_b200.engine.batch import StepEntry
    monkeypatch.setattr(shared, "STRETCH", 7)
    directory = model_dirs[name]
    model = load_model(directory, dtype="bfloat16")
    page, vocab = 8, model.spec.vocab_size
    rng = np.random.default_rng(53)
    prefix = helpers.random_tokens(rng, 11 * page + 3, vocab)
    tails = [helpers.random_tokens(rng, n, vocab) for n in (1, 9, 30, 5, 2, 14)]
    runner, seqs = started(model, prefix, tails, page)
    steps = runner.shared_prefix
    steps.after, steps.always = 2, True
    histories, graphs = [prefix + tail for tail in tails], []

    def decode(which):
        new = [int(rng.integers(vocab)) for _ in which]
        runner.step_and_sample([StepEntry(seqs[r], [t], [0]) for r, t in zip(which, new)], [0.0] * len(which), [0.0] * len(which))
        for r, t in zip(which, new):
            histories[r].append(t)
        graph = steps._graph
        if graph is not None:
            assert runner.last_decode_graph is graph and graph.ctx.shared is not None
            if graph not in graphs:
                graphs.append(graph)
            logits = graph.last_logits.float().cpu().numpy()
            for row, r in enumerate(which):
                assert float(np.abs(logits[row] - helpers.plain_logits(directory, histories[r])[-1]).max()) <= tolerance(model, "bfloat16")
        return graph

    made = [decode([0, 1, 2, 3, 4, 5]) for _ in range(19)]
    assert made[0] is None and made[1] is not None                  # the second step of the same requests
    assert [made.index(g) for g in graphs] == [1, 9, 17]            # a plan serves its own step and seven behind it
    assert [decode([5, 3, 1]) is None for _ in range(3)] == [True, False, False]
    assert len(graphs) == 4 and steps.steps == 22
    # other steps in between, and a request that was taken back further than its plan's first step
    assert decode([5, 3, 1]) is graphs[3]
    seqs[3].length -= 5
    del histories[3][-5:]
    assert decode([5, 3, 1]) is not graphs[3] and len(graphs) == 5
    steps.always = False
    assert decode([0, 1]) is None and decode([0, 1]) is None        # it does not pay here
    runner.check_status()


@pytest.mark.parametrize("ahead", [False, True])
def test_pages_reserved_beyond_a_captured_step(model_dirs, ahead):
    """Between two decode steps over a capture the caller reserves more pages than the capture's tables hold: the steps go on, over a capture
    made for them."""
    from sprout_lm_b200 import load_model
    from sprout_lm_b200.engine.batch import StepEntry
    directory = model_dirs["wide"]
    model = load_model(directory, dtype="bfloat16")
    page, vocab = 8, model.spec.vocab_size
    rng = np.random.default_rng(67)
    prefix = helpers.random_tokens(rng, 11 * page + 3, vocab)
    tails = [helpers.random_tokens(rng, n, vocab) for n in (1, 9, 30)]
    runner, seqs = started(model, prefix, tails, page)
    steps = runner.shared_prefix
    steps.after = 2
    histories, graphs = [prefix + tail for tail in tails], []
    new = [int(t) for t in rng.integers(vocab, size=3)]
    for i in range(8):
        if i == 4:
            assert runner.reserve(seqs[1], steps._graph.table_pages * page + 1)
        then = ([StepEntry(seq, [0], [0]) for seq in seqs], [0.0] * 3, [0.0] * 3, [0, 1, 2]) if ahead else None
        sampled = runner.step_and_sample([StepEntry(seq, [t], [0]) for seq, t in zip(seqs, new)], [0.0] * 3, [0.0] * 3, then=then)
        for history, t in zip(histories, new):
            history.append(t)
        new = sampled
        graphs.append(steps._graph)
    assert graphs[2] is graphs[3] is not None and graphs[5] is not graphs[3] and graphs[5] is graphs[7] is not None
    assert runner.ahead_used > 0 or not ahead
    for tail, history in zip(tails, histories):
        at = len(prefix) + len(tail) + 1                  # what the model said behind each of its tokens
        assert nearly_greedy(model, directory, history[:at], history[at:], "bfloat16")
    runner.check_status()


def test_captured_generation_with_shared_prompts(model_dirs, monkeypatch):
    """The same through the scheduler, whose steps are launched ahead."""
    from sprout_lm_b200 import EngineOptions, generate, load_model, make_engine
    from sprout_lm_b200.engine import shared
    monkeypatch.setattr(shared, "STRETCH", 11)
    model = load_model(model_dirs["B"], dtype="bfloat16")
    rng = np.random.default_rng(59)
    prefix = helpers.random_tokens(rng, 80, 509)
    prompts = [prefix + helpers.random_tokens(rng, n, 509) for n in (1, 20, 9, 33)]
    engine = make_engine(model, EngineOptions(block_size=8, num_blocks=160, max_sequences=4, max_batch_tokens=64, prefill_chunk_size=48, shared_prefix=True))
    runner = engine.runner
    runner.shared_prefix.always, runner.shared_prefix.after = True, 2
    runner.shared_prefix.plans = lambda entries, replayed: None     # captured ones alone
    generate(model, prompts[:1], max_new_tokens=1, ignore_eos=True, engine=engine)      # publishes the prefix
    results = generate(model, prompts, max_new_tokens=40, ignore_eos=True, engine=engine)
    assert runner.shared_prefix.steps >= 30 and runner.ahead_used >= 20
    for prompt, result in zip(prompts, results):
        assert len(result["output"]) == 40 and nearly_greedy(model, model_dirs["B"], prompt, result["output"], "bfloat16")


def test_captured_generation_in_a_pool_too_small(model_dirs, monkeypatch):
    """Requests come, end and are thrown out and readmitted with other pages while captures over the shared ones are made and dropped."""
    from sprout_lm_b200 import EngineOptions, generate, load_model, make_engine
    from sprout_lm_b200.engine import shared
    monkeypatch.setattr(shared, "STRETCH", 5)
    model = load_model(model_dirs["B"], dtype="bfloat16")
    rng = np.random.default_rng(61)
    prefix = helpers.random_tokens(rng, 80, 509)
    prompts = [prefix + helpers.random_tokens(rng, n, 509) for n in (1, 20, 9, 33, 14, 5, 27)]
    engine = make_engine(model, EngineOptions(block_size=8, num_blocks=34, max_sequences=5, max_batch_tokens=64, prefill_chunk_size=48, shared_prefix=True))
    steps = engine.runner.shared_prefix
    steps.always, steps.after = True, 2
    generate(model, prompts[:1], max_new_tokens=1, ignore_eos=True, engine=engine)      # publishes the prefix
    results = generate(model, prompts, max_new_tokens=30, ignore_eos=True, engine=engine)
    assert steps.steps > 0 and any(e["type"] == "preempted" for e in engine.trace)
    for prompt, result in zip(prompts, results):
        assert len(result["output"]) == 30 and nearly_greedy(model, model_dirs["B"], prompt, result["output"], "bfloat16")
    engine.runner.check_status()


def test_plans_are_taken_where_they_pay(model_dirs):
    """Without ``always``: not for a tiny model's short prompt."""
    from sprout_lm_b200 import load_model
    from sprout_lm_b200.engine.batch import StepEntry
    model = load_model(model_dirs["A"], dtype="bfloat16")
    rng = np.random.default_rng(43)
    prefix = helpers.random_tokens(rng, 64, 256)
    runner, seqs = started(model, prefix, [[1], [2], [3]], 16)
    runner.shared_prefix.always = False
    entries = [StepEntry(seq, [5], [0]) for seq in seqs]
    assert runner.shared_prefix.plans(entries, replayed=True) is None
    runner.shared_prefix.always = True
    assert list(runner.shared_prefix.plans(entries, replayed=True)) == [(4, 2, 16)]
    assert runner.shared_prefix.plans([StepEntry(seqs[0], [5], [0])], replayed=True) is None
    assert runner.shared_prefix.plans([StepEntry(seqs[0], [5] * 17, [0]), entries[1]], replayed=False) is None


def test_refusals(model_dirs):
    from sprout_lm_b200 import ModelRunner, load_model
    from sprout_lm_b200.engine.batch import StepEntry
    from sprout_lm_b200.engine.step import StepError
    model = load_model(model_dirs["A"], dtype="bfloat16")
    runner = ModelRunner(model, num_pages=20, page_tokens=16, max_requests=2)
    seq = runner.new_sequence()
    assert runner.reserve(seq, 10)
    entry = StepEntry(seq, [1, 2, 3], [])
    for bad in (dict(temperatures=[]), dict(accept=[0.1] * 2), dict(draw=[0.1] * 4), dict(draft_logits=torch.zeros(1, 256, device="cuda")),
                dict(entries=[StepEntry(seq, [], [])], accept=[], draw=[]), dict(entries=[StepEntry(seq, [1, 2, 999], [])])):
        given = dict(entries=[entry], temperatures=[0.0], accept=[0.1] * 3, draw=[0.1] * 3)
        given.update(bad)
        with pytest.raises(StepError):
            runner.step_and_verify(**given)
    assert seq.length == 0
    runner.manager.state_slot_count = 1
    with pytest.raises(StepError, match="per-request state"):
        runner.step_and_verify([entry], [0.0], [0.1] * 3, [0.1] * 3)
