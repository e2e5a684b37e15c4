"""Verification of drafted tokens against a plain implementation in 64 bits, request by request.

Results are whole numbers and have to be equal.  The kernel's running sums are off by about 1e-12 of the total (64-bit sums of
exponentials good to 1e-12), so a draw can come out differently only where it lands that close to a border between two tokens: with 24-bit
uniform numbers and a few thousand draws that does not happen by chance, and the fixed seeds here do not meet it."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture()
def status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def softmax64(row, temperature):
    z = row.astype(np.float64) / float(temperature)
    e = np.exp(z - z.max())
    return e / e.sum()


def draw_from(weights, w):
    sums = np.cumsum(weights)
    place = int(np.searchsorted(sums, float(w) * sums[-1], side="right"))
    return place if place < len(weights) else int(np.flatnonzero(weights)[-1])


def plain(logits, drafts, counts, draft_logits, temperatures, accept, draw):
    """(tokens, accepted, status bits) by the definition."""
    tokens, accepted, bits, at, drafted = [], [], 0, 0, 0
    vocab = logits.shape[1]
    for r, n in enumerate(counts):
        answer, stood = [-1] * (n + 1), n
        temperature = temperatures[r] if temperatures is not None else 0.0
        for i in range(n + 1):
            row, x = logits[at + i], int(drafts[at + i])
            stood = i
            if not np.isfinite(row).all():
                bits |= 4
                break
            if i < n and not 0 <= x < vocab:
                bits |= 2
                break
            if not temperature > 0:
                best = int(np.flatnonzero(row == row.max())[0])
                if i < n and x == best:
                    answer[i] = x
                    continue
                answer[i] = best
                break
            p = softmax64(row, temperature)
            if i < n:
                if draft_logits is None:
                    q = np.zeros_like(p)
                    q[x] = 1.0
                else:
                    if not np.isfinite(draft_logits[drafted + i]).all():
                        bits |= 4
                        break
                    q = softmax64(draft_logits[drafted + i], temperature)
                if float(accept[at + i]) * q[x] < p[x]:
                    answer[i] = x
                    continue
                rest = np.maximum(p - q, 0.0)
                p = rest if rest.sum() > 0 else p
            answer[i] = draw_from(p, draw[at + i])
            break
        tokens += answer
        accepted.append(stood)
        at, drafted = at + n + 1, drafted + n
    return tokens, accepted, bits


def case(counts, vocab, seed, model=True, greedy=False, spread=2.0, noise=0.7):
    rng = np.random.default_rng(seed)
    rows = sum(counts) + len(counts)
    logits = (rng.standard_normal((rows, vocab)) * spread).astype(np.float32)
    temperatures = np.array([0.0 if greedy and r % 3 == 2 else rng.choice([0.5, 0.8, 1.0, 1.7]) for r in range(len(counts))], dtype=np.float32)
    drafts = np.full(rows, -7, dtype=np.int32)           # a request's last entry is not read
    draft_logits = [] if model else None
    at = 0
    for r, n in enumerate(counts):
        for i in range(n):
            d = logits[at + i] + (rng.standard_normal(vocab) * noise).astype(np.float32)
            if model:
                draft_logits.append(d)
            t = temperatures[r]
            drafts[at + i] = int(np.argmax(logits[at + i])) if t == 0 and rng.random() < 0.7 else rng.choice(vocab, p=softmax64(d, max(t, 0.5)))
        at += n + 1
    if model:
        draft_logits = np.stack(draft_logits) if draft_logits else np.zeros((0, vocab), dtype=np.float32)
    uniform = rng.integers(0, 1 << 24, (2, rows)).astype(np.float32) / np.float32(1 << 24)
    return dict(logits=logits, drafts=drafts, counts=list(counts), draft_logits=draft_logits, temperatures=temperatures, accept=uniform[0], draw=uniform[1])


def on_device(c, pad=0, shift=0):
    """The arguments of ``verify``; rows of the logits ``pad`` apart and ``shift`` elements off their allocation's start."""
    def matrix(a):
        if a is None:
            return None
        rows, vocab = a.shape
        whole = torch.full((rows * (vocab + pad) + shift,), float("nan"), device=DEV)
        view = whole[shift:].view(rows, vocab + pad)[:, :vocab]
        view.copy_(torch.from_numpy(a))
        return view
    start = np.cumsum([0] + [n + 1 for n in c["counts"]]).astype(np.int32)
    vector = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV) if a is not None else None
    return (matrix(c["logits"]), vector(c["drafts"]), vector(start)), dict(draft_logits=matrix(c["draft_logits"]), temperatures=vector(c["temperatures"]),
                                                                          accept=vector(c["accept"]), draw=vector(c["draw"]))


def check(c, status, pad=0, shift=0):
    from sprout_lm_b200 import sampling
    args, more = on_device(c, pad, shift)
    tokens, accepted = sampling.verify(*args, status, **more)
    want_tokens, want_accepted, bits = plain(c["logits"], c["drafts"], c["counts"], c["draft_logits"], c["temperatures"], c["accept"], c["draw"])
    assert accepted.tolist() == want_accepted
    assert tokens.tolist() == want_tokens
    assert int(status.item()) == bits
    return want_tokens, want_accepted


@pytest.mark.parametrize("vocab", [1, 2, 5, 509, 4095, 4096, 4097, 33001])
@pytest.mark.parametrize("model", [True, False])
def test_against_plain(vocab, model, status):
    counts = [3, 0, 1, 5, 2, 0, 4]
    check(case(counts, vocab, seed=vocab, model=model, greedy=True), status)


@pytest.mark.parametrize("model", [True, False])
def test_many_requests_and_long_drafts(model, status):
    rng = np.random.default_rng(3)
    counts = [int(n) for n in rng.integers(0, 9, 150)] + [8, 9, 17, 40]
    c = case(counts, 700, seed=11, model=model, noise=0.2)
    tokens, accepted = check(c, status)
    assert any(a == n for a, n in zip(accepted, counts) if n) and any(a < n for a, n in zip(accepted, counts))


@pytest.mark.parametrize("model", [True, False])
def test_a_vocabulary_of_a_million(model, status):
    """More runs of a row than the drawing block holds in shared memory."""
    check(case([2, 0, 1], 1100003, 41, model=model, spread=0.5), status)


@pytest.mark.parametrize("counts", [[4, 0, 8, 1], [4, 0, 8, 1, 3, 2, 6, 5] * 3])
def test_the_same_call_many_times(counts, status):
    """Which block is done last, where that one draws, changes from call to call; nothing else does."""
    from sprout_lm_b200 import sampling
    c = case(counts, 50021, 42)
    args, more = on_device(c)
    calls = [sampling.verify(*args, status, **more) for _ in range(200)]
    want_tokens, want_accepted, bits = plain(c["logits"], c["drafts"], c["counts"], c["draft_logits"], c["temperatures"], c["accept"], c["draw"])
    assert int(status.item()) == bits == 0
    assert all(tokens.tolist() == want_tokens and accepted.tolist() == want_accepted for tokens, accepted in calls)


def test_all_stand_and_none_stands(status):
    """Drafts that the target would draw for certain stand to the end over several batches of rows; drafts it cannot draw never do."""
    vocab, n = 200, 21
    logits = np.full((2 * (n + 1), vocab), -50.0, dtype=np.float32)
    drafts = np.arange(2 * (n + 1), dtype=np.int32) % vocab
    logits[np.arange(2 * (n + 1)), drafts] = 50.0
    drafts[n + 1:] = (drafts[n + 1:] + 1) % vocab
    c = dict(logits=logits, drafts=drafts, counts=[n, n], draft_logits=None, temperatures=np.array([1.0, 1.0], np.float32),
             accept=np.full(2 * (n + 1), 0.999, np.float32), draw=np.full(2 * (n + 1), 0.5, np.float32))
    _, accepted = check(c, status)
    assert accepted == [n, 0]


@pytest.mark.parametrize("pad,shift", [(1, 0), (4, 0), (3, 1), (0, 3)])
def test_strides_and_alignment(pad, shift, status):
    check(case([2, 4, 0, 3], 9001, seed=5), status, pad, shift)


def test_every_place_of_the_distribution(status):
    """Uniform numbers across [0, 1), ends included: a looked-up draft that falls, and the place behind the last draft."""
    vocab, count = 6, 256
    base = case([1] * count, vocab, seed=2, model=False)
    base["logits"][:] = base["logits"][:1]
    base["temperatures"][:] = 1.0
    base["draw"][:] = np.repeat(np.arange(count) / np.float32(count), 2)
    base["draw"][-2:] = 1 - 2.0 ** -24
    base["accept"][:] = 0.0
    base["accept"][::4] = 1 - 2.0 ** -24
    tokens, accepted = check(base, status)
    assert set(tokens[1::2]) | set(tokens[0::2]) >= set(range(vocab))


def test_equal_distributions(status):
    """p = q: every draft stands whatever the number, and where a draft is put that q cannot draw, nothing is left of p - q."""
    c = case([4] * 12, 5000, seed=9, noise=0.0)
    c["accept"][:] = 1 - 2.0 ** -24
    _, accepted = check(c, status)
    assert accepted == [4] * 12


@pytest.mark.parametrize("counts,vocab", [([1, 3], 5000), ([1] * 40, 12000), ([2], 1100003), ([2] * 3, 1100003)])
def test_nothing_left_of_the_difference(counts, vocab, status):
    """Equal rows and numbers of 1, at which the first draft falls all the same: p - q is zero everywhere, and the token is drawn from p.  The
    last summing block draws for few requests, a launch of its own for many; beyond 256 runs the sums stay in memory."""
    c = case(counts, vocab, seed=17, noise=0.0)
    c["accept"][:] = 1.0
    tokens, accepted = check(c, status)
    assert accepted == [0] * len(counts) and all(t >= 0 for t in np.array(tokens)[np.cumsum([0] + [n + 1 for n in counts])[:-1]])


@pytest.mark.parametrize("noise", [1e-6, 1e-5, 1e-4])
def test_close_distributions(noise, status):
    """Draft rows that differ from the target's by little.  The sums that decide are off by at most (3 d + 12) 2^-24 of themselves, d the mean of
    (max - logit) / T: a draft whose u q / p is further than both rows' from 1 falls or stands as the definition has it, and the token
    of one that falls has something left of p - q and lies within the two rows' (of p, over what is left in all) of where the exact
    running sum has the draw."""
    count, vocab, t = 600, 20000, 0.9
    rng = np.random.default_rng(5)
    row = rng.standard_normal(vocab).astype(np.float32)
    near = (row + (noise * rng.standard_normal(vocab)).astype(np.float32)).astype(np.float32)
    p, q = softmax64(row, t), softmax64(near, t)
    rel = sum((3 * float((w * (l.max() - l.astype(np.float64)) / t).sum()) + 12) * 2.0 ** -24 for l, w in ((row, p), (near, q)))
    # drafts all over p / q, each with numbers on both sides of where it falls
    by_ratio = np.argsort(p / q)
    drafts = np.zeros(2 * count, np.int32)
    drafts[::2] = by_ratio[np.linspace(0, vocab - 1, count).astype(int)]
    accept = np.zeros(2 * count, np.float32)
    accept[::2] = np.where(np.arange(count) % 3 == 0, 1 - 2.0 ** -24, (p / q)[drafts[::2]] * (1 + rng.choice([-4, 4], count) * rel))
    draw = (np.arange(2 * count) / (2.0 * count)).astype(np.float32)
    c = dict(logits=np.broadcast_to(row, (2 * count, vocab)).copy(), drafts=drafts, counts=[1] * count, draft_logits=np.broadcast_to(near, (count, vocab)).copy(),
             temperatures=np.full(count, t, np.float32), accept=accept, draw=draw)
    from sprout_lm_b200 import sampling
    args, more = on_device(c)
    tokens, accepted = (x.cpu().numpy() for x in sampling.verify(*args, status, **more))
    assert int(status.item()) == 0
    x = drafts[::2]
    far = accept[::2].astype(np.float64) * q[x] / p[x] - 1.0
    clear = np.abs(far) > rel
    assert clear.sum() > count / 4 and (accepted == (far < 0))[clear].all()
    fell = np.flatnonzero(accepted == 0)
    left = np.maximum(p - q, 0.0)
    sums = np.concatenate([[0.0], np.cumsum(left)])
    assert len(fell) > 50
    for r in fell:
        token, target = int(tokens[2 * r]), float(draw[2 * r]) * sums[-1]
        assert p[token] > q[token]
        assert sums[token] - 2 * rel <= target <= sums[token + 1] + 2 * rel


def test_drafted_token_with_all_the_weight(status):
    """A looked-up draft of probability 1 that falls all the same (a number of 1): drawn from p, the draft itself."""
    vocab = 4100
    logits = np.full((2, vocab), -1e30, dtype=np.float32)
    logits[:, 77] = 3.0
    c = dict(logits=logits, drafts=np.array([77, 0], np.int32), counts=[1], draft_logits=None, temperatures=np.array([1.0], np.float32),
             accept=np.array([1.0, 0.0], np.float32), draw=np.array([0.3, 0.3], np.float32))
    tokens, accepted = check(c, status)
    assert (tokens, accepted) == ([77, -1], [0])


@pytest.mark.parametrize("size", [1e3, 1e9, 3e38])
def test_large_logits(size, status):
    """Logits far from zero: the differences decide."""
    c = case([3, 2, 0], 9000, seed=14)
    for name in ("logits", "draft_logits"):
        c[name] = (c[name] + np.float32(size)).astype(np.float32)
    check(c, status)


@pytest.mark.parametrize("temperature", [1e-38, 1e-3, 1e30, float("inf")])
def test_extreme_temperatures(temperature, status):
    c = case([3, 2, 0], 5000, seed=4)
    c["temperatures"][:] = temperature
    with np.errstate(over="ignore"):
        check(c, status)


def test_masked_logits(status):
    """Tokens masked with the type's lowest value have no probability; they neither stand nor are drawn."""
    c = case([3] * 20, 4500, seed=6)
    lowest = np.finfo(np.float32).min
    c["logits"][:, 100:] = lowest
    c["draft_logits"][:, 50:] = lowest
    for i, row in enumerate(r for r in range(80) if r % 4 != 3):
        c["drafts"][row] = i % 50 if i % 5 else 3000      # a draft the target masks
    tokens, _ = check(c, status)
    assert all(t < 100 for t in tokens)
    c["temperatures"][:] = 0.0
    check(c, status)


def test_ties_go_to_the_lowest_index(status):
    c = case([3, 0, 2], 9000, seed=8)
    c["temperatures"][:] = 0.0
    c["logits"][:, [4100, 17, 8999]] = 90.0
    c["drafts"][:] = [17, 17, 4100, 0, 0, 17, 8999, 0]
    tokens, accepted = check(c, status)
    assert accepted == [2, 0, 1] and tokens[:4] == [17, 17, 17, -1]


def test_greedy_without_temperatures(status):
    c = case([3, 1, 0], 600, seed=8)
    c.update(temperatures=None, accept=None, draw=None)
    check(c, status)


def test_flagged_rows(status):
    """A row with a non-finite logit, or a draft outside the vocabulary, ends the request's tokens where it is reached; rows behind the
    first draft that falls may hold anything."""
    for bad in (np.nan, np.inf, -np.inf):
        c = case([4, 4, 4], 5000, seed=21, noise=0.0)
        c["accept"][:] = 0.0                              # everything stands up to what is flagged
        c["logits"][2, 4321] = bad
        c["draft_logits"][4 + 1, 7] = bad
        _, accepted = check(c, status)
        assert accepted == [2, 1, 4] and int(status.item()) == 4
        status.zero_()
    c = case([4, 4], 5000, seed=22, noise=0.0)
    c["accept"][:] = 0.0
    c["drafts"][1], c["drafts"][5] = 5000, -1
    _, accepted = check(c, status)
    assert accepted == [1, 0] and int(status.item()) == 2
    status.zero_()
    c = case([4], 5000, seed=23, model=False)
    c["drafts"][0] = int(np.argmin(c["logits"][0]))
    c["accept"][:] = 1 - 2.0 ** -24
    c["logits"][1:] = np.nan
    c["drafts"][1] = 123456
    _, accepted = check(c, status)
    assert accepted == [0] and int(status.item()) == 0


def test_rows_of_nobody_stay(status):
    """Rows behind the last request's are left as they were, and a request whose rows lie outside the step's is flagged."""
    from sprout_lm_b200 import kernels
    c = case([2, 1], 300, seed=1, model=False)
    args, more = on_device(c)
    out = torch.full((5,), 99, dtype=torch.int32, device=DEV)
    accepted = torch.full((1,), 99, dtype=torch.int32, device=DEV)
    more["temperatures"] = more["temperatures"][:1].contiguous()
    kernels.verify_drafts(args[0], args[1], args[2][:2].contiguous(), status, out=out, accepted=accepted, **more)
    assert out[3:].tolist() == [99, 99] and accepted.tolist() != [99] and int(status.item()) == 0
    for start in ([0, 6], [-1, 3], [3, 3], [4, 2]):
        out.fill_(99)
        kernels.verify_drafts(args[0], args[1], torch.tensor(start, dtype=torch.int32, device=DEV), status, out=out, accepted=accepted, **more)
        assert out.tolist() == [99] * 5 and accepted.tolist() == [-1] and int(status.item()) == 64
        status.zero_()


@pytest.mark.parametrize("greedy", [False, True])
def test_no_row_of_the_result_is_left_unwritten(greedy, status):
    """Rows that are no request's, or of a request whose rows lie outside the step's, are -1 in tokens that the call makes: memory that held
    something else before shows nothing of it."""
    from sprout_lm_b200 import sampling
    c = case([2, 1, 3, 0, 4], 3000, seed=3, model=False)
    args, more = on_device(c)
    more = {} if greedy else {name: t for name, t in more.items() if t is not None}
    whole, _ = sampling.verify(*args, status, **more)
    whole, starts = whole.tolist(), args[2].tolist()
    rows = args[1].numel()
    for change in (lambda s: s[:4], lambda s: s[1:], lambda s: [*s[:5], rows + 1], lambda s: [-1, *s[1:]], lambda s: [*s[:2], s[1], *s[3:]]):
        start = change(list(starts))
        requests = len(start) - 1
        torch.cuda.synchronize()
        for n in (rows, requests):                        # what the call is likely to be given by the allocator
            torch.full((n,), 1234567, dtype=torch.int32, device=DEV)
        status.zero_()
        per_request = {name: t[:requests].contiguous() if name == "temperatures" else t for name, t in more.items()}
        if start[0] == starts[1] and not greedy:
            per_request["temperatures"] = more["temperatures"][1:].contiguous()
        tokens, accepted = sampling.verify(args[0], args[1], torch.tensor(start, dtype=torch.int32, device=DEV), status, **per_request)
        want, flagged = [-1] * rows, 0
        for r, (a, b) in enumerate(zip(start, start[1:])):
            if 0 <= a < b <= rows:
                if a in starts and b in starts and starts.index(b) == starts.index(a) + 1:
                    want[a:b] = whole[a:b]
                else:
                    want[a:b] = tokens[a:b].tolist()      # rows of two requests taken as one's: written, whatever the answer
                    assert 1234567 not in want[a:b]
            else:
                flagged = 64
                assert int(accepted[r]) == -1
        assert tokens.tolist() == want and int(status.item()) & 64 == flagged


def test_distribution_of_the_first_token(status):
    """Whatever the draft model, the first emitted token is distributed as the target's: 40,000 requests, each frequency within five
    standard deviations (the binomial's)."""
    from sprout_lm_b200 import sampling
    count, vocab = 40000, 8
    rng = np.random.default_rng(31)
    p_row, q_row = (rng.standard_normal(vocab).astype(np.float32) * 1.5 for _ in range(2))
    p, q = softmax64(p_row, 0.9), softmax64(q_row, 0.9)
    drafts = np.full(2 * count, -1, np.int32)
    drafts[::2] = rng.choice(vocab, count, p=q)
    uniform = torch.from_numpy(rng.random((2, 2 * count)).astype(np.float32).clip(0, 1 - 2.0 ** -24)).to(DEV)
    start = torch.arange(0, 2 * count + 1, 2, dtype=torch.int32, device=DEV)
    tokens, accepted = sampling.verify(torch.from_numpy(p_row).to(DEV).expand(2 * count, vocab), torch.from_numpy(drafts).to(DEV), start, status,
                                       draft_logits=torch.from_numpy(q_row).to(DEV).repeat(count, 1),
                                       temperatures=torch.full((count,), 0.9, device=DEV), accept=uniform[0], draw=uniform[1])
    seen = np.bincount(tokens[::2].cpu().numpy(), minlength=vocab) / count
    assert (np.abs(seen - p) <= 5 * np.sqrt(p * (1 - p) / count)).all()
    stands = np.minimum(p, q).sum()
    assert abs(accepted.float().mean().item() - stands) <= 5 * np.sqrt(stands * (1 - stands) / count)


def test_captured_and_on_another_stream(status):
    """A captured call replayed with other numbers, two captures side by side, and a call on a stream of its own give what eager calls give."""
    from sprout_lm_b200 import sampling
    cases = [case([3, 0, 5, 2], 9000, seed=s, greedy=True) for s in (41, 42, 43)]
    eager = []
    for c in cases:
        args, more = on_device(c)
        eager.append([t.clone() for t in sampling.verify(*args, status, **more)])
    args, more = on_device(cases[0])
    graphs = []
    torch.cuda.synchronize()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = sampling.verify(*args, status, **more)
        graphs.append((graph, held))
    for c, want in zip(cases, eager):
        fresh, extra = on_device(c)
        assert fresh[2].tolist() == args[2].tolist()
        for mine, new in list(zip(args, fresh)) + [(more[k], extra[k]) for k in more]:
            mine.copy_(new)
        for graph, held in graphs:
            graph.replay()
        for graph, held in graphs:
            assert all(torch.equal(a, b) for a, b in zip(held, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = sampling.verify(*args, status, **more)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, eager[-1]))


def test_refusals(status):
    from sprout_lm_b200 import kernels
    c = case([2, 1], 300, seed=1)
    args, more = on_device(c)
    out, accepted = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (5, 2))

    def refused(match, **changes):
        given = dict(logits=args[0], drafts=args[1], row_start=args[2], out=out, accepted=accepted, status=status, **more)
        given.update(changes)
        with pytest.raises(kernels.KernelError, match=match):
            kernels.verify_drafts(**given)

    refused("CUDA tensor", logits=args[0].cpu())
    refused("must be torch.float32", draft_logits=more["draft_logits"].double())
    refused("must be torch.float32", logits=args[0].double())
    refused("unit inner stride", logits=args[0].t())
    refused("at least one request", row_start=args[2][:1])
    refused("drafts must be contiguous int32", drafts=args[1].long())
    refused("drafts must be contiguous int32", drafts=args[1][:3])
    refused("out must be contiguous int32", out=torch.zeros(10, dtype=torch.int32, device=DEV)[::2])
    refused("accepted must be", accepted=out)
    refused("go together", draw=None)
    refused("go together", temperatures=None)
    refused("temperatures must be", temperatures=more["temperatures"].double())
    refused("accept must be", accept=more["accept"][:2])
    refused("a row per draft", draft_logits=more["draft_logits"][:2])
    refused("a row per draft", draft_logits=more["draft_logits"][:, :200].contiguous())
    refused("share memory", out=args[1])
    refused("share memory", accepted=out[:2])
    assert int(status.item()) == 0
