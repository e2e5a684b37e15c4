"""Operators of serving steps that check drafted tokens and share a prompt, as timed cases.

* ``attention``: attention of a step's tokens over the paged cache where requests hold the same leading pages (a common
  system prompt, several answers to one question): one token a request, or a few drafted ones.  The prefix's keys and values
  are needed once for all requests that share them.
* ``verify``: drafted tokens against the target's probabilities, with given random numbers: which drafts stand, and the
  token after the last of them.

Sizes are those of the benchmark's model shapes (heads, key/value heads, head size; vocabularies of the configurations).
How long the requests are follows from the case alone, what their tensors hold from the seed.
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
SHAPES = {"0.5b": (14, 2, 64), "7b": (28, 4, 128), "14b": (40, 8, 128)}     # heads, key/value heads, head size
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # three answers to one short prompt: the smallest call, where launches and latency count
        {"name": "few-short", "kind": "attention", "shape": "0.5b", "dtype": "bf16", "page": 16, "requests": 3, "tokens": 1, "groups": 1,
         "prefix": 700, "own": 40},
        # a small model's busy server behind one system prompt
        {"name": "shared-64", "kind": "attention", "shape": "0.5b", "dtype": "bf16", "page": 16, "requests": 64, "tokens": 1, "groups": 1,
         "prefix": 4096, "own": 600},
        # long conversations behind a shared prompt: most keys are the requests' own
        {"name": "mostly-own-32", "kind": "attention", "shape": "14b", "dtype": "bf16", "page": 16, "requests": 32, "tokens": 1, "groups": 1,
         "prefix": 1024, "own": 3300},
        # drafted tokens checked: up to six tokens a request
        {"name": "drafts-24", "kind": "attention", "shape": "7b", "dtype": "bf16", "page": 16, "requests": 24, "tokens": 6, "groups": 1,
         "prefix": 2000, "own": 500},
        # several prompts, each with answers of its own, groups of uneven sizes
        {"name": "groups-90", "kind": "attention", "shape": "0.5b", "dtype": "bf16", "page": 32, "requests": 90, "tokens": 2, "groups": 6,
         "prefix": 5000, "own": 300},
        # many requests over one long document: the largest call, a matrix product's worth of arithmetic
        {"name": "long-256", "kind": "attention", "shape": "7b", "dtype": "bf16", "page": 16, "requests": 256, "tokens": 1, "groups": 1,
         "prefix": 32768, "own": 400},
        # the 32-bit path
        {"name": "float32-12", "kind": "attention", "shape": "0.5b", "dtype": "f32", "page": 16, "requests": 12, "tokens": 3, "groups": 1,
         "prefix": 1500, "own": 200},
        # one user, drafts looked up in the text: no draft distribution
        {"name": "lookup-1", "kind": "verify", "vocab": 151936, "requests": 1, "drafts": 4, "model": False, "greedy": False},
        # a small batch with a draft model's logits
        {"name": "model-8", "kind": "verify", "vocab": 151936, "requests": 8, "drafts": 5, "model": True, "greedy": False},
        # the largest: a busy server's batch with a draft model, some requests greedy
        {"name": "model-64", "kind": "verify", "vocab": 152064, "requests": 64, "drafts": 8, "model": True, "greedy": True},
        # a batch with a smaller vocabulary, looked-up drafts, some requests greedy
        {"name": "lookup-48", "kind": "verify", "vocab": 32768, "requests": 48, "drafts": 6, "model": False, "greedy": True},
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    if rng.random() < 0.4:
        return {"kind": "verify", "vocab": rng.choice([32768, 151936, 152064, _spread(rng, 509, 152064), _spread(rng, 509, 152064)]),
                "requests": _spread(rng, 1, 64), "drafts": rng.randint(1, 8), "model": rng.random() < 0.6, "greedy": rng.random() < 0.4}
    requests = _spread(rng, 2, 256)
    case = {"kind": "attention", "shape": rng.choice(list(SHAPES)), "dtype": "f32" if rng.random() < 0.12 else "bf16",
            "page": rng.choice([8, 16, 16, 32, 64]), "requests": requests, "tokens": rng.choice([1, 1, 2, rng.randint(3, 8)]),
            "groups": min(requests, rng.choice([1, 1, 2, rng.randint(3, 9)])), "prefix": _spread(rng, 100, 32768), "own": _spread(rng, 8, 3300)}
    if case["dtype"] == "f32":
        case.update(shape="0.5b", requests=min(requests, 16), groups=min(case["groups"], 3), prefix=min(case["prefix"], 4000), own=min(case["own"], 1000))
    # no more than the largest listed case, in arithmetic and in bytes
    largest = work(listed()[5])
    while True:
        w = work(case)
        if w["flops"] <= largest["flops"] and w["bytes"] <= largest["bytes"] and _visited(case) <= 256 * 33200 * 4:
            return case
        case["prefix"] = max(64, case["prefix"] * 2 // 3)
        case["own"] = max(8, case["own"] * 2 // 3)
        case["requests"] = max(2, case["requests"] * 7 // 8)
        case["groups"] = min(case["groups"], case["requests"])


# ---------------------------------------------------------------------------------- lengths
def _rng(case):
    return random.Random("/".join(str(case[k]) for k in sorted(case) if k != "name"))


def _attention_lengths(case):
    """Per request: its group, the tokens cached beyond the prefix, the tokens it brings; per group: the prefix (whole pages)."""
    rng, page = _rng(case), case["page"]
    groups = case["groups"]
    cuts = sorted(rng.sample(range(1, case["requests"]), groups - 1)) if groups > 1 else []
    group = [sum(r >= c for c in cuts) for r in range(case["requests"])]
    rng.shuffle(group)
    own = [rng.randint(0, case["own"]) for _ in range(case["requests"])]
    tokens = [rng.randint(1, case["tokens"]) for _ in range(case["requests"])]
    prefix = [max(1, (case["prefix"] if groups == 1 else rng.randint(case["prefix"] // 2, case["prefix"])) // page) * page for _ in range(groups)]
    return group, own, tokens, prefix


def _visited(case):
    """(request, key) places that a form without the sharing reads, times the key/value heads."""
    group, own, tokens, prefix = _attention_lengths(case)
    return sum(prefix[g] + o + t for g, o, t in zip(group, own, tokens)) * SHAPES[case["shape"]][1]


def _verify_lengths(case):
    rng = _rng(case)
    drafts = [rng.randint(0, case["drafts"]) for _ in range(case["requests"])]
    drafts[0] = case["drafts"]
    temperatures = [0.0 if case["greedy"] and r % 3 == 2 else rng.choice([0.6, 0.8, 1.0]) for r in range(case["requests"])]
    return drafts, temperatures


def work(case):
    if case["kind"] == "verify":
        drafts, _ = _verify_lengths(case)
        rows = sum(drafts) + case["requests"]
        read = rows + (sum(drafts) if case["model"] else 0)
        # a softmax over every row (a difference, a product, an exponential, a sum)
        return {"bytes": 4 * read * case["vocab"] + 16 * rows, "flops": 4 * read * case["vocab"]}
    heads, kv_heads, dim = SHAPES[case["shape"]]
    size = 2 if case["dtype"] == "bf16" else 4
    group, own, tokens, prefix = _attention_lengths(case)
    keys = sum(prefix) + sum(own) + sum(tokens)
    pairs = sum(t * (prefix[g] + o) + t * (t + 1) // 2 for g, o, t in zip(group, own, tokens))
    return {"bytes": size * (2 * keys * kv_heads * dim + 2 * sum(tokens) * heads * dim), "flops": 4 * pairs * heads * dim}


# ---------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    generator = torch.Generator(device=DEVICE).manual_seed(seed)
    return (_prepare_verify if case["kind"] == "verify" else _prepare_attention)(case, generator)


def _prepare_attention(case, generator):
    heads, kv_heads, dim = SHAPES[case["shape"]]
    dtype, page = TYPES[case["dtype"]], case["page"]
    group, own_keys, tokens, prefix = _attention_lengths(case)
    requests = case["requests"]
    contexts = [prefix[g] + o + t for g, o, t in zip(group, own_keys, tokens)]
    # the pool as a server has it after a while: pages in any order
    own_pages = [-(-(o + t) // page) for o, t in zip(own_keys, tokens)]
    total = sum(prefix) // page + sum(own_pages) + 8
    free = torch.randperm(total, generator=generator, device=DEVICE).tolist()
    shared = [[free.pop() for _ in range(n // page)] for n in prefix]
    tables = [shared[group[r]] + [free.pop() for _ in range(own_pages[r])] for r in range(requests)]
    width = max(len(t) for t in tables)
    table = torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.int32)
    q_start = torch.tensor([0] + tokens, dtype=torch.int32).cumsum(0, dtype=torch.int32)
    positions = torch.cat([torch.arange(c - t, c, dtype=torch.int32) for c, t in zip(contexts, tokens)])

    def normal(*shape):
        return torch.randn(*shape, generator=generator, device=DEVICE, dtype=torch.float32)

    qkv = normal(sum(tokens), (heads + 2 * kv_heads) * dim)
    qkv[:, :heads * dim] *= 1.0 + torch.rand(sum(tokens), 1, generator=generator, device=DEVICE)     # some queries attend more sharply than others
    state = {"case": case, "tables": tables, "contexts": contexts, "tokens": tokens, "q": qkv.to(dtype)[:, :heads * dim],
             "k": normal(total, kv_heads, page, dim).to(dtype), "v": normal(total, kv_heads, page, dim).to(dtype),
             "block_table": table.to(DEVICE), "positions": positions.to(DEVICE)}
    if own:
        from sprout_lm_b200 import kernels
        # the step's plan, made once a step and used by all layers
        state["plan"] = kernels.shared_prefix_plan(table.numpy(), q_start.numpy(), contexts, page, heads, kv_heads, dim, dtype, DEVICE)
        state["status"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    return state


def _prepare_verify(case, generator):
    drafts, temperatures = _verify_lengths(case)
    rows, vocab = sum(drafts) + case["requests"], case["vocab"]

    def normal(*shape):
        return torch.randn(*shape, generator=generator, device=DEVICE, dtype=torch.float32)

    def uniform(n):
        # 24 bits, as the engine's own numbers
        return torch.randint(0, 1 << 24, (n,), generator=generator, device=DEVICE).float() / float(1 << 24)

    # a wide floor and a few likely tokens a row
    logits = 2.0 * normal(rows, vocab)
    likely = torch.randint(0, vocab, (rows, 24), generator=generator, device=DEVICE)
    logits.scatter_(1, likely, 11.0 + 5.0 * torch.rand(rows, 24, generator=generator, device=DEVICE))
    start = [0]
    for n in drafts:
        start.append(start[-1] + n + 1)
    drafted = [start[r] + i for r, n in enumerate(drafts) for i in range(n)]
    of_row = torch.tensor([t if t > 0 else 1.0 for r, n in enumerate(drafts) for t in [temperatures[r]] * n], device=DEVICE)
    tokens = torch.full((rows,), -1, dtype=torch.int32, device=DEVICE)
    draft_logits = None
    if drafted:
        at = torch.tensor(drafted, device=DEVICE)
        picked = torch.empty(len(drafted), dtype=torch.int64, device=DEVICE)
        if case["model"]:
            draft_logits = torch.empty(len(drafted), vocab, dtype=torch.float32, device=DEVICE)
        for i, row in enumerate(drafted):
            scores = logits[row]
            if case["model"]:
                scores = torch.add(scores, normal(vocab), alpha=0.7, out=draft_logits[i])
            noise = -torch.log(-torch.log(torch.rand(vocab, generator=generator, device=DEVICE).clamp_(1e-7, 1 - 1e-7)))
            picked[i] = torch.argmax(scores / of_row[i] + noise)
        if not case["model"]:
            # what a look-up finds is often right and often not
            guess = torch.randint(0, vocab, (len(drafted),), generator=generator, device=DEVICE)
            picked = torch.where(torch.rand(len(drafted), generator=generator, device=DEVICE) < 0.7, picked, guess)
        greedy = torch.tensor([temperatures[r] == 0 for r, n in enumerate(drafts) for _ in range(n)], device=DEVICE)
        best = torch.stack([logits[row].argmax() for row in drafted])
        picked = torch.where(greedy & (torch.rand(len(drafted), generator=generator, device=DEVICE) < 0.8), best, picked)
        tokens[at] = picked.to(torch.int32)
    state = {"case": case, "counts": drafts, "host_temperatures": temperatures, "logits": logits, "draft_logits": draft_logits, "drafts": tokens,
             "row_start": torch.tensor(start, dtype=torch.int32, device=DEVICE), "temperatures": torch.tensor(temperatures, device=DEVICE),
             "accept": uniform(rows), "draw": uniform(rows)}
    if own:
        state["status"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    return state


# ---------------------------------------------------------------------------------- one pass
def run(state):
    if state["case"]["kind"] == "verify":
        return _own_verify(state) if own else _plain_verify(state)
    return _own_attention(state) if own else _plain_attention(state)


def _own_attention(state):
    from sprout_lm_b200 import kernels
    heads, kv_heads, dim = SHAPES[state["case"]["shape"]]
    q = state["q"]
    out = torch.empty((q.shape[0], heads * dim), dtype=q.dtype, device=q.device)
    kernels.attention_shared_prefix(q, state["k"], state["v"], state["block_table"], state["positions"], state["plan"], out, state["status"])
    return out


def _own_verify(state):
    from sprout_lm_b200 import sampling
    return sampling.verify(state["logits"], state["drafts"], state["row_start"], state["status"], draft_logits=state["draft_logits"],
                           temperatures=state["temperatures"], accept=state["accept"], draw=state["draw"])


def _plain_attention(state):
    """A request at a time: gather its keys and values, scores, softmax, weighted sum; 32 bits, rounded once."""
    heads, kv_heads, dim = SHAPES[state["case"]["shape"]]
    group = heads // kv_heads
    q, page = state["q"], state["case"]["page"]
    out = torch.empty((q.shape[0], heads * dim), dtype=q.dtype, device=q.device)
    at = 0
    for r, (context, n) in enumerate(zip(state["contexts"], state["tokens"])):
        pages = state["block_table"][r, :-(-context // page)].long()
        k = state["k"][pages].transpose(0, 1).reshape(kv_heads, -1, dim)[:, :context].float()
        v = state["v"][pages].transpose(0, 1).reshape(kv_heads, -1, dim)[:, :context].float()
        rows = q[at:at + n].float().view(n, kv_heads, group, dim).permute(1, 0, 2, 3).reshape(kv_heads, n * group, dim)
        scores = torch.matmul(rows, k.transpose(1, 2)) * (1.0 / math.sqrt(dim))
        if n > 1:
            limit = torch.arange(context - n, context, device=q.device).repeat_interleave(group)
            scores.masked_fill_(torch.arange(context, device=q.device)[None, None, :] > limit[None, :, None], -math.inf)
        scores = torch.exp(scores - scores.amax(-1, keepdim=True))
        mixed = torch.matmul(scores, v) / scores.sum(-1, keepdim=True)
        out[at:at + n] = mixed.view(kv_heads, n, group, dim).permute(1, 0, 2, 3).reshape(n, heads * dim).to(q.dtype)
        at += n
    return out


def _plain_verify(state):
    """A request at a time: softmax of its rows, which drafts stand, and the inverse of the cumulative distribution at the draw.  64 bits:
    a sum over a vocabulary decides between neighbouring tokens."""
    drafts, draft_logits = state["drafts"], state["draft_logits"]
    rows, vocab = state["logits"].shape
    tokens = torch.full((rows,), -1, dtype=torch.int32, device=DEVICE)
    accepted = torch.empty(len(state["counts"]), dtype=torch.int32, device=DEVICE)
    index = torch.arange(vocab, device=DEVICE)
    at = drafted_at = 0
    for r, n in enumerate(state["counts"]):
        logits, x = state["logits"][at:at + n + 1], drafts[at:at + n].long()
        temperature = state["host_temperatures"][r]
        step = torch.arange(n + 1, device=DEVICE)
        if temperature == 0:
            best = torch.where(logits == logits.amax(-1, keepdim=True), index, vocab).amin(-1)
            stands = (x == best[:n]).long()
            count = stands.cumprod(0).sum()
            last = best[count]
        else:
            scaled = logits.double() / temperature
            weight = torch.exp(scaled - scaled.amax(-1, keepdim=True))
            p = weight / weight.sum(-1, keepdim=True)
            q = torch.zeros_like(p)                                  # the place after the last draft has nothing to take away
            if draft_logits is not None:
                scaled = draft_logits[drafted_at:drafted_at + n].double() / temperature
                weight = torch.exp(scaled - scaled.amax(-1, keepdim=True)) if n else scaled
                q[:n] = weight / weight.sum(-1, keepdim=True)
            else:
                q[step[:n], x] = 1.0
            stands = (state["accept"][at:at + n].double() * q[step[:n], x] < p[step[:n], x]).long()
            count = stands.cumprod(0).sum()
            left = (p[count] - q[count]).clamp(min=0)
            left = torch.where(left.sum() > 0, left, p[count])
            sums = left.cumsum(0)
            target = state["draw"][at + count].double() * sums[-1]
            last = torch.searchsorted(sums, target, right=True).clamp(max=vocab - 1)
        kept = torch.where(step < count, torch.nn.functional.pad(x, (0, 1)), -1)
        tokens[at:at + n + 1] = torch.where(step == count, last, kept).to(torch.int32)
        accepted[r] = count
        at, drafted_at = at + n + 1, drafted_at + n
    return tokens, accepted


# ---------------------------------------------------------------------------------- from the definition, in 64 bits
def exact(case, seed):
    global own
    before, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before
    return (_exact_verify if case["kind"] == "verify" else _exact_attention)(state)


def _exact_attention(state):
    heads, kv_heads, dim = SHAPES[state["case"]["shape"]]
    page, device = state["case"]["page"], state["q"].device
    outputs, at = [], 0
    for table, context, n in zip(state["tables"], state["contexts"], state["tokens"]):
        place = torch.arange(context, device=device)
        page_of = torch.tensor(table, device=device)[place // page]
        k, v = state["k"][page_of, :, place % page].double(), state["v"][page_of, :, place % page].double()        # [context, kv_heads, dim]
        q = state["q"][at:at + n].double().reshape(n, kv_heads, heads // kv_heads, dim)
        scores = torch.einsum("tghd,cgd->tghc", q, k) / dim ** 0.5
        hidden = place[None, :] > torch.arange(context - n, context, device=device)[:, None]
        scores = scores.masked_fill(hidden[:, None, None, :], -torch.inf)
        weights = torch.exp(scores - torch.logsumexp(scores, -1, keepdim=True))
        outputs.append(torch.einsum("tghc,cgd->tghd", weights, v).reshape(n, heads * dim))
        at += n
    return torch.cat(outputs)


def _exact_verify(state):
    import numpy as np
    tokens, accepted = [], []
    x_all, u, w = (state[name].cpu().numpy() for name in ("drafts", "accept", "draw"))
    at = drafted_at = 0
    for r, n in enumerate(state["counts"]):
        temperature, answer, stood = state["host_temperatures"][r], [-1] * (n + 1), n
        for i in range(n + 1):
            l = state["logits"][at + i].double().cpu().numpy()
            x = int(x_all[at + i])
            if temperature == 0:
                best = int(np.flatnonzero(l == l.max())[0])
                if i < n and x == best:
                    answer[i] = x
                    continue
                answer[i], stood = best, i
                break
            p = np.exp(l / temperature - np.logaddexp.reduce(l / temperature))
            if i < n:
                q = np.zeros_like(p)
                if state["draft_logits"] is None:
                    q[x] = 1.0
                else:
                    d = state["draft_logits"][drafted_at + i].double().cpu().numpy() / temperature
                    q = np.exp(d - np.logaddexp.reduce(d))
                if float(u[at + i]) * q[x] < p[x]:
                    answer[i] = x
                    continue
                left = np.maximum(p - q, 0.0)
                p = left if left.sum() > 0 else p
            sums = np.cumsum(p)
            answer[i], stood = min(int(np.searchsorted(sums, float(w[at + i]) * sums[-1], side="right")), len(p) - 1), i
            break
        tokens += answer
        accepted.append(stood)
        at, drafted_at = at + n + 1, drafted_at + n
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(accepted, dtype=torch.int32)
