"""What the requests of one served batch bring of their own, measured on one MI355X: low-rank adapters
beside a projection that all share, and the pick of each request's next token by its own temperature,
top-k, top-p and min-p from a given random number.

``listed`` holds the measured cases, ``draw`` spreads over the same ranges. Widths, batches, vocabularies
and chunks of prompts are those of the benchmark's configurations (Qwen3-0.6B and 4B) and of the cases of
the operators over a paged cache; ranks are generic. All inputs come from the seed through torch's
generators; lengths, adapters and settings come from the case alone.

With ``own`` false the operators run in their plain form, elementary torch operations in 32 bits (weights
of tokens and their running sums, next to which a pick falls, in 64) rounded once at the end; with ``own``
true through the library's entry points.
"""
import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32


def _package():
    if "llm_inference_amd" not in sys.modules:
        home = ROOT / "llm-inference_amd"
        spec = importlib.util.spec_from_file_location(
            "llm_inference_amd", home / "__init__.py", submodule_search_locations=[str(home)])
        module = importlib.util.module_from_spec(spec)
        sys.modules["llm_inference_amd"] = module
        spec.loader.exec_module(module)
    return sys.modules["llm_inference_amd"]


# ---- cases ----

def _project(**c):
    return dict(dict(kind="project", chunks=0, new=1, spare=0, product=True, residual=False), **c)


def _pick(**c):
    return dict(dict(kind="pick", masked=False), **c)


def listed():
    return [
        # one conversation's next token through the 0.6B query projection, its own small adapter: the smallest
        _project(name="project_token", n_in=1024, n_out=2048, seqs=1, rank=8, adapters=4, mix=1),
        # the next token of 64 conversations through the 4B query projection, most with an adapter of their own
        _project(name="project_batch", n_in=2560, n_out=4096, seqs=64, rank=16, adapters=48, mix=2),
        # the next token of 17 conversations through the 4B down projection, added to the residual stream
        _project(name="project_down", n_in=9728, n_out=2560, seqs=17, rank=64, adapters=6, residual=True, mix=3),
        # the rows of five prompts through the 4B gate projection: the largest product
        _project(name="project_prompts", n_in=2560, n_out=9728, seqs=5, chunks=5, new=1500, rank=32, adapters=4, mix=4),
        # chunks of two prompts beside the next tokens of 20 conversations, 4B down projection, padded batch
        _project(name="project_mixed", n_in=9728, n_out=2560, seqs=22, chunks=2, new=511, rank=64, adapters=9,
                 residual=True, spare=14, mix=5),
        # adapters alone, added to a 4B query/key/value projection that was computed without them
        _project(name="project_beside", n_in=2560, n_out=6144, seqs=3, chunks=3, new=701, rank=128, adapters=3,
                 product=False, residual=True, mix=6),
        # the 4B output head for 64 conversations, no adapters: the most bytes
        _project(name="project_head", n_in=2560, n_out=151936, seqs=64, rank=0, adapters=0, mix=7),
        # a token pick for one conversation: temperature, top-k and top-p
        _pick(name="pick_row", rows=1, vocab=151936, settings="common", mix=8),
        # picks for 64 conversations with settings of every kind, greedy ones among them, half with a token mask
        _pick(name="pick_batch", rows=64, vocab=151936, settings="any", masked=True, mix=9),
        # picks from whole distributions, temperature alone
        _pick(name="pick_open", rows=16, vocab=151936, settings="open", mix=10),
        # many conversations over a vocabulary whose rows are not aligned
        _pick(name="pick_many", rows=200, vocab=32003, settings="common", mix=11),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    by_name = {c["name"]: work(c) for c in listed()}
    while True:
        mix = rng.randrange(1 << 20)
        if rng.random() < 0.35:
            c = _pick(rows=_log(rng, 1, 256), vocab=_log(rng, 100, 151936), masked=rng.random() < 0.4,
                      settings=rng.choice(["common", "any", "open"]), mix=mix)
            if work(c)["bytes"] <= by_name["pick_batch"]["bytes"]:
                return c
            continue
        seqs = _log(rng, 1, 128)
        c = _project(n_in=8 * _log(rng, 8, 1216), n_out=_log(rng, 16, 19456), seqs=seqs, mix=mix,
                     chunks=rng.choice([0, 0, rng.randint(0, seqs), min(seqs, 2)]), new=_log(rng, 1, 2048),
                     rank=rng.choice([8, 16, 16, 24, 32, 64, 128]), adapters=_log(rng, 1, 64),
                     spare=rng.choice([0, 0, rng.randint(1, 30)]), product=rng.random() < 0.85,
                     residual=rng.random() < 0.5)
        if rng.random() < 0.7:  # most models' widths are whole
            c["n_out"] = -(-c["n_out"] // 64) * 64
        if rng.random() < 0.1:
            c.update(rank=0, adapters=0, product=True)
        cost = work(c)
        if sum(_lengths(c)) > 4096 or cost["flops"] > by_name["project_prompts"]["flops"]:
            continue
        if cost["bytes"] <= by_name["project_head"]["bytes"]:
            return c


def _lengths(c):
    """New rows of each sequence; the first of those with a prompt's chunk has the most."""
    r = random.Random(c["mix"])
    spread = [r.random() for _ in range(c["seqs"])]
    return [(c["new"] if i == 0 else 1 + int(a * (c["new"] - 1))) if i < c["chunks"] else 1
            for i, a in enumerate(spread)]


def _adapters(c):
    """The adapter of each sequence, -1 for about one in eight; the first sequence has one."""
    r = random.Random(c["mix"] + 1)
    picks = [(r.random(), r.randrange(max(c["adapters"], 1))) for _ in range(c["seqs"])]
    return [a if i == 0 or p > 0.125 else -1 for i, (p, a) in enumerate(picks)]


def _settings(c):
    """(temperature, top_k, top_p, min_p) of each row."""
    r = random.Random(c["mix"])
    rows = []
    for _ in range(c["rows"]):
        if c["settings"] == "open":
            rows.append((1.0, 0, 1.0, 0.0))
        elif c["settings"] == "common":
            rows.append((r.uniform(0.5, 1.0), r.choice([20, 40, 50]), r.uniform(0.8, 0.95), 0.0))
        else:
            rows.append((r.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.4]), r.choice([0, 0, 1, 20, 50, 1000]),
                         r.choice([1.0, 1.0, 0.5, 0.9, 0.95]), r.choice([0.0, 0.0, 0.02, 0.1])))
    return rows


def work(c):
    if c["kind"] == "pick":
        return dict(bytes=c["rows"] * (2 * c["vocab"] + 4 + 4 + 20), flops=4 * c["rows"] * c["vocab"])
    n_in, n_out, lengths = c["n_in"], c["n_out"], _lengths(c)
    rows = sum(lengths)
    used = _adapters(c) if c["adapters"] else []
    adapted = sum(n for n, a in zip(lengths, used) if a >= 0)
    weights = len(set(used) - {-1}) * c["rank"] * (n_in + n_out) + (n_in * n_out if c["product"] else 0)
    io = rows * n_out * (2 if c["residual"] else 1) + (rows if c["product"] else adapted) * n_in
    return dict(bytes=2 * (weights + io),
                flops=2 * (rows * n_in * n_out if c["product"] else 0) + 2 * adapted * c["rank"] * (n_in + n_out))


# ---- inputs ----

def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.empty(*shape, dtype=BF16, device="cuda").normal_(0.0, std, generator=g)

    def column(values, dtype):
        return torch.tensor(values, dtype=dtype, device="cuda")

    s = dict(c=c, ws=None)
    if c["kind"] == "pick":
        rows, vocab = c["rows"], c["vocab"]
        x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.5
        # some tokens that fit, far above the others
        likely = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
        x.scatter_add_(1, likely, torch.rand(rows, 24, generator=g, device="cuda") * 10 + 4)
        if c["masked"]:  # every other row: a grammar allows about half of the tokens
            x[::2].masked_fill_(torch.rand(x[::2].shape, generator=g, device="cuda") < 0.5, -math.inf)
        temperature, top_k, top_p, min_p = zip(*_settings(c))
        s.update(logits=x.to(BF16), u=torch.rand(rows, generator=g, device="cuda"),
                 token=torch.empty(rows, dtype=I32, device="cuda"), logprob=torch.empty(rows, device="cuda"),
                 temperature=column(temperature, F32), top_k=None, top_p=None, min_p=None)
        if c["settings"] != "open":
            s.update(top_k=column(top_k, I32), top_p=column(top_p, F32))
        if c["settings"] == "any":
            s["min_p"] = column(min_p, F32)
        if own:
            floats = _package().sample_rows_workspace_floats(rows, vocab)
            s["ws"] = torch.empty(max(floats, 1), device="cuda")
        return s
    n_in, n_out, rank = c["n_in"], c["n_out"], c["rank"]
    starts = [0]
    for n in _lengths(c):
        starts.append(starts[-1] + n)
    rows = starts[-1] + c["spare"]
    s.update(x=normal(rows, n_in), out=torch.zeros(rows, n_out, dtype=BF16, device="cuda"), starts=starts,
             w=normal(n_out, n_in, std=n_in ** -0.5) if c["product"] else None,
             residual=normal(rows, n_out) if c["residual"] else None, lora_a=None, lora_b=None, lora_scale=None,
             q_start=None, adapter=None)
    if c["adapters"]:
        s.update(lora_a=normal(c["adapters"], rank, n_in, std=n_in ** -0.5),
                 lora_b=normal(c["adapters"], n_out, rank, std=0.5 * rank ** -0.5),
                 lora_scale=torch.rand(c["adapters"], generator=g, device="cuda") * 1.5 + 0.5,
                 q_start=column(starts, I32), adapter=column(_adapters(c), I32))
    if own:  # the workspace that a program keeps for these calls
        floats = _package().lora_projection_workspace_floats(rows, n_out, n_in, rank)
        s["ws"] = torch.empty(max(floats, 1), device="cuda")
    return s


# ---- one pass ----

def run(s):
    if s["c"]["kind"] == "pick":
        (_pick_own if own else _pick_plain)(s)
        return dict(token=s["token"], logprob=s["logprob"])
    (_project_own if own else _project_plain)(s)
    return s["out"]


def _project_own(s):
    _package().lora_projection_forward(
        s["out"], s["x"], s["w"], s["lora_a"], s["lora_b"], s["lora_scale"], s["q_start"], s["adapter"],
        residual=s["residual"], ws=s["ws"])


def _pick_own(s):
    _package().sample_rows_forward(
        s["token"], s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"],
        logprob=s["logprob"], ws=s["ws"])


def _project_plain(s):
    c, starts = s["c"], s["starts"]
    rows = starts[-1] if c["adapters"] else s["x"].shape[0]  # rows behind the last sequence stay
    x = s["x"][:rows].to(F32)
    y = x @ s["w"].to(F32).T if c["product"] else torch.zeros(rows, c["n_out"], device="cuda")
    at = {}
    for i, a in enumerate(_adapters(c) if c["adapters"] else []):
        if a >= 0:
            at.setdefault(a, []).append(slice(starts[i], starts[i + 1]))
    for a, parts in at.items():  # each adapter once, for the rows of all its sequences
        low = torch.cat([x[p] for p in parts]) @ s["lora_a"][a].to(F32).T
        more = (low * s["lora_scale"][a]) @ s["lora_b"][a].to(F32).T
        for p, part in zip(parts, more.split([p.stop - p.start for p in parts])):
            y[p] += part
    if c["residual"]:
        y += s["residual"][:rows]
    s["out"][:rows] = y.to(BF16)


def _pick_plain(s):
    x, order = (s["logits"].to(F64) + 0.0).sort(dim=1, descending=True, stable=True)
    temperature = s["temperature"].to(F64)[:, None]
    greedy = temperature <= 0
    weights = torch.exp((x - x[:, :1]) / torch.where(greedy, 1.0, temperature))
    place = torch.arange(x.shape[1], device="cuda")
    kept = x > -math.inf
    kept &= ~greedy | (place == 0)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        kept &= (k <= 0) | (place < k)
    weights = weights * kept
    if s["top_p"] is not None:
        p = s["top_p"].to(F64)[:, None]
        upto = weights.cumsum(1)
        kept &= (p >= 1) | (place == 0) | (upto - weights < p * upto[:, -1:])
        weights = weights * kept
    if s["min_p"] is not None:
        weights = weights * ((weights >= s["min_p"].to(F64)[:, None]) | (place == 0))
    upto = weights.cumsum(1)
    total = upto[:, -1:]
    pick = (upto <= s["u"].to(F64)[:, None] * total).sum(1, keepdim=True)
    s["token"].copy_(order.gather(1, pick)[:, 0])
    s["logprob"].copy_(torch.log(weights.gather(1, pick) / total)[:, 0])


# ---- the same from the definitions, in 64 bits ----

def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "pick":
        tokens, logprobs = [], []
        settings = _settings(c)
        for r in range(c["rows"]):
            temperature, top_k, top_p, min_p = settings[r]
            top_p, min_p, temperature = (float(torch.tensor(v, dtype=F32)) for v in (top_p, min_p, temperature))
            x = s["logits"][r].to(F64)
            # values one by one, largest first, and the tokens that have each
            values, which, counts = torch.unique(x, return_inverse=True, return_counts=True)
            values, counts = values.flip(0), counts.flip(0).to(F64)
            there = values > -math.inf
            values, counts = values[there], counts[there]
            if temperature <= 0:
                values, counts, w = values[:1], counts[:1].clamp(max=1), torch.ones(1, dtype=F64, device="cuda")
            else:
                w = ((values - values[0]) / temperature).exp()
            if top_k > 0:
                before = counts.cumsum(0) - counts
                counts = torch.minimum(counts, (top_k - before).clamp(min=0))
            if top_p < 1:
                before = (counts * w).cumsum(0) - counts * w
                target = top_p * (counts * w).sum()
                counts = torch.minimum(counts, torch.ceil((target - before) / w).clamp(min=0))
                counts[0] = counts[0].clamp(min=1)
            fine = w >= min_p
            fine[0] = True
            counts = torch.where(fine, counts, 0.0)
            mass = counts * w
            target = s["u"][r].to(F64) * mass.sum()
            group = int((mass.cumsum(0) <= target).sum())
            nth = int(torch.floor((target - mass[:group].sum()) / w[group]))
            nth = max(0, min(nth, int(counts[group]) - 1))
            tokens.append(int(torch.nonzero(x == values[group])[nth]))
            logprobs.append(float(torch.log(w[group] / mass.sum())))
        return dict(token=torch.tensor(tokens, dtype=I32, device="cuda"),
                    logprob=torch.tensor(logprobs, dtype=F64, device="cuda"))
    out = s["out"].to(F64)
    owners = _adapters(c) if c["adapters"] else [-1]
    edges = s["starts"] if c["adapters"] else [0, s["x"].shape[0]]
    w = s["w"].to(F64).T.contiguous() if c["product"] else None
    for a, first, last in zip(owners, edges, edges[1:]):
        x = s["x"][first:last].to(F64)
        y = s["residual"][first:last].to(F64) if c["residual"] else torch.zeros_like(out[first:last])
        if c["product"]:
            y = torch.addmm(y, x, w)
        if a >= 0:
            delta = s["lora_b"][a].to(F64) @ (s["lora_a"][a].to(F64) @ x.T.contiguous())
            y = y + s["lora_scale"][a].to(F64) * delta.T
        out[first:last] = y
    return out
