"""sample_rows_forward (include/llm_amd/batch.h) against its definition in 64 bits, token by token."""
import math

import numpy as np
import pytest

F32 = 2.0 ** -24  # half a step of fp32, relative to the value


def order_of(x):
    """The tokens that can be taken, largest logit first, equal ones by lowest token."""
    x = np.where(x == 0, 0.0, x)
    tokens = np.flatnonzero(~np.isnan(x) & (x > -np.inf))
    return tokens[np.argsort(-x[tokens], kind="stable")]


def defined(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob, distance of u from the nearest edge between two tokens)"""
    order = order_of(x)
    if len(order) == 0:
        return -1, -np.inf, 1.0
    if not temperature > 0:
        return order[0], 0.0, 1.0
    y = x[order]
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        w = np.where(y == y[0], 1.0, np.exp((y - y[0]) / np.float64(temperature)) if y[0] < np.inf else 0.0)
    keep = np.ones(len(order), bool)
    edges = []
    if top_k > 0:
        keep[top_k:] = False
    if top_p < 1:
        s = np.cumsum(w * keep)
        target = top_p * s[-1]
        edges.append(np.abs(s - target).min() / s[-1])
        keep &= np.concatenate([[True], s[:-1] < target])
    if min_p > 0:
        keep &= np.concatenate([[True], w[1:] >= min_p])
    w = w * keep
    s = np.cumsum(w)
    if math.isnan(u):
        return order[0], math.log(w[0] / s[-1]), 1.0
    edges.append(np.abs(s - u * s[-1]).min() / s[-1])
    past = np.flatnonzero(s > u * s[-1])
    at = past[0] if len(past) else np.flatnonzero(w > 0)[-1]
    return order[at], math.log(w[at] / s[-1]), min(edges)


def run(gpu, logits, c, ws="own", stream=None):
    """c: columns of settings (numpy, or None). (tokens, logprobs)"""
    import torch
    d = {k: None if v is None else torch.from_numpy(np.asarray(v)).cuda() for k, v in c.items()}
    rows, vocab = logits.shape
    out = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    logprob = torch.full((rows,), 7.0, device="cuda")
    if ws == "own":
        ws = torch.full((gpu.sample_rows_workspace_floats(rows, vocab),), math.nan, device="cuda")
    gpu.sample_rows_forward(out, logits, **d, logprob=logprob, ws=ws, stream=stream)
    torch.cuda.synchronize()
    return out.cpu().numpy(), logprob.cpu().numpy().astype(np.float64)


def check(got, logits, c, exact_edges=False):
    tokens, logprobs = got
    x = logits.float().cpu().numpy().astype(np.float64)
    for r in range(len(x)):
        setting = {k: float(v[r]) if k != "top_k" else int(v[r]) for k, v in c.items() if v is not None}
        token, logprob, edge = defined(x[r], **setting)
        # sums of V terms in any order differ by less than V steps of 2^-53; inputs with ties on purpose have
        # sums that are exact in 64 bits
        assert exact_edges or edge > x.shape[1] * 2.0 ** -52 or tokens[r] == token, "an unlucky input: u on an edge"
        assert tokens[r] == token, (r, tokens[r], token, setting)
        if np.isinf(logprob):
            assert logprobs[r] == logprob
        else:  # ln in 64 bits of sums that differ by V 2^-52, then one rounding
            assert abs(logprobs[r] - logprob) <= F32 * abs(logprob) + x.shape[1] * 2.0 ** -50


def make(rng, rows, **on):
    c = dict(u=rng.random(rows).astype(np.float32), temperature=None, top_k=None, top_p=None, min_p=None)
    if on.get("temperature"):
        c["temperature"] = rng.choice([0.0, 0.2, 0.7, 1.0, 1.3, 50.0], rows).astype(np.float32)
    if on.get("top_k"):
        c["top_k"] = rng.choice([-3, 0, 1, 2, 7, 40, 1000, 2 ** 31 - 1], rows).astype(np.int32)
    if on.get("top_p"):
        c["top_p"] = rng.choice([-1.0, 0.0, 0.1, 0.5, 0.9, 0.999, 1.0, 2.0, np.nan], rows).astype(np.float32)
    if on.get("min_p"):
        c["min_p"] = rng.choice([-1.0, 0.0, 1e-4, 0.05, 0.5, 1.0, 3.0, np.nan], rows).astype(np.float32)
    return c


ALL = dict(temperature=True, top_k=True, top_p=True, min_p=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 7), (4, 64), (7, 1003), (2, 8192), (40, 5001), (3, 32003),
                                        (2, 151936), (300, 129), (3, 65537), (70, 20000), (17, 151937)])
@pytest.mark.parametrize("on", [{}, dict(temperature=True), dict(top_k=True), dict(top_p=True), dict(min_p=True), ALL],
                         ids=lambda on: "+".join(on) if len(on) < 4 else "all")
def test_picks_against_the_definition(gpu, rows, vocab, on):
    import torch
    rng = np.random.default_rng(rows * 1000 + vocab + len(on))
    logits = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32) * 3).cuda().bfloat16()
    c = make(rng, rows, **on)
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1000, 20001])
def test_many_random_numbers(gpu, vocab):
    """The same row with random numbers over the whole range, the ends among them: every token that they fall on."""
    import torch
    rng = np.random.default_rng(1)
    row = torch.from_numpy(rng.standard_normal((1, vocab)).astype(np.float32) * 2).cuda().bfloat16()
    logits = row.expand(500, vocab).contiguous()
    c = make(rng, 500)
    c["u"][:4] = 0, 2.0 ** -24, 1 - 2.0 ** -24, 2.0 ** -149
    check(run(gpu, logits, c), logits, c)
    c["u"][:5] = 1.0, 7.0, -1.0, -0.0, np.nan  # outside of what is asked for: the last, the first
    c["top_k"] = rng.integers(1, 30, 500).astype(np.int32)
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [5, 4096, 151936])
@pytest.mark.parametrize("value", [0.0, -1e4, 1e-39, -3.3895e38])
def test_equal_logits(gpu, vocab, value):
    """All of one weight, more of them than 16 bits count: the order is that of the tokens, and every sum is exact."""
    import torch
    rng = np.random.default_rng(2)
    logits = torch.full((40, vocab), value, device="cuda").bfloat16()
    if value == 0.0:
        logits[:, ::3] = -0.0
    c = make(rng, 40, **dict(ALL, min_p=False))
    c["u"] = (rng.integers(0, 64, 40) / 64).astype(np.float32)
    c["top_p"] = (rng.integers(0, 65, 40) / 64).astype(np.float32)
    check(run(gpu, logits, c), logits, c, exact_edges=True)


@pytest.mark.gpu
@pytest.mark.parametrize("first,second", [(1.0, 1.0078125), (1.0078125, 1.015625), (-1.0, -1.0078125), (2.0, -2.0)])
def test_counts_past_16_bits(gpu, first, second):
    """Two values, neighbours among them, each of more tokens than 16 bits count, up to exactly 2^16 and one less."""
    import torch
    rng = np.random.default_rng(3)
    rows = []
    for n, m in [(65535, 65536), (65536, 65535), (65536, 65536), (65537, 131072), (70000, 200001), (131071, 1)]:
        row = np.zeros(300000, np.float32) - np.inf
        where = rng.permutation(300000)
        row[where[:n]], row[where[n:n + m]] = first, second
        rows += [row] * 6
    logits = torch.from_numpy(np.stack(rows)).cuda().bfloat16()
    c = make(rng, len(rows))
    c["top_k"] = rng.integers(60000, 140000, len(rows)).astype(np.int32)
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(130, 140000), (2, 600000), (1, 524225), (3, 524224), (127, 65536), (128, 16384)])
def test_rows_with_and_without_slices(gpu, rows, vocab):
    """Both sides of the sizes from which rows are cut and slices are too many, with counts past 16 bits."""
    import torch
    rng = np.random.default_rng(vocab)
    logits = torch.from_numpy(rng.choice([1.0, 1.0, 2.0, -1.0], (rows, vocab)).astype(np.float32)).cuda().bfloat16()
    logits[0] = 3.0
    c = make(rng, rows)
    c["top_k"] = rng.integers(1, vocab, rows).astype(np.int32)
    check(run(gpu, logits, c), logits, c)
    logits = (torch.randn(rows, vocab, device="cuda") * 3).bfloat16()
    c = make(rng, rows, **ALL)
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
def test_every_value(gpu):
    """Every bf16 value once, in a random order, NaN and infinities among them; then every one that is finite."""
    import torch
    rng = np.random.default_rng(4)
    bits = np.stack([rng.permutation(1 << 16) for _ in range(12)]).astype(np.uint16)
    logits = torch.from_numpy(bits.view(np.int16)).cuda().view(torch.bfloat16)
    c = make(rng, 12, top_k=True)
    check(run(gpu, logits, c), logits, c)
    logits = torch.where(logits.isinf(), torch.full_like(logits, -math.inf), logits)
    for temperature in (1.0, 1e36, 1e38, np.inf):
        c["temperature"] = np.full(12, temperature, np.float32)
        check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
def test_small_values_and_wide_ranges(gpu):
    """Values next to zero that differ by less than any weight shows, and rows over the whole exponent range."""
    import torch
    rng = np.random.default_rng(5)
    tiny = rng.standard_normal((8, 9000)) * 1e-30
    wide = np.exp(rng.uniform(-80, 80, (8, 9000))) * rng.choice([-1, 1], (8, 9000))
    logits = torch.from_numpy(np.concatenate([tiny, wide]).astype(np.float32)).cuda().bfloat16()
    c = make(rng, 16, top_k=True)
    c["temperature"] = np.array([1.0, 1e-30] * 4 + [1.0, 1e30, 1e34, 1e-3] * 2, np.float32)
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [3, 700, 40000])
def test_rows_with_little_to_take(gpu, vocab):
    """Nothing but -inf and NaN: -1; one token; the type's lowest value as a mask; infinities."""
    import torch
    rng = np.random.default_rng(6)
    x = np.full((9, vocab), -np.inf, np.float32)
    x[1] = np.nan
    x[2, ::2] = np.nan
    x[3, vocab // 2] = -5.0
    x[4] = -3.3895e38
    x[5] = -3.3895e38
    x[5, vocab - 1] = 2.0
    x[6] = rng.standard_normal(vocab)
    x[6, ::3] = np.nan
    x[7] = rng.standard_normal(vocab)
    x[7, 1::2] = np.inf
    x[8] = rng.standard_normal(vocab)
    x[8, -1] = np.inf
    logits = torch.from_numpy(x).cuda().bfloat16()
    for on in ({}, ALL, dict(temperature=True)):
        c = make(rng, 9, **on)
        got = run(gpu, logits, c)
        check(got, logits, c)
        assert (got[0][:3] == -1).all()
    c["temperature"][:] = np.inf  # every finite logit weighs the same, but nothing beside +inf
    check(run(gpu, logits, c), logits, c)
    c["temperature"][:] = np.nan
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", range(8))
@pytest.mark.parametrize("vocab", [9, 1000, 30011])
def test_rows_apart_and_unaligned(gpu, shift, vocab):
    """Rows of a wider buffer from any element on; what lies beside them, larger, is not taken."""
    import torch
    rng = np.random.default_rng(shift)
    wide = torch.full((5, vocab + 19), 99.0, device="cuda", dtype=torch.bfloat16)
    logits = wide[:, shift:shift + vocab]
    logits.copy_(torch.from_numpy(rng.standard_normal((5, vocab)).astype(np.float32)))
    c = make(rng, 5, **ALL)
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
def test_the_last_of_many_equal_tokens(gpu):
    """The token is found among equal ones at both ends of the row."""
    import torch
    logits = torch.full((66, 151936), -1.0, device="cuda").bfloat16()
    logits[:, :3] = 5.0
    logits[:, -3:] = 5.0
    logits[:, 75000:75002] = 5.0
    c = dict(u=(np.arange(66) % 8 / 8).astype(np.float32), top_k=np.full(66, 8, np.int32))
    check(run(gpu, logits, c), logits, c, exact_edges=True)


@pytest.mark.gpu
def test_without_logprob_and_workspaces_of_larger_calls(gpu):
    import torch
    rng = np.random.default_rng(7)
    ws = torch.full((gpu.sample_rows_workspace_floats(64, 151936),), math.nan, device="cuda")
    for rows, vocab in [(64, 151936), (1, 151936), (64, 5), (33, 70001), (1, 1), (8, 151936)]:
        assert gpu.sample_rows_workspace_floats(rows, vocab) <= ws.numel()
        logits = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32)).cuda().bfloat16()
        c = make(rng, rows, **ALL)
        got = run(gpu, logits, c, ws=ws)
        check(got, logits, c)
        out = torch.zeros(rows, dtype=torch.int32, device="cuda")
        d = {k: torch.from_numpy(v).cuda() for k, v in c.items()}
        gpu.sample_rows_forward(out, logits, **d, ws=ws)
        assert np.array_equal(out.cpu().numpy(), got[0])


def test_workspace_grows_with_the_sizes(pkg):
    rng = np.random.default_rng(8)
    for _ in range(300):
        rows, vocab = int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 22))
        floats = pkg.sample_rows_workspace_floats(rows, vocab)
        for _ in range(5):
            assert pkg.sample_rows_workspace_floats(rng.integers(0, rows + 1), rng.integers(1, vocab + 1)) <= floats


@pytest.mark.gpu
def test_captured_on_another_stream(gpu):
    """A graph follows logits, settings and random numbers as they change."""
    import torch
    rng = np.random.default_rng(9)
    rows, vocab = 6, 90000
    logits = torch.zeros(rows, vocab, device="cuda", dtype=torch.bfloat16)
    d = {k: torch.from_numpy(v).cuda() for k, v in make(rng, rows, **ALL).items()}
    out, logprob = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
    ws = torch.empty(gpu.sample_rows_workspace_floats(rows, vocab), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        gpu.sample_rows_forward(out, logits, **d, logprob=logprob, ws=ws)
    for _ in range(4):
        c = make(rng, rows, **ALL)
        for k, v in c.items():
            d[k].copy_(torch.from_numpy(v))
        logits.copy_(torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32) * 3))
        graph.replay()
        torch.cuda.synchronize()
        check((out.cpu().numpy(), logprob.cpu().numpy().astype(np.float64)), logits, c)


@pytest.mark.gpu
def test_two_streams_at_once(gpu):
    import torch
    rng = np.random.default_rng(10)
    streams = [torch.cuda.Stream() for _ in range(2)]
    calls = []
    for i in range(8):
        logits = torch.from_numpy(rng.standard_normal((3, 100000)).astype(np.float32) * 3).cuda().bfloat16()
        c = make(rng, 3, **ALL)
        d = {k: torch.from_numpy(v).cuda() for k, v in c.items()}
        out, logprob = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, device="cuda")
        ws = torch.empty(gpu.sample_rows_workspace_floats(3, 100000), device="cuda")
        calls.append((logits, c, d, out, logprob, ws))
    torch.cuda.synchronize()
    for i, (logits, c, d, out, logprob, ws) in enumerate(calls):
        gpu.sample_rows_forward(out, logits, **d, logprob=logprob, ws=ws, stream=streams[i % 2])
    torch.cuda.synchronize()
    for logits, c, d, out, logprob, ws in calls:
        check((out.cpu().numpy(), logprob.cpu().numpy().astype(np.float64)), logits, c)


@pytest.mark.parametrize("at,value,message", [
    (0, None, "must not be null"), (2, None, "must not be null"), (7, None, "must not be null"), (9, -1, "rows -1"),
    (9, (1 << 20) + 1, "rows 1048577"), (10, 0, "vocab 0"), (10, (1 << 22) + 1, "vocab 4194305"), (11, 999, "overlap"),
    (8, 0x1004, "16-byte aligned"), (8, None, "16-byte aligned")])
def test_refusals(pkg, at, value, message):
    p = 0x1000
    args = [p, p, p, p, p, p, p, p, p, 2, 1000, 1000, None]
    args[at] = value
    if at == 8:  # so large that a workspace is needed
        args[9:12] = 1, 151936, 151936
    L = pkg.lib()
    L.llm_clear_error()
    L.sample_rows_forward(*args)
    got = L.llm_last_error()
    L.llm_clear_error()
    assert got and message in got.decode()


def test_no_rows_is_no_error(pkg):
    L = pkg.lib()
    L.llm_clear_error()
    L.sample_rows_forward(None, None, None, None, None, None, None, None, None, 0, 1000, 1000, None)
    assert L.llm_last_error() is None
    for rows, vocab in [(-1, 5), (5, 0), (5, 1 << 23)]:
        with pytest.raises(pkg.LlmError, match="is not in"):
            pkg.sample_rows_workspace_floats(rows, vocab)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_wrapper_refusals(gpu, monkeypatch, native):
    import torch
    if not native:
        monkeypatch.setattr(gpu, "_native", None)
    x = torch.randn(2, 151936, device="cuda").bfloat16()
    i, f = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, device="cuda")
    ws = torch.empty(gpu.sample_rows_workspace_floats(2, 151936), device="cuda")
    for args, message in [
            (dict(out=i.long()), "out must be torch.int32"), (dict(out=i[:1]), "out must be contiguous of shape"),
            (dict(logits=x.float()), "logits must be torch.bfloat16"), (dict(logits=x[0]), "logits must have shape"),
            (dict(logits=x.T), "contiguous rows"), (dict(logits=x.cpu()), "must be a tensor on the GPU"),
            (dict(u=f.double()), "u must be torch.float32"), (dict(u=None), "must not be null"),
            (dict(temperature=f[:1]), "temperature must be"), (dict(top_k=f), "top_k must be torch.int32"),
            (dict(top_p=0.9), "top_p must be a tensor"), (dict(min_p=i), "min_p must be"), (dict(logprob=i), "logprob must be"),
            (dict(ws=None), "ws holds 0 floats"), (dict(ws=ws[1:]), "ws holds"), (dict(ws=ws.double()), "ws must be")]:
        with pytest.raises(gpu.LlmError, match=message):
            gpu.sample_rows_forward(**dict(dict(out=i, logits=x, u=f, ws=ws), **args))
    gpu.sample_rows_forward(i, x, f, ws=ws)  # and no error is left
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [3, 700, 40000, 151936])
def test_random_numbers_of_one_and_more(gpu, vocab):
    """No running sum passes them: the last token of positive weight, also where the first one's weight is the whole sum in
    64 bits, and where those behind weigh nothing."""
    import torch
    rng = np.random.default_rng(11)
    x = np.full((12, vocab), -60.0, np.float32)  # e^-60 is less than half a step of 1
    x[:, vocab // 2] = 0.0
    x[1, :vocab // 3 + 1] = -700.0
    x[2] = rng.choice([-60.0, -2000.0], vocab)  # e^-2000 is 0
    x[2, vocab // 2] = 0.0
    x[3] = -2000.0
    x[3, vocab // 2] = 1.0
    x[4, vocab - 1] = np.inf
    x[5] = rng.standard_normal(vocab)
    x[6:] = x[:6]
    logits = torch.from_numpy(x).cuda().bfloat16()
    for u in (1.0, 7.0, np.inf):
        c = make(rng, 12)
        c["u"] = np.full(12, u, np.float32)
        check(run(gpu, logits, c), logits, c, exact_edges=True)
        c["top_k"] = np.tile([0, 1, 2, 5, 600, 1], 2).astype(np.int32)
        check(run(gpu, logits, c), logits, c, exact_edges=True)
        c["min_p"] = np.repeat([0.0, 1e-30], 6).astype(np.float32)
        check(run(gpu, logits, c), logits, c, exact_edges=True)
        c["top_p"] = np.full(12, 0.75, np.float32)
        c["temperature"] = np.full(12, 1.5, np.float32)
        check(run(gpu, logits, c), logits, c, exact_edges=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,cut", [
    (1, 16384, False), (64, 32003, False), (1, 49151, False), (1, 49152, True), (64, 50257, True), (65, 65536, False),
    (65, 98303, False), (65, 98304, True), (127, 151936, True), (128, 151936, False)])
def test_rows_are_cut_where_that_is_shorter(gpu, rows, vocab, cut):
    """Rows that a workgroup each counts in less time than two launches take are left whole: these do without a workspace."""
    import torch
    rng = np.random.default_rng(rows + vocab)
    logits = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32) * 3).cuda().bfloat16()
    c = make(rng, rows, **ALL)
    ws = torch.full((max(gpu.sample_rows_workspace_floats(rows, vocab), 4),), math.nan, device="cuda")
    check(run(gpu, logits, c, ws=ws), logits, c)
    assert bool(ws.isnan().all()) == (not cut)
