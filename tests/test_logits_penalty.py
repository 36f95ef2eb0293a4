"""logits_penalty_forward (include/llm_amd/paged.h) against its definition in 64 bits, token by token."""
import math

import numpy as np
import pytest

HALF_STEP = 2.0 ** -8   # of bf16, relative to the value
F32 = 2.0 ** -24        # half a step of fp32


def defined(logits, c):
    """(value, bound on the fp32 error: one rounding per operation, of values no larger than the sum of
    the operands' sizes)."""
    rows, vocab = logits.shape
    out = logits.astype(np.float64)
    size = np.abs(out)
    for r in range(rows):
        n = 0 if c["tokens"] is None else max(0, min(c["tokens"].shape[1], int(c["token_len"][r])))
        ids = [] if n == 0 else c["tokens"][r, :n].tolist()
        prompt = 0 if c["prompt_len"] is None else int(c["prompt_len"][r])
        f, p = (0.0 if c[k] is None else float(c[k][r]) for k in ("frequency", "presence"))
        answers = {}
        for i, t in enumerate(ids):
            if i >= prompt:
                answers[t] = answers.get(t, 0) + 1
        for t in set(ids):
            if 0 <= t < vocab and c["repetition"] is not None:
                x, rep = out[r, t], float(c["repetition"][r])
                out[r, t] = x / rep if x > 0 else x * rep
                size[r, t] = abs(out[r, t])
        for t, k in answers.items():
            if 0 <= t < vocab:
                out[r, t] -= f * k + p
                size[r, t] += abs(f * k) + abs(p)
        if c["bias_tokens"] is not None:
            m = c["bias_tokens"].shape[1] if c["bias_len"] is None else max(0, min(c["bias_tokens"].shape[1], int(c["bias_len"][r])))
            last = {int(t): float(v) for t, v in zip(c["bias_tokens"][r, :m], c["bias"][r, :m])}
            for t, v in last.items():
                if 0 <= t < vocab:
                    out[r, t] += v
                    size[r, t] += abs(v)
        if c["allowed"] is not None:
            words = c["allowed"][r].astype(np.int64) & 0xffffffff
            t = np.arange(vocab)
            out[r, (words[t // 32] >> (t % 32)) & 1 == 0] = -np.inf
    return out, 8 * F32 * size


def make(rng, rows, vocab, history, biases, mask, odd=False):
    c = dict.fromkeys(["tokens", "prompt_len", "token_len", "repetition", "frequency", "presence", "bias_tokens",
                       "bias", "bias_len", "allowed"])
    if history:
        few = rng.integers(0, vocab, max(1, history // 3))  # most tokens more than once
        c["tokens"] = rng.choice(few, (rows, history)).astype(np.int32)
        c["token_len"] = rng.integers(0, history + 1, rows).astype(np.int32)
        c["token_len"][0] = history
        c["prompt_len"] = (c["token_len"] * rng.random(rows)).astype(np.int32)
        c["repetition"] = rng.uniform(0.8, 1.6, rows).astype(np.float32)
        c["frequency"], c["presence"] = (rng.uniform(-0.3, 0.8, rows).astype(np.float32) for _ in range(2))
        if odd:  # ids that are no tokens, lengths past the row and below nothing
            c["tokens"][:, ::5] = rng.choice([-1, vocab, 2 ** 31 - 1, -2 ** 31], c["tokens"][:, ::5].shape)
            c["token_len"][-1], c["prompt_len"][-1] = history + 9, -4
            if rows > 2:
                c["token_len"][1], c["prompt_len"][2] = -3, history + 50
    if biases:
        c["bias_tokens"] = rng.integers(0, vocab, (rows, biases)).astype(np.int32)
        c["bias_tokens"][:, -1] = c["bias_tokens"][:, 0]  # the same token twice: the last counts
        c["bias"] = rng.uniform(-9, 9, (rows, biases)).astype(np.float32)
        if odd:
            c["bias_len"] = rng.integers(-1, biases + 3, rows).astype(np.int32)
            c["bias_tokens"][:, biases // 2] = vocab + 3
    if mask:
        c["allowed"] = rng.integers(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32))).astype(np.int32)
        c["allowed"][0, :] = 0  # a row whose mask leaves nothing
    return c


def run(gpu, logits, c, out=None, stream=None):
    import torch
    d = {k: None if v is None else torch.from_numpy(v).cuda() for k, v in c.items()}
    out = torch.zeros_like(logits) if out is None else out
    gpu.logits_penalty_forward(out, logits, **d, stream=stream)
    torch.cuda.synchronize()
    return out


def check(out, logits, c):
    import torch
    got = out.float().cpu().numpy().astype(np.float64)
    want, err = defined(logits.float().cpu().numpy(), c)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    got, want, err = got[fine], want[fine], err[fine]
    off = np.abs(got - want) - (HALF_STEP * (np.abs(want) + err) + err)
    assert (off <= 0).all(), f"{(off > 0).sum()} of {off.size} off by up to {off.max():.3g} more than allowed"


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 7), (3, 31), (2, 1000), (5, 1003), (1, 4096), (2, 4097), (3, 8191),
                                        (1, 151936), (7, 32003), (70, 2049)])
@pytest.mark.parametrize("history,biases,mask,odd", [(0, 0, False, False), (1, 1, True, False), (300, 0, False, True),
                                                     (0, 40, True, True), (700, 33, True, True)])
def test_penalties_against_the_definition(gpu, rows, vocab, history, biases, mask, odd):
    import torch
    rng = np.random.default_rng(rows * 1000 + vocab)
    logits = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32) * 4).cuda().bfloat16()
    c = make(rng, rows, vocab, history, biases, mask, odd)
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 200])
def test_biases_of_tokens_with_one_place(gpu, rows):
    """Tokens whose biases begin their search at the same places, each several times, the first tokens of a
    slice and the last among them."""
    import torch
    rng = np.random.default_rng(3)
    logits = torch.randn(rows, 20000, device="cuda").bfloat16()
    c = make(rng, rows, 20000, 50, 512, True)
    near = np.concatenate([np.arange(0, 20000, 1024), np.arange(1023, 20000, 1024), np.arange(1022, 20000, 2048), [8191, 8192]])
    c["bias_tokens"] = rng.choice(near, (rows, 512)).astype(np.int32)
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
def test_a_long_history_of_few_tokens(gpu):
    import torch
    rng = np.random.default_rng(1)
    logits = torch.randn(2, 5000, device="cuda").bfloat16()
    c = make(rng, 2, 5000, 40000, 0, False)
    c["tokens"] = rng.choice([3, 4999, 17], (2, 40000)).astype(np.int32)
    c["frequency"] = np.full(2, 1e-3, np.float32)
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
@pytest.mark.parametrize("history,biases", [(100, 512), (100, 513), (33000, 512), (40000, 2000), (32767, 1), (32768, 1)])
@pytest.mark.parametrize("vocab", [40, 5000, 70001])
def test_many_biases_and_long_histories(gpu, history, biases, vocab):
    """Both sides of the sizes from which counts and biases take more room; every bias in one place; one token
    counted 32767 times and more."""
    import torch
    rng = np.random.default_rng(7)
    logits = torch.randn(3, vocab, device="cuda").bfloat16()
    c = make(rng, 3, vocab, history, biases, True, True)
    c["bias_tokens"][1] = rng.integers(0, 30, biases)
    c["tokens"][2], c["token_len"][2], c["prompt_len"][2], c["frequency"][2] = 7, history, 0, 1e-3
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,history,biases,slices", [(64, 65544, 700, 600, 9), (64, 70001, 300, 513, 9),
                                                              (32, 65544, 32768, 600, 17), (64, 65544, 32800, 40, 9)])
def test_penalties_of_many_rows(gpu, rows, vocab, history, biases, slices):
    """So many rows that the slices are the largest: 8192 tokens, 4096 where counts of 32 bits and a word per
    token for the biases share the memory."""
    import torch
    assert rows * slices >= 512 and -(-vocab // (4096 if slices == 17 else 8192)) == slices
    rng = np.random.default_rng(history + biases)
    logits = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32) * 4).cuda().bfloat16()
    c = make(rng, rows, vocab, history, biases, True, True)
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
@pytest.mark.parametrize("off", ["repetition", "frequency", "presence", "prompt_len"])
def test_each_part_can_be_off(gpu, off):
    import torch
    rng = np.random.default_rng(2)
    logits = torch.randn(3, 777, device="cuda").bfloat16()
    c = make(rng, 3, 777, 200, 5, True)
    c[off] = None
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1, 5])
@pytest.mark.parametrize("vocab", [1000, 1001, 20000])
def test_rows_apart_unaligned_and_in_place(gpu, shift, vocab):
    """Rows of a wider buffer from any element on; what lies between the rows stays; out may be logits."""
    import torch
    rng = np.random.default_rng(4)
    c = make(rng, 4, vocab, 100, 9, True, True)
    for in_place in (False, True):
        wide = torch.randn(4, vocab + 13, device="cuda").bfloat16()
        before = wide.clone()
        logits = wide[:, shift:shift + vocab]
        target = torch.full((4, vocab + 21), 7.0, device="cuda", dtype=torch.bfloat16)
        out = logits if in_place else target[:, 2 * shift:2 * shift + vocab]
        run(gpu, logits, c, out)
        check(out, before[:, shift:shift + vocab], c)
        rest = wide if in_place else target
        keep = before if in_place else torch.full_like(target, 7.0)
        first = shift if in_place else 2 * shift
        assert torch.equal(rest[:, :first], keep[:, :first]) and torch.equal(rest[:, first + vocab:], keep[:, first + vocab:])


@pytest.mark.gpu
def test_infinities_and_nan(gpu):
    """Infinite and NaN logits go through the arithmetic; a masked token is -inf whatever it was."""
    import torch
    rng = np.random.default_rng(5)
    x = rng.standard_normal((2, 3000)).astype(np.float32)
    x[:, ::7], x[:, 1::11], x[:, 2::13], x[:, 3::17] = np.inf, -np.inf, np.nan, -0.0
    logits = torch.from_numpy(x).cuda().bfloat16()
    c = make(rng, 2, 3000, 2000, 50, True)
    c["bias"][:, 3], c["bias"][:, 4] = -np.inf, np.inf
    check(run(gpu, logits, c), logits, c)


@pytest.mark.gpu
def test_captured_with_a_growing_history(gpu):
    import torch
    rng = np.random.default_rng(6)
    logits = torch.randn(2, 9000, device="cuda").bfloat16()
    c = make(rng, 2, 9000, 64, 4, True)
    d = {k: None if v is None else torch.from_numpy(v).cuda() for k, v in c.items()}
    out = torch.zeros_like(logits)
    gpu.logits_penalty_forward(out, logits, **d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.logits_penalty_forward(out, logits, **d)
    for n in (0, 1, 30, 64):
        d["token_len"].fill_(n)
        c["token_len"] = np.full(2, n, np.int32)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check(out, logits, c)


@pytest.mark.gpu
def test_then_a_pick(gpu):
    """The picks that a sampler makes of the row: banned tokens are never drawn or taken."""
    import torch
    logits = torch.zeros(1, 50000, device="cuda").bfloat16()
    logits[0, 123] = 9.0
    allowed = torch.zeros(1, 1563, dtype=torch.int32, device="cuda")
    allowed[0, 1000 // 32] = 1 << (1000 % 32)
    allowed[0, 123 // 32] |= -2 ** 31 if 123 % 32 == 31 else 1 << (123 % 32)
    bias_tokens = torch.tensor([[123]], dtype=torch.int32, device="cuda")
    bias = torch.tensor([[-math.inf]], device="cuda")
    out, token = torch.empty_like(logits), torch.zeros(1, dtype=torch.int32, device="cuda")
    gpu.logits_penalty_forward(out, logits, bias_tokens=bias_tokens, bias=bias, allowed=allowed)
    gpu.argmax_forward(token, out[0], 50000)
    assert int(token) == 1000
    gpu.sample_forward(token, out[0], 50000, 1.0, 0.999)
    assert int(token) == 1000


@pytest.mark.parametrize("at,value,message", [
    (0, None, "must not be null"), (1, None, "must not be null"), (12, -1, "rows -1"), (12, 70000, "rows 70000"),
    (13, 0, "vocab 0"), (13, 1 << 29, "vocab"), (4, None, "token_len"), (14, -1, "token_stride"), (9, None, "biases need"),
    (15, -2, "bias_stride"), (16, 31, "allowed_stride 31"), (17, 999, "overlap"), (18, 5, "overlap")])
def test_refusals(pkg, at, value, message):
    p = 0x1000
    args = [p, p, p, p, p, p, p, p, p, p, p, p, 2, 1000, 8, 8, 32, 1000, 1000, None]
    args[at] = value
    L = pkg.lib()
    L.llm_clear_error()
    L.logits_penalty_forward(*args)
    got = L.llm_last_error()
    L.llm_clear_error()
    assert got and message in got.decode()


def test_in_place_needs_one_stride(pkg):
    p, L = 0x1000, pkg.lib()
    L.llm_clear_error()
    L.logits_penalty_forward(p, p, *[None] * 10, 2, 1000, 0, 0, 0, 1000, 1008, None)
    assert "in place" in L.llm_last_error().decode()
    L.llm_clear_error()
    L.logits_penalty_forward(p, p, *[None] * 10, 0, 1000, 0, 0, 0, 1000, 1000, None)  # no rows: nothing to do
    assert L.llm_last_error() is None


def test_too_many_biases_are_refused(pkg):
    p, L = 0x1000, pkg.lib()
    L.llm_clear_error()
    L.logits_penalty_forward(p, p, p, p, p, p, p, p, p, p, p, p, 2, 1000, 8, (1 << 22) + 1, 32, 1000, 1000, None)
    got = L.llm_last_error()
    L.llm_clear_error()
    assert got and "bias_stride 4194305" in got.decode()


@pytest.mark.gpu
def test_wrapper_refusals(gpu):
    import torch
    x = torch.randn(2, 100, device="cuda").bfloat16()
    i = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    f = torch.zeros(2, device="cuda")
    for args, message in [
            (dict(out=x.float()), "out must be torch.bfloat16"), (dict(out=x[:1]), "out must have shape"),
            (dict(logits=x.cpu()), "logits must be a tensor on the GPU"), (dict(tokens=i.long(), token_len=n), "tokens must be torch.int32"),
            (dict(tokens=i[:1], token_len=n), "tokens must be contiguous of shape"), (dict(tokens=i), "token_len"),
            (dict(repetition=f.half()), "repetition must be torch.float32"), (dict(bias_tokens=i), "biases need"),
            (dict(bias_tokens=i, bias=f), "bias must be"), (dict(allowed=i[:, :3].contiguous()), "allowed_stride 3"),
            (dict(allowed=i.float()), "allowed must be")]:
        with pytest.raises(gpu.LlmError, match=message):
            gpu.logits_penalty_forward(**dict(dict(out=torch.empty_like(x), logits=x), **args))
