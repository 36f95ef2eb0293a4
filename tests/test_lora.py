"""lora_projection_forward (include/llm_amd/batch.h) against its definition in 64 bits."""
import math

import numpy as np
import pytest

HALF_STEP = 2.0 ** -8   # of bf16, relative to the value
F32 = 2.0 ** -24        # half a step of fp32


def _normal(g, *shape, std=1.0):
    import torch
    return (torch.randn(*shape, generator=g, device="cuda") * std).bfloat16()


def make(seed, lengths, n_in, n_out, rank=16, adapters=3, which=None, spare=0, product=True, residual=False, scale=True):
    """Sequences of these lengths; `which` adapter each one has (a random one, -1 among them)."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    rows = sum(lengths) + spare
    c = dict(x=_normal(g, rows, n_in), w=None, lora_a=None, lora_b=None, lora_scale=None, q_start=None, adapter=None,
             residual=None)
    if product:
        c["w"] = _normal(g, n_out, n_in, std=n_in ** -0.5)
    if residual:
        c["residual"] = _normal(g, rows, n_out)
    if adapters:
        if which is None:
            which = rng.integers(-1, adapters, len(lengths))
        c["lora_a"] = _normal(g, adapters, rank, n_in, std=n_in ** -0.5)
        c["lora_b"] = _normal(g, adapters, n_out, rank, std=rank ** -0.5)
        if scale:
            c["lora_scale"] = torch.rand(adapters, generator=g, device="cuda") * 2 - 0.5
        c["q_start"] = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda")
        c["adapter"] = torch.tensor(np.asarray(which), dtype=torch.int32, device="cuda")
    return c


def defined(c, rows, n_out):
    """(value, bound on the error in 32 bits, rows that are written). A sum of K terms has K roundings, each of
    at most half a step of a partial sum, without a common sign: 4 sqrt(K) half steps of the sum of sizes."""
    import torch
    x = c["x"].double()
    out = torch.zeros(rows, n_out, dtype=torch.float64, device="cuda")
    err = torch.zeros_like(out)
    if c["w"] is not None:
        w = c["w"].double().T.contiguous()
        out += x @ w
        err += 4 * math.sqrt(w.shape[0]) * F32 * (x.abs() @ w.abs())
    written = torch.ones(rows, dtype=torch.bool, device="cuda")
    if c["lora_a"] is not None:
        written[:] = False
        starts = c["q_start"].clamp(0, rows).tolist()
        for s, a in enumerate(c["adapter"].tolist()):
            own = slice(starts[s], max(starts[s], starts[s + 1]))
            written[own] = True
            if not 0 <= a < c["lora_a"].shape[0] or own.stop == own.start:
                continue
            at, bt = (c[k][a].double().T.contiguous() for k in ("lora_a", "lora_b"))
            f = 1.0 if c["lora_scale"] is None else float(c["lora_scale"][a])
            low, size = f * (x[own] @ at), abs(f) * (x[own].abs() @ at.abs())
            out[own] += low @ bt
            # what the sum of low is off by, a rounding by the scale, its 16 bits, and the sum over the rank
            off = 4 * math.sqrt(at.shape[0]) * F32 * size + F32 * low.abs() + 2.0 ** -17 * low.abs()
            err[own] += off @ bt.abs() + 4 * math.sqrt(2 * bt.shape[0]) * F32 * (low.abs() @ bt.abs())
    if c["residual"] is not None:
        out += c["residual"].double()
    return out, err + 2 * F32 * out.abs(), written


def run(gpu, c, out=None, ws="own", stream=None):
    import torch
    rows = c["x"].shape[0]
    rank = 0 if c["lora_a"] is None else c["lora_a"].shape[1]
    if ws == "own":
        floats = gpu.lora_projection_workspace_floats(rows, out.shape[1], c["x"].shape[1], rank)
        ws = torch.full((floats,), math.nan, device="cuda")
    torch.cuda.synchronize()
    gpu.lora_projection_forward(out, **c, ws=ws, stream=stream)
    torch.cuda.synchronize()
    return out


def check(out, c, before=7.0):
    import torch
    want, err, written = defined(c, *out.shape)
    got = out.double()
    assert (got[~written] == before).all(), "a row of no sequence was written"
    got, want, err = got[written], want[written], err[written]
    assert torch.equal(got.isnan(), want.isnan())
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    off = (got - want).abs()[fine] - (HALF_STEP * (want.abs() + err) + err)[fine]
    assert (off <= 0).all(), f"{int((off > 0).sum())} of {off.numel()} off by up to {float(off.max()):.3g} more than allowed"


def both(gpu, c, n_out, **kw):
    import torch
    out = torch.full((c["x"].shape[0], n_out), 7.0, device="cuda", dtype=torch.bfloat16)
    check(run(gpu, c, out, **kw), c)
    return out


SHAPES = [(8, 1), (8, 16), (64, 64), (72, 65), (1024, 2048), (2560, 1000), (1000, 257), (4096, 192), (520, 7), (2504, 3000)]


@pytest.mark.gpu
@pytest.mark.parametrize("n_in,n_out", SHAPES)
@pytest.mark.parametrize("lengths", [[1], [1] * 5, [1] * 64, [3, 0, 17, 1], [65], [130, 1, 1, 0, 77], [1] * 129 + [40],
                                     [600, 1, 2, 3, 500, 1, 1], [2100]], ids=lambda l: f"{len(l)}s{sum(l)}")
def test_projection_against_the_definition(gpu, n_in, n_out, lengths):
    rank = [8, 16, 24, 64][(n_in + len(lengths)) // 8 % 4]
    both(gpu, make(n_in + n_out, lengths, n_in, n_out, rank, spare=sum(lengths) % 3, residual=n_out % 2 == 0), n_out)


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 96, 128, 200, 256])
@pytest.mark.parametrize("lengths", [[1, 1, 1], [40, 1, 0, 9], [1] * 200, [700, 333, 1, 1, 600]],
                         ids=lambda l: f"{len(l)}s{sum(l)}")
def test_every_rank(gpu, rank, lengths):
    both(gpu, make(rank, lengths, 136, 320, rank, adapters=7), 320)
    both(gpu, make(rank, lengths, 136, 320, rank, adapters=7, product=False, residual=True), 320)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[1], [1] * 20, [33, 1, 700], [2048, 5]], ids=lambda l: f"{len(l)}s{sum(l)}")
@pytest.mark.parametrize("product,residual,scale,adapters", [
    (True, False, True, 0), (True, True, True, 0), (False, False, True, 4), (False, True, False, 4), (True, False, False, 4),
    (False, True, True, 0), (False, False, True, 0)])
def test_each_part_can_be_off(gpu, lengths, product, residual, scale, adapters):
    for n_out in (256, 333):
        both(gpu, make(1, lengths, 264, n_out, 16, adapters, product=product, residual=residual, scale=scale), n_out)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[1] * 70, [200, 1, 1, 900, 3]], ids=lambda l: f"{len(l)}s{sum(l)}")
def test_which_adapter(gpu, lengths):
    """None for all, the same for all, outside of the adapters, and one for every sequence."""
    for which in (-1, 0, 2, 3, 2 ** 31 - 1, -2 ** 31):
        both(gpu, make(2, lengths, 128, 192, which=[which] * len(lengths)), 192)
    both(gpu, make(3, lengths, 128, 192, 8, adapters=len(lengths), which=np.random.default_rng(0).permutation(len(lengths))), 192)


@pytest.mark.gpu
@pytest.mark.parametrize("starts", [[0, 0, 0, 0], [5, 9, 9, 30], [-4, 3, 50, 99], [60, 70, 80, 90], [0, 20, 40, 40]])
@pytest.mark.parametrize("repeat", [1, 40])
def test_rows_of_no_sequence_stay(gpu, starts, repeat):
    """Rows before the first sequence and behind the last, starts outside of the rows, sequences of no row."""
    import torch
    c = make(4, [41 * repeat], 64, 128)
    c["q_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda") * repeat
    c["adapter"] = torch.tensor([1, -1, 2], dtype=torch.int32, device="cuda")
    both(gpu, c, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[1] * 9, [70, 3], [900, 400]], ids=lambda l: f"{len(l)}s{sum(l)}")
@pytest.mark.parametrize("n_out,shift", [(128, 0), (128, 3), (136, 8), (101, 1)])
def test_slices_of_wider_rows_and_in_place(gpu, lengths, n_out, shift):
    """x, out and residual as slices of wider rows; what lies beside out stays; residual may be out."""
    import torch
    c = make(5, lengths, 128, n_out, residual=True, spare=2)
    rows = c["x"].shape[0]
    x = torch.full((rows, 128 + 24), math.nan, device="cuda", dtype=torch.bfloat16)
    x[:, 16:144] = c["x"]
    c["x"] = x[:, 16:144]
    wide = torch.full((rows, n_out + 19), 7.0, device="cuda", dtype=torch.bfloat16)
    out = wide[:, shift:shift + n_out]
    apart = torch.full((rows, n_out + 5), math.nan, device="cuda", dtype=torch.bfloat16)
    apart[:, 2:2 + n_out] = c["residual"]
    c["residual"] = apart[:, 2:2 + n_out]
    check(run(gpu, c, out), c)
    assert (wide[:, :shift] == 7).all() and (wide[:, shift + n_out:] == 7).all()
    expected = out.clone()
    out.copy_(c["residual"])
    expected[-2:] = out[-2:]
    run(gpu, dict(c, residual=out), out)
    assert torch.equal(out, expected)
    assert (wide[:, :shift] == 7).all() and (wide[:, shift + n_out:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[1] * 40, [1, 300, 1, 250, 4], [700, 1, 1, 1, 700]], ids=lambda l: f"{len(l)}s{sum(l)}")
@pytest.mark.parametrize("where", ["x", "lora_a", "lora_b", "lora_scale", "residual"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_no_number_reaches_other_rows(gpu, lengths, where, bad):
    """NaN and infinities of one row, or of one adapter, stay with the rows that have them; those of adapters that
    no sequence has, and of rows of no sequence, reach none."""
    import torch
    which = [i % 3 for i in range(len(lengths))]
    n_in, n_out = 200, 272
    c = make(6, lengths, n_in, n_out, 16, adapters=5, which=which, residual=True, spare=3)
    if where == "x":
        c["x"][sum(lengths) // 2, 77] = bad
        c["x"][-1] = bad
    elif where == "residual":
        c["residual"][sum(lengths) // 2, 77] = bad
        c["residual"][-1] = bad
    elif where == "lora_a":
        c["lora_a"][1, 5, 199] = bad
        c["lora_a"][4] = bad
    elif where == "lora_b":
        c["lora_b"][1, 133, 5] = bad
        c["lora_b"][1, 271] = bad
        c["lora_b"][4] = bad
    else:
        c["lora_scale"][1] = bad
        c["lora_scale"][4] = bad
    out = torch.full((c["x"].shape[0], n_out), 7.0, device="cuda", dtype=torch.bfloat16)
    run(gpu, c, out)
    clean = dict(c)
    for k in ("x", "residual", "lora_a", "lora_b", "lora_scale"):
        clean[k] = torch.nan_to_num(c[k], 0.0, 0.0, 0.0)
    touched = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    starts = c["q_start"].tolist()
    for s, a in enumerate(which):
        if a == 1 and where.startswith("lora"):
            if where == "lora_b":
                touched[starts[s]:starts[s + 1], [133, 271]] = True
            else:
                touched[starts[s]:starts[s + 1]] = True
    if where == "x":
        touched[sum(lengths) // 2] = True
    if where == "residual":
        touched[sum(lengths) // 2, 77] = True
    assert not out[touched].isfinite().any()
    if where == "lora_b" and not math.isnan(bad):  # an infinity times a number that is not zero
        s = which.index(1)
        low = c["x"][starts[s]].double() @ c["lora_a"][1].double().T * float(c["lora_scale"][1])
        assert float(out[starts[s], 133]) == bad * float(torch.sign(low[5]))
    want, err, written = defined(clean, *out.shape)
    fine = written[:, None] & ~touched
    off = (out.double() - want).abs() - (HALF_STEP * (want.abs() + err) + err)
    assert (off[fine] <= 0).all()
    assert (out[~written] == 7).all()


@pytest.mark.gpu
def test_large_values(gpu):
    """What overflows becomes an infinity of its sign, and what lies just below the range of 32 bits does not."""
    import torch
    for lengths in ([3], [700, 2]):
        c = make(7, lengths, 64, 128, 8, adapters=1, which=[0] * len(lengths), product=False, scale=False)
        c["x"].fill_(2.0 ** 60)
        c["lora_a"].fill_(2.0 ** 60)
        c["lora_b"].fill_(2.0 ** -100)
        out = torch.zeros(sum(lengths), 128, device="cuda", dtype=torch.bfloat16)
        run(gpu, c, out)
        assert (out == 2.0 ** (126 - 100 + 3)).all()
        c["lora_b"].fill_(-1.0)
        run(gpu, c, out)  # 8 x 2^126
        assert (out == -math.inf).all()
        c["x"].fill_(2.0 ** 120)
        run(gpu, c, out)  # the low product is infinite already
        assert (out == -math.inf).all()


@pytest.mark.gpu
def test_a_workspace_for_the_largest_call(gpu):
    import torch
    ws = torch.full((gpu.lora_projection_workspace_floats(2500, 640, 512, 64),), math.nan, device="cuda")
    for lengths, rank in [([2500], 64), ([1], 8), ([64], 64), ([1] * 300, 16), ([1300], 64), ([500, 1], 32), ([17], 64)]:
        assert gpu.lora_projection_workspace_floats(sum(lengths), 640, 512, rank) <= ws.numel()
        both(gpu, make(8, lengths, 512, 640, rank), 640, ws=ws)


def test_workspace_grows_with_the_sizes(pkg):
    rng = np.random.default_rng(8)
    for _ in range(300):
        n, n_out, n_in = (int(2 ** rng.uniform(0, k)) for k in (13, 18, 12))
        rank = 8 * int(rng.integers(0, 33))
        floats = pkg.lora_projection_workspace_floats(n, n_out, 8 * n_in, rank)
        for _ in range(8):
            fewer, lower = int(rng.integers(0, n + 1)), 8 * int(rng.integers(0, rank // 8 + 1))
            assert pkg.lora_projection_workspace_floats(fewer, n_out, 8 * n_in, lower) <= floats


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [6, 300, 1100])
def test_captured_with_lengths_and_adapters_that_change(gpu, rows):
    import torch
    rng = np.random.default_rng(9)
    c = make(9, [rows] + [0] * 5, 256, 384, 16, adapters=4, residual=True)
    out = torch.full((rows, 384), 7.0, device="cuda", dtype=torch.bfloat16)
    ws = torch.empty(gpu.lora_projection_workspace_floats(rows, 384, 256, 16), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        gpu.lora_projection_forward(out, **c, ws=ws)
    for _ in range(4):
        starts = np.concatenate([[0], np.sort(rng.integers(0, rows + 1, 6))])
        c["q_start"].copy_(torch.from_numpy(starts.astype(np.int32)))
        c["adapter"].copy_(torch.from_numpy(rng.integers(-1, 4, 6).astype(np.int32)))
        c["x"].copy_(torch.randn(c["x"].shape, device="cuda"))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        check(out, c)
        first = out.clone()
        run(gpu, c, out.fill_(7.0), ws=ws)
        assert torch.equal(out, first)


@pytest.mark.gpu
def test_two_streams_at_once_give_the_same_as_one(gpu):
    import torch
    streams = [torch.cuda.Stream() for _ in range(2)]
    cases = [make(i, lengths, 512, 320, 16) for i, lengths in enumerate([[1] * 8, [900], [1] * 100, [300, 1, 1], [64], [1] * 8])]
    def fresh(c):
        rows = c["x"].shape[0]
        return (torch.full((rows, 320), 7.0, device="cuda", dtype=torch.bfloat16),
                torch.empty(gpu.lora_projection_workspace_floats(rows, 320, 512, 16), device="cuda"))
    alone = []
    for c in cases:
        out, ws = fresh(c)
        alone.append(run(gpu, c, out, ws=ws))
        check(out, c)
    buffers = [fresh(c) for c in cases]
    torch.cuda.synchronize()
    for i, (c, (out, ws)) in enumerate(zip(cases, buffers)):
        gpu.lora_projection_forward(out, **c, ws=ws, stream=streams[i % 2])
    torch.cuda.synchronize()
    for (out, _), want in zip(buffers, alone):
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_weights_past_32_bit_offsets(gpu):
    """More than 2^31 elements of w, of lora_b and between the first rows of out and its last."""
    import torch
    n_out, n_in = (1 << 22) - 24, 520
    w = torch.zeros(n_out, n_in, device="cuda", dtype=torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(0)
    w[-300:] = _normal(g, 300, n_in)
    b = torch.zeros(40, n_out, 16, device="cuda", dtype=torch.bfloat16)
    b[-1, -300:] = _normal(g, 300, 16)
    a = _normal(g, 40, 16, n_in, std=n_in ** -0.5)
    for rows in (3, 600):
        c = dict(x=_normal(g, rows, n_in), w=w, lora_a=a, lora_b=b, lora_scale=None, residual=None,
                 q_start=torch.tensor([0, rows], dtype=torch.int32, device="cuda"),
                 adapter=torch.tensor([39], dtype=torch.int32, device="cuda"))
        out = torch.empty(rows, n_out, device="cuda", dtype=torch.bfloat16)
        run(gpu, c, out)
        part = dict(c, w=w[-300:].contiguous(), lora_b=b[:, -300:].contiguous())
        check(out[:, -300:].contiguous(), part)
        assert not out[:, :-300].any()


@pytest.mark.gpu
@pytest.mark.parametrize("n_seqs", [1, 5])
def test_a_serving_step(gpu, n_seqs):
    """The operators of a step as they are used together: projections with adapters, norms and rotation into pages,
    attention over them, the output projection onto the residual stream, the head, penalties and the pick; the
    logits against the same in 64 bits, where only the roundings between operators are repeated."""
    import torch
    rng = np.random.default_rng(n_seqs)
    hidden, heads, kv_heads, dim, vocab, page, rank = 256, 4, 2, 64, 1003, 16, 8
    lengths = [1] * (n_seqs - 1) + [37]
    tokens, width = sum(lengths), (heads + 2 * kv_heads) * dim
    qkv = make(n_seqs, lengths, hidden, width, rank)
    c_out = make(n_seqs + 50, lengths, heads * dim, hidden, rank, residual=True)
    c_out.update(q_start=qkv["q_start"], residual=qkv["x"])
    head = make(n_seqs + 99, lengths, hidden, vocab, adapters=0)
    out = torch.zeros(tokens, width, device="cuda", dtype=torch.bfloat16)
    floats = max(gpu.lora_projection_workspace_floats(tokens, n, k, r)
                 for n, k, r in ((width, hidden, rank), (hidden, heads * dim, rank), (vocab, hidden, 0)))
    ws = torch.empty(max(floats, 1), device="cuda")
    gpu.lora_projection_forward(out, **qkv, ws=ws)
    check(out, qkv)
    rows = out.view(tokens, heads + 2 * kv_heads, dim)
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]
    pages = [-(-n // page) for n in lengths]
    table = torch.full((n_seqs, max(pages)), -1, dtype=torch.int32, device="cuda")
    for i, n in enumerate(pages):
        table[i, :n] = torch.arange(sum(pages[:i]), sum(pages[:i + 1]))
    kv_len = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    caches = [torch.zeros(sum(pages), page, kv_heads, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    norm = torch.ones(dim, device="cuda", dtype=torch.bfloat16)
    inv_freq, factor = gpu.rope_frequencies(dim, 1e4)
    turned = torch.zeros(tokens, heads, dim, device="cuda", dtype=torch.bfloat16)
    gpu.qk_norm_rope_paged(turned, q, k, v, norm, norm, inv_freq.cuda(), *caches, table, qkv["q_start"], kv_len, 1e-6, factor)
    floats = gpu.attention_paged_workspace_floats(tokens, n_seqs, heads, kv_heads, dim, 37, 37)
    attended = torch.zeros_like(turned)
    gpu.attention_paged_forward(attended, turned, *caches, table, qkv["q_start"], kv_len,
                                torch.empty(max(floats, 1), device="cuda"), dim ** -0.5, 37, 37)
    c_out["x"] = attended.view(tokens, heads * dim)
    stream = torch.full((tokens, hidden), 7.0, device="cuda", dtype=torch.bfloat16)
    gpu.lora_projection_forward(stream, **c_out, ws=ws)
    check(stream, c_out)
    last = (torch.cumsum(kv_len, 0) - 1).long()
    head["x"] = stream[last]
    logits = torch.zeros(n_seqs, vocab, device="cuda", dtype=torch.bfloat16)
    gpu.lora_projection_forward(logits, **head, ws=ws)
    check(logits, head)
    history = torch.from_numpy(rng.integers(0, vocab, (n_seqs, 30)).astype(np.int32)).cuda()
    full = torch.full((n_seqs,), 30, dtype=torch.int32, device="cuda")
    half = torch.full((n_seqs,), 0.5, device="cuda")
    gpu.logits_penalty_forward(logits, logits, history, None, full, half * 2.5, half, half)
    token, logprob = torch.zeros(n_seqs, dtype=torch.int32, device="cuda"), torch.zeros(n_seqs, device="cuda")
    u = torch.from_numpy(rng.random(n_seqs).astype(np.float32)).cuda()
    k20 = torch.full((n_seqs,), 20, dtype=torch.int32, device="cuda")
    gpu.sample_rows_forward(token, logits, u, half * 1.6, k20, half * 1.8, None, logprob)
    torch.cuda.synchronize()
    x = logits.double()
    top, order = x.sort(dim=1, descending=True, stable=True)
    p = torch.softmax(top[:, :20] / (half * 1.6).double()[:, None], 1)
    p = p * (p.cumsum(1) - p < (half * 1.8).double()[:, None])
    want = (p.cumsum(1) <= u.double()[:, None] * p.sum(1, keepdim=True)).sum(1)
    assert torch.equal(token.long(), order.gather(1, want[:, None])[:, 0])
    assert torch.allclose(logprob.double(), torch.log(p.gather(1, want[:, None])[:, 0] / p.sum(1)), atol=1e-6)


def _call(pkg, lora=(), **args):
    p = 0x1000
    batch = pkg.LoraBatch(**dict(dict(a=p, b=p, scale=p, q_start=p, adapter=p, n_seqs=2, n_adapters=2, rank=16), **dict(lora)))
    import ctypes
    base = dict(out=0x2000, x=p, w=p, residual=None, lora=ctypes.byref(batch), ws=p, n_tokens=4, n_out=64, n_in=128,
                out_stride=64, x_stride=128, residual_stride=64, stream=None)
    L = pkg.lib()
    L.llm_clear_error()
    L.lora_projection_forward(*dict(base, **args).values())
    got = L.llm_last_error()
    L.llm_clear_error()
    return got.decode() if got else None


@pytest.mark.parametrize("args,message", [
    (dict(out=None), "must not be null"), (dict(x=None), "must not be null"), (dict(n_tokens=-1), "n_tokens -1"),
    (dict(n_tokens=(1 << 20) + 1), "n_tokens"), (dict(n_out=0), "n_out 0"), (dict(n_out=1 << 23), "n_out"),
    (dict(n_in=0), "n_in 0"), (dict(n_in=12, x_stride=16), "n_in 12"), (dict(x=0x1008), "16-byte aligned"),
    (dict(w=0x1002), "16-byte aligned"), (dict(x_stride=120), "x are 120"), (dict(x_stride=132), "x are 132"),
    (dict(out_stride=63), "overlap"), (dict(residual=0x3000, residual_stride=60), "overlap"),
    (dict(residual=0x2000, residual_stride=72), "in place"), (dict(out=0x1000), "must not be x"),
    (dict(ws=None), "ws must be"), (dict(ws=0x1004), "ws must be"), (dict(lora=dict(rank=0)), "rank 0"),
    (dict(lora=dict(rank=12)), "rank 12"), (dict(lora=dict(rank=264)), "rank 264"), (dict(lora=dict(rank=-8)), "rank -8"),
    (dict(lora=dict(n_seqs=0)), "n_seqs 0"), (dict(lora=dict(n_seqs=1 << 21)), "n_seqs 2097152"),
    (dict(lora=dict(n_adapters=0)), "n_adapters 0"), (dict(lora=dict(a=None)), "a, b, q_start"),
    (dict(lora=dict(b=0x1008)), "16-byte aligned"), (dict(lora=dict(q_start=None)), "a, b, q_start"),
    (dict(lora=dict(adapter=None)), "a, b, q_start")])
def test_refusals(pkg, args, message):
    assert message in _call(pkg, **args)


def test_no_rows_is_no_error(pkg):
    assert _call(pkg, n_tokens=0, out=None, x=None, ws=None) is None
    for sizes in [(-1, 8, 8, 8), (1, 0, 8, 8), (1, 8, 4, 8), (1, 8, 8, 7), (1, 8, 8, 264)]:
        with pytest.raises(pkg.LlmError, match="is not"):
            pkg.lora_projection_workspace_floats(*sizes)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_wrapper_refusals(gpu, monkeypatch, native):
    import torch
    if not native:
        monkeypatch.setattr(gpu, "_native", None)
    c = make(11, [2, 3], 64, 96, residual=True)
    out = torch.zeros(5, 96, device="cuda", dtype=torch.bfloat16)
    ws = torch.empty(gpu.lora_projection_workspace_floats(5, 96, 64, 16), device="cuda")
    for args, message in [
            (dict(out=out.float()), "out must be torch.bfloat16"), (dict(out=out[0]), "out must have two"),
            (dict(out=out[:4]), "out must have shape"), (dict(x=c["x"].cpu()), "x must be a tensor on the GPU"),
            (dict(x=c["x"].T), "must have|contiguous rows"), (dict(w=c["w"][:, :32].contiguous()), "w must be contiguous of shape"),
            (dict(w=c["w"].half()), "w must be"), (dict(residual=c["residual"][:, :8]), "residual must have shape"),
            (dict(lora_a=None), "lora_a is None"), (dict(lora_b=None), "lora_b is None"), (dict(q_start=None), "q_start is None"),
            (dict(adapter=None), "adapter is None"), (dict(lora_a=None, lora_b=None, q_start=None, adapter=None), "lora_a is None"),
            (dict(lora_a=c["lora_a"][0]), "lora_a must have shape"), (dict(lora_b=c["lora_b"][:2]), "lora_b must be contiguous"),
            (dict(lora_scale=c["lora_scale"].double()), "lora_scale must be"), (dict(q_start=c["q_start"][:2]), "q_start must be"),
            (dict(adapter=c["adapter"].long()), "adapter must be torch.int32"), (dict(ws=None), "ws holds 0 floats"),
            (dict(ws=ws[4:-1]), "ws holds"), (dict(ws=3), "ws must be a tensor"), (dict(out=c["x"][:, :32], w=None, lora_b=c["lora_b"][:, :32].contiguous(), residual=None), "must not be x")]:
        with pytest.raises(gpu.LlmError, match=message):
            gpu.lora_projection_forward(**dict(dict(c, out=out, ws=ws), **args))
    gpu.lora_projection_forward(out, **c, ws=ws)  # and no error is left
    torch.cuda.synchronize()
    check(out, c, 0.0)


@pytest.mark.gpu
def test_raw_bits_and_the_general_way_give_the_same(gpu, monkeypatch):
    import torch
    c = make(12, [2, 30], 64, 96, residual=True)
    want = both(gpu, c, 96)
    raw = {k: v.view(torch.int16) if v is not None and v.dtype == torch.bfloat16 else v for k, v in c.items()}
    for use_native in (True, False):
        with monkeypatch.context() as m:
            if not use_native:
                m.setattr(gpu, "_native", None)
            for form in (c, raw):
                assert torch.equal(run(gpu, form, torch.full_like(want, 7.0)), want)


@pytest.fixture
def force(gpu):
    """force(shape, splits, join): the plan of the calls until the test ends. The number of shapes."""
    L = gpu.lib()
    yield L.llm_lora_force
    L.llm_lora_force(-1, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", range(9))
@pytest.mark.parametrize("splits", [1, 2, 7])
@pytest.mark.parametrize("join", [False, True])
def test_every_way_to_compute(gpu, force, shape, splits, join):
    """Every tile with and without splits, its adapters as steps of the product or joined: ragged rows and columns, sums
    that end within a step, fewer steps than stages, no product, no adapters."""
    import torch
    assert force(shape, splits, int(join)) == 9
    for n_in, n_out, lengths, rank, spare in [(136, 270, [3, 1, 0, 300, 1, 1, 40], 24, 3), (8, 1, [5, 17], 8, 0),
                                              (1000, 515, [1] * 70 + [2, 3, 4], 40, 0), (512, 192, [257], 128, 1),
                                              (72, 1030, [600, 600], 16, 0)]:
        for kw in (dict(residual=True), dict(product=False), dict(adapters=0)):
            c = make(n_in + len(lengths), lengths, n_in, n_out, rank, **dict(dict(adapters=5), **kw), spare=spare)
            both(gpu, c, n_out)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", range(9))
@pytest.mark.parametrize("splits,join", [(1, 0), (3, 0), (1, 1), (3, 1)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_no_number_of_an_adapter_in_every_way(gpu, force, shape, splits, join, bad):
    """Elements of an adapter's b that are no numbers, in each way to compute: only the rows of its sequences, in their
    columns; infinities of the right sign also where the low product is a bf16 exactly, so that its remainder is zero."""
    import torch
    force(shape, splits, join)
    lengths, which = [40, 1, 1, 90, 2, 1, 30], [0, 1, 2, 1, -1, 3, 2]
    c = make(21, lengths, 200, 280, 16, adapters=4, which=which, residual=True, spare=2, scale=False)
    clean = {k: v if v is None else v.clone() for k, v in c.items()}
    c["lora_b"][1, 33, 5] = bad
    c["lora_b"][1, 279, 15] = bad
    c["lora_a"][1, 5].zero_()
    c["lora_a"][1, 5, 0] = 1.0
    c["x"][:, 0] = 3.0  # low[5] is 3
    clean["lora_a"], clean["x"] = c["lora_a"], c["x"]
    clean["lora_b"][1, 33, 5] = clean["lora_b"][1, 279, 15] = 0
    out = torch.full((c["x"].shape[0], 280), 7.0, device="cuda", dtype=torch.bfloat16)
    run(gpu, c, out)
    touched = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    starts = c["q_start"].tolist()
    for s, a in enumerate(which):
        if a == 1:
            touched[starts[s]:starts[s + 1], [33, 279]] = True
            if not math.isnan(bad):
                assert (out[starts[s]:starts[s + 1], 33] == bad).all()
    assert not out[touched].isfinite().any()
    want, err, written = defined(clean, *out.shape)
    fine = written[:, None] & ~touched
    off = (out.double() - want).abs() - (HALF_STEP * (want.abs() + err) + err)
    assert (off[fine] <= 0).all() and (out[~written] == 7).all()


@pytest.mark.gpu
def test_starts_that_decrease_stay_within_the_rows(gpu, force):
    """What the documentation does not allow reads and writes nothing outside of the call's tensors: rows of
    sequences that do not overlap are right, whatever the others hold."""
    import torch
    for shape, join in ((4, 0), (4, 1), (8, 1), (0, 0)):
        force(shape, 2, join)
        c = make(22, [60], 128, 192, 8, adapters=3)
        c["q_start"] = torch.tensor([0, 20, 10, 55, 2 ** 31 - 1, -5, 60], dtype=torch.int32, device="cuda")
        c["adapter"] = torch.tensor([0, 1, 2, 0, 1, 2], dtype=torch.int32, device="cuda")
        wide = torch.full((64, 200), 7.0, device="cuda", dtype=torch.bfloat16)
        run(gpu, c, wide[2:62, 4:196])
        assert (wide[:2] == 7).all() and (wide[62:] == 7).all() and (wide[:, :4] == 7).all() and (wide[:, 196:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,rank", [(1, 8), (1, 16), (2, 8)])
@pytest.mark.parametrize("n_in,n_out", [(8, 1), (72, 19), (1024, 2048), (520, 515), (2560, 1030)])
def test_one_or_two_rows(gpu, rows, rank, n_in, n_out):
    """The sizes of a single launch: sequences of one and two rows, empty ones around them, up to 64 of them and one more,
    rows of no sequence, no adapter, each part off."""
    import torch
    for lengths, which in [([rows], [1]), ([0, 1] + [0] * 61 + [rows - 1], [0, 2] + [1] * 61 + [3]), ([0] * 40 + [rows], None),
                           ([0] * 64 + [rows], None), ([1] * rows, [-1, 7][:rows]), ([0, 0], [0, 1])]:
        spare = rows - sum(lengths)
        for kw in (dict(residual=True), dict(product=False, residual=True), dict(product=False), dict(scale=False)):
            c = make(len(lengths) + n_in, lengths, n_in, n_out, rank, adapters=4, which=which, spare=spare, **kw)
            both(gpu, c, n_out)
    for starts in ([0, 1], [1, rows], [-3, 9], [2 ** 31 - 1, -1], [rows, 0]):
        c = make(5, [rows], n_in, n_out, rank, adapters=2, which=[1], residual=True)
        c["q_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        both(gpu, c, n_out)


@pytest.mark.gpu
@pytest.mark.parametrize("product", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_no_number_in_one_of_two_rows(gpu, product, bad):
    """A row, an adapter's a, b or scale that are no numbers, beside a row that has none of it."""
    import torch
    for where in ("x", "lora_a", "lora_b", "lora_scale"):
        c = make(9, [1, 1], 264, 70, 8, adapters=2, which=[1, 0], product=product, residual=True)
        clean = {k: v if v is None else v.clone() for k, v in c.items()}
        dict(x=lambda t: t[0, 3:4], lora_a=lambda t: t[1, 2, 5:6], lora_b=lambda t: t[1, 33, 5:6],
             lora_scale=lambda t: t[1:2])[where](c[where]).fill_(bad)
        out = torch.zeros(2, 70, device="cuda", dtype=torch.bfloat16)
        run(gpu, c, out)
        want = torch.zeros_like(out)
        run(gpu, clean, want)
        assert torch.equal(out[1], want[1]) and not out[0, 33].isfinite()
    c["adapter"][1] = -1  # without an adapter and, without w, the residual alone
    c["x"][1, 3] = bad
    run(gpu, c, out)
    assert product or torch.equal(out[1], c["residual"][1])


@pytest.mark.gpu
@pytest.mark.parametrize("shape,join", [(-1, 0)] + [(s, j) for s in range(9) for j in (0, 1)])
@pytest.mark.parametrize("last", [1.0, 1.5])
def test_low_products_at_the_end_of_the_range(gpu, force, shape, join, last):
    """Finite in 32 bits, but past the largest bf16 by half its step and more: 8 (255 2^120 + last 2^119) 2^-100 is exact in
    32 bits, and the nearest bf16 (the even one, where last is 1) is 2^31."""
    import torch
    force(shape, 1, join)
    for lengths in ([1], [3], [20, 1, 40], [300, 2]):
        c = make(7, lengths, 64, 130, 8, adapters=1, which=[0] * len(lengths), product=False, scale=False)
        for k in ("x", "lora_a"):
            c[k].zero_()
        sign = torch.where(torch.arange(sum(lengths), device="cuda") % 3 == 1, -1.0, 1.0)
        c["x"][:, :2] = sign[:, None] * 2.0 ** 64
        c["lora_a"][:, :, 0] = 255 * 2.0 ** 56
        c["lora_a"][:, :, 1] = last * 2.0 ** 55
        c["lora_b"].fill_(2.0 ** -100)
        out = torch.zeros(sum(lengths), 130, device="cuda", dtype=torch.bfloat16)
        run(gpu, c, out)
        assert (out == sign[:, None] * 2.0 ** 31).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,splits,join", [(-1, 0, 0)] + [(s, n, j) for s in range(9) for n, j in ((1, 0), (3, 0), (1, 1))])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_infinite_low_products_meet_infinities(gpu, force, shape, splits, join, bad):
    """An element of b that is no number, where the low product that it meets is infinite: their product, as in 64 bits."""
    import torch
    force(shape, splits, join)
    for lengths, which in ([[1], [1]], [[1, 1], [0, 1]], [[40, 1, 1, 90, 2, 1, 30], [0, 1, 2, 1, -1, 3, 2]]):
        c = make(23, lengths, 200, 280, 8, adapters=4, which=which, residual=True, scale=False)
        rows = sum(lengths)
        sign = torch.where(torch.arange(rows, device="cuda") % 3 == 1, -1.0, 1.0)
        c["x"][:, 0] = 3 * sign
        c["lora_a"][1, 5, 0] = math.inf  # low[5] is an infinity of x[:, 0]'s sign
        c["lora_b"][1, :, 5] = torch.where(c["lora_b"][1, :, 5] == 0, 1.0, c["lora_b"][1, :, 5])
        clean = defined(dict(c, lora_a=c["lora_a"].nan_to_num(0, 0, 0)), rows, 280)
        c["lora_b"][1, 33, 5] = bad
        out = torch.full((rows, 280), 7.0, device="cuda", dtype=torch.bfloat16)
        run(gpu, c, out)
        starts = c["q_start"].tolist()
        for s, a in enumerate(which):
            own = slice(starts[s], starts[s + 1])
            if a == 1:
                want = sign[own, None] * c["lora_b"][1, :, 5].float() * math.inf
                assert torch.equal(out[own].isnan(), want.isnan())
                assert torch.equal(out[own].float().nan_to_num(), want.nan_to_num())
            else:
                value, err, _ = (t[own] if t.dim() == 2 else t for t in clean)
                assert ((out[own].double() - value).abs() <= HALF_STEP * (value.abs() + err) + err).all()


@pytest.mark.parametrize("n_out", [250000, 1 << 22])  # of the first, 2^31 to 2^32 threads with most tiles
@pytest.mark.parametrize("adapters", [False, True])
def test_products_of_too_many_threads(pkg, n_out, adapters):
    """Refused before anything is launched, low in front of the product neither."""
    sizes = dict(n_tokens=1 << 20, n_out=n_out, out_stride=n_out)
    if adapters:
        message = _call(pkg, **sizes)
    else:
        L, p = pkg.lib(), 0x1000
        L.llm_clear_error()
        L.lora_projection_forward(0x2000, p, p, None, None, p, 1 << 20, n_out, 128, n_out, 128, n_out, None)
        message = L.llm_last_error().decode()
        L.llm_clear_error()
    assert "too much for one launch" in message


def test_sequences_of_too_many_threads(pkg):
    assert "too many for one launch" in _call(pkg, lora=dict(n_seqs=1 << 20), n_in=1 << 15, x_stride=1 << 15)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,rank,n_in,n_out,product,one", [
    (1, 8, 1024, 2048, True, True), (1, 8, 4096, 2560, True, True), (1, 16, 2560, 4096, True, True), (2, 8, 1024, 2048, True, True),
    (1, 16, 1024, 8192, False, True), (1, 8, 9728, 16, True, False), (1, 8, 9728, 256, True, False), (1, 16, 9728, 1024, True, False),
    (1, 16, 4096, 1024, True, False), (1, 8, 1 << 16, 16, True, False), (1, 8, 1 << 20, 16, True, False), (2, 8, 4096, 257, True, False),
    (2, 8, 9728, 16, True, False), (1, 8, 9728, 64, False, False), (2, 8, 1 << 16, 16, False, False), (1, 8, 512, 9728, False, False)])
def test_a_single_launch_where_it_is_shorter(gpu, rows, rank, n_in, n_out, product, one):
    """Few columns of a long sum are not left to a workgroup each, nor so many columns that the workgroups take turns. The
    single launch does without the workspace."""
    import torch
    c = make(rows + n_in, [1] * rows, n_in, n_out, rank, adapters=2, which=[1, 0][:rows], product=product, residual=True)
    ws = torch.full((gpu.lora_projection_workspace_floats(rows, n_out, n_in, rank),), math.nan, device="cuda")
    both(gpu, c, n_out, ws=ws)
    assert bool(ws.isnan().all()) == one


@pytest.mark.gpu
def test_a_plan_for_tests_stays_with_its_thread(gpu, force):
    """The plan that a test forces is not another thread's: that one's single launch leaves the workspace alone."""
    import threading
    import torch
    c = make(31, [1], 1024, 64, 8, adapters=2, which=[1])
    floats = gpu.lora_projection_workspace_floats(1, 64, 1024, 8)
    ws = [torch.full((floats,), math.nan, device="cuda") for _ in range(2)]
    force(4, 2, 0)
    both(gpu, c, 64, ws=ws[0])
    failed = []

    def other():
        try:
            both(gpu, c, 64, ws=ws[1])
        except BaseException as e:
            failed.append(e)
    thread = threading.Thread(target=other)
    thread.start()
    thread.join()
    assert not failed and not ws[0].isnan().all() and ws[1].isnan().all()


@pytest.mark.parametrize("rows,n_out,n_in,rank,n_seqs,large", [
    (1344, 6144, 2560, 0, 0, True), (1344, 6144, 2560, 32, 5, True), (1324, 1040, 4976, 0, 0, True), (1600, 2560, 9728, 0, 0, True),
    (1987, 6144, 2560, 16, 2, True), (64, 4096, 2560, 16, 64, False), (64, 151936, 2560, 0, 0, False), (17, 2560, 9728, 64, 17, False)])
def test_tiles_of_few_rows_are_for_few_rows(pkg, rows, n_out, n_in, rank, n_seqs, large):
    """Shapes 5 to 8 have up to 64 rows and read w past the caches, as often as there are such rows of tiles: 114 us in place
    of 50 for the first of these calls."""
    assert (pkg.lib().llm_lora_plan(rows, n_out, n_in, rank, n_seqs, 4 if rank else 0) < 5) == large
