"""Operators over a paged KV cache (include/llm_amd/paged.h) against their definitions in 64 bits: the
QK-norm + RoPE that writes pages, the attention over pages, both together with the logits' penalties as a
serving loop runs them, in captured graphs too; and what they refuse."""
import ctypes
import math

import numpy as np
import pytest

HALF_STEP = 2.0 ** -8   # of bf16, relative to the value
F32 = 2.0 ** -24        # half a step of fp32


# ---------------------------------------------------------------- batches

class Batch:
    """Sequences (new rows, cached tokens with them) over a shuffled pool. Slots that hold no token of
    a sequence hold NaN and infinities."""

    def __init__(self, seqs, kv_heads, dim, page, seed, lead=0, trail=0, extra_pages=3, layout="pages"):
        import torch
        self.seqs, self.kv_heads, self.dim, self.page = seqs, kv_heads, dim, page
        self.rng = np.random.default_rng(seed)
        g = self.g = torch.Generator().manual_seed(seed)
        need = [max(0, -(-n // page)) for _, n in seqs]
        self.pages = sum(need) + extra_pages
        self.table_pages = max(need + [1]) + 1
        order = torch.randperm(self.pages, generator=g)
        table = torch.full((len(seqs), self.table_pages), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n].int()
            at += n
        self.table = table
        starts = [lead]
        for new, _ in seqs:
            starts.append(starts[-1] + new)
        self.starts, self.tokens = starts, starts[-1] + trail
        self.q_start = torch.tensor(starts, dtype=torch.int32)
        self.kv_len = torch.tensor([n for _, n in seqs], dtype=torch.int32)
        bad = torch.tensor([math.nan, math.inf, -math.inf])
        self.k, self.v = (bad[torch.randint(0, 3, (self.pages, page, kv_heads, dim), generator=g)].bfloat16()
                          for _ in range(2))
        for s, (_, n) in enumerate(seqs):
            for p in range(max(0, n)):
                slot = self.slot(s, p)
                if slot:
                    self.k[slot], self.v[slot] = self.normal(kv_heads, dim), self.normal(kv_heads, dim)
        self.layout = layout

    def normal(self, *shape, std=1.0):
        import torch
        return (torch.randn(*shape, generator=self.g) * std).bfloat16()

    def slot(self, s, p):
        if p < 0 or p // self.page >= self.table.shape[1]:
            return None
        page = int(self.table[s, p // self.page])
        return (page, p % self.page) if 0 <= page < self.pages else None

    def rows(self):
        """(row, sequence, position) of every row of a sequence."""
        for s, (new, n) in enumerate(self.seqs):
            for i in range(new):
                yield self.starts[s] + i, s, n - new + i

    def pools(self):
        """The caches on the GPU, dense or as views of one pool that holds both (by page, by kv head)."""
        import torch
        if self.layout == "pages":
            return self.k.cuda(), self.v.cuda()
        both = torch.empty(self.pages, 2, self.kv_heads, self.page, self.dim, dtype=torch.bfloat16, device="cuda")
        k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
        k.copy_(self.k)
        v.copy_(self.v)
        return k, v

    def where(self):
        return self.table.cuda(), self.q_start.cuda(), self.kv_len.cuda()


def bits(t):
    import torch
    return t.contiguous().view(torch.int16).cpu()


def workspace(gpu, b, heads, max_q, max_kv):
    import torch
    n = gpu.attention_paged_workspace_floats(b.tokens, len(b.seqs), heads, b.kv_heads, b.dim, max_q, max_kv)
    return torch.full((max(n, 1),), math.nan, device="cuda")


# ---------------------------------------------------------------- QK-norm + RoPE into pages

def rotated(x, weight, pos, inv_freq, scale, interleaved, eps):
    """(value, a bound on its fp32 arithmetic's error) of one row's heads [heads, dim] in 64 bits."""
    x = x.double().numpy()
    dim = x.shape[-1]
    err = 8 * F32
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.double().numpy()
        err += (dim / 2 + 8) * F32  # the sum of squares under the root, then root, quotient and products
    n = 2 * len(inv_freq)
    i = np.arange(n // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n // 2)
    angle = pos * inv_freq
    c, s = np.cos(angle) * scale, np.sin(angle) * scale
    y, size = x.copy(), np.abs(x)
    y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
    size[:, a] = size[:, b] = (size[:, a] + size[:, b]) * abs(scale)
    return y, err * size


def close(got, want, err):
    """got is bf16 of a value within err of want."""
    got = got.double().numpy()
    off = np.abs(got - want) - (HALF_STEP * (np.abs(want) + err) + err)
    assert (off <= 0).all(), f"{(off > 0).sum()} of {off.size} off by up to {off.max():.3g} more than allowed"


APPEND = [
    # heads, kv heads, dim, rotary, interleaved, norm, page, sequences (new, cached), layout
    (16, 8, 128, 128, False, True, 16, [(1, 261)], "pages"),
    (32, 8, 128, 128, False, True, 16, [(1, 1), (1, 16), (1, 17), (1, 300)], "pages"),
    (5, 1, 128, 128, True, True, 7, [(19, 40), (0, 9), (1, 3)], "heads"),
    (6, 2, 64, 32, True, False, 1, [(33, 33)], "pages"),
    (3, 3, 64, 64, False, True, 32, [(70, 131), (2, 65)], "heads"),
    (4, 4, 256, 256, False, True, 16, [(9, 9), (17, 100)], "pages"),
    (8, 2, 256, 16, True, True, 128, [(130, 130)], "heads"),
    (9, 3, 128, 48, False, False, 24, [(3, 25), (25, 25)], "pages"),
    # sequences longer in new rows than in cached tokens: the first rows' positions are negative
    (2, 1, 64, 64, False, True, 16, [(5, 2), (3, 0), (2, 2)], "pages"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(APPEND)))
@pytest.mark.parametrize("fused", [False, True])
def test_append_against_the_definition(gpu, case, fused):
    import torch
    heads, kv_heads, dim, rotary, interleaved, norm, page, seqs, layout = APPEND[case]
    b = Batch(seqs, kv_heads, dim, page, 100 + case, lead=2, trail=3, layout=layout)
    # one page of the first sequence is not there
    gone = case % 2 == 1 and seqs[0][1] > page
    if gone:
        b.table[0, 0] = b.pages if case % 4 == 1 else -7
    rows = b.normal(b.tokens, heads + 2 * kv_heads, dim)
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]
    qn, kn = (b.normal(dim), b.normal(dim)) if norm else (None, None)
    kind = [gpu.ROPE_PLAIN, gpu.ROPE_LINEAR, gpu.ROPE_YARN][case % 3]
    inv_freq, scale = gpu.rope_frequencies(rotary, 1e4 if case % 2 else 1e6, kind, 4.0 if kind else 1.0, 4096)
    kc, vc = b.pools()
    dev = [t.cuda() for t in (q, k, v)]
    if fused:
        whole = rows.cuda()
        dev = [whole[:, :heads], whole[:, heads:heads + kv_heads], whole[:, heads + kv_heads:]]
    q_out = torch.full((b.tokens, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    gpu.qk_norm_rope_paged(q_out, *dev, qn.cuda() if norm else None, kn.cuda() if norm else None,
                           inv_freq.cuda(), kc, vc, *b.where(), 1e-6, scale, interleaved=interleaved)
    got_q, got_k, got_v = q_out.cpu(), kc.cpu(), vc.cpu()
    written = torch.zeros(b.pages, page, dtype=torch.bool)
    mine = torch.zeros(b.tokens, dtype=torch.bool)
    for t, s, p in b.rows():
        mine[t] = True
        close(got_q[t], *rotated(q[t], qn, p, inv_freq.numpy(), scale, interleaved, 1e-6))
        slot = b.slot(s, p)
        if slot:
            written[slot] = True
            close(got_k[slot], *rotated(k[t], kn, p, inv_freq.numpy(), scale, interleaved, 1e-6))
            assert torch.equal(bits(got_v[slot]), bits(v[t]))
    assert (got_q[~mine] == 7).all()
    for got, before in ((got_k, b.k), (got_v, b.v)):
        assert torch.equal(bits(got[~written]), bits(before[~written]))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim,rotary,interleaved,norm,seqs", [
    (32, 8, 128, 128, False, True, [(1500, 1700), (1, 5), (31, 31)]), (35, 7, 64, 32, True, False, [(2601, 2601)]),
    (6, 3, 256, 256, True, True, [(1200, 1200), (0, 4), (601, 640)]), (12, 4, 128, 48, False, False, [(4100, 4100)])])
def test_append_of_many_rows(gpu, heads, kv_heads, dim, rotary, interleaved, norm, seqs):
    """So many rows that a wave takes several groups of a row's heads, of q, k and v among each other."""
    import torch
    page = 16
    groups = -(-heads * dim // 512) + 2 * -(-kv_heads * dim // 512)
    assert sum(n for n, _ in seqs) * groups // 6144 >= 2
    b = Batch([], kv_heads, dim, page, 47)
    b.seqs, need = seqs, [-(-n // page) for _, n in seqs]
    b.pages = sum(need) + 2
    b.table = torch.full((len(seqs), max(need)), -1, dtype=torch.int32)
    order = torch.randperm(b.pages, generator=b.g).int()
    for s, n in enumerate(need):
        b.table[s, :n] = order[sum(need[:s]):sum(need[:s]) + n]
    b.starts = [sum(n for n, _ in seqs[:s]) for s in range(len(seqs) + 1)]
    b.tokens = b.starts[-1] + 1
    b.q_start, b.kv_len = (torch.tensor(x, dtype=torch.int32) for x in (b.starts, [n for _, n in seqs]))
    rows = b.normal(b.tokens, heads + 2 * kv_heads, dim)
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]
    qn, kn = (b.normal(dim), b.normal(dim)) if norm else (None, None)
    inv_freq, scale = gpu.rope_frequencies(rotary, 1e6, gpu.ROPE_YARN, 4.0, 4096)
    kc, vc = (torch.full((b.pages, page, kv_heads, dim), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    whole = rows.cuda()
    q_out = torch.full((b.tokens, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    gpu.qk_norm_rope_paged(q_out, whole[:, :heads], whole[:, heads:heads + kv_heads], whole[:, heads + kv_heads:],
                           qn.cuda() if norm else None, kn.cuda() if norm else None, inv_freq.cuda(), kc, vc,
                           *b.where(), 1e-6, scale, interleaved=interleaved)
    got_q, got_k, got_v = q_out.cpu(), kc.cpu(), vc.cpu()
    written = torch.zeros(b.pages, page, dtype=torch.bool)
    for t, s, p in b.rows():
        slot = b.slot(s, p)
        written[slot] = True
        close(got_q[t], *rotated(q[t], qn, p, inv_freq.numpy(), scale, interleaved, 1e-6))
        close(got_k[slot], *rotated(k[t], kn, p, inv_freq.numpy(), scale, interleaved, 1e-6))
        assert torch.equal(got_v[slot], v[t])
    assert (got_q[-1] == 7).all() and (got_k[~written] == 7).all() and (got_v[~written] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_far_positions_and_in_place(gpu, interleaved):
    """A long context's last rows (positions around 2^20): the angle's 64 bits; q_out may be q."""
    import torch
    heads, dim, page, far = 4, 128, 64, (1 << 20) + 5
    b = Batch([(3, 3)], 2, dim, page, 5)
    b.seqs = [(3, far)]
    b.kv_len = torch.tensor([far], dtype=torch.int32)
    table = torch.full((1, far // page + 1), -1, dtype=torch.int32)
    table[0, -1] = 2
    table[0, -2] = 1
    b.table, b.table_pages = table, table.shape[1]
    q, k, v = b.normal(3, heads, dim), b.normal(3, 2, dim), b.normal(3, 2, dim)
    inv_freq, scale = gpu.rope_frequencies(dim, 1e6)
    kc, vc = b.pools()
    q_dev = q.cuda()
    gpu.qk_norm_rope_paged(q_dev, q_dev, k.cuda(), v.cuda(), None, None, inv_freq.cuda(), kc, vc, *b.where(),
                           1e-6, interleaved=interleaved)
    for t, s, p in b.rows():
        close(q_dev[t].cpu(), *rotated(q[t], None, p, inv_freq.numpy(), 1.0, interleaved, 0))
        slot = b.slot(s, p)
        close(kc.cpu()[slot], *rotated(k[t], None, p, inv_freq.numpy(), 1.0, interleaved, 0))
        assert torch.equal(bits(vc.cpu()[slot]), bits(v[t]))


def test_rope_frequencies(pkg):
    """Closed forms: the powers; divided pairs; YaRN's ends and its ramp, which is straight in the pair."""
    j = np.arange(64)
    base = 1e6 ** (-2.0 * j / 128)
    got, scale = pkg.rope_frequencies(128, 1e6)
    assert scale == 1.0 and np.allclose(got.numpy(), base, rtol=1e-14, atol=0)
    got, scale = pkg.rope_frequencies(128, 1e6, pkg.ROPE_LINEAR, 8.0)
    assert scale == 1.0 and np.allclose(got.numpy(), base / 8, rtol=1e-14, atol=0)
    got, scale = pkg.rope_frequencies(128, 1e6, pkg.ROPE_YARN, 4.0, 32768)
    assert scale == pytest.approx(0.1 * math.log(4) + 1, rel=1e-6)
    turns = 32768 * base / (2 * math.pi)
    share = (base - got.numpy()) / (base - base / 4)  # 0: left as it is, 1: divided
    assert np.allclose(share[turns > 32 * 1.3], 0, atol=1e-12) and np.allclose(share[turns < 0.7], 1, atol=1e-12)
    inner = (share > 1e-9) & (share < 1 - 1e-9)
    assert inner.sum() > 8 and np.allclose(np.diff(share[inner]), np.diff(share[inner])[0], atol=1e-9)
    for args in [(0, 1e4), (7, 1e4), (64, 1.0), (64, math.nan), (64, 1e4, 3), (64, 1e4, 1, 0.5),
                 (64, 1e4, 2, math.inf, 4096), (64, 1e4, 2, 2.0, 0)]:
        with pytest.raises(pkg.LlmError, match="rope_frequencies"):
            pkg.rope_frequencies(*args)


@pytest.mark.parametrize("theta,trained,share", [(1e4, 1, 1), (1e4, 4, 1), (1e6, 6, 1), (10.0, 32768, 0), (1.5, 100000, 0)])
def test_yarn_where_all_pairs_are_slow_or_fast(pkg, theta, trained, share):
    """None turns once over the trained length: all are divided. All turn more than 32 times: all are left."""
    base = theta ** (-2.0 * np.arange(32) / 64)
    turns = trained * base / (2 * math.pi)
    assert (turns < 1).all() if share else (turns > 32).all()
    got, scale = pkg.rope_frequencies(64, theta, pkg.ROPE_YARN, 4.0, trained)
    assert scale == pytest.approx(0.1 * math.log(4) + 1, rel=1e-6)
    assert np.allclose(got.numpy(), base / 4 if share else base, rtol=1e-14, atol=0)


# ---------------------------------------------------------------- attention over pages

def attended(b, q, scale, window):
    """(value, a bound on the error before the last rounding) in 64 bits, row by row and key by key that
    the row sees; rows of no sequence None. The bound: every weight is off by its rounding to bf16 and
    by twice its score's error (the dot's fp32 sums, then the largest score's), the sums in fp32."""
    k, v = b.k.double().numpy(), b.v.double().numpy()
    q = q.double().numpy()
    heads, dim = q.shape[1:]
    out, err = np.zeros(q.shape), np.zeros(q.shape)
    for t, s, p in b.rows():
        first = max(0, p - window + 1) if window else 0
        slots = [b.slot(s, i) for i in range(first, p + 1)]
        slots = [x for x in slots if x]
        if not slots:
            continue
        pages, at = np.array(slots).T
        for h in range(heads):
            kk, vv = (x[pages, at, h // (heads // b.kv_heads)] for x in (k, v))
            with np.errstate(all="ignore"):
                score = kk @ q[t, h] * scale
                keep = score != -np.inf
                if not keep.any():
                    continue
                score, kk, vv = score[keep], kk[keep], vv[keep]
                w = np.exp(score - score.max())
                w /= w.sum()
                out[t, h] = w @ vv
                off = 2 * (dim * F32 * (np.abs(kk) @ np.abs(q[t, h])).max() * scale + 8 * F32 * np.abs(score).max())
                err[t, h] = (HALF_STEP + off + (len(w) + 64) * F32) * (w @ np.abs(vv))
    return out, err


def attend(gpu, b, q, scale, window=0, max_q=None, max_kv=None, pools=None, ws=None, out=None):
    import torch
    heads = q.shape[1]
    max_q = max_q or max([new for new, _ in b.seqs] + [1])
    max_kv = max_kv or max([n for _, n in b.seqs] + [1])
    kc, vc = pools or b.pools()
    ws = workspace(gpu, b, heads, max_q, max_kv) if ws is None else ws
    out = torch.full((b.tokens, heads, b.dim), 7.0, dtype=torch.bfloat16, device="cuda") if out is None else out
    gpu.attention_paged_forward(out, q.cuda(), kc, vc, *b.where(), ws, scale, max_q, max_kv, window=window)
    return out


def check_attend(b, out, q, scale, window):
    import torch
    got = out.cpu()
    want, err = attended(b, q, scale, window)
    mine = [t for t, _, _ in b.rows()]
    fine = np.isfinite(want[mine])
    assert np.array_equal(fine, np.isfinite(got[mine].double().numpy())), "finite elsewhere than the definition"
    close(got[mine][torch.from_numpy(fine)], want[mine][fine], err[mine][fine])
    other = np.setdiff1d(np.arange(b.tokens), mine)
    assert (got[other] == 7).all(), "rows of no sequence were written"


ATTEND = [
    # heads, kv heads, dim, page, window, sequences (new, cached), layout
    (16, 8, 128, 16, 0, [(1, 261)], "pages"),
    (16, 8, 128, 16, 0, [(1, 1)], "pages"),
    (32, 8, 128, 16, 0, [(1, 1), (1, 31), (1, 32), (1, 33), (1, 64), (1, 65), (1, 700), (1, 129)], "pages"),
    (4, 4, 128, 1, 0, [(1, 77), (1, 5)], "heads"),
    (7, 1, 128, 24, 0, [(1, 500), (3, 130), (4, 4)], "pages"),
    (40, 1, 64, 16, 0, [(1, 300), (2, 90)], "heads"),
    (6, 2, 64, 7, 50, [(1, 200), (13, 149), (1, 20)], "pages"),
    (8, 2, 256, 16, 0, [(1, 90), (1, 257), (5, 40)], "pages"),
    (2, 2, 256, 128, 33, [(70, 200)], "heads"),
    (8, 2, 128, 64, 0, [(200, 333)], "pages"),
    (4, 4, 64, 32, 0, [(129, 129), (1, 400), (64, 64), (65, 300)], "heads"),
    (24, 4, 64, 16, 100, [(150, 400), (131, 131)], "pages"),
    (12, 3, 128, 16, 1, [(40, 80), (1, 9)], "pages"),
    (16, 8, 128, 32, 0, [(127, 300), (1, 17), (0, 50), (1, 900), (30, 30)], "heads"),
    (6, 1, 256, 20, 0, [(90, 311)], "pages"),
    # nothing cached, nothing new, more new rows than cached tokens: rows that see nothing
    (4, 2, 128, 16, 0, [(1, 0), (0, 0), (5, 2), (1, 1), (2, -3)], "pages"),
    (4, 2, 64, 16, 4, [(40, 7), (70, 40)], "pages"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention_against_the_definition(gpu, case):
    heads, kv_heads, dim, page, window, seqs, layout = ATTEND[case]
    b = Batch(seqs, kv_heads, dim, page, 200 + case, lead=1, trail=2, layout=layout)
    q = b.normal(b.tokens, heads, dim, std=1.5)
    scale = 1 / math.sqrt(dim)
    check_attend(b, attend(gpu, b, q, scale, window), q, scale, window)


@pytest.mark.gpu
@pytest.mark.parametrize("max_q,max_kv", [(1, 1), (1, 4000), (400, 1), (5000, 100000), (33, 70000)])
@pytest.mark.parametrize("case", [2, 4, 9, 13])
def test_attention_whatever_the_expected_lengths(gpu, case, max_q, max_kv):
    """The expected lengths split the work and nothing else: shorter and longer ones than the batch has."""
    heads, kv_heads, dim, page, window, seqs, layout = ATTEND[case]
    b = Batch(seqs, kv_heads, dim, page, 300 + case, lead=1, trail=2, layout=layout)
    q = b.normal(b.tokens, heads, dim, std=1.5)
    scale = 1 / math.sqrt(dim)
    check_attend(b, attend(gpu, b, q, scale, window, max_q, max_kv), q, scale, window)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [[(5, 2), (8, 3), (1, 40)], [(70, 40), (40, 7)]])
@pytest.mark.parametrize("window", [2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1])
def test_attention_window_past_every_length(gpu, seqs, window):
    """A window past any position is none, for rows whose positions are negative beside others too."""
    b = Batch(seqs, 2, 64, 16, 21)
    q = b.normal(b.tokens, 4, 64)
    check_attend(b, attend(gpu, b, q, 0.125, window), q, 0.125, window)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,dim,heads", [([(1, 9000)], 128, 4), ([(1, 70000), (1, 3)], 64, 2),
                                            ([(3, 5000), (1, 2500), (1, 1)], 256, 2), ([(150, 6000)], 128, 2)])
def test_attention_long_histories(gpu, seqs, dim, heads):
    """Split over the keys: a peak of the scores late, early and in the middle of the history."""
    import torch
    b = Batch(seqs, 1, dim, 64, 7)
    q = b.normal(b.tokens, heads, dim)
    for p, size in ((3, 6.0), (seqs[0][1] // 2, 9.0), (seqs[0][1] - 1, 12.0)):
        b.k[b.slot(0, p)] = (q[0, 0].float() * size / 4).bfloat16()
    scale = 1 / math.sqrt(dim)
    out = attend(gpu, b, q, scale)
    check_attend(b, out, q, scale, 0)
    again = attend(gpu, b, q, scale)
    assert torch.equal(bits(out), bits(again))  # the joins have one order


@pytest.mark.gpu
@pytest.mark.parametrize("dim,page", [(64, 32), (128, 16), (128, 5), (256, 16)])
@pytest.mark.parametrize("window", [0, 2500])
def test_attention_split_chunks_beside_single_tokens(gpu, dim, page, window):
    """Chunks whose keys are split over workgroups and joined, single tokens beside them, a page gone."""
    b = Batch([(150, 6000), (1, 5000), (40, 3000), (0, 100), (1, 2), (33, 40)], 1, dim, page, 41, lead=1, trail=1)
    b.table[0, 2000 // page], b.table[1, 4000 // page] = -1, b.pages
    q = b.normal(b.tokens, 2, dim, std=1.5)
    scale = 1 / math.sqrt(dim)
    check_attend(b, attend(gpu, b, q, scale, window), q, scale, window)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,window,dim", [([(40, 100), (1, 100), (1, 65)], 0, 128),
                                             ([(40, 100), (1, 100), (1, 65)], 21, 64),
                                             ([(200, 230)], 0, 128), ([(200, 230)], 30, 256)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", ["k", "v"])
def test_attention_bad_values_stay_with_the_rows_that_see_them(gpu, seqs, window, dim, bad, which):
    """A NaN or an infinity in a key or value: rows in front of its position and past its window are what
    they are without it; pages that are not there are not seen."""
    heads, kv_heads = 4, 2
    b = Batch(seqs, kv_heads, dim, 16, 11)
    q = b.normal(b.tokens, heads, dim)
    last = seqs[0][1] - 1
    for p, h, d in ((last, 0, 3), (last - 20, 1, dim - 1), (last - 7, 0, dim // 2)):
        getattr(b, which)[b.slot(0, p) + (h, d)] = bad
    b.table[0, 1] = -1
    if len(seqs) > 1:
        b.table[1, 2] = b.pages + 5
    scale = 1 / math.sqrt(dim)
    check_attend(b, attend(gpu, b, q, scale, window), q, scale, window)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,window,dim,page", [
    ([(1, 1)], 0, 128, 16), ([(1, 40), (2, 70)], 0, 64, 16), ([(1, 300), (5, 300), (1, 33)], 40, 128, 5),
    ([(1, 9000)], 0, 128, 64), ([(3, 5000), (1, 2500)], 0, 256, 16), ([(70, 200)], 0, 128, 16),
    ([(40, 600), (1, 600)], 0, 64, 16), ([(150, 6000)], 200, 256, 64)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_attention_infinite_values_that_every_row_sees(gpu, seqs, window, dim, page, bad):
    """An infinity among the values that all rows of a sequence see makes an infinity of its sign, both signs in
    one element no number, and other elements are what they are without it: for few and for many rows, split or
    not, whatever the position weighs (here down to e^-60)."""
    import torch
    heads, kv_heads, scale = 4, 2, 1 / math.sqrt(dim)
    b = Batch(seqs, kv_heads, dim, page, 43)
    q = b.normal(b.tokens, heads, dim)
    q[:, :, 0] = 4.0
    for s, (new, n) in enumerate(seqs):
        seen = list(range(max(0, n - window) if window else 0, n - new + 1))  # by every row of the sequence
        for p in seen[-3:]:
            b.v[b.slot(s, p) + (0, 3)] = bad
        b.v[b.slot(s, seen[-1]) + (1, dim - 1)] = bad
        b.v[b.slot(s, seen[0]) + (1, dim // 2)] = bad
        if len(seen) > 1:
            b.v[b.slot(s, seen[0]) + (0, 9)], b.v[b.slot(s, seen[-1]) + (0, 9)] = bad, -bad
            b.k[b.slot(s, seen[0]) + (1, 0)] = -15 / scale  # 60 below where it would be
    out = attend(gpu, b, q, scale, window)
    got, (want, err) = out.cpu().double().numpy(), attended(b, q, scale, window)
    fine = np.isfinite(want)
    assert 0 < (~fine).sum() < fine.size // 4
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True), "other infinities than the definition"
    close(out.cpu()[torch.from_numpy(fine)], want[fine], err[fine])


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,window,dim", [([(4, 60), (1, 30)], 0, 128), ([(4, 60), (30, 90)], 9, 64),
                                             ([(200, 230)], 0, 128), ([(200, 230)], 30, 256)])
@pytest.mark.parametrize("key", [math.nan, 1e38, 20.0])
def test_attention_bad_keys_with_bad_values(gpu, seqs, window, dim, key):
    """A key and a value that are no numbers at one position, or a key far ahead of every other there: rows
    that do not see it are what they are without it."""
    heads, kv_heads = 4, 2
    b = Batch(seqs, kv_heads, dim, 16, 12)
    q = b.normal(b.tokens, heads, dim).abs()
    for s, (new, n) in enumerate(seqs):
        for p in (n - 1, n - 3, n - new // 2, n - 26):
            b.k[b.slot(s, p)] = key
            b.v[b.slot(s, p)] = math.nan
    scale = 1 / math.sqrt(dim)
    check_attend(b, attend(gpu, b, q, scale, window), q, scale, window)


@pytest.mark.gpu
def test_attention_scores_of_minus_infinity(gpu):
    """A score of -inf weighs nothing; a row of none but those gives zeros, as one that sees nothing."""
    b = Batch([(1, 40), (70, 90), (1, 30)], 2, 64, 16, 13)
    q = b.normal(b.tokens, 4, 64)
    q[:, :, 5] = 1.0
    for s, p in [(0, 3), (0, 39), (1, 20), (1, 60), (1, 89)] + [(2, p) for p in range(30)]:
        b.k[b.slot(s, p)] = 0
        b.k[b.slot(s, p) + (slice(None), 5)] = -math.inf
    out = attend(gpu, b, q, 0.125)
    check_attend(b, out, q, 0.125, 0)
    assert (out[-1] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-30, 1.0, 3e4])
def test_attention_extreme_scores(gpu, size):
    """Scores far apart (one key takes it all), tiny, and a large scale."""
    import torch
    b = Batch([(1, 200), (70, 70)], 2, 128, 16, 17)
    q = (b.normal(b.tokens, 4, 128).float() * size).bfloat16()
    if size > 1:  # one key ahead of the others by more than any rounding of the scores
        for s, n in ((0, 200), (1, 70)):
            for p in range(n):
                b.k[b.slot(s, p)] = (torch.ones(2, 128) * (1.0 if p == 0 else -1.0)).bfloat16()
        q = q.abs()
    for scale in (1 / math.sqrt(128), 4.0):
        if size == 1.0 and scale == 4.0:
            continue  # sums of many near-equal large scores: the bound is of no use
        check_attend(b, attend(gpu, b, q, scale), q, scale, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("count,max_q", [(130, 1), (130, 40), (5000, 1)])
def test_many_sequences(gpu, count, max_q):
    """More sequences than lanes, most of them short, some without rows, some with many."""
    rng = np.random.default_rng(count)
    seqs = [(int(n), int(n + k)) for n, k in zip(rng.integers(0, 2 if count > 1000 else 3, count), rng.integers(0, 6, count))]
    if max_q > 1:
        seqs[70], seqs[129], seqs[0] = (40, 90), (33, 33), (0, 0)
    b = Batch(seqs, 1, 64, 4, 31, lead=3, trail=1)
    rows = b.normal(b.tokens, 4, 64)
    q_out, (kc, vc) = rows[:, :2].contiguous().cuda(), b.pools()
    inv_freq, scale = gpu.rope_frequencies(64, 1e4)
    gpu.qk_norm_rope_paged(q_out, q_out, rows[:, 2:3].cuda(), rows[:, 3:].cuda(), None, None, inv_freq.cuda(), kc, vc,
                           *b.where(), 1e-6, scale)
    b.k, b.v, q = kc.cpu(), vc.cpu(), q_out.cpu()
    for t, s, p in b.rows():
        close(q[t], *rotated(rows[t, :2], None, p, inv_freq.numpy(), 1.0, False, 0))
        close(b.k[b.slot(s, p)], *rotated(rows[t, 2:3], None, p, inv_freq.numpy(), 1.0, False, 0))
        assert np.array_equal(bits(b.v[b.slot(s, p)]), bits(rows[t, 3:]))
    check_attend(b, attend(gpu, b, q, 0.2, 0, max_q, 90, pools=(kc, vc)), q, 0.2, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 5)])
def test_lengths_past_the_table(gpu, dim, page):
    """Tokens past the end of the table's row, by a little or as far as numbers go, are neither written nor seen;
    lengths below nothing see nothing."""
    import torch
    b = Batch([(2, 60), (1, 33), (70, 100), (1, 5), (3, 40)], 2, dim, page, 37)
    keep = 40 // page
    b.table = b.table[:, :keep].contiguous()
    b.seqs[1], b.seqs[3] = (1, 1 << 30), (1, -(1 << 30))
    b.kv_len = torch.tensor([60, 2 ** 31 - 1, 100, -2 ** 31, 40], dtype=torch.int32)
    q, k, v = b.normal(b.tokens, 4, dim), b.normal(b.tokens, 2, dim), b.normal(b.tokens, 2, dim)
    kc, vc = b.pools()
    gpu.qk_norm_rope_paged(torch.empty_like(q, device="cuda"), q.cuda(), k.cuda(), v.cuda(), None, None,
                           gpu.rope_frequencies(dim, 1e4)[0].cuda(), kc, vc, *b.where(), 1e-6)
    written = torch.zeros(b.pages, page, dtype=torch.bool)
    for t, s, p in b.rows():
        if b.slot(s, p):
            written[b.slot(s, p)] = True
    assert written.any()
    got_k, got_v = kc.cpu(), vc.cpu()
    assert torch.equal(bits(got_k[~written]), bits(b.k[~written])) and torch.equal(bits(got_v[~written]), bits(b.v[~written]))
    # what every row sees lies in the table's keep * page positions, whatever its own
    b.k, b.v = got_k, got_v
    far = Batch.rows
    b.rows = lambda: ((t, s, min(p, keep * page - 1)) for t, s, p in far(b))
    check_attend(b, attend(gpu, b, q, 0.1, 0, 70, 100, pools=(kc, vc)), q, 0.1, 0)


@pytest.mark.gpu
def test_attention_pools_past_32_bits(gpu):
    """Pages past 2^31 elements and 2^32 bytes of the pool, written and read."""
    import torch
    kv_heads, dim, page = 8, 128, 64
    b = Batch([(1, 200), (90, 120)], kv_heads, dim, page, 19)
    pages = (1 << 31) // (page * kv_heads * dim) + 40
    far = torch.arange(b.pages, dtype=torch.int32) + (pages - b.pages)
    kc, vc = (torch.empty(pages, page, kv_heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kc[far[0]:], vc[far[0]:] = b.k.cuda(), b.v.cuda()
    q, k, v = b.normal(b.tokens, 16, dim), b.normal(b.tokens, kv_heads, dim), b.normal(b.tokens, kv_heads, dim)
    inv_freq, scale = gpu.rope_frequencies(dim, 1e6)
    table = torch.where(b.table >= 0, b.table + int(far[0]), b.table).cuda()
    q_out = torch.empty_like(q, device="cuda")
    gpu.qk_norm_rope_paged(q_out, q.cuda(), k.cuda(), v.cuda(), None, None, inv_freq.cuda(), kc, vc, table,
                           b.q_start.cuda(), b.kv_len.cuda(), 1e-6)
    b.k, b.v = kc[far[0]:].cpu(), vc[far[0]:].cpu()
    for t, s, p in b.rows():
        close(b.k[b.slot(s, p)], *rotated(k[t], None, p, inv_freq.numpy(), 1.0, False, 0))
        assert torch.equal(bits(b.v[b.slot(s, p)]), bits(v[t]))
    out = torch.full((b.tokens, 16, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    ws = workspace(gpu, b, 16, 90, 200)
    gpu.attention_paged_forward(out, q_out, kc, vc, table, b.q_start.cuda(), b.kv_len.cuda(), ws, 0.09, 90, 200)
    check_attend(b, out, q_out.cpu(), 0.09, 0)


@pytest.mark.gpu
def test_attention_strided_rows(gpu):
    """q from one projection's rows, out into a wider buffer's rows, whose rest stays."""
    import torch
    b = Batch([(3, 50), (40, 70)], 2, 64, 16, 23, trail=1)
    q = b.normal(b.tokens, 4, 64)
    rows = torch.zeros(b.tokens, 8, 64, dtype=torch.bfloat16, device="cuda")
    rows[:, :4] = q.cuda()
    wide = torch.full((b.tokens, 6, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    kc, vc = b.pools()
    gpu.attention_paged_forward(wide[:, :4], rows[:, :4], kc, vc, *b.where(), workspace(gpu, b, 4, 40, 70), 0.125, 40, 70)
    check_attend(b, wide[:, :4].contiguous(), q, 0.125, 0)
    assert (wide[:, 4:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads,dim,new,past,window", [(3, 64, 1456, 0, 0), (3, 128, 1450, 30, 60), (5, 256, 840, 3, 0)])
def test_attention_of_more_workgroups_than_the_device_has_cus(gpu, kv_heads, dim, new, past, window):
    """Whole tiles without splits, more of them than CUs but not twice as many, an odd number: every row of every
    tile, against 64 bits a kv head at a time."""
    import torch
    group, page, n = 8, 16, new + past
    units = -(-new * group // 128) * kv_heads
    assert 256 < units < 512 and units % 2
    scale = 1 / math.sqrt(dim)
    g = torch.Generator().manual_seed(dim)

    def normal(*shape):
        return torch.randn(*shape, generator=g).bfloat16()

    pages = -(-n // page)
    q, k, v = normal(new, kv_heads * group, dim), normal(pages, page, kv_heads, dim), normal(pages, page, kv_heads, dim)
    table = torch.randperm(pages, generator=g).int()[None]
    where = [t.cuda() for t in (table, torch.tensor([0, new], dtype=torch.int32), torch.tensor([n], dtype=torch.int32))]
    floats = gpu.attention_paged_workspace_floats(new, 1, kv_heads * group, kv_heads, dim, new, n)
    out = torch.zeros(new, kv_heads * group, dim, dtype=torch.bfloat16, device="cuda")
    gpu.attention_paged_forward(out, q.cuda(), k.cuda(), v.cuda(), *where, torch.empty(max(floats, 1), device="cuda"),
                                scale, new, n, window=window)
    got = out.cpu()
    at, key = np.arange(past, n)[:, None], np.arange(n)[None]
    hidden = (key > at) | ((key <= at - window) if window else False)
    for h in range(kv_heads):
        kk, vv = (x[table[0].long(), :, h].reshape(-1, dim)[:n].double().numpy() for x in (k, v))
        for j in range(h * group, (h + 1) * group):
            qq = q[:, j].double().numpy()
            score = np.where(hidden, -np.inf, qq @ kk.T * scale)
            off = 2 * (dim * F32 * (np.abs(qq) @ np.abs(kk).T).max(-1) * scale
                       + 8 * F32 * np.abs(np.where(hidden, 0, score)).max(-1))[:, None]
            w = np.exp(score - score.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            close(got[:, j], w @ vv, (HALF_STEP + off + (n + 64) * F32) * (w @ np.abs(vv)))


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,window,dim,page", [([(1, 261)], 0, 128, 16), ([(1, 40), (4, 300), (1, 900)], 0, 64, 16),
                                                  ([(1, 3000), (1, 10)], 0, 256, 16), ([(2, 700), (3, 90)], 64, 128, 7)])
def test_few_rows_keep_what_their_weights_rounding_leaves(gpu, seqs, window, dim, page):
    """A call whose sequences all have few rows: each weight is a bf16 and a bf16 of the rest, off by half a
    step of half a step at most, so the bound has 2^-16 where that of many rows has 2^-8."""
    b = Batch(seqs, 2, dim, page, 53)
    q, scale = b.normal(b.tokens, 8, dim), 1 / math.sqrt(dim)
    out = attend(gpu, b, q, scale, window)
    want, err = attended(b, q, scale, window)
    b.v = b.v.abs()
    close(out.cpu(), want, err - (HALF_STEP - HALF_STEP ** 2) * attended(b, q, scale, window)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_calls_stay_within_the_workspace_of_their_sizes(gpu, dim):
    """What lies behind the floats that each of several calls asks for is left as it is."""
    import torch
    heads, kv_heads = 8, 2
    for seqs in ([(1, 9000)], [(40, 3000)], [(200, 5000)], [(1, 3000), (3, 900), (1, 1)], [(60, 2000), (1, 4000), (2, 10)],
                 [(600, 2500), (33, 900)]):
        b = Batch([(0, 0)], kv_heads, dim, 64, 59)
        n = [-(-have // 64) for _, have in seqs]
        b.table = torch.arange(sum(n)).int()[None].expand(len(seqs), -1).contiguous()  # a pool that all share
        k, v = (torch.randn(sum(n), 64, kv_heads, dim, device="cuda").bfloat16() for _ in range(2))
        starts = [sum(new for new, _ in seqs[:s]) for s in range(len(seqs) + 1)]
        where = [t.cuda() for t in (b.table, torch.tensor(starts).int(), torch.tensor([have for _, have in seqs]).int())]
        q = torch.randn(starts[-1], heads, dim, device="cuda").bfloat16()
        max_q, max_kv = max(new for new, _ in seqs), max(have for _, have in seqs)
        for q_told, kv_told in ((max_q, max_kv), (1, max_kv), (max_q, 700), (2 * max_q, 40960)):
            need = gpu.attention_paged_workspace_floats(starts[-1], len(seqs), heads, kv_heads, dim, q_told, kv_told)
            ws = torch.full((need + (1 << 20),), 7.0, device="cuda")
            gpu.attention_paged_forward(torch.empty_like(q), q, k, v, *where, ws[:need], 0.1, q_told, kv_told)
            assert (ws[need:] == 7).all()


# ---------------------------------------------------------------- together

@pytest.mark.gpu
def test_serving_loop_with_captured_steps(gpu):
    """Two prompts (one in two chunks), then tokens: rows into pages, attention over them, penalties and
    the pick. The whole against 64 bits; the token steps once eagerly and once as one captured graph that
    is replayed as lengths grow, with other work between, equal to the eager ones bit for bit."""
    import torch
    heads, kv_heads, dim, page, vocab, steps = 8, 2, 128, 16, 1003, 5
    rng = torch.Generator().manual_seed(3)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=rng) * std).bfloat16()

    prompts, pages = [70, 21], 14
    table = torch.randperm(pages, generator=rng).int().view(2, 7)
    inv_freq, scale_r = gpu.rope_frequencies(dim, 1e6, gpu.ROPE_YARN, 4.0, 64)
    qn, kn = normal(dim, std=0.1) + 1, normal(dim, std=0.1) + 1
    head = normal(vocab, heads * dim, std=0.05).cuda()
    total = [p + steps for p in prompts]
    rows = [[normal(n, h, dim) for n in total] for h in (heads, kv_heads, kv_heads)]

    def run(captured):
        kc, vc = (torch.zeros(pages, page, kv_heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        history = torch.zeros(2, 16, dtype=torch.int32, device="cuda")
        lens = torch.zeros(2, dtype=torch.int32, device="cuda")
        prompt_len = torch.ones(2, dtype=torch.int32, device="cuda")
        rep, freq = torch.full((2,), 1.3, device="cuda"), torch.full((2,), 0.4, device="cuda")
        d = [qn.cuda(), kn.cuda(), inv_freq.cuda()]
        outs, picks, all_logits, turned = [], [], [], []

        def layer(q, k, v, where, out, ws, max_q):
            gpu.qk_norm_rope_paged(q, q, k, v, *d, kc, vc, *where, 1e-6, scale_r)
            gpu.attention_paged_forward(out, q, kc, vc, *where, ws, 0.09, max_q, 112)

        # chunks: 40 + 0 rows, then 30 + 21
        for spans in [((0, 40), (0, 0)), ((40, 70), (0, 21))]:
            q, k, v = (torch.cat([rows[i][s][a:e] for s, (a, e) in enumerate(spans)]).cuda() for i in range(3))
            n = [e - a for a, e in spans]
            where = (table.cuda(), torch.tensor([0, n[0], n[0] + n[1]], dtype=torch.int32).cuda(),
                     torch.tensor([e for _, e in spans], dtype=torch.int32).cuda())
            ws = torch.empty(max(1, gpu.attention_paged_workspace_floats(sum(n), 2, heads, kv_heads, dim, 40, 112)), device="cuda")
            out = torch.empty_like(q)
            layer(q, k, v, where, out, ws, 40)
            outs.append(out.cpu())
            turned.append(q.cpu())
        # token steps: fixed buffers
        q, k, v = (torch.empty(2, h, dim, dtype=torch.bfloat16, device="cuda") for h in (heads, kv_heads, kv_heads))
        where = (table.cuda(), torch.arange(3, dtype=torch.int32).cuda(), torch.tensor(prompts, dtype=torch.int32).cuda())
        ws = torch.empty(max(1, gpu.attention_paged_workspace_floats(2, 2, heads, kv_heads, dim, 1, 112)), device="cuda")
        out = torch.empty_like(q)
        logits, raw = (torch.empty(2, vocab, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        pick = torch.zeros(2, dtype=torch.int32, device="cuda")

        def step():
            layer(q, k, v, where, out, ws, 1)
            for s in range(2):
                gpu.gemv_forward(raw[s], head, out[s], vocab, heads * dim)
            gpu.logits_penalty_forward(logits, raw, history, prompt_len, lens, rep, freq)
            for s in range(2):
                gpu.argmax_forward(pick[s:s + 1], logits[s], vocab)

        graph = None
        for i in range(steps):
            for buffer, source in ((q, rows[0]), (k, rows[1]), (v, rows[2])):
                buffer.copy_(torch.stack([source[s][prompts[s] + i] for s in range(2)]))
            where[2].add_(1)
            if captured and graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    step()
            if graph:
                graph.replay()
            else:
                step()
            torch.cuda.synchronize()
            outs.append(out.cpu())
            turned.append(q.cpu())
            all_logits.append((raw.cpu(), logits.cpu()))
            picks.append(pick.cpu())
            history[:, i] = pick
            lens.add_(1)
        return outs, turned, picks, all_logits, kc.cpu(), vc.cpu()

    eager, again = run(False), run(True)
    for x, y in zip(eager, again):
        for a, c in zip(*((z,) if torch.is_tensor(z) else (z,) for z in (x, y))):
            pairs = zip(a, c) if isinstance(a, (list, tuple)) else [(a, c)]
            for m, n in pairs:
                m, n = (m, n) if isinstance(m, tuple) else ((m,), (n,))
                assert all(torch.equal(u.view(torch.int16) if u.dtype == torch.bfloat16 else u,
                                       w.view(torch.int16) if w.dtype == torch.bfloat16 else w) for u, w in zip(m, n))
    outs, turned, picks, all_logits, kc, vc = eager

    # the attention of every row against 64 bits, over the caches that the loop wrote
    b = Batch([(total[s], total[s]) for s in range(2)], kv_heads, dim, page, 1)
    b.table, b.table_pages, b.pages, b.k, b.v = table, 7, pages, kc, vc

    def in_order(x):  # rows of the chunks and steps by sequence and position
        return torch.cat([x[0], x[1][:30]] + [o[:1] for o in x[2:]] + [x[1][30:]] + [o[1:] for o in x[2:]])

    q = in_order(turned)
    for t, s, p in b.rows():
        close(q[t], *rotated(rows[0][s][p], qn, p, inv_freq.numpy(), scale_r, False, 1e-6))
        close(kc[b.slot(s, p)], *rotated(rows[1][s][p], kn, p, inv_freq.numpy(), scale_r, False, 1e-6))
    close(in_order(outs), *attended(b, q, 0.09, 0))

    # the picks: penalties by their definition on the loop's own logits, the lowest index of the largest
    for i, (raw, logits) in enumerate(all_logits):
        for s in range(2):
            x = raw[s].double()
            before = [int(picks[j][s]) for j in range(i)]
            for t in set(before):
                x[t] = x[t] / float(np.float32(1.3)) if x[t] > 0 else x[t] * float(np.float32(1.3))
                n = before[1:].count(t)
                x[t] -= float(np.float32(0.4)) * n
            close(logits[s], x.numpy(), 8 * F32 * (np.abs(x.numpy()) + 4))
            assert int(picks[i][s]) == int(torch.nonzero(logits[s] == logits[s].max())[0])


@pytest.mark.gpu
def test_two_captured_graphs_and_streams(gpu):
    """Two graphs with a workspace each, replayed at once on two streams, with eager work on a third; every
    replay equal to the eager result."""
    import torch
    made = []
    for seed, seqs, heads in ((1, [(1, 3000), (1, 40)], 8), (2, [(1, 700), (60, 900)], 4)):
        b = Batch(seqs, 2, 128, 16, seed)
        q = b.normal(b.tokens, heads, 128).cuda()
        max_q, max_kv = max(n for n, _ in seqs), max(n for _, n in seqs)
        ws, out, pools, where = workspace(gpu, b, heads, max_q, max_kv), torch.zeros_like(q), b.pools(), b.where()
        args = (q, *pools, *where, ws, 0.09, max_q, max_kv)
        gpu.attention_paged_forward(out, *args)
        want = out.clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gpu.attention_paged_forward(out, *args)
        made.append((graph, out, want, args))
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(4):
        torch.cuda.synchronize()
        for (graph, out, _, _), stream in zip(made, streams):
            with torch.cuda.stream(stream):
                out.zero_()
                graph.replay()
        torch.randn(1000, 1000, device="cuda").sum()
        torch.cuda.synchronize()
        for _, out, want, args in made:
            assert torch.equal(bits(out), bits(want))
            out.fill_(3)
            torch.cuda.synchronize()
            gpu.attention_paged_forward(out, *args, stream=streams[0])
            torch.cuda.synchronize()
            assert torch.equal(bits(out), bits(want))


# ---------------------------------------------------------------- refusals

def record(pkg, **change):
    base = dict(key_cache=0x1000, value_cache=0x1000, page_stride=2048, slot_stride=128, head_stride=64,
                page_table=0x1000, q_start=0x1000, kv_len=0x1000, n_seqs=2, n_pages=4, page_size=16,
                table_pages=3, n_kv_heads=2, head_dim=64)
    base.update(change)
    return pkg.PagedBatch(**base)


BATCHES = [
    (dict(head_dim=96), "head_dim 96"), (dict(n_kv_heads=0), "n_kv_heads 0"), (dict(n_kv_heads=3), "multiple of n_kv_heads 3"),
    (dict(n_seqs=0), "n_seqs 0"), (dict(n_pages=-1), "n_pages -1"), (dict(page_size=0), "page_size 0"),
    (dict(table_pages=0), "table_pages 0"), (dict(key_cache=None), "null"), (dict(kv_len=None), "null"),
    (dict(value_cache=0x1002), "16-byte aligned"), (dict(slot_stride=100), "multiples of 8"),
    (dict(page_size=(1 << 20) + 1), "over 1048576"), (dict(n_seqs=(1 << 20) + 1), "n_seqs 1048577"),
    (dict(page_stride=-2048), "may be negative"), (dict(slot_stride=(1 << 26) + 8), "over 2^26"),
    (dict(slot_stride=56), "overlap"),
]


def refused(pkg, fn, *args):
    L = pkg.lib()
    L.llm_clear_error()
    getattr(L, fn)(*args)
    message = L.llm_last_error()
    L.llm_clear_error()
    return message.decode() if message else ""


@pytest.mark.parametrize("change,message", BATCHES)
def test_batches_that_are_refused(pkg, change, message):
    b = ctypes.byref(record(pkg, **change))
    p = 0x1000
    assert message in refused(pkg, "qk_norm_rope_paged", p, p, p, p, None, None, p, b, 4, 4, 64, 0, 1e-6, 1.0,
                              256, 256, 128, 128, None)
    assert message in refused(pkg, "attention_paged_forward", p, p, b, p, 4, 4, 1, 100, 0, 0.1, 256, 256, None)


@pytest.mark.parametrize("at,value,message", [
    (0, None, "q_out is null"), (2, 0x1008, "k must be 16-byte aligned"), (4, 0x1002, "norm weights"),
    (6, None, "inv_freq"), (6, 0x1004, "inv_freq"), (7, None, "no batch"), (8, -1, "n_tokens -1"),
    (9, 0, "n_heads 0"), (10, 24, "rotary_dim 24"), (10, 0, "rotary_dim 0"), (10, 80, "rotary_dim 80"),
    (14, 248, "rows of q_out"), (15, 260, "rows of q "), (16, 64, "rows of k"), (17, 0, "rows of v")])
def test_append_refusals(pkg, at, value, message):
    p, b = 0x1000, record(pkg)
    args = [p, p, p, p, None, None, p, ctypes.byref(b), 4, 4, 64, 0, 1e-6, 1.0, 256, 256, 128, 128, None]
    args[at] = value
    assert message in refused(pkg, "qk_norm_rope_paged", *args)


@pytest.mark.parametrize("at,value,message", [
    (0, None, "out is null"), (1, 0x1004, "q must be 16-byte aligned"), (2, None, "no batch"), (3, 0x1004, "ws must be"),
    (4, 1 << 25, "n_tokens"), (5, 5, "multiple of n_kv_heads"), (6, 0, "max_q_len 0"), (7, -4, "max_kv_len -4"),
    (8, -1, "window -1"), (9, 0.0, "scale 0"), (9, -1.0, "scale -1"), (9, math.nan, "scale nan"), (9, math.inf, "scale inf"),
    (10, 128, "rows of out"), (11, 257, "rows of q")])
def test_attention_refusals(pkg, at, value, message):
    p, b = 0x1000, record(pkg)
    args = [p, p, ctypes.byref(b), p, 4, 4, 1, 100, 0, 0.1, 256, 256, None]
    args[at] = value
    assert message in refused(pkg, "attention_paged_forward", *args)


def test_append_where_it_would_write_over_itself(pkg):
    p = 0x1000
    for change in (dict(head_stride=56), dict(head_stride=0), dict(page_stride=0)):
        assert "overlap" in refused(pkg, "qk_norm_rope_paged", p, p, p, p, None, None, p, ctypes.byref(record(pkg, **change)),
                                    4, 4, 64, 0, 1e-6, 1.0, 256, 256, 128, 128, None)
    assert "in place" in refused(pkg, "qk_norm_rope_paged", p, p, p, p, None, None, p, ctypes.byref(record(pkg)),
                                 4, 4, 64, 0, 1e-6, 1.0, 264, 256, 128, 128, None)


def test_attention_in_place_and_overflowing_scales_are_refused(pkg):
    p, b = 0x1000, ctypes.byref(record(pkg))
    assert "out must not be q" in refused(pkg, "attention_paged_forward", p, p, b, p, 4, 4, 1, 100, 0, 0.1, 256, 256, None)
    assert "not positive and finite" in refused(pkg, "attention_paged_forward", 0x9000, p, b, p, 4, 4, 1, 100, 0, 3e38, 256, 256, None)


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (16, 8, 128), (16, 4, 256), (24, 4, 64), (40, 1, 64),
                                                (7, 7, 128), (600, 300, 64)])
def test_workspace_of_the_largest_call_serves_smaller_ones(pkg, heads, kv_heads, dim):
    """The count does not fall as a size grows, nor does it grow without end."""
    def floats(*sizes):
        n_tokens, n_seqs, max_q, max_kv = sizes
        return pkg.attention_paged_workspace_floats(n_tokens, n_seqs, heads, kv_heads, dim, max_q, max_kv)

    assert floats(2048, 1, 2048, 8192) >= floats(512, 1, 512, 8192) > 0
    rng = np.random.default_rng(heads)
    most = [65536, 4096, 65536, 1 << 20]
    for _ in range(3000):
        large = [int(math.exp(rng.uniform(0, math.log(n + 1)))) for n in most]
        small = [int(rng.integers(1, n + 1)) if rng.random() < 0.6 else n for n in large]
        assert floats(*small) <= floats(*large), (small, large)
    for i in range(4):  # one size by one, the others in the middle
        sizes = [600, 20, 300, 9000]
        counts = []
        for n in list(range(1, 700)) + [1000, 2000, 4096]:
            sizes[i] = n
            counts.append(floats(*sizes))
        assert counts == sorted(counts)
    assert floats(*most) <= (4096 * 32 + 2048 * 128) * (dim + 2)


def test_more_workgroups_than_a_launch_has_are_refused(pkg):
    """On the host, by the library's own message: 2^24 workgroups of 256 threads and more."""
    p, n = 0x1000, 1 << 20
    for kv_heads in (16, 17, 31):
        b = ctypes.byref(record(pkg, n_seqs=n, n_kv_heads=kv_heads, slot_stride=64 * kv_heads, page_stride=1024 * kv_heads))
        assert "too many for one launch" in refused(pkg, "attention_paged_forward", 0x9000, p, b, p, n, kv_heads, 1, 100, 0,
                                                    0.1, 64 * kv_heads, 64 * kv_heads, None)


def test_no_rows_is_no_launch(pkg):
    p, b = 0x1000, record(pkg)
    assert refused(pkg, "qk_norm_rope_paged", p, p, p, p, None, None, p, ctypes.byref(b), 0, 4, 64, 0, 1e-6, 1.0,
                   256, 256, 128, 128, None) == ""
    assert refused(pkg, "attention_paged_forward", p, p, ctypes.byref(b), p, 0, 4, 1, 100, 0, 0.1, 256, 256, None) == ""


@pytest.mark.gpu
def test_wrapper_refusals(gpu):
    import torch
    b = Batch([(2, 20), (1, 5)], 2, 64, 16, 1)
    kc, vc = b.pools()
    q, k, v = (b.normal(3, h, 64).cuda() for h in (4, 2, 2))
    where, f = b.where(), gpu.rope_frequencies(64, 1e4)[0].cuda()
    good = dict(q_out=torch.empty_like(q), q=q, k=k, v=v, q_norm_w=None, k_norm_w=None, inv_freq=f, key_cache=kc,
                value_cache=vc, page_table=where[0], q_start=where[1], kv_len=where[2], eps=1e-6)
    gpu.qk_norm_rope_paged(**good)
    for change, message in [
            (dict(q=q.cpu()), "q must be a tensor on the GPU"), (dict(k=k.float()), "k must be torch.bfloat16"),
            (dict(v=v[:2]), "v must have shape"), (dict(q_out=q.transpose(0, 1).contiguous().transpose(0, 1)), "q_out must be contiguous"),
            (dict(key_cache=kc[:2]), "same shape and strides"), (dict(page_table=where[0].long()), "page_table must be torch.int32"),
            (dict(q_start=where[1][:2]), "q_start must be contiguous of shape"), (dict(kv_len=where[2][:1]), "kv_len must be"),
            (dict(inv_freq=f.float()), "inv_freq must be torch.float64"), (dict(inv_freq=f[:3].contiguous()), "rotary_dim 6"),
            (dict(q_norm_w=torch.ones(32, device="cuda", dtype=torch.bfloat16)), "q_norm_w must be")]:
        with pytest.raises(gpu.LlmError, match=message):
            gpu.qk_norm_rope_paged(**dict(good, **change))
    need = gpu.attention_paged_workspace_floats(3, 2, 4, 2, 64, 2, 100000)
    good = dict(out=torch.empty_like(q), q=q, key_cache=kc, value_cache=vc, page_table=where[0], q_start=where[1],
                kv_len=where[2], ws=torch.empty(max(need, 1), device="cuda"), scale=0.1, max_q_len=2, max_kv_len=100000)
    gpu.attention_paged_forward(**good)
    for change, message in [
            (dict(out=q.float()), "out must be torch.bfloat16"), (dict(q=q[:, :3]), "out must have shape|n_heads 3"),
            (dict(ws=good["ws"].half()), "ws must be torch.float32"), (dict(scale=0.0), "scale"), (dict(window=-1), "window"),
            (dict(max_kv_len=0), "max_kv_len")]:
        with pytest.raises(gpu.LlmError, match=message):
            gpu.attention_paged_forward(**dict(good, **change))
    if need:
        with pytest.raises(gpu.LlmError, match=f"ws holds {need - 1} floats"):
            gpu.attention_paged_forward(**dict(good, ws=good["ws"][:need - 1]))
        with pytest.raises(gpu.LlmError, match="ws holds 0 floats"):
            gpu.attention_paged_forward(**dict(good, ws=None))
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_wrappers_name_what_is_no_tensor(gpu):
    """What is no tensor is refused by the library's own error, whatever else it is."""
    import torch
    b = Batch([(2, 20), (1, 5)], 2, 64, 16, 1)
    kc, vc = b.pools()
    q, k, v = (b.normal(3, h, 64).cuda() for h in (4, 2, 2))
    where, f = b.where(), gpu.rope_frequencies(64, 1e4)[0].cuda()
    append = dict(q_out=torch.empty_like(q), q=q, k=k, v=v, q_norm_w=None, k_norm_w=None, inv_freq=f, key_cache=kc,
                  value_cache=vc, page_table=where[0], q_start=where[1], kv_len=where[2], eps=1e-6)
    attend = dict(out=torch.empty_like(q), q=q, key_cache=kc, value_cache=vc, page_table=where[0], q_start=where[1],
                  kv_len=where[2], ws=workspace(gpu, b, 4, 2, 9000), scale=0.1, max_q_len=2, max_kv_len=9000)
    ids, n = torch.zeros(2, 5, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    x = torch.zeros(2, 100, dtype=torch.bfloat16, device="cuda")
    penalty = dict(out=x, logits=x, tokens=ids, token_len=n, bias_tokens=ids, bias=ids.float(), allowed=ids)
    for call, good, names, none in (
            (gpu.qk_norm_rope_paged, append, ["q_out", "q", "k", "v", "inv_freq", "key_cache", "value_cache", "page_table",
                                              "q_start", "kv_len", "q_norm_w"], True),
            (gpu.attention_paged_forward, attend, ["out", "q", "key_cache", "value_cache", "page_table", "q_start", "kv_len",
                                                   "ws"], True),
            (gpu.logits_penalty_forward, penalty, ["out", "logits"], True),
            (gpu.logits_penalty_forward, penalty, ["tokens", "token_len", "bias_tokens", "bias", "allowed"], False)):
        for name in names:
            for value in [[1, 2], 7] + ([None] if none and name != "q_norm_w" else []):
                with pytest.raises(gpu.LlmError):
                    call(**dict(good, **{name: value}))
    with pytest.raises(gpu.LlmError, match="page_table must be a tensor on the GPU"):
        gpu.attention_paged_forward(**dict(attend, page_table=None))
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_an_error_from_before_is_reported(gpu, monkeypatch, native):
    """An error that an earlier call of the library left is reported by the next call, once."""
    import torch
    if not native:
        monkeypatch.setattr(gpu, "_native", None)
    b = Batch([(1, 20)], 2, 64, 16, 1)
    q, (kc, vc), where = b.normal(1, 4, 64).cuda(), b.pools(), b.where()
    out, x = torch.empty_like(q), torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda")
    f, k = gpu.rope_frequencies(64, 1e4)[0].cuda(), q[:, :2]
    for call in (lambda: gpu.attention_paged_forward(out, q, kc, vc, *where, None, 0.1, 1, 20),
                 lambda: gpu.qk_norm_rope_paged(out, q, k, k, None, None, f, kc, vc, *where, 1e-6),
                 lambda: gpu.logits_penalty_forward(x, x)):
        gpu.lib().attention_paged_workspace_floats(1, 1, 4, 3, 64, 1, 20)  # no such heads
        with pytest.raises(gpu.LlmError, match="4 heads on 3"):
            call()
        call()
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_native_and_general_way_are_one(gpu, monkeypatch):
    """The native launchers and the general ctypes way: the same results from the same arguments, and the
    same refusals."""
    import torch
    b = Batch([(3, 50), (40, 70), (1, 9000)], 2, 64, 16, 29, layout="heads")
    rows = b.normal(b.tokens, 8, 64).cuda()
    norm, f = b.normal(64).cuda(), gpu.rope_frequencies(32, 1e4)[0].cuda()
    x = torch.randn(3, 1001, device="cuda").bfloat16()
    ids, n = torch.randint(0, 1001, (3, 40), device="cuda", dtype=torch.int32), torch.tensor([40, 3, 0], device="cuda", dtype=torch.int32)
    results = []
    for general in (False, True):
        with monkeypatch.context() as m:
            if general:
                m.setattr(gpu, "_native", None)
            kc, vc = b.pools()
            q_out = torch.zeros(b.tokens, 4, 64, device="cuda", dtype=torch.int16)
            out, z = torch.zeros_like(q_out, dtype=torch.bfloat16), torch.zeros_like(x)
            ws = workspace(gpu, b, 4, 40, 9000)
            where, bias = b.where(), ids.float()  # kept until the other stream has read them
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            gpu.qk_norm_rope_paged(q_out, rows[:, :4], rows[:, 4:6], rows[:, 6:], norm, norm, f, kc, vc, *where, 1e-5,
                                   1.5, True, side)
            gpu.attention_paged_forward(out, q_out, kc, vc, *where, ws, 0.25, 40, 9000, window=60, stream=side.cuda_stream)
            gpu.logits_penalty_forward(z, x, ids, n, n, bias_tokens=ids, bias=bias, stream=side)
            torch.cuda.synchronize()
            refusals = []
            for call in (lambda: gpu.attention_paged_forward(out, q_out, kc, vc, *where, ws, 1, 40, 9000, -1),
                         lambda: gpu.attention_paged_forward(out, q_out, kc, vc, *where, None, 0.1, 40, 9000),
                         lambda: gpu.qk_norm_rope_paged(q_out, rows[:, :4], rows[:, 4:6], rows[:, 6:], None, None, f[:4], kc, vc, *where, 1e-5),
                         lambda: gpu.logits_penalty_forward(z, x[:, :1000], ids, n, n)):
                with pytest.raises(gpu.LlmError) as e:
                    call()
                refusals.append(str(e.value))
            results.append(([bits(t) for t in (q_out, out, z, kc, vc)], refusals))
    assert results[0][1] == results[1][1]
    assert all(torch.equal(a, c) for a, c in zip(results[0][0], results[1][0]))
