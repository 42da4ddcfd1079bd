"""GPU parity of the attention operators with their formulas in 64 bits (attention_reference.py
derives the bounds): packed prompts forward and backward, the paged cache and attention over it."""
import math

import numpy as np
import pytest

from futhark_amd import Kernels, heads

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import attention_reference as ref  # noqa: E402

DEV = "cuda"
MARK = 7.0  # what outputs hold before a call


@pytest.fixture(scope="module")
def K():
    return Kernels()


def view(x):
    return heads(x.data_ptr(), x.stride(0), x.stride(1))


def randn(gen, t, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(ref.DTYPE[t])


def generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def segments(lens, gaps):
    """(first, length) pairs with gaps[i] rows before segment i, and the rows in all (some behind
    the last)."""
    segs, at = [], 0
    for i, n in enumerate(lens):
        at += gaps[i % len(gaps)]
        segs.append((at, n))
        at += n
    return segs, at + gaps[0] + 3


def device_segments(segs):
    return (torch.tensor([s[0] for s in segs], dtype=torch.int64, device=DEV),
            torch.tensor([s[1] for s in segs], dtype=torch.int64, device=DEV))


def stream():
    return torch.cuda.current_stream().cuda_stream


class Problem:
    """One packed batch; layout "rows" is [rows][heads][dim], "heads" is [heads][rows][dim],
    "fused" has q, k and v as parts of one row."""

    def __init__(self, t, h, hk, dim, q_lens, k_lens=None, causal=True, layout="rows", gaps=(0,), seed=0,
                 spread=1.0):
        gen = generator(seed)
        self.t, self.h, self.hk, self.dim, self.causal = t, h, hk, dim, causal
        self.segs_q, self.nq = segments(q_lens, gaps)
        self.segs_k, self.nk = segments(q_lens if k_lens is None else k_lens, gaps)
        self.scale = 1 / math.sqrt(dim)

        def make(rows, n, scale=1.0):
            if layout == "heads":
                return randn(gen, t, n, rows, dim, scale=scale).transpose(0, 1)
            return randn(gen, t, rows, n, dim, scale=scale)

        if layout == "fused":
            x = randn(gen, t, self.nq, h + 2 * hk, dim, scale=spread)
            self.q, self.k, self.v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
        else:
            self.q, self.k, self.v = make(self.nq, h, spread), make(self.nk, hk, spread), make(self.nk, hk)
        self.dout = make(self.nq, h)
        self.out, self.dq, self.dk, self.dv = (torch.full_like(x, MARK) for x in (self.q, self.q, self.k, self.v))
        self.lse = torch.full((self.nq, h), MARK, dtype=torch.float32, device=DEV)
        self.qo, self.ql = device_segments(self.segs_q)
        self.ko, self.kl = device_segments(self.segs_k)
        self.failure = torch.zeros(1, dtype=torch.int32, device=DEV)

    def args(self):
        return (self.t, view(self.q), self.nq, view(self.k), view(self.v), self.nk, self.h, self.hk, self.dim,
                self.qo.data_ptr(), self.ql.data_ptr(), self.ko.data_ptr(), self.kl.data_ptr(), len(self.segs_q),
                self.scale, int(self.causal), view(self.out))

    def forward(self, K, lse=True):
        K.attention(stream(), *self.args(), self.lse.data_ptr() if lse else None, self.failure.data_ptr(), 5)

    def backward(self, K):
        size = K.attention_grad_workspace_bytes(self.nq, self.nk, self.h, self.hk, self.dim, len(self.segs_q))
        self.workspace = torch.full((max(size, 1),), 0xff, dtype=torch.uint8, device=DEV)
        K.attention_grad(stream(), *self.args(), self.lse.data_ptr(), view(self.dout), view(self.dq), view(self.dk),
                         view(self.dv), self.workspace.data_ptr(), size, self.failure.data_ptr(), 5)

    def check_forward(self, lse=True):
        out, l, tol_o, tol_l = ref.forward(self.t, self.q, self.k, self.v, self.segs_q, self.segs_k, self.scale,
                                           self.causal)
        outside = out.isnan()
        assert bool((self.out[outside] == MARK).all()), "rows in no segment were written"
        ref.within(self.out, out, tol_o)
        if lse:
            assert bool((self.lse[l.isnan()] == MARK).all())
            ref.within(self.lse, l, tol_l)
        assert self.failure.item() == 0

    def check_backward(self):
        grads, tols = ref.gradient(self.t, self.q, self.k, self.v, self.dout, self.segs_q, self.segs_k, self.scale,
                                   self.causal)
        for got, want, tol in zip((self.dq, self.dk, self.dv), grads, tols):
            assert bool((got[want.isnan()] == MARK).all()), "rows in no segment were written"
            ref.within(got, want, tol)
        assert self.failure.item() == 0


RAGGED = [1, 0, 2, 63, 64, 65, 31, 33, 127, 128, 129, 200, 0]
PROMPTS = [
    # type, heads, kv_heads, dim, q lengths, k lengths (None: the same), causal, layout, gaps
    ("bf16", 2, 1, 128, RAGGED, None, True, "rows", (0,)),
    ("f16", 2, 2, 64, RAGGED, None, True, "rows", (3, 0, 1)),
    ("f16", 3, 1, 128, RAGGED, None, False, "fused", (0, 2)),
    ("bf16", 4, 2, 64, RAGGED, None, False, "heads", (1,)),
    ("bf16", 1, 1, 8, [1], None, True, "rows", (0,)),
    ("f16", 1, 1, 8, [5, 70], None, False, "rows", (0,)),
    ("bf16", 5, 1, 72, [130, 17], None, True, "fused", (0,)),
    ("f16", 6, 2, 96, [257], None, True, "heads", (0,)),
    ("bf16", 16, 1, 120, [90, 3], None, True, "rows", (5,)),
    ("f16", 128, 1, 64, [7, 40], None, True, "rows", (0,)),
    ("bf16", 127, 1, 16, [70], None, True, "rows", (0,)),
    ("bf16", 8, 8, 128, [513, 1030], None, True, "rows", (0,)),
    ("f16", 8, 2, 64, [1537], None, True, "rows", (0,)),
    # rows with nothing to see, queries behind cached keys, keys nobody asks
    ("bf16", 2, 1, 128, [100, 70, 5, 9, 0, 130], [40, 0, 1, 200, 30, 129], True, "rows", (0,)),
    ("f16", 4, 1, 64, [100, 70, 5, 9, 0, 300], [40, 0, 1, 200, 30, 131], True, "rows", (2,)),
    ("bf16", 2, 2, 40, [3, 260], [700, 0], False, "rows", (0,)),
    ("f16", 6, 3, 128, [1, 1, 1], [1, 900, 64], True, "rows", (0,)),
]


@pytest.mark.parametrize("i", range(len(PROMPTS)))
def test_prompts_forward(K, i):
    p = Problem(*PROMPTS[i], seed=i)
    p.forward(K)
    p.check_forward()
    lse = p.lse.clone()
    p.out.fill_(MARK)
    p.lse.fill_(MARK)
    p.forward(K, lse=False)
    p.check_forward(lse=False)
    assert bool((p.lse == MARK).all()) and lse.shape == p.lse.shape


@pytest.mark.parametrize("i", range(len(PROMPTS)))
def test_prompts_backward(K, i):
    p = Problem(*PROMPTS[i], seed=100 + i)
    p.forward(K)
    p.backward(K)
    p.check_backward()


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_wide_scores(K, t, dim):
    """Scores spread over hundreds: weights of one, weights that vanish, maxima that move late."""
    p = Problem(t, 4, 2, dim, [300, 129], spread=6.0, seed=3)
    order = torch.arange(p.nk, device=DEV, dtype=torch.float32) / 100
    p.k.copy_((p.k.float() * order[:, None, None]).to(p.k.dtype))  # later keys have larger scores
    p.forward(K)
    p.check_forward()
    p.backward(K)
    p.check_backward()


def test_gradient_against_differences(K):
    """The derivative of sum(out * dout) along a direction, by central differences in 64 bits."""
    p = Problem("f16", 4, 2, 64, [70, 33], [90, 20], seed=9)
    p.forward(K)
    p.backward(K)
    gen = generator(10)
    grads, tols = ref.gradient(p.t, p.q, p.k, p.v, p.dout, p.segs_q, p.segs_k, p.scale, p.causal)
    for i, name in enumerate("qkv"):
        d = torch.randn(getattr(p, name).shape, generator=gen, device=DEV, dtype=torch.float64)

        def loss(step):
            x = {n: getattr(p, n).double() for n in "qkv"}
            x[name] = x[name] + step * d
            out = ref.forward(p.t, x["q"], x["k"], x["v"], p.segs_q, p.segs_k, p.scale, p.causal)[0]
            return float(torch.nansum(out * p.dout.double()))

        h = 1e-4  # third derivatives times h^2 stay below 1e-6 of the sum's terms
        slope = (loss(h) - loss(-h)) / (2 * h)
        got = (p.dq, p.dk, p.dv)[i].double()
        inside = ~grads[i].isnan()
        along = float((got * d)[inside].sum())
        tol = float((tols[i] * d.abs())[inside].sum()) * 0.2 + 1e-4
        # 0.2: errors of thousands of elements with random signs add like their root; a wrong
        # factor or sign moves the sum by far more
        assert abs(along - slope) <= tol, (name, along, slope, tol)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 65504.0])
def test_keys_that_are_not_seen_have_no_effect(K, causal, bad):
    """NaN and infinities in rows behind a sequence, between sequences and, under a causal mask, in
    the future of a row change nothing for that row."""
    lens = [37, 100, 129, 64]
    clean = Problem("f16", 4, 2, 64, lens, causal=causal, gaps=(2, 5), seed=21)
    dirty = Problem("f16", 4, 2, 64, lens, causal=causal, gaps=(2, 5), seed=21)
    inside = torch.zeros(clean.nk, dtype=torch.bool, device=DEV)
    for f, n in clean.segs_k:
        inside[f:f + n] = True
    dirty.k[~inside] = bad
    dirty.v[~inside] = bad
    clean.forward(K)
    dirty.forward(K)
    clean.check_forward()
    assert torch.equal(clean.out, dirty.out) and torch.equal(clean.lse, dirty.lse)
    if not causal:
        return
    for hole in (20, 36):  # token `hole` of every sequence long enough: rows before it are untouched
        for x in ("k", "v"):
            d = Problem("f16", 4, 2, 64, lens, causal=True, gaps=(2, 5), seed=21)
            for f, n in d.segs_k:
                getattr(d, x)[f + hole, :, 3] = bad
            d.forward(K)
            for f, n in d.segs_k:
                assert torch.equal(clean.out[f:f + hole], d.out[f:f + hole]), (hole, x)
                if bad != 65504.0 and x == "v":  # and rows from it on see it
                    assert not bool(d.out[f + hole:f + n, :, 3].isfinite().any())
                    rest = [c for c in range(64) if c != 3]
                    assert torch.equal(d.out[f + hole:f + n][..., rest], clean.out[f + hole:f + n][..., rest])


def test_broken_segments_are_reported_and_left_out(K):
    for which, seg, what in [("ql", 1, -1), ("ql", 2, 1 << 40), ("qo", 1, -5), ("qo", 2, 3), ("kl", 1, -7),
                             ("ko", 0, 1 << 62), ("kl", 2, 1 << 62), ("ko", 1, -(1 << 63)), ("ql", 0, (1 << 63) - 1)]:
        p = Problem("bf16", 2, 1, 64, [40, 50, 60], gaps=(1,), seed=30)
        getattr(p, which)[seg] = what
        p.forward(K)
        assert p.failure.item() == 5, (which, seg, what)
        f, n = p.segs_q[seg]
        assert bool((p.out[f:f + n] == MARK).all())
        p.failure.zero_()
        p.backward(K)
        assert p.failure.item() == 5, (which, seg, what)
        if seg > 0:  # the segment before the broken one has its values
            q = Problem("bf16", 2, 1, 64, [40, 50, 60], gaps=(1,), seed=30)
            q.forward(K)
            a, b = q.segs_q[0]
            assert torch.equal(q.out[a:a + b], p.out[a:a + b])


def test_without_a_failure_word_and_without_segments(K):
    p = Problem("bf16", 2, 1, 64, [40], seed=31)
    p.ql[0] = -1
    K.attention(stream(), *p.args(), None, None, 0)
    torch.cuda.synchronize()
    assert bool((p.out == MARK).all())
    p = Problem("bf16", 2, 1, 64, [0, 0], seed=31)
    p.forward(K)
    p.backward(K)
    p.check_forward()
    p.check_backward()


def test_repeated_rows_of_keys(K):
    """Strides of 0 in what is read: every head shares one key head's memory."""
    p = Problem("f16", 4, 4, 64, [50], seed=32)
    k1, v1 = randn(generator(1), "f16", p.nk, 64), randn(generator(2), "f16", p.nk, 64)
    p.k, p.v = k1[:, None].expand(-1, 4, -1), v1[:, None].expand(-1, 4, -1)
    p.forward(K)
    p.check_forward()
    p.backward(K)
    p.check_backward()


def test_many_segments(K):
    lens = [(7 * i) % 5 for i in range(1000)]
    p = Problem("bf16", 2, 2, 64, lens, gaps=(0, 1), seed=33)
    p.forward(K)
    p.check_forward()
    p.backward(K)
    p.check_backward()


def test_another_stream_and_the_same_bits_again(K):
    p = Problem("bf16", 8, 2, 128, [400, 77], seed=34)
    p.forward(K)
    p.backward(K)
    first = [x.clone() for x in (p.out, p.lse, p.dq, p.dk, p.dv)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in (p.out, p.dq, p.dk, p.dv, p.lse):
            x.fill_(MARK)
        p.forward(K)
        p.backward(K)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, (p.out, p.lse, p.dq, p.dk, p.dv)):
        assert torch.equal(a, b)


def test_captured_and_replayed(K):
    p = Problem("f16", 4, 2, 64, [150, 30], seed=35)
    size = K.attention_grad_workspace_bytes(p.nq, p.nk, p.h, p.hk, p.dim, 2)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device=DEV)

    def step():
        K.attention(stream(), *p.args(), p.lse.data_ptr(), p.failure.data_ptr(), 5)
        K.attention_grad(stream(), *p.args(), p.lse.data_ptr(), view(p.dout), view(p.dq), view(p.dk), view(p.dv),
                         ws.data_ptr(), size, p.failure.data_ptr(), 5)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (1, 2, 3):
        for i, x in enumerate((p.q, p.k, p.v, p.dout)):
            x.copy_(randn(generator(10 * seed + i), "f16", *x.shape))
        p.ql[0], p.kl[0] = 150 - 10 * seed, 150 - 10 * seed  # lengths may change between replays
        p.segs_q[0] = p.segs_k[0] = (0, 150 - 10 * seed)
        for x in (p.out, p.dq, p.dk, p.dv, p.lse):
            x.fill_(MARK)
        graph.replay()
        torch.cuda.synchronize()
        p.check_forward()
        p.check_backward()


# ------------------------------------------------------------------------ the paged cache
class Cache:
    def __init__(self, t, h, hk, dim, page, new, past, gaps=(0,), seed=0, extra_cols=0):
        gen = generator(seed)
        self.t, self.h, self.hk, self.dim, self.page, self.past = t, h, hk, dim, page, past
        self.segs, self.n = segments(new, gaps)
        need = [-(-(n + p) // page) for n, p in zip(new, past)]
        self.cols, self.pages = max(need) + extra_cols, sum(need) + 2
        order = torch.randperm(self.pages, generator=gen, device=DEV).cpu().numpy()
        table = np.full((len(new), self.cols), -1, np.int32)  # places no sequence needs are out of range
        at = 0
        for s, c in enumerate(need):
            table[s, :c] = order[at:at + c]
            at += c
        self.table = torch.from_numpy(table).to(DEV)
        self.kp, self.vp = (randn(gen, t, self.pages, hk, page, dim) for _ in range(2))
        self.q, self.k, self.v = (randn(gen, t, self.n, x, dim) for x in (h, hk, hk))
        self.out = torch.full_like(self.q, MARK)
        self.lse = torch.full((self.n, h), MARK, dtype=torch.float32, device=DEV)
        self.offsets, self.lens = device_segments(self.segs)
        self.past_lens = torch.tensor(past, dtype=torch.int64, device=DEV)
        self.failure = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.scale = 1 / math.sqrt(dim)
        size = Kernels().attention_paged_workspace_bytes(self.n, h, hk, dim, len(new), page, self.cols)
        self.size, self.workspace = size, torch.full((max(size, 1),), 0xff, dtype=torch.uint8, device=DEV)

    def cache(self):
        return (self.kp.data_ptr(), self.vp.data_ptr(), self.pages, self.page, self.table.data_ptr(), self.cols)

    def append(self, K, freqs, rot, interleaved, q=True, q_out=None):
        q_out = self.out if q_out is None else q_out
        K.kv_append(stream(), self.t, view(self.q) if q else None, view(q_out) if q else None, view(self.k),
                    view(self.v), self.n, self.h, self.hk, self.dim, self.offsets.data_ptr(), self.lens.data_ptr(),
                    len(self.segs), self.past_lens.data_ptr(), freqs.data_ptr() if rot else None, rot,
                    int(interleaved), *self.cache(), self.failure.data_ptr(), 6)

    def attend(self, K, q=None, lse=True):
        q = self.q if q is None else q
        K.attention_paged(stream(), self.t, view(q), self.n, self.h, self.hk, self.dim, self.offsets.data_ptr(),
                          self.lens.data_ptr(), len(self.segs), self.past_lens.data_ptr(), self.scale, *self.cache(),
                          view(self.out), self.lse.data_ptr() if lse else None, self.workspace.data_ptr(), self.size,
                          self.failure.data_ptr(), 6)

    def gathered(self):
        """Keys and values of all sequences, packed, and their segments."""
        ks, vs, segs, at = [], [], [], 0
        for s, ((_, n), p) in enumerate(zip(self.segs, self.past)):
            ids = self.table[s, :-(-(n + p) // self.page)].long()
            for pages, out in ((self.kp, ks), (self.vp, vs)):
                x = pages[ids].transpose(1, 2).reshape(-1, self.hk, self.dim)[:n + p]
                out.append(x)
            segs.append((at, n + p))
            at += n + p
        return torch.cat(ks), torch.cat(vs), segs

    def check(self, q=None):
        k, v, segs = self.gathered()
        out, lse, tol_o, tol_l = ref.forward(self.t, self.q if q is None else q, k, v, self.segs, segs, self.scale, True)
        assert bool((self.out[out.isnan()] == MARK).all()) and bool((self.lse[lse.isnan()] == MARK).all())
        ref.within(self.out, out, tol_o)
        ref.within(self.lse, lse, tol_l)
        assert self.failure.item() == 0

    def positions(self):
        pos = torch.full((self.n,), -1, dtype=torch.int64, device=DEV)
        for (f, n), p in zip(self.segs, self.past):
            pos[f:f + n] = torch.arange(p, p + n, device=DEV)
        return pos


PAGED = [
    # type, heads, kv_heads, dim, page, new tokens, cached tokens, gaps, extra columns
    ("bf16", 4, 1, 128, 16, [1, 1, 1, 1], [0, 1, 15, 700], (0,), 0),
    ("f16", 8, 8, 64, 16, [1, 1, 1], [31, 32, 33], (0,), 5),
    ("bf16", 6, 2, 96, 32, [1, 0, 1, 1], [1000, 7, 63, 64], (1, 0), 0),
    ("f16", 3, 1, 72, 1, [1, 2], [40, 129], (0,), 1),
    ("bf16", 32, 1, 128, 64, [1, 1], [257, 2000], (0,), 0),
    ("f16", 40, 1, 64, 8, [1, 1, 3], [5, 300, 90], (0,), 0),
    ("bf16", 128, 1, 64, 16, [1, 4], [200, 77], (0,), 0),
    ("f16", 8, 2, 64, 4, [5, 9, 0, 2], [100, 0, 50, 1027], (2,), 0),
    ("bf16", 4, 4, 128, 128, [70, 1, 200], [300, 90, 0], (0, 3), 2),
    ("f16", 6, 2, 128, 2, [129, 64], [63, 128], (0,), 0),
    ("bf16", 5, 1, 8, 16, [33], [0], (0,), 0),
    ("f16", 8, 1, 64, 256, [300, 30], [5000, 1], (0,), 40),
    ("bf16", 8, 2, 128, 16, [1], [20000], (0,), 0),       # a long axis and few rows
    ("f16", 4, 1, 64, 32, [3], [9001], (0,), 300),
    ("bf16", 2, 1, 64, 16, [1] * 300, [(37 * i) % 90 for i in range(300)], (0,), 0),
]


@pytest.mark.parametrize("i", range(len(PAGED)))
def test_paged(K, i):
    *p, gaps, extra = PAGED[i]
    c = Cache(*p, gaps=gaps, seed=200 + i, extra_cols=extra)
    c.attend(K)
    c.check()
    c.out.fill_(MARK)
    before = c.lse.clone()
    c.lse.fill_(MARK)
    c.attend(K, lse=False)
    assert bool((c.lse == MARK).all())
    c.lse.copy_(before)
    c.check()


@pytest.mark.parametrize("i", [0, 2, 3, 8, 11, 12])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_slots_past_the_end_have_no_effect(K, i, bad):
    *p, gaps, extra = PAGED[i]
    a, b = (Cache(*p, gaps=gaps, seed=300 + i, extra_cols=extra) for _ in range(2))
    used = torch.zeros(b.pages, b.page, dtype=torch.bool, device=DEV)
    for s, ((_, n), past) in enumerate(zip(b.segs, b.past)):
        pos = torch.arange(n + past, device=DEV)
        used[b.table[s].long()[pos // b.page], pos % b.page] = True
    for x in (b.kp, b.vp):
        x.masked_fill_(~used[:, None, :, None], bad)
    a.attend(K)
    b.attend(K)
    assert torch.equal(a.out, b.out) and torch.equal(a.lse, b.lse)
    b.check()


@pytest.mark.parametrize("i", range(len(PAGED)))
@pytest.mark.parametrize("rot,interleaved", [(1.0, False), (0.5, True), (0.0, False)])
def test_append(K, i, rot, interleaved):
    *p, gaps, extra = PAGED[i]
    c = Cache(*p, gaps=gaps, seed=400 + i, extra_cols=extra)
    rot = 2 * int(rot * c.dim / 2)
    freqs = torch.tensor([10000.0 ** (-2 * j / max(rot, 1)) for j in range(rot // 2)], dtype=torch.float32, device=DEV)
    kp, vp = c.kp.clone(), c.vp.clone()
    c.append(K, freqs, rot, interleaved)
    check_append(c, kp, vp, freqs, rot, interleaved)
    # without queries, and with queries rotated where they are
    c.kp.copy_(kp)
    c.vp.copy_(vp)
    c.out.fill_(MARK)
    c.append(K, freqs, rot, interleaved, q=False)
    assert bool((c.out == MARK).all())
    q = c.q.clone()
    c.append(K, freqs, rot, interleaved, q_out=c.q)
    c.out, c.q = c.q, q
    pos = c.positions()
    assert torch.equal(c.out[pos < 0], q[pos < 0])
    c.out[pos < 0] = MARK
    check_append(c, kp, vp, freqs, rot, interleaved)


def check_append(c, kp, vp, freqs, rot, interleaved):
    pos = c.positions()
    assert bool((c.out[pos < 0] == MARK).all())
    want_q = torch.where((pos < 0)[:, None, None], MARK, ref.rotate(c.q, pos.clamp(min=0), freqs, rot, interleaved))
    want_k, want_v, k = kp.double(), vp.double(), ref.rotate(c.k, pos.clamp(min=0), freqs, rot, interleaved)
    for s, ((f, n), past) in enumerate(zip(c.segs, c.past)):
        at = torch.arange(past, past + n, device=DEV)
        ids = c.table[s].long()[at // c.page]
        want_k[ids, :, at % c.page] = k[f:f + n]
        want_v[ids, :, at % c.page] = c.v[f:f + n].double()
    # one rounding of the result; sine, cosine, two products and a sum in f32 stay within
    # 4 * 2^-24 * (|a| + |b|), components here being below 8; f16 subnormals: half a step
    for got, want in ((c.out, want_q), (c.kp, want_k)):
        ref.within(got, want, ref.U[c.t] * want.abs() + 4 * 2.0 ** -24 * 16 + ref.tiny(c.t))
    assert torch.equal(c.vp.double(), want_v)
    assert c.failure.item() == 0


@pytest.mark.parametrize("past", [1 << 20, (1 << 24) + 1, (1 << 30) + 12345])
def test_angles_of_far_positions(K, past):
    """Positions whose product with a frequency keeps few bits of the angle in 32 bits.  The table
    names pages only where the new tokens go."""
    page = 1 << 22
    t, n = "f16", 5
    cols = (past + n) // page + 1
    q, k, v = (randn(generator(s), t, n, 1, 64) for s in range(3))
    out = torch.zeros_like(q)
    kp, vp = (torch.zeros(2, 1, page, 64, dtype=torch.float16, device=DEV) for _ in range(2))
    table = torch.full((1, cols), -1, dtype=torch.int32, device=DEV)
    table[0, past // page] = 1
    table[0, (past + n - 1) // page] = 1
    off, lens = device_segments([(0, n)])
    pl = torch.tensor([past], dtype=torch.int64, device=DEV)
    fail = torch.zeros(1, dtype=torch.int32, device=DEV)
    freqs = torch.tensor([10000.0 ** (-j / 32) for j in range(32)], dtype=torch.float32, device=DEV)
    K.kv_append(stream(), t, view(q), view(out), view(k), view(v), n, 1, 1, 64, off.data_ptr(), lens.data_ptr(), 1,
                pl.data_ptr(), freqs.data_ptr(), 64, 0, kp.data_ptr(), vp.data_ptr(), 2, page, table.data_ptr(), cols,
                fail.data_ptr(), 1)
    pos = torch.arange(past, past + n, device=DEV)
    for got, want in ((out, ref.rotate(q, pos, freqs, 64, False)),
                      (kp[1, 0, pos % page].unsqueeze(1), ref.rotate(k, pos, freqs, 64, False))):
        ref.within(got, want, ref.U[t] * want.abs() + 4 * 2.0 ** -24 * 16 + ref.tiny(t))
    assert fail.item() == 0


def test_bad_pages_and_lengths_are_reported(K):
    freqs = torch.ones(32, dtype=torch.float32, device=DEV)
    for what in ("page high", "page low", "past negative", "past high", "past huge", "len"):
        c = Cache("f16", 2, 1, 64, 16, [4, 5, 3], [30, 20, 40], seed=50)
        if what == "page high":
            c.table[1, 1] = c.pages
        elif what == "page low":
            c.table[1, 1] = -3
        elif what == "len":
            c.lens[1] = -5
        else:
            c.past_lens[1] = {"past negative": -1, "past high": c.cols * 16 - 4, "past huge": (1 << 63) - 1}[what]
        kp, vp = c.kp.clone(), c.vp.clone()
        c.append(K, freqs, 64, False)
        assert c.failure.item() == 6, what
        if what == "page high" or what == "page low":  # tokens 20..24 go to page 1: none is stored
            mine = c.table[1].clone()
            mine = mine[(mine >= 0) & (mine < c.pages)].long()
            assert torch.equal(kp[mine], c.kp[mine]) and torch.equal(vp[mine], c.vp[mine])
        c.failure.zero_()
        c.out.fill_(MARK)
        c.attend(K)
        assert c.failure.item() == 6, what
        f, n = c.segs[1]
        if "page" not in what:
            assert bool((c.out[f:f + n] == MARK).all()), what
        good = Cache("f16", 2, 1, 64, 16, [4, 5, 3], [30, 20, 40], seed=50)
        good.append(K, freqs, 64, False)
        good.attend(K)
        f, n = c.segs[0]
        assert torch.equal(good.out[f:f + n], c.out[f:f + n]), what


def test_a_table_without_columns(K):
    c = Cache("f16", 2, 1, 64, 16, [1], [3], seed=51)
    c.cols = 0
    c.attend(K)
    assert c.failure.item() == 6
    assert bool((c.out == MARK).all())


def test_prompt_then_tokens_as_a_server_runs_them(K):
    """The prompt's keys go into the cache, attention over the packed prompt and attention over the
    cache agree with the formulas; then tokens one at a time, captured once and replayed."""
    t, h, hk, dim, page, rot = "bf16", 8, 2, 128, 16, 128
    new, steps = [50, 1, 129], 4
    freqs = torch.tensor([10000.0 ** (-j / 64) for j in range(64)], dtype=torch.float32, device=DEV)
    c = Cache(t, h, hk, dim, page, new, [0, 0, 0], seed=60, extra_cols=1)
    table = torch.arange(c.pages, device=DEV, dtype=torch.int32)
    spare = [i for i in table.tolist() if i not in c.table.flatten().tolist()]
    for s in range(3):  # one more page for each sequence, from a cache that is made larger
        c.table[s, -(-new[s] // page)] = c.pages + s
    assert len(spare) == 2
    c.kp, c.vp = (torch.cat([x, torch.zeros(3, *x.shape[1:], dtype=x.dtype, device=DEV)]) for x in (c.kp, c.vp))
    c.pages += 3
    q_rot = torch.full_like(c.q, MARK)
    c.append(K, freqs, rot, False, q_out=q_rot)
    c.attend(K, q=q_rot)
    c.check(q=q_rot)
    paged = c.out.clone()
    k, v, segs = c.gathered()
    p = Problem(t, h, hk, dim, new, seed=61)
    p.q, p.k, p.v = q_rot[:sum(new)].contiguous(), k, v
    p.nq = p.nk = sum(new)
    p.out = torch.full_like(p.q, MARK)
    p.lse = torch.full((p.nq, h), MARK, dtype=torch.float32, device=DEV)
    p.forward(K)
    p.check_forward()
    assert paged[:sum(new)].shape == p.out.shape
    # one token of each sequence at a time
    d = Cache(t, h, hk, dim, page, [1, 1, 1], new, seed=62)
    d.kp, d.vp, d.pages, d.table, d.cols = c.kp, c.vp, c.pages, c.table, c.cols
    d.size = K.attention_paged_workspace_bytes(d.n, h, hk, dim, 3, page, d.cols)
    d.workspace = torch.empty(max(d.size, 1), dtype=torch.uint8, device=DEV)
    q_rot = torch.full_like(d.q, MARK)

    def step():
        d.append(K, freqs, rot, False, q_out=q_rot)
        d.attend(K, q=q_rot)

    before = d.kp.clone(), d.vp.clone()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    d.kp.copy_(before[0])
    d.vp.copy_(before[1])
    for i in range(steps):
        for j, x in enumerate((d.q, d.k, d.v)):
            x.copy_(randn(generator(70 + 10 * i + j), t, *x.shape))
        d.out.fill_(MARK)
        d.lse.fill_(MARK)
        q_rot.fill_(MARK)
        graph.replay()
        torch.cuda.synchronize()
        pos = d.positions()
        live = pos >= 0
        want = ref.rotate(d.q, pos.clamp(min=0), freqs, rot, False)
        ref.within(q_rot[live], want[live], ref.U[t] * want[live].abs() + 4 * 2.0 ** -24 * 16)
        d.check(q=q_rot)
        d.past = [n + 1 for n in d.past]
        d.past_lens += 1


def test_with_the_arrays_of_a_context(ctx, K):
    """The same operators on a Futhark context's arrays and stream, next to its own entry points."""
    from futhark_amd import datagen as dg
    n, h, dim = 96, 4, 64
    x = dg.normal_f32(80, 3 * n * h * dim).reshape(3, n, h * dim)
    bits = dg.to_f16_bits(x)
    q, k, v = (ctx.new("f16_3d", bits[i][None]) for i in range(3))
    out = ctx.new("f16_3d", np.zeros((1, n, h * dim), np.uint16))
    offsets, lens = ctx.new("i64_1d", np.array([0, 40], np.int64)), ctx.new("i64_1d", np.array([40, n - 40], np.int64))
    arr = [heads(a.device_ptr, h * dim, dim) for a in (q, k, v, out)]
    K.attention(ctx.stream, "f16", arr[0], n, arr[1], arr[2], n, h, h, dim, offsets.device_ptr, lens.device_ptr,
                offsets.device_ptr, lens.device_ptr, 2, 1 / math.sqrt(dim), 1, arr[3], None, None, 0)
    got = torch.from_numpy(out.values().view(np.float16).reshape(n, h, dim).copy())
    tq, tk, tv = (torch.from_numpy(bits[i].view(np.float16).reshape(n, h, dim).copy()) for i in range(3))
    want, _, tol, _ = ref.forward("f16", tq, tk, tv, [(0, 40), (40, n - 40)], [(0, 40), (40, n - 40)],
                                  1 / math.sqrt(dim), True)
    ref.within(got, want, tol)
    # scores of a product of the same arrays: the context's own matmul after the attention
    prod = ctx.call("bmm_f16", ["f32_3d"], out, ctx.new("f16_3d", np.ascontiguousarray(bits[1].T)[None])).values()[0]
    a, b = got.reshape(n, -1).double().numpy(), tk.reshape(n, -1).double().numpy()
    assert np.all(np.abs(prod - a @ b.T) <= 1e-5 * (np.abs(a) @ np.abs(b).T))
    for y in (q, k, v, out, offsets, lens):
        y.free()


def test_rows_of_nothing_but_nan(K):
    """A query row of NaN, and a row whose only key is NaN, come out as NaN, not as a row that
    sees nothing; the others are what they are."""
    p = Problem("bf16", 4, 2, 64, [100, 70, 1], seed=90)
    bounds = ref.forward(p.t, p.q, p.k, p.v, p.segs_q, p.segs_k, p.scale, True)
    p.q[40, 1] = float("nan")
    p.k[170, 0] = float("nan")  # the one key of the last sequence, of query heads 0 and 1
    p.forward(K)
    only_these_are_nan([(40, 1), (170, 0), (170, 1)], p.out[:171], p.lse[:171], *(x[:171] for x in bounds))


@pytest.mark.parametrize("t,h,hk,dim,page,new,past", [
    ("f16", 4, 2, 64, 16, [1, 1], [300, 40]),         # a block a unit
    ("bf16", 8, 2, 128, 16, [1, 2], [20000, 70]),     # keys split over waves
    ("f16", 4, 4, 64, 64, [200, 40], [30, 0]),        # many rows
    ("bf16", 4, 1, 128, 64, [70, 40], [9000, 500]),   # many rows, keys split
])
def test_paged_rows_of_nothing_but_nan(K, t, h, hk, dim, page, new, past):
    c = Cache(t, h, hk, dim, page, new, past, seed=91)
    k, v, segs = c.gathered()
    n = sum(new)
    bounds = ref.forward(t, c.q, k, v, c.segs, segs, c.scale, True)
    c.q[0, 1] = float("nan")
    c.attend(K)
    only_these_are_nan([(0, 1)], c.out[:n], c.lse[:n], *(x[:n] for x in bounds))


def only_these_are_nan(rows, out, lse, want, want_lse, tol_o, tol_l):
    bad = torch.zeros(lse.shape, dtype=torch.bool, device=DEV)
    for r, h in rows:
        bad[r, h] = True
    assert bool(out[bad].isnan().all()) and bool(lse[bad].isnan().all())
    ref.within(out[~bad], want[~bad], tol_o[~bad])
    ref.within(lse[~bad], want_lse[~bad], tol_l[~bad])


@pytest.mark.parametrize("h,new,past", [(16, [1, 1], [100, 1]), (4, [200, 3], [70, 9])])
def test_pages_past_32_bit_offsets(K, h, new, past):
    """A cache of 2^31 elements and more, its last pages in use."""
    hk, dim, page = 4, 128, 64
    c = Cache("bf16", h, hk, dim, page, new, past, seed=92)
    n_pages = (1 << 31) // (hk * page * dim) + c.pages
    kp, vp = (torch.empty(n_pages, hk, page, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    kp[-c.pages:], vp[-c.pages:] = c.kp, c.vp
    c.table = torch.where(c.table >= 0, c.table + (n_pages - c.pages), c.table)
    c.kp, c.vp, c.pages = kp, vp, n_pages
    freqs = torch.tensor([10000.0 ** (-j / 64) for j in range(64)], dtype=torch.float32, device=DEV)
    q_rot = torch.empty_like(c.q)
    c.append(K, freqs, dim, False, q_out=q_rot)
    pos = c.positions()
    live = pos >= 0
    want = ref.rotate(c.k, pos.clamp(min=0), freqs, dim, False)
    at = [(c.table[s].long()[(past[s] + i) // page], (past[s] + i) % page, f + i)
          for s, (f, n) in enumerate(c.segs) for i in range(n)]
    got = torch.stack([c.kp[p, :, slot] for p, slot, _ in at])
    rows = want[[r for _, _, r in at]]
    ref.within(got, rows, ref.U["bf16"] * rows.abs() + 4 * 2.0 ** -24 * 16 + ref.tiny("bf16"))
    assert int(live.sum()) == len(at)
    q_rot[~live] = 0
    c.attend(K, q=q_rot)
    c.check(q=q_rot)


def test_rows_past_32_bit_offsets(K):
    """Parts of rows 2^26 elements apart: the last row begins past 2^31 elements."""
    h, hk, dim, n, stride = 4, 2, 64, 40, 1 << 26
    p = Problem("f16", h, hk, dim, [30, 10], seed=93)
    whole = torch.empty((n - 1) * stride + 4096, dtype=torch.float16, device=DEV)

    def far(x, at):
        y = whole.as_strided((n, x.shape[1], dim), (stride, dim, 1), at)
        y.copy_(x[:n])
        return y

    at = 0
    for name in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        x = getattr(p, name)
        setattr(p, name, far(x, at))
        at += x.shape[1] * dim
    p.nq = p.nk = n
    p.lse = p.lse[:n].contiguous()
    p.forward(K)
    p.backward(K)
    p.check_forward()
    p.check_backward()


@pytest.mark.parametrize("h,hk,dim", [(4, 2, 64), (8, 1, 128)])
def test_key_tiles_whose_rows_are_split(K, h, hk, dim):
    """Few key tiles and many rows: the sums of a tile come from several blocks."""
    p = Problem("bf16", h, hk, dim, [2100, 40], seed=94)
    p.forward(K)
    p.backward(K)
    p.check_backward()


@pytest.mark.parametrize("t,h,hk,dim,page,new,past", [
    ("f16", 4, 2, 80, 1, [3, 7], [90, 11]),
    ("bf16", 4, 2, 96, 2, [3, 7, 1], [900, 11, 31]),
    ("f16", 40, 1, 64, 8, [1, 1, 1], [33, 900, 0]),
    ("bf16", 6, 2, 128, 16, [70, 130], [9, 600]),
])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_of_later_tokens_have_no_effect(K, t, h, hk, dim, page, new, past, bad):
    """What the last new token of a sequence has in the cache does not reach the tokens before it."""
    a, b = (Cache(t, h, hk, dim, page, new, past, seed=95) for _ in range(2))
    for s, (n, p) in enumerate(zip(new, past)):
        pos = p + n - 1
        for x in (b.kp, b.vp):
            x[b.table[s, pos // page].long(), :, pos % page] = bad
    a.attend(K)
    a.check()
    b.attend(K)
    for f, n in a.segs:
        assert torch.equal(a.out[f:f + n - 1], b.out[f:f + n - 1])
        assert torch.equal(a.lse[f:f + n - 1], b.lse[f:f + n - 1])
        assert not bool(b.out[f + n - 1].isfinite().any())


def test_two_graphs_and_two_streams(K):
    """Captured calls of two sequences of steps, each with its own workspace, replayed on two
    streams at once."""
    caches = [Cache("bf16", 8, 2, 128, 16, [1, 1, 1], [5000, 40, 900], seed=96 + i) for i in range(2)]
    graphs = []
    for c in caches:
        c.attend(K)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.attend(K)
        graphs.append(g)
    sides = [torch.cuda.Stream() for _ in caches]
    for _ in range(3):
        for c in caches:
            c.q.copy_(-c.q)
            c.out.fill_(MARK)
            c.lse.fill_(MARK)
        torch.cuda.synchronize()
        for g, s in zip(graphs, sides):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for c in caches:
            c.check()


@pytest.mark.parametrize("dim", [40, 72])
def test_split_key_tiles_of_odd_heads(K, dim):
    p = Problem("f16", 12, 2, dim, [1300, 7, 300], [1300, 200, 90], seed=97)
    p.forward(K)
    p.check_forward()
    p.backward(K)
    p.check_backward()


def test_bad_pages_and_lengths_of_many_rows(K):
    """The same as above for the kernel that takes many rows, its keys split."""
    for what in ("page high", "past negative", "past high", "past huge", "len"):
        c, good = (Cache("bf16", 2, 1, 64, 16, [70, 90, 65], [3000, 20, 40], seed=98) for _ in range(2))
        if what == "page high":
            c.table[1, 3] = c.pages
        elif what == "len":
            c.lens[1] = 1 << 40
        else:
            c.past_lens[1] = {"past negative": -1, "past high": c.cols * 16 - 89, "past huge": (1 << 63) - 1}[what]
        c.attend(K)
        assert c.failure.item() == 6, what
        good.attend(K)
        good.check()
        kept = [0] if what == "len" else [0, 2]  # a length past the end breaks the segment behind it too
        for s in kept:
            f, n = c.segs[s]
            assert torch.equal(good.out[f:f + n], c.out[f:f + n]), (what, s)
        f, n = c.segs[1]
        if what != "page high":
            assert bool((c.out[f:f + n] == MARK).all()), what


@pytest.mark.parametrize("t,h,hk,dim,page,new,past", [
    ("bf16", 8, 2, 128, 16, [1] * 9, [1500, 3, 900, 0, 31, 1023, 64, 1499, 700]),       # a short line
    ("f16", 16, 4, 64, 16, [1] * 9, [2500, 3, 900, 0, 31, 1023, 64, 2499, 700]),
    ("bf16", 32, 8, 128, 16, [1] * 70, [(61 * i) % 1900 for i in range(70)]),            # units fill half of the waves
    ("f16", 24, 8, 64, 32, [1, 3, 9, 2, 0, 7] * 6, [(331 * i) % 2200 for i in range(36)]),
    ("bf16", 32, 32, 128, 16, [1] * 40, [(97 * i) % 1200 for i in range(40)]),           # more units than waves
])
def test_lines_of_all_lengths(K, t, h, hk, dim, page, new, past):
    c = Cache(t, h, hk, dim, page, new, past, seed=99)
    c.attend(K)
    c.check()


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("h,hk,dim,q_lens,k_lens,causal", [
    (4, 2, 128, [1] * 70, None, True),               # sequences of one token
    (3, 1, 64, [1, 1, 1], None, False),
    (16, 2, 72, [1] * 9, [1] * 9, True),
    (5, 5, 8, [1], None, True),
    (2, 1, 128, [2100, 3, 130], [1, 1, 1], False),   # many rows on one key, split into parts
    (12, 4, 40, [700], [1], False),
    (4, 2, 64, [40, 1, 200], [1, 1, 1], True),       # rows of nothing before the row of one key
])
def test_rows_of_one_key_have_no_gradient(K, t, h, hk, dim, q_lens, k_lens, causal):
    """A row that sees one key has the weight 1 whatever its score is: the derivative of the score is
    zero, and with it dq and dk, not the difference of two roundings."""
    p = Problem(t, h, hk, dim, q_lens, k_lens, causal, seed=101, spread=3.0)
    p.forward(K)
    p.backward(K)
    p.check_backward()
    for x, segs in ((p.dq, p.segs_q), (p.dk, p.segs_k)):
        for f, n in segs:
            assert not bool(x[f:f + n].any())


@pytest.mark.parametrize("t,h,hk,dim", [("bf16", 8, 2, 128), ("f16", 6, 6, 64), ("f16", 5, 1, 96)])
def test_first_rows_of_sequences_have_no_gradient(K, t, h, hk, dim):
    """The same for the first row of a causal sequence, beside rows that see more, and for the row that
    sees the first key behind rows that see nothing."""
    q_lens, k_lens = [2, 64, 300, 1, 90, 130], [2, 64, 300, 1, 40, 129]
    p = Problem(t, h, hk, dim, q_lens, k_lens, seed=102)
    p.forward(K)
    p.backward(K)
    p.check_backward()
    for (f, n), (_, kn) in zip(p.segs_q, p.segs_k):
        assert not bool(p.dq[f:f + n - kn + 1].any())
        assert n == 1 or bool(p.dq[f + n - kn + 1:f + n].any(-1).all())


# --------------------------------------------------------- segments that break the rules
def kept_segments(offsets, lens, n):
    """The numbers of the segments that are not left out, by the header's rules."""
    kept, reach = [], 0
    for i, (f, l) in enumerate(zip(offsets, lens)):
        inside = 0 <= f <= n and 0 <= l <= n - f
        ok = inside and f >= reach
        if i > 0:
            pf, pl = offsets[i - 1], lens[i - 1]
            ok = ok and 0 <= pf <= n and 0 <= pl <= n - pf
        if ok:
            kept.append(i)
        if inside:
            reach = max(reach, f + l)
    return kept


# A broken segment and what comes behind it, in units of rows from the first one on.
BROKEN = {
    "overlap behind an overlap": [(0, 10), (5, 1), (6, 10), (16, 2)],
    "far behind it": [(0, 20), (2, 1), (3, 1), (4, 0), (4, 9), (13, 4), (17, 8), (25, 3)],
    "outside": [(0, 10), (4, 1 << 40), (6, 10), (16, 2)],
    "negative": [(0, 10), (4, -1), (6, 10), (16, 2), (18, 1)],
    "backwards": [(4, 10), (0, 4), (4, 10), (14, 2)],
}


def broken_segments(what, m, unit, at=None):
    """m segments of `unit` rows, some of none, with the broken ones from number `at` on; offsets and
    lengths, and the rows they need."""
    at = m // 2 if at is None else at
    offsets, lens, first = [], [], 0
    for i in range(at):
        offsets.append(first)
        lens.append(0 if i % 7 == 3 else unit)
        first += lens[-1]
    for f, l in BROKEN[what]:
        offsets.append(first + f * unit)
        lens.append(l * unit if abs(l) < 1 << 30 else l)
    first = offsets[-1] + lens[-1]
    while len(offsets) < m:
        offsets.append(first)
        lens.append(unit)
        first += unit
    return offsets, lens, first


@pytest.mark.parametrize("what", BROKEN)
@pytest.mark.parametrize("m,unit,at", [(8, 7, 0), (40, 3, None), (200, 2, 62), (200, 2, 63), (300, 1, 127)])
def test_segments_that_overlap_are_left_out(K, what, m, unit, at):
    """Of segments that overlap the first counts, however many broken ones lie between."""
    offsets, lens, rows = broken_segments(what, m, unit, at)
    rows += 3
    kept = kept_segments(offsets, lens, rows)
    assert 0 < len(kept) < len(offsets)
    t, h, hk, dim = "bf16", 4, 2, 64
    p = Problem(t, h, hk, dim, [rows], seed=110)
    rows = p.nq
    for x in (p.qo, p.ko):
        x.resize_(len(offsets)).copy_(torch.tensor(offsets))
    for x in (p.ql, p.kl):
        x.resize_(len(lens)).copy_(torch.tensor(lens))
    p.segs_q = p.segs_k = list(zip(offsets, lens))
    p.forward(K)
    p.backward(K)
    assert p.failure.item() == 5
    p.failure.zero_()
    p.segs_q = p.segs_k = [(offsets[i], lens[i]) for i in kept_segments(offsets, lens, rows)]
    p.check_forward()
    p.check_backward()


def broken_cache(t, h, hk, dim, page, what, m, unit, at, past_of, extra_cols, seed):
    offsets, lens, rows = broken_segments(what, m, unit, at)
    new = [l if 0 <= l < 1 << 30 else unit for l in lens]
    c = Cache(t, h, hk, dim, page, new, [past_of(i) for i in range(len(new))], seed=seed, extra_cols=extra_cols)
    assert c.n >= rows
    c.offsets.copy_(torch.tensor(offsets))
    c.lens.copy_(torch.tensor(lens))
    return c, kept_segments(offsets, lens, c.n), list(zip(offsets, lens))


def only_kept(c, kept, segs):
    assert c.failure.item() == 6
    c.failure.zero_()
    c.segs, c.past, c.table = [segs[i] for i in kept], [c.past[i] for i in kept], c.table[kept]


@pytest.mark.parametrize("what", BROKEN)
@pytest.mark.parametrize("h,hk,dim,m,unit,at,most_past,extra_cols", [
    (4, 2, 64, 12, 1, 0, 300, 0),        # a block a unit
    (4, 2, 128, 80, 1, 61, 90, 0),       # the same, several batches of segments
    (4, 2, 64, 12, 1, 3, 1900, 99),      # a short line
    (8, 8, 64, 200, 1, 100, 1700, 0),    # a line, a sequence a thread
    (2, 1, 64, 700, 1, 254, 90, 99),     # a line, several sequences a thread
    (8, 8, 64, 700, 1, 440, 120, 99),
    (4, 2, 64, 12, 40, 3, 90, 0),        # many rows
    (4, 2, 128, 80, 33, 62, 300, 0),     # the same, tiles in the order of the segments
])
def test_cached_segments_that_overlap_are_left_out(K, what, h, hk, dim, m, unit, at, most_past, extra_cols):
    c, kept, segs = broken_cache("f16", h, hk, dim, 16, what, m, unit, at, lambda i: (37 * i) % most_past, extra_cols, 111)
    assert 0 < len(kept) < len(segs)
    c.attend(K)
    only_kept(c, kept, segs)
    c.check()


@pytest.mark.parametrize("what", BROKEN)
@pytest.mark.parametrize("m,unit,at", [(12, 5, 0), (80, 3, 62), (700, 1, 318), (700, 2, 400)])
def test_appended_segments_that_overlap_are_left_out(K, what, m, unit, at):
    c, kept, segs = broken_cache("f16", 2, 1, 64, 16, what, m, unit, at, lambda i: (11 * i) % 50, 0, 112)
    freqs = torch.tensor([10000.0 ** (-j / 32) for j in range(32)], dtype=torch.float32, device=DEV)
    kp, vp = c.kp.clone(), c.vp.clone()
    c.append(K, freqs, 64, False)
    only_kept(c, kept, segs)
    check_append(c, kp, vp, freqs, 64, False)


@pytest.mark.parametrize("which,what", [("kl", 1 << 40), ("ko", -1), ("ql", 1), ("qo", 2)])
def test_gradient_without_query_rows_reports_broken_segments(K, which, what):
    """Keys nobody asks have gradients of zero, written by the second kernel alone."""
    for broken in (False, True):
        p = Problem("bf16", 4, 2, 64, [0, 0, 0], [40, 50, 60], seed=113)
        p.nq = 0
        if broken:
            getattr(p, which)[1] = what
        p.backward(K)
        assert p.failure.item() == (5 if broken else 0)
        kept = [0] if broken else [0, 1, 2]  # the one behind a segment outside the rows is left out too
        for x in (p.dk, p.dv):
            for f, n in [p.segs_k[i] for i in kept]:
                assert bool((x[f:f + n] == 0).all())
            if broken:
                f, n = p.segs_k[1]
                assert bool((x[f:f + n] == MARK).all())
        assert bool((p.dq == MARK).all())


@pytest.mark.parametrize("n", [1, 100])  # few rows; many rows, whose keys are split
def test_the_longest_table(K, n):
    """2^31 - 2^20 positions, the same page over and over: a page's slot counts as often as it is seen.
    (f32 sums of a part, of chunk = 2^31 / 512 keys here: weights chunk / 2 additions in a row, outputs
    at most 17 / 16 chunk, each off by 2^-24 of what it adds to.)"""
    t, dim, page, cols = "bf16", 8, 1 << 20, 2047
    k, v = randn(generator(120), t, page, dim), (randn(generator(121), t, page, dim, scale=0.1).float() + 1).to(ref.DTYPE[t])
    q = randn(generator(122), t, n, 1, dim)
    out, lse = torch.full_like(q, MARK), torch.full((n, 1), MARK, dtype=torch.float32, device=DEV)
    table = torch.zeros(1, cols, dtype=torch.int32, device=DEV)
    off, lens = device_segments([(0, n)])
    past = torch.tensor([cols * page - n], dtype=torch.int64, device=DEV)
    fail = torch.zeros(1, dtype=torch.int32, device=DEV)
    scale = 1 / math.sqrt(dim)
    size = K.attention_paged_workspace_bytes(n, 1, 1, dim, 1, page, cols)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device=DEV)
    K.attention_paged(stream(), t, view(q), n, 1, 1, dim, off.data_ptr(), lens.data_ptr(), 1, past.data_ptr(), scale,
                      k.data_ptr(), v.data_ptr(), 1, page, table.data_ptr(), cols, view(out), lse.data_ptr(),
                      ws.data_ptr(), size, fail.data_ptr(), 1)
    kd, vd = k.double(), v.double()
    chunk = 2 ** 31 / 512
    for i in sorted({0, n // 2, n - 1}):
        s = kd @ q[i, 0].double() * scale
        times = cols - (torch.arange(page, device=DEV) >= page - n + i + 1).double()
        w = times * torch.exp(s - s.max())
        o, l = (w @ vd) / w.sum(), s.max() + torch.log(w.sum())
        rel = chunk / 2 * 2.0 ** -24 + chunk * 17 / 16 * 2.0 ** -24 + 4 * ref.U[t]
        assert bool(((out[i, 0].double() - o).abs() <= rel * o.abs()).all()), (i, out[i, 0], o)
        assert abs(lse[i, 0].item() - l.item()) <= -math.log(1 - chunk / 2 * 2.0 ** -24) + 0.01, (i, lse[i, 0], l)
    assert fail.item() == 0


@pytest.mark.parametrize("t,h,hk,dim,page,new,past", [
    ("f16", 16, 4, 64, 16, [1, 1, 1, 1], [500, 3, 1535, 90]),
    ("bf16", 32, 8, 128, 16, [1, 2, 0, 1], [1000, 3, 500, 1023]),
])
def test_one_launch_without_a_workspace(K, t, h, hk, dim, page, new, past):
    c = Cache(t, h, hk, dim, page, new, past, seed=130)
    assert c.size == 0
    K.attention_paged(stream(), t, view(c.q), c.n, h, hk, dim, c.offsets.data_ptr(), c.lens.data_ptr(), len(c.segs),
                      c.past_lens.data_ptr(), c.scale, *c.cache(), view(c.out), c.lse.data_ptr(), None, 0,
                      c.failure.data_ptr(), 6)
    c.check()


# ------------------------------------------------------- ways that calls above do not take
@pytest.mark.parametrize("t,h,hk,dim,m,most_past", [
    ("f16", 2, 1, 64, 300, 200),     # more sequences than threads of a block, a short line
    ("bf16", 16, 8, 64, 300, 200),   # the same with more units than waves
    ("bf16", 4, 2, 128, 600, 330),
    ("f16", 6, 2, 96, 1025, 90),
])
def test_few_rows_of_many_sequences(K, t, h, hk, dim, m, most_past):
    """A thread of a block counts several sequences; some are empty, one does not fit its table."""
    new = [[1, 0, 1, 2, 1, 1, 3][i % 7] for i in range(m)]
    c = Cache(t, h, hk, dim, 16, new, [(53 * i) % most_past for i in range(m)], gaps=(0, 1, 0), seed=140, extra_cols=99)
    c.attend(K)
    c.check()
    bad = 2 * m // 3 - (2 * m // 3) % 7  # of one new token
    c.past_lens[bad] = c.cols * 16
    c.out.fill_(MARK)
    c.lse.fill_(MARK)
    c.attend(K)
    assert c.failure.item() == 6
    c.failure.zero_()
    f, n = c.segs[bad]
    assert n == 1 and bool((c.out[f:f + n] == MARK).all()) and bool((c.lse[f:f + n] == MARK).all())
    keep = [i for i in range(m) if i != bad]
    c.segs, c.past, c.table = [c.segs[i] for i in keep], [c.past[i] for i in keep], c.table[keep]
    c.check()


@pytest.mark.parametrize("t,h,hk,dim,new,past", [
    ("bf16", 8, 2, 64, [(17 * i) % 80 for i in range(70)], [(211 * i) % 2000 for i in range(70)]),  # keys split
    ("f16", 4, 1, 128, [40 + i % 9 for i in range(90)], [(97 * i) % 1500 for i in range(90)]),
    ("f16", 64, 64, 128, [700, 3, 690], [100, 0, 310]),  # tiles of few sequences fill the chip
])
def test_many_rows_in_the_order_of_the_segments(K, t, h, hk, dim, new, past):
    c = Cache(t, h, hk, dim, 16, new, past, gaps=(0, 2), seed=141)
    c.attend(K)
    c.check()


@pytest.mark.parametrize("t,h,hk,dim,lens,causal", [
    ("bf16", 4, 1, 128, [i % 6 for i in range(79)] + [2000], True),   # parts, more segments than lanes
    ("f16", 8, 2, 64, [2300] + [(5 * i) % 9 for i in range(99)], False),
    ("f16", 32, 32, 128, [2100, 20], True),                           # parts, many key heads
])
def test_split_key_tiles_in_the_order_of_the_segments(K, t, h, hk, dim, lens, causal):
    p = Problem(t, h, hk, dim, lens, causal=causal, seed=142)
    p.forward(K)
    p.check_forward()
    p.backward(K)
    p.check_backward()


# ------------------------------------------------------------------- ways against each other
@pytest.mark.parametrize("i", range(len(PROMPTS)))
def test_without_lse_the_same_bits(K, i):
    p = Problem(*PROMPTS[i], seed=i)
    p.forward(K)
    out = p.out.clone()
    p.out.fill_(MARK)
    p.forward(K, lse=False)
    assert torch.equal(out, p.out)


@pytest.mark.parametrize("i", range(len(PAGED)))
def test_paged_without_lse_the_same_bits(K, i):
    *p, gaps, extra = PAGED[i]
    c = Cache(*p, gaps=gaps, seed=200 + i, extra_cols=extra)
    c.attend(K)
    out = c.out.clone()
    c.out.fill_(MARK)
    c.attend(K, lse=False)
    assert torch.equal(out, c.out)


@pytest.mark.parametrize("t,h,hk,dim,page,new,past", [
    ("bf16", 8, 2, 128, 16, [50, 1, 129], [0, 0, 0]),
    ("f16", 4, 4, 64, 32, [1, 1, 1], [300, 0, 2000]),
    ("bf16", 6, 2, 96, 8, [5, 200], [90, 700]),
])
def test_paged_and_packed_agree(K, t, h, hk, dim, page, new, past):
    """The same attention over the cache and over its keys packed: within the sum of both bounds."""
    c = Cache(t, h, hk, dim, page, new, past, seed=143)
    c.attend(K)
    c.check()
    k, v, segs = c.gathered()
    p = Problem(t, h, hk, dim, new, [n + s for n, s in zip(new, past)], seed=144)
    assert p.segs_q == c.segs and p.segs_k == segs
    p.q, p.k, p.v, p.nk = c.q, k, v, k.shape[0]
    p.forward(K)
    p.check_forward()
    want, lse, tol_o, tol_l = ref.forward(t, p.q, k, v, c.segs, segs, c.scale, True)
    live = ~lse.isnan()
    ref.within(c.out[live], p.out[live].double(), 2 * tol_o[live])
    ref.within(c.lse[live], p.lse[live].double(), 2 * tol_l[live])


def test_a_serving_and_a_training_step_with_the_arrays_of_a_context(ctx, K):
    """Cache append, attention over the cache and the gradient on a Futhark context's arrays and
    stream; the context reads the results with its own calls."""
    from futhark_amd import datagen as dg
    h, hk, dim, page, lens = 4, 2, 64, 16, [40, 23]
    n, offsets = sum(lens), [0, 40]
    cols = max(-(-x // page) for x in lens)
    pages = cols * len(lens) + 1
    sizes = {"q": h, "k": hk, "v": hk, "dout": h}
    bits = {x: dg.to_f16_bits(dg.normal_f32(90 + i, n * c * dim).reshape(1, n, c * dim))
            for i, (x, c) in enumerate(sizes.items())}
    arr = {x: ctx.new("f16_3d", b) for x, b in bits.items()}
    for x, like in (("rotated", "q"), ("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v")):
        arr[x] = ctx.new("f16_3d", np.zeros_like(bits[like]))
    for x in ("kp", "vp"):
        arr[x] = ctx.new("f16_3d", np.zeros((pages * hk, page, dim), np.uint16))
    table = np.arange(pages - 1, dtype=np.int32)[::-1].copy()
    freqs = np.array([10000.0 ** (-j / 32) for j in range(32)], np.float32)
    off, ln, zero = (ctx.new("i64_1d", np.array(x, np.int64)) for x in (offsets, lens, [0, 0]))
    tab, fr, lse = ctx.new("i32_1d", table), ctx.new("f32_1d", freqs), ctx.new("f32_1d", np.zeros(n * h, np.float32))
    fail = ctx.new("i32_1d", np.zeros(1, np.int32))
    m, scale, width = 2, 1 / math.sqrt(dim), {**sizes, "rotated": h, "out": h, "dq": h, "dk": hk, "dv": hk}

    def V(x):
        return heads(arr[x].device_ptr, width[x] * dim, dim)

    seg = (off.device_ptr, ln.device_ptr)
    cache = (arr["kp"].device_ptr, arr["vp"].device_ptr, pages, page, tab.device_ptr, cols)
    size = K.attention_paged_workspace_bytes(n, h, hk, dim, m, page, cols)
    ws = ctx.new("u8_1d", np.zeros(max(size, 1), np.uint8))
    K.kv_append(ctx.stream, "f16", V("q"), V("rotated"), V("k"), V("v"), n, h, hk, dim, *seg, m, zero.device_ptr,
                fr.device_ptr, dim, 0, *cache, fail.device_ptr, 7)
    K.attention_paged(ctx.stream, "f16", V("rotated"), n, h, hk, dim, *seg, m, zero.device_ptr, scale, *cache, V("out"),
                      lse.device_ptr, ws.device_ptr, size, fail.device_ptr, 7)

    def host(x):
        return torch.from_numpy(arr[x].values().view(np.float16).reshape(n, -1, dim).copy())

    pos = torch.cat([torch.arange(x) for x in lens])
    f = torch.from_numpy(freqs)
    q, k, v = (torch.from_numpy(bits[x].view(np.float16).reshape(n, -1, dim).copy()) for x in "qkv")
    for x, want in (("rotated", ref.rotate(q, pos, f, dim, False)),):
        ref.within(host(x), want, ref.U["f16"] * want.abs() + 4 * 2.0 ** -24 * 16 + ref.tiny("f16"))
    stored = torch.from_numpy(arr["kp"].values().view(np.float16).reshape(pages, hk, page, dim).copy())
    kd = torch.cat([stored[table[s * cols:(s + 1) * cols]].transpose(1, 2).reshape(-1, hk, dim)[:x]
                    for s, x in enumerate(lens)])
    want = ref.rotate(k, pos, f, dim, False)
    ref.within(kd, want, ref.U["f16"] * want.abs() + 4 * 2.0 ** -24 * 16 + ref.tiny("f16"))
    segs = list(zip(offsets, lens))
    want, _, tol, _ = ref.forward("f16", host("rotated"), kd, v, segs, segs, scale, True)
    ref.within(host("out"), want, tol)
    # a training step on the prompts as they are
    size = K.attention_grad_workspace_bytes(n, n, h, hk, dim, m)
    ws2 = ctx.new("u8_1d", np.zeros(size, np.uint8))
    args = ("f16", V("q"), n, V("k"), V("v"), n, h, hk, dim, *seg, *seg, m, scale, 1, V("out"))
    K.attention(ctx.stream, *args, lse.device_ptr, fail.device_ptr, 7)
    K.attention_grad(ctx.stream, *args, lse.device_ptr, V("dout"), V("dq"), V("dk"), V("dv"), ws2.device_ptr, size,
                     fail.device_ptr, 7)
    dout = torch.from_numpy(bits["dout"].view(np.float16).reshape(n, h, dim).copy())
    grads, tols = ref.gradient("f16", q, k, v, dout, segs, segs, scale, True)
    for x, want, tol in zip(("dq", "dk", "dv"), grads, tols):
        ref.within(host(x), want, tol)
    assert fail.values()[0] == 0
    for x in (*arr.values(), off, ln, zero, tab, fr, lse, fail, ws, ws2):
        x.free()
