"""Attention of a ragged batch's new tokens over the paged cache
(gptoss_attn_chunk, chunk.attend_chunks) against softmax attention in 64 bits.

Tolerances, element by element, from the arithmetic alone.  With p the softmax
weights and den their sum with the sink's:
  P is rounded to bf16 (2^-9 of itself), or in 8 bits split into two e4m3 terms
  (2^-8, and 2^-18 of the row's largest, which may sit 2^2 below the top of a
  term's range: 2^-16); Q's split moves a score by up to 2^-18 of the largest
  product, below 2^-11 here: a little more than 2^-8 of P in all.  The output is
  rounded once (2^-9).
  |o - exact| <= 1.25 * 2^-8 * sum p |v| / den + 2^-16 * max p * sum |v| / den
                 + 2^-9 |o| + 1e-6
lse: fp32 sums of up to a few thousand terms (1e-4), in 8 bits Q's split too
(5e-4).
"""
import importlib
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

chunk = importlib.import_module("gpt-oss-tvm_b200.chunk")
_lib = importlib.import_module("gpt-oss-tvm_b200._lib")
D, PAGE = 64, 16


def quantise(x):
    """bf16 rows [rows, heads, 64] as an 8-bit pool, by the definition."""
    a = x.double().abs().amax(-1)
    e = torch.ceil(torch.log2(a.clamp(min=1e-300) / 448.0)).clamp(-60, 60)
    q = (x.double() * torch.exp2(-e).unsqueeze(-1)).float().to(torch.float8_e4m3fn)
    code = (e + 127).to(torch.uint8).reshape(-1, PAGE, x.shape[1]).transpose(1, 2).contiguous()
    return q, code.view(torch.float8_e8m0fnu)


def dequantise(q, code):
    e = code.view(torch.uint8).transpose(1, 2).reshape(q.shape[:2]).double() - 127
    return q.float().double() * torch.exp2(e).unsqueeze(-1)


class Case:
    """Inputs of one call, and its exact answer."""

    def __init__(self, ql, kl, hq=64, hkv=8, window=0, f8=False, sinks=True, seed=0, ring=None, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        n = len(ql)
        self.ql, self.kl, self.hq, self.hkv, self.window = ql, kl, hq, hkv, window
        stride = max(1, -(-max(max(kl), 1) // PAGE)) if ring is None else ring
        self.table = torch.randperm(n * stride, generator=g).to(torch.int32).reshape(n, stride)
        self.stride = stride
        rows = n * stride * PAGE
        self.k = (torch.randn(rows, hkv, D, generator=g) * scale).to(torch.bfloat16)
        self.v = torch.randn(rows, hkv, D, generator=g).to(torch.bfloat16)
        self.ks = self.vs = None
        if f8:
            (self.k, self.ks), (self.v, self.vs) = quantise(self.k), quantise(self.v)
        self.q = torch.randn(sum(ql), hq, D, generator=g).to(torch.bfloat16)
        self.sinks = torch.randn(hq, generator=g).to(torch.bfloat16) if sinks else None
        self.rows = torch.arange(n, dtype=torch.int32)
        start = [0]
        for x in ql:
            start.append(start[-1] + x)
        self.q_start, self.kv_len = torch.tensor(start, dtype=torch.int32), torch.tensor(kl, dtype=torch.int32)

    def gpu(self):
        for name in ("table", "k", "v", "ks", "vs", "q", "sinks", "rows", "q_start", "kv_len"):
            t = getattr(self, name)
            if t is not None:
                setattr(self, name, t.cuda())
        return self

    def run(self, **kw):
        a = dict(max_q=max(max(self.ql), 1), window=self.window, sinks=self.sinks, k_scale=self.ks, v_scale=self.vs,
                 return_lse=True)
        a.update(kw)
        out = chunk.attend_chunks(self.q, self.k, self.v, self.table, self.rows, self.q_start, self.kv_len, **a)
        torch.cuda.synchronize()
        return out

    def exact(self):
        """(o, lse, tolerance of o) in 64 bits; masked keys are left out, so what they hold does not matter."""
        k = dequantise(self.k, self.ks) if self.ks is not None else self.k.double()
        v = dequantise(self.v, self.vs) if self.vs is not None else self.v.double()
        T, grp, dev = sum(self.ql), self.hq // self.hkv, self.q.device
        o = torch.zeros(T, self.hq, D, dtype=torch.float64, device=dev)
        lse = torch.full((T, self.hq), -math.inf, dtype=torch.float64, device=dev)
        tol = torch.full((T, self.hq, D), 1e-6, dtype=torch.float64, device=dev)
        at = 0
        for b, (n, L) in enumerate(zip(self.ql, self.kl)):
            for i in range(n):
                pos = L - n + i
                lo = max(0, pos - self.window + 1) if self.window else 0
                if pos >= lo and pos >= 0:
                    j = torch.arange(lo, pos + 1, device=dev)
                    row = self.table[b].long()[(j // PAGE) % self.stride] * PAGE + j % PAGE
                    kk, vv = k[row].repeat_interleave(grp, 1), v[row].repeat_interleave(grp, 1)
                    s = torch.einsum("hd,jhd->hj", self.q[at].double(), kk) / 8.0
                    lse[at] = torch.logsumexp(s, -1) / math.log(2.0)
                    m = s.amax(-1, keepdim=True)
                    p = torch.exp(s - m)
                    den = p.sum(-1)
                    if self.sinks is not None:
                        den = den + torch.exp(self.sinks.double() - m[:, 0])
                    o[at] = torch.einsum("hj,jhd->hd", p, vv) / den[:, None]
                    av = vv.abs()
                    tol[at] += (1.25 * 2.0 ** -8 * torch.einsum("hj,jhd->hd", p, av) + 2.0 ** -16 * av.sum(0)) \
                        / den[:, None] + 2.0 ** -9 * o[at].abs()
                at += 1
        return o, lse, tol

    def check(self, **kw):
        o, lse = self.run(**kw)
        eo, el, tol = self.exact()
        assert bool(torch.isfinite(o).all())
        over = ((o.double() - eo).abs() - tol).max().item() if o.numel() else 0.0
        assert over <= 0, f"o is {over:.3e} beyond its tolerance"
        seen = torch.isfinite(el)
        assert torch.equal(torch.isfinite(lse), seen) and bool((lse[~seen] == -math.inf).all())
        d = (lse.double() - el)[seen].abs().max().item() if bool(seen.any()) else 0.0
        assert d <= (5e-4 if self.ks is not None else 1e-4), f"lse is {d:.3e} off"
        return o, lse


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("ql,kl", [
    ([1], [1]), ([1], [16]), ([1], [17]), ([1], [129]), ([1], [1000]),           # one token, page and tile edges
    ([1, 1, 1, 1], [1, 127, 128, 257]), ([2], [2]), ([3, 1, 2], [300, 40, 513]),  # small chunks
    ([5, 4, 1], [260, 129, 700]), ([8, 3], [8, 900]), ([6], [255]),               # 48 and 64 rows
    ([9], [9]), ([33, 7], [33, 400]), ([70], [333]), ([130, 1, 40], [130, 600, 41]),  # past 64 rows: longer tiles
    ([0, 3, 0, 5], [0, 90, 50, 5]), ([0, 20], [10, 20]),                          # sequences without new tokens
])
def test_ragged_chunks(ql, kl, f8):
    Case(ql, kl, f8=f8, seed=len(ql) + sum(kl)).gpu().check()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("hq,hkv,q", [(8, 8, 1), (8, 8, 5), (8, 8, 40), (12, 4, 3), (10, 2, 2), (5, 1, 3), (3, 3, 30),
                                      (16, 1, 1), (32, 2, 2), (28, 4, 4), (64, 1, 1), (64, 2, 2), (40, 8, 50)])
def test_head_groups(hq, hkv, q, f8):
    Case([q, 1], [q + 130, 77], hq=hq, hkv=hkv, f8=f8, seed=hq + q).gpu().check()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("q", [1, 4, 7, 40])
@pytest.mark.parametrize("window", [1, 15, 16, 128, 1000])
def test_window(window, q, f8):
    Case([q, q], [300 + q, q], window=window, f8=f8, seed=window + q).gpu().check()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("q", [1, 5, 30])
def test_window_ring(q, f8):
    """Pages in a ring that holds window + chunk - 1 keys and the page being
    filled, gone round several times."""
    ring = -(-(128 + q - 1) // PAGE) + 1
    Case([q, 1, q], [1000, 140, 129 + q], window=128, f8=f8, ring=ring, seed=q).gpu().check()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("q", [1, 5, 20])
def test_rows_that_see_nothing(q, f8):
    """Chunks longer than their sequence: tokens before position 0 give zeros and -inf."""
    c = Case([q + 2, q, q], [q, 0, q + 40], f8=f8, seed=3 * q).gpu()
    o, lse = c.check()
    assert bool((o[:2] == 0).all()) and bool((lse[:2] == -math.inf).all())
    assert bool((o[q + 2:2 * q + 2] == 0).all())


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("q,window", [(1, 0), (5, 0), (5, 100), (40, 0), (40, 100)])
def test_hidden_keys_may_hold_anything(q, window, f8):
    """NaN and infinities beyond the last position, before the window and in
    pages of nobody change no bit."""
    c = Case([q], [250], window=window, f8=f8, seed=q, ring=20).gpu()
    o, lse = c.check()
    j = torch.arange(20 * PAGE, device="cuda")
    hidden = (j >= 250) | (j < (250 - q - window + 1 if window else 0))
    rows = (c.table[0].long()[j // PAGE] * PAGE + j % PAGE)[hidden]
    if f8:
        for t, s in ((c.k, c.ks), (c.v, c.vs)):
            t.view(torch.uint8)[rows] = 0x7F
            t.view(torch.uint8)[rows[::2]] = 0xFF
            s.view(torch.uint8)[rows // PAGE, :, rows % PAGE] = 255
    else:
        for t in (c.k, c.v):
            t[rows] = math.nan
            t[rows[::2]] = -math.inf
    o2, lse2 = c.run()
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("f8", [False, True])
def test_a_nan_key_stays_with_those_who_see_it(f8):
    c = Case([3, 2], [100, 60], f8=f8, seed=5).gpu()
    row = int(c.table[0, 98 // PAGE]) * PAGE + 98 % PAGE   # position 98: tokens 1 and 2 of the first chunk
    if f8:
        c.ks.view(torch.uint8)[row // PAGE, 2, row % PAGE] = 255
    else:
        c.k[row, 2, 7] = math.nan
    o, _ = c.run()
    bad = torch.zeros(5, 64, dtype=torch.bool, device="cuda")
    bad[1:3, 16:24] = True   # kv head 2 serves heads 16..23
    assert torch.equal(torch.isnan(o).any(-1), bad)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("q,window", [(1, 0), (4, 0), (7, 0), (40, 0), (100, 0), (5, 20), (40, 20)])
def test_a_value_that_is_not_finite_stays_with_those_who_see_it(q, window, value, f8):
    """Also when it is a later token's of the same chunk: the rows before it
    keep their bits, the rows from it on are NaN (in the window), sums and
    other heads are untouched."""
    L = 150 + q
    c = Case([q, 2], [L, 60], f8=f8, window=window, seed=q).gpu()
    o, lse = c.run()
    for at in (q // 2, q - 1):
        pos = L - q + at
        row = int(c.table[0, pos // PAGE]) * PAGE + pos % PAGE
        keep = [t.clone() if t is not None else None for t in (c.v, c.vs)]
        if f8:
            c.vs.view(torch.uint8)[row // PAGE, 2, row % PAGE] = 255
            c.v.view(torch.uint8)[row, 2] = 0x7F
        else:
            c.v[row, 2, 7] = value
        o2, lse2 = c.run()
        c.v, c.vs = keep
        sees = torch.zeros(q + 2, 64, dtype=torch.bool, device="cuda")
        sees[at:(min(q, at + window) if window else q), 16:24] = True
        assert bool(((lse - lse2).abs() <= 1e-4).all())
        assert torch.equal(o[~sees], o2[~sees])
        assert not bool(torch.isfinite(o2[sees][:, 7]).any())


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("q", [1, 5, 40])
def test_large_scores_and_moving_reference(q, f8):
    """Scores that rise along the keys by hundreds (the reference of a row
    moves again and again) and keys that differ by powers of two in size."""
    c = Case([q], [600], f8=False, seed=q).gpu()
    ramp = torch.linspace(0.05, 12.0, c.k.shape[0], device="cuda")
    j = torch.arange(600, device="cuda")
    rows = c.table[0].long()[j // PAGE] * PAGE + j % PAGE
    u = c.q[0, 0].float() / c.q[0, 0].float().norm()
    c.k[rows] = (u * ramp[:600, None, None] * 4 + 0.1 * c.k[rows].float()).to(torch.bfloat16)
    c.v[rows] = (c.v[rows].float() * torch.exp2((j % 23 - 11).float())[:, None, None]).to(torch.bfloat16)
    if f8:
        (c.k, c.ks), (c.v, c.vs) = quantise(c.k), quantise(c.v)
    c.check()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("q", [1, 4, 20])
def test_strided_queries(q, f8):
    """q as a slice of a wider projection, and an output the caller brings."""
    c = Case([q, q], [200, 90], f8=f8, seed=q + 1).gpu()
    o, lse = c.run()
    wide = torch.full((2 * q, 80, D), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[:, :64] = c.q
    c.q = wide[:, :64]
    out = torch.empty(2 * q, 64, D, dtype=torch.bfloat16, device="cuda")
    o2, lse2 = c.run(out=out)
    assert o2 is out and torch.equal(o, out) and torch.equal(lse, lse2)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("ql,kl", [([1] * 9, [3000] * 9), ([5, 2], [4000, 7]), ([200], [3000])])
def test_same_bits_again_and_on_another_stream(ql, kl, f8):
    """Keys split over CTAs are joined in their own order: repeated calls, calls
    on another stream and calls with a wrong idea of the longest chunk agree."""
    c = Case(ql, kl, f8=f8, seed=1).gpu()
    o, lse = c.check()
    for _ in range(3):
        o2, lse2 = c.run()
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o3, lse3 = c.run()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(o, o3) and torch.equal(lse, lse3)
    c.check(max_q=1)      # a longer chunk than the hint says
    c.check(max_q=5000)


def test_lengths_change_under_a_captured_graph():
    c = Case([3, 1, 2], [600, 90, 301], seed=9).gpu()
    ws = chunk.ChunkWorkspace("cuda")
    out = torch.empty_like(c.q)
    kw = dict(max_q=3, sinks=c.sinks, out=out, workspace=ws)
    args = (c.q, c.k, c.v, c.table, c.rows, c.q_start, c.kv_len)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        chunk.attend_chunks(*args, **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        chunk.attend_chunks(*args, **kw)
    for kl in ([600, 90, 301], [3, 600, 2], [17, 1, 128]):
        c.kl = kl
        c.kv_len.copy_(torch.tensor(kl, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        eo, _, tol = c.exact()
        assert ((out.double() - eo).abs() <= tol).all()
    assert ws.error() == 0


@pytest.mark.parametrize("f8", [False, True])
def test_pools_beyond_32_bit_offsets(f8):
    """Pages whose values lie more than 2^31 elements into the pool."""
    pages = (1 << 31) // (PAGE * 8 * D) + 64
    c = Case([2, 40], [50, 45], f8=f8, seed=2, ring=4)
    big = []
    for t, s in ((c.k, c.ks), (c.v, c.vs)):
        z = torch.zeros(pages * PAGE, 8, D, dtype=torch.uint8 if f8 else torch.bfloat16, device="cuda")
        z[-t.shape[0]:] = (t.view(torch.uint8) if f8 else t).cuda()
        codes = None
        if f8:
            z = z.view(torch.float8_e4m3fn)
            codes = torch.full((pages, 8, PAGE), 127, dtype=torch.uint8, device="cuda")
            codes[-s.shape[0]:] = s.view(torch.uint8).cuda()
            codes = codes.view(torch.float8_e8m0fnu)
        big.append((z, codes))
    c.gpu()
    o, lse = c.check()
    n = c.k.shape[0] // PAGE
    (c.k, c.ks), (c.v, c.vs) = big
    c.table = c.table + (pages - n)
    o2, lse2 = c.run()
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_pages_and_rows_outside_the_pool_are_not_read():
    c = Case([2, 1, 1], [100, 50, 40], seed=4).gpu()
    o, lse = c.run()
    c.rows[1] = 99                      # no such row of the table: the chunk sees nothing
    c.table[2, 3:] = 1 << 26            # pages the third sequence does not reach
    o2, lse2 = c.run()
    assert torch.equal(o[:2], o2[:2]) and torch.equal(o[3], o2[3]) and bool((o2[2] == 0).all())
    assert bool((lse2[2] == -math.inf).all())


def test_refusals():
    c = Case([2], [40], seed=1).gpu()
    f = Case([2], [40], f8=True, seed=1).gpu()
    args = (c.q, c.k, c.v, c.table, c.rows, c.q_start, c.kv_len)

    def no(match, *a, **kw):
        kw = {"max_q": 2, **kw}
        with pytest.raises((ValueError, _lib.GptossError), match=match):
            chunk.attend_chunks(*a, **kw)

    def but(i, t):
        return args[:i] + (t,) + args[i + 1:]

    no("q must be", *but(0, c.q.float()))
    no("q must be", *but(0, c.q.cpu()))
    no("heads and values must be dense", *but(0, c.q.transpose(0, 1)))
    no("multiple of 8 elements", *but(0, torch.zeros(2 * 4100, dtype=torch.bfloat16, device="cuda")
                                      .as_strided((2, 64, 64), (4100, 64, 1))))
    no("page pools are", *but(1, c.k[:-1]))
    no("differ in shape", *but(2, c.v[:PAGE]))
    no("bfloat16 or float8", c.q, c.k.half(), c.v.half(), *args[3:])
    no("need k_scale", c.q, f.k, f.v, *args[3:])
    no("scales of this pool", c.q, f.k, f.v, *args[3:], k_scale=f.ks[:1], v_scale=f.vs)
    no("no scales", *args, k_scale=f.ks, v_scale=f.vs)
    no("page_table", *but(3, c.table.long()))
    no("seq_rows", *but(4, c.rows.long()))
    no("q_start", *but(5, c.q_start[:1]))
    no("kv_len", *but(6, c.kv_len.cpu()))
    no("do not fit", *but(0, torch.zeros(2, 60, 64, dtype=torch.bfloat16, device="cuda")))
    no("sinks", *args, sinks=c.sinks.float())
    no("out must be", *args, out=torch.empty(2, 64, 64, device="cuda"))
    no("sm_scale", *args, sm_scale=0.0)
    no("sm_scale", *args, sm_scale=math.nan)
    no("max_q", *args, max_q=0)
    n = 1025
    no("0..1024 chunks", c.q, c.k, c.v, c.table, torch.zeros(n, dtype=torch.int32, device="cuda"),
       torch.zeros(n + 1, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"))
    assert torch.isfinite(c.run()[0]).all()  # and the context still works


def test_no_sequences_and_no_tokens():
    c = Case([2], [40], seed=1).gpu()
    e = torch.zeros(0, dtype=torch.int32, device="cuda")
    o = chunk.attend_chunks(c.q[:0], c.k, c.v, c.table, e, c.q_start[:1], e, max_q=1)
    assert o.shape == (0, 64, 64)


# Few short chunks share a kernel with the long ones; with many sequences they have their own.
def many(q, window, f8, n=24, ring=None):
    g = torch.Generator().manual_seed(100 * q + window)
    ql = [q] + torch.randint(0, q + 1, (n - 1,), generator=g).tolist()
    kl = [150 + q] + [max(a + b, 0) for a, b in zip(ql[1:], torch.randint(-2, 400, (n - 1,), generator=g).tolist())]
    return Case(ql, kl, window=window, f8=f8, seed=q + window, ring=ring).gpu()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("window", [0, 1, 100])
@pytest.mark.parametrize("q", [1, 2, 3, 4, 5, 6, 7, 8, 9])
def test_many_sequences(q, window, f8):
    many(q, window, f8).check()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("q,window", [(2, 0), (4, 0), (6, 100), (8, 0), (8, 20)])
def test_many_sequences_hidden_and_not_finite(q, window, f8):
    """Hidden keys of the first sequence change no bit; a value that is not
    finite makes the rows that see it NaN and leaves all others their bits."""
    c = many(q, window, f8, ring=30)
    o, lse = c.check()
    L = 150 + q
    j = torch.arange(30 * PAGE, device="cuda")
    hidden = (j >= L) | (j < (L - q - window + 1 if window else 0))
    rows = (c.table[0].long()[j // PAGE] * PAGE + j % PAGE)[hidden]
    for t, s in ((c.k, c.ks), (c.v, c.vs)):
        if f8:
            t.view(torch.uint8)[rows] = 0x7F
            s.view(torch.uint8)[rows // PAGE, :, rows % PAGE] = 255
        else:
            t[rows] = math.nan
    o2, lse2 = c.run()
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    at = q // 2
    row = int(c.table[0, (L - q + at) // PAGE]) * PAGE + (L - q + at) % PAGE
    if f8:
        c.vs.view(torch.uint8)[row // PAGE, 2, row % PAGE] = 255
    else:
        c.v[row, 2, 7] = math.inf
    o2, lse2 = c.run()
    sees = torch.zeros(o.shape[:2], dtype=torch.bool, device="cuda")
    sees[at:(min(q, at + window) if window else q), 16:24] = True
    assert torch.equal(o[~sees], o2[~sees]) and bool(((lse - lse2).abs()[torch.isfinite(lse)] <= 1e-4).all())
    assert not bool(torch.isfinite(o2[sees][:, 7]).any())


@pytest.mark.parametrize("hq,hkv,q", [(8, 8, 20), (12, 4, 14), (10, 2, 8), (64, 1, 1), (40, 8, 6)])
@pytest.mark.parametrize("f8", [False, True])
def test_many_sequences_head_groups(hq, hkv, q, f8):
    Case([q] * 40, [q + 7 * b for b in range(40)], hq=hq, hkv=hkv, f8=f8, seed=hq + q).gpu().check()


@pytest.mark.parametrize("q", [1, 4, 40])
def test_infinite_scores_make_their_rows_nan(q):
    """A key of +infinity in one dim: the rows with a positive query there have an infinite score, and
    infinity - infinity is no number; those with a negative one do not weigh it at all."""
    c = Case([q], [200], seed=q).gpu()
    pos = 200 - q   # every token sees it
    row = int(c.table[0, pos // PAGE]) * PAGE + pos % PAGE
    before = c.k[row, 3].clone()
    c.k[row, 3, 9] = math.inf
    o, lse = c.run()
    up = torch.zeros(q, 64, dtype=torch.bool, device="cuda")
    up[:, 24:32] = c.q[:, 24:32, 9] > 0
    assert bool(torch.isnan(o[up]).all()) and bool(torch.isfinite(o[~up]).all())
    c.k[row, 3] = before
    c.check()
