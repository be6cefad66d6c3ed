"""Chunk attention where its number formats end: weights far below a row's
largest, queries and scores that are not finite, windows beyond every key."""
import importlib
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from test_chunk_gpu import Case, D, PAGE, dequantise, quantise  # noqa: E402

chunk = importlib.import_module("gpt-oss-tvm_b200.chunk")


def one_context(n, q, k, v, f8, hq=64):
    """A Case of n sequences that share one context, k and v [positions, heads, 64] bf16, q new tokens each."""
    length, hkv, _ = k.shape
    c = Case([q] * n, [length] * n, hq=hq, hkv=hkv, sinks=False, ring=1)
    c.stride = length // PAGE
    c.table = torch.arange(c.stride, dtype=torch.int32).repeat(n, 1)
    c.k, c.v = k, v
    if f8:
        (c.k, c.ks), (c.v, c.vs) = quantise(k), quantise(v)
    return c


# 8 bits: P is two e4m3 terms in units that a row's largest weight sets to 2^3.5, and that follow a key tile's largest
# down when it is below 1.  A term's rounding leaves 2^-8 of P, the 16-bit value that is split 2^-11, and what is too
# small for a term's normal range 2^-14.8 of a unit: 2^-18.3 of the row's largest, for each key of a tile (256 at most) until
# the units have followed.  bf16: 2^-9 of P.
SPLIT = 1.02 * (2.0 ** -8 + 2.0 ** -11)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("v0", [-1.0, -16.0])
@pytest.mark.parametrize("length", [8192, 32768])
@pytest.mark.parametrize("q", [1, 4, 6, 8])
def test_a_dominant_key_before_a_long_tail(q, length, v0, f8):
    """One key 7 to 16 nats above thousands of equal ones, whose small weights
    are together as large as its own; 16, 32, 48 and 64 rows a unit."""
    for nats in (7.0, 8.0, 9.0, 10.0, 12.0, 16.0):
        k, v = torch.zeros(length, 8, D), torch.ones(length, 8, D)
        k[0], v[0] = nats / 8.0, v0
        c = one_context(24, q, k.bfloat16(), v.bfloat16(), f8)
        c.q = torch.ones_like(c.q)
        o, _ = c.gpu().run()
        for i in range(q):
            tail, top = length - q + i, math.exp(nats)
            den = top + tail
            exact = (v0 * top + tail) / den
            tiles = 2 * 256 * 2.0 ** -18 * (top * abs(v0) + tail / 128) / den
            tol = SPLIT * (abs(v0) * top + tail) / den + tiles + 2.0 ** -9 * abs(exact) + 2e-6
            worst = (o[i::q].double() - exact).abs().max().item()
            assert worst <= tol, f"{nats} nats, token {i}: {worst:.3e} off, {tol:.3e} allowed"


@pytest.mark.parametrize("q", [1, 4, 6, 8, 40])
@pytest.mark.parametrize("low", [6.0, 40.0, 90.0])
def test_key_tiles_of_very_different_weight(q, low):
    """Blocks of keys up to `low` nats below the largest, in no order, so that a
    row's units move up and down: 2^-8 of each key's own weight and 2^-18 of the
    row's largest (times 2, by which a V row's values may differ from its power
    of two)."""
    g = torch.Generator().manual_seed(int(low) + q)
    length, n = 3200, 24 if q < 40 else 2
    off = (torch.rand(length // 32, generator=g) * -low).repeat_interleave(32)
    off[0] = 3.0  # one key on top of all
    k = torch.randn(length, 8, D, generator=g) * 0.5
    k[:, :, :8] = off[:, None, None]
    v = torch.randn(length, 8, D, generator=g) + 1.0
    c = one_context(n, q, k.bfloat16(), v.bfloat16(), True)
    c.q = torch.randn(c.q.shape, generator=g).bfloat16()
    c.q[..., :8] = 1.0
    c.gpu()
    o, lse = c.run()
    kk, vv = dequantise(c.k, c.ks), dequantise(c.v, c.vs)
    rep = 64 // 8
    for b in range(0, n, max(1, n // 4)):
        for i in range(q):
            m = length - q + i + 1
            kr, vr = kk[:m].repeat_interleave(rep, 1), vv[:m].repeat_interleave(rep, 1)
            s = torch.einsum("hd,jhd->hj", c.q[b * q + i].double(), kr) / 8.0
            p = torch.softmax(s, -1)
            exact = torch.einsum("hj,jhd->hd", p, vr)
            av = torch.einsum("hj,jhd->hd", p, vr.abs())
            top = (p * vr.abs().amax(-1).t()).amax(-1)
            # Q's terms move a score by 2^-18 of the largest product, below 2^-11 in base e
            tol = (SPLIT + 2.0 ** -11) * av + (2 * m * 2.0 ** -18) * top[:, None] + 2.0 ** -9 * exact.abs() + 2e-6
            over = ((o[b * q + i].double() - exact).abs() - tol).max().item()
            assert over <= 0, f"o is {over:.3e} beyond its tolerance"
            want = torch.logsumexp(s, -1) / math.log(2.0)
            assert (lse[b * q + i].double() - want).abs().max().item() <= 5e-4


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("q", [1, 4, 5, 6, 8, 40])
def test_a_query_that_is_not_finite_stays_with_its_row(q, value):
    """8 bits: the rows of a unit share one scale for their queries, which the
    finite values alone decide: the other rows keep their bits, also when one of
    them is the largest by far."""
    c = Case([q] * 24, [200] * 24, f8=True, seed=q).gpu()
    big = q * 8 - 1 if q < 5 else 32   # row of the unit: token, head of the group
    c.q[big // 8, big % 8] *= 2.0 ** 10
    o, lse = c.run()
    assert bool(torch.isfinite(o).all())
    c.q[0, 0, ::2] = value
    o2, lse2 = c.run()
    assert bool(torch.isnan(o2[0, 0]).all())
    o2[0, 0], lse2[0, 0] = o[0, 0], lse[0, 0]
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("n", [1, 24])
@pytest.mark.parametrize("q", [1, 2, 4, 6, 8, 40])
def test_scores_of_minus_infinity_weigh_nothing(q, n):
    """Every key of the first tiles scores -infinity: those keys weigh nothing.
    A row that has no other key gets zeros and an lse of -infinity, whichever
    kernel runs."""
    length = 700
    c = Case([q] * n, [length] * n, seed=q).gpu()
    j = torch.arange(512, device="cuda")
    rows = torch.cat([c.table[b].long()[j // PAGE] * PAGE + j % PAGE for b in range(n)])
    c.k[rows] = 0
    c.k[rows, :, 9] = -math.inf
    c.q[..., 9] = c.q[..., 9].abs() + 0.1
    o, lse = c.run()
    # the same call without those keys: a window that ends behind them (less for the chunk's later tokens)
    assert bool(torch.isfinite(o).all()) and bool(torch.isfinite(lse).all())
    w = Case([q] * n, [length] * n, seed=q).gpu()
    w.q = c.q
    exact_k = w.k.clone()
    exact_k[rows] = 0
    exact_k[rows, :, 9] = -1000.0 / 0.1  # 1250 nats below: no weight in 64 bits either
    w.k = exact_k.to(torch.bfloat16)
    eo, el, tol = w.exact()
    assert bool(((o.double() - eo).abs() <= tol).all())
    assert (lse.double() - el).abs().max().item() <= 1e-4
    c.kv_len.fill_(300)
    c.kl = [300] * n
    c.k[...] = 0
    c.k[..., 9] = -math.inf
    o, lse = c.run()
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("n", [1, 24])
@pytest.mark.parametrize("q", [1, 4, 8, 40])
def test_scores_of_minus_infinity_in_8_bits(q, n):
    """8-bit keys are finite; queries and keys of 2^60 and more bring their
    product beyond fp32."""
    c = Case([q] * n, [300] * n, f8=False, seed=q).gpu()
    c.k[...] = 0
    c.k[..., 9] = -(2.0 ** 68)
    c.q[...] = 0
    c.q[..., 9] = 2.0 ** 70
    (c.k, c.ks), (c.v, c.vs) = quantise(c.k), quantise(c.v)
    o, lse = c.run()
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())


def captured(c, out):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        chunk.attend_chunks(c.q, c.k, c.v, c.table, c.rows, c.q_start, c.kv_len, max_q=max(c.ql), sinks=c.sinks,
                            k_scale=c.ks, v_scale=c.vs, out=out)
    return g


@pytest.mark.parametrize("f8", [False, True])
def test_captured_calls_without_a_workspace_are_their_own(f8):
    """Each captured call brings its memory and its zeros: graphs replay in any
    order, at the same time on two streams, and leave nothing to later calls."""
    known = set(chunk._workspaces)
    a, b = Case([4, 1], [5000, 30], f8=f8, seed=1).gpu(), Case([300], [5200], f8=f8, seed=2).gpu()
    for x in (a, b):
        x.run()
    torch.cuda.synchronize()
    eager = set(chunk._workspaces)
    oa, ob = torch.empty_like(a.q), torch.empty_like(b.q)
    ga, gb = captured(a, oa), captured(b, ob)
    # whatever the memory of a workspace held that a capture left behind
    for key in set(chunk._workspaces) - eager - known:
        chunk._workspaces[key].buf.fill_(0xFF)
    wa, wb = a.run()[0], b.run()[0]
    s = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(20):
        oa.fill_(math.nan)
        ob.fill_(math.nan)
        torch.cuda.synchronize()
        for g, st in ((gb, s[1]), (ga, s[0]))[::1 if rep % 2 else -1]:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(ob, wb) and torch.equal(oa, wa), f"replay {rep}"
    assert set(chunk._workspaces) == eager | known


def test_a_workspace_is_not_made_under_capture():
    """Its zeros would be a node of that graph, run only when that graph is."""
    t = torch.zeros(4, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="captur"):
            chunk.ChunkWorkspace("cuda")
        t.add_(1)
    g.replay()
    assert float(t[0]) == 1.0


def test_a_model_s_scratch_has_no_workspace_of_a_capture():
    att = importlib.import_module("gpt-oss-tvm_b200.attention")
    scratch, t, g = att.DecodeScratch("cuda"), torch.zeros(4, device="cuda"), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t.add_(1)
        assert scratch.chunk() is None
    ws = scratch.chunk()
    assert isinstance(ws, chunk.ChunkWorkspace) and ws.error() == 0 and scratch.chunk() is ws


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 128, 2 ** 30, 4097])
@pytest.mark.parametrize("ql,kl", [([1], [300]), ([5], [260]), ([6] * 24, [130 + b for b in range(24)]),
                                   ([6] * 3, [130, 200, 300]), ([4] * 5, [4, 130, 129, 300, 255]),
                                   ([40, 3], [290, 290]), ([400] * 3, [401, 700, 400])])
def test_a_window_beyond_every_key_is_none(ql, kl, window, f8):
    c = Case(ql, kl, f8=f8, seed=len(ql), window=0).gpu()
    o, lse = c.run()
    o2, lse2 = c.run(window=window)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("kv_dtype", ["float8_e4m3", "bfloat16"])
def test_more_sequences_than_one_call_takes(kv_dtype):
    """A layer over 1030 sequences: a decode step (8 bit) and a chunk each, against
    the same layer over the first and the last of them alone."""
    att, cfgm = (importlib.import_module("gpt-oss-tvm_b200." + n) for n in ("attention", "config"))
    cfg = cfgm.GPTOssConfig(num_hidden_layers=2, num_experts=16, vocab_size=64, context_window_size=1024)
    n, g = chunk.MAX_CHUNKS + 6, torch.Generator(device="cuda").manual_seed(1)
    block = att.AttentionBlock(cfg, layer_idx=1)
    for w in (block.qkv_weight, block.out_weight):
        w.copy_(torch.randn(w.shape, generator=g, device="cuda") * 0.02)
    x = [torch.randn(1, n, cfg.hidden_size, generator=g, device="cuda").bfloat16().cpu() for _ in range(2)]
    picked = [0, 1, chunk.MAX_CHUNKS - 1, chunk.MAX_CHUNKS, n - 1]

    def steps(rows):
        c = att.KVCache(cfg, len(rows), 32, 2, kv_dtype=kv_dtype, max_chunk=2)
        out = []
        for i, t in enumerate(x):
            ids = list(range(len(rows)))
            if i and c.f8:
                pos, mode = c.begin_forward(ids, [1] * len(rows)), "decode"
            else:
                pos, mode = c.begin_chunks(ids, [1] * len(rows)), "chunk"
            y = block.forward(t[:, rows].cuda(), c, pos, mode)[0]
            out.append(y.float().cpu().reshape(len(rows), cfg.hidden_size))
        return out

    tol = 2e-2  # bf16 attention and projections, as in the tests of the layers
    for many, few in zip(steps(list(range(n))), steps(picked)):
        assert many.shape == (n, cfg.hidden_size)
        assert float((many[picked] - few).abs().max()) <= tol * float(few.abs().max())


@pytest.mark.parametrize("nats", [5.0, 70.0, 140.0])
@pytest.mark.parametrize("q", [1, 4, 6])
def test_values_of_zero_on_top(q, nats):
    """8 bits: rows of zeros have the smallest power of two, which P takes in and
    the sum takes out again, 2^60 of it: keys with such rows far above all others,
    before and between them."""
    length = 4000
    k, v = torch.zeros(length, 8, D), torch.ones(length, 8, D)
    top = torch.zeros(length, dtype=torch.bool)
    top[:300], top[2000:2010] = True, True
    k[top], v[top] = nats / 8.0, 0.0
    c = one_context(24, q, k.bfloat16(), v.bfloat16(), True)
    c.q = torch.ones_like(c.q)
    nats = 8 * float(dequantise(c.k, c.ks)[0, 0, 0])  # as the pages hold the key
    o, lse = c.gpu().run()
    for i in range(q):
        m = length - q + i + 1 - 310
        den = 310 * math.exp(nats) + m
        assert (o[i::q].double() - m / den).abs().max().item() <= (SPLIT + 2.0 ** -9) * m / den + 1e-6
        assert (lse[i::q].double() - math.log2(den)).abs().max().item() <= 5e-4
