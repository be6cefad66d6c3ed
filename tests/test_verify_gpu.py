"""Draft verification (gptoss_verify_drafts) against the definition in 64 bits.

An accept test is u q < p with p within 1e-5 of itself of the exact softmax
(fp32 exp and division, weights in steps of 2^-40 of the largest over up to
2 x 10^5 values: 2 x 10^5 * 2^-40 < 2e-7 in all); the draws are made so that no
test lies nearer than 1e-4 to its threshold.  A drawn token's exact cumulative
interval must hold the draw to within 1e-4 of the whole."""
import importlib
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

verify = importlib.import_module("gpt-oss-tvm_b200.verify")
_lib = importlib.import_module("gpt-oss-tvm_b200._lib")


def make(counts, V, seed, probs, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, n = sum(counts), len(counts)
    z = (torch.randn(T, V, generator=g, device="cuda") * 2).to(dtype)
    q = torch.softmax(z.float() + torch.randn(T, V, generator=g, device="cuda"), -1) if probs else None
    tok = torch.randint(0, V, (T,), generator=g, device="cuda")
    if T > 1:
        tok[1:] = (q if probs else torch.softmax(z.float(), -1))[:-1].multinomial(1, generator=g)[:, 0]
    start = [0]
    for c in counts:
        start.append(start[-1] + c)
    return (z, tok.to(torch.int32), torch.tensor(start, dtype=torch.int32, device="cuda"),
            torch.rand(T, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda"), q)


def check(z, tok, start, ua, un, q, temperature):
    T, V = z.shape
    p = torch.softmax(z.double() / temperature, -1)
    st = start.tolist()
    # no accept test on the edge: move its draw away
    if T > 1:
        x = tok[1:].long()
        thr = p[:-1].gather(1, x[:, None])[:, 0] / (q[:-1].gather(1, x[:, None])[:, 0].double() if q is not None else 1.0)
        near = (ua[:-1].double() - thr).abs() < 1e-4
        ua[:-1][near] = torch.where(thr[near] > 0.5, thr[near] - 0.25, thr[near] + 0.25).float()
    acc, nxt = verify.verify_drafts(z, tok, start, ua, un, temperature=temperature, draft_probs=q)
    for b in range(len(st) - 1):
        r0, r1 = st[b], st[b + 1]
        if r1 <= r0:
            assert int(acc[b]) == 0 and int(nxt[b]) == -1
            continue
        a = 0
        while a < r1 - r0 - 1:
            x = int(tok[r0 + a + 1])
            qx = float(q[r0 + a, x]) if q is not None else 1.0
            if not float(ua[r0 + a]) * qx < float(p[r0 + a, x]):
                break
            a += 1
        assert int(acc[b]) == a, f"sequence {b}"
        w = p[r0 + a].clone()
        if a < r1 - r0 - 1:
            if q is not None:
                w = (w - q[r0 + a].double()).clamp(min=0)
            else:
                w[int(tok[r0 + a + 1])] = 0
        c = torch.cumsum(w, 0) / w.sum()
        t = int(nxt[b])
        assert 0 <= t < V and float(w[t]) > 0
        u = float(un[b])
        lo, hi = (float(c[t - 1]) if t else 0.0), float(c[t])
        assert lo - 1e-4 <= u <= hi + 1e-4, (b, t, lo, u, hi)


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("V", [1, 2, 33, 255, 256, 257, 1000, 5003, 50257])
def test_against_the_definition(V, probs):
    if V == 1 and probs:
        pytest.skip("one token: nothing is left to draw from")
    for seed, t in ((0, 1.0), (1, 0.6)):
        check(*make([1, 4, 2, 1, 6], V, seed, probs), t)


@pytest.mark.parametrize("probs", [False, True])
def test_full_vocabulary(probs):
    check(*make([5, 3], 201088, 3, probs), 0.7)


def test_bf16_logits_and_strided_rows():
    z, tok, start, ua, un, _ = make([3, 4], 1000, 5, False, torch.bfloat16)
    check(z, tok, start, ua, un, None, 1.0)
    wide = torch.zeros(7, 1003, dtype=torch.bfloat16, device="cuda")
    wide[:, :1000] = z
    a = verify.verify_drafts(z, tok, start, ua, un)
    b = verify.verify_drafts(wide[:, :1000], tok, start, ua, un)
    f = verify.verify_drafts(z.float(), tok, start, ua, un)
    for y in (b, f):
        assert torch.equal(a[0], y[0]) and torch.equal(a[1], y[1])


@pytest.mark.parametrize("V", [7, 300, 201088])
def test_greedy_takes_the_lowest_index(V):
    z = torch.zeros(6, V, device="cuda")
    z[0, [V - 1, 3]] = 5.0          # a tie: 3
    z[1, 2] = 1.0
    z[2, 4] = math.inf
    z[3] = -math.inf                # all the same: 0
    z[4, V - 2] = 7.0
    z[5, 5] = math.nan              # counts as -inf: 0
    tok = torch.tensor([1, 3, 2, 4, 0, 6], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")
    acc, nxt = verify.verify_drafts(z, tok, start, temperature=0.0)
    # rows 0, 1 accept 3 and 2, row 2 gives 4; row 3 accepts 0, row 4 has V - 2 and not 6
    assert acc.tolist() == [2, 1] and nxt.tolist() == [4, V - 2]


def test_certain_draws():
    """u = 0 accepts whatever has weight, u near 1 takes the last token with weight; drafts outside the vocabulary
    or without weight are not accepted."""
    V = 100
    z = torch.full((4, V), -math.inf, device="cuda")
    z[:, 10], z[:, 20] = 0.0, 0.0
    start = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    zero, one = torch.zeros(4, device="cuda"), torch.full((1,), 1 - 2.0 ** -24, device="cuda")
    for tok, acc, nxt in (([0, 10, 20, 10], 3, 20), ([0, 10, 30, 10], 1, 20), ([0, -5, 10, 10], 0, 20),
                          ([0, V, 10, 10], 0, 20), ([0, 20, 20, 11], 2, 20)):
        a, t = verify.verify_drafts(z, torch.tensor(tok, dtype=torch.int32, device="cuda"), start, zero, one)
        assert (int(a[0]), int(t[0])) == (acc, nxt)
    # the only token with weight is rejected: the row's own weights are what is left
    z[:, 20] = -math.inf
    a, t = verify.verify_drafts(z, torch.tensor([0, 10, 10, 10], dtype=torch.int32, device="cuda"), start,
                                torch.ones(4, device="cuda"), one)
    assert (int(a[0]), int(t[0])) == (0, 10)
    # nothing left of p - q: p itself
    q = torch.zeros(4, V, device="cuda")
    q[:, 10] = 1.0
    a, t = verify.verify_drafts(z, torch.tensor([0, 10, 10, 10], dtype=torch.int32, device="cuda"), start,
                                torch.ones(4, device="cuda"), one, draft_probs=q)
    assert (int(a[0]), int(t[0])) == (0, 10)


@pytest.mark.parametrize("value,want", [(math.nan, 3), (-math.inf, 3), (math.inf, 6)])
def test_values_that_are_no_numbers(value, want):
    z = torch.full((1, 9), -math.inf, device="cuda")
    z[0, 3] = 1.0
    z[0, 6] = value
    a, t = verify.verify_drafts(z, torch.zeros(1, dtype=torch.int32, device="cuda"),
                                torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.zeros(1, device="cuda"),
                                torch.full((1,), 0.5, device="cuda"))
    assert (int(a[0]), int(t[0])) == (0, want)


def test_empty_sequences_and_no_rows():
    z, tok, start, ua, un, _ = make([2, 0, 3], 500, 1, False)
    check(z, tok, start, ua, un, None, 1.0)
    e = torch.zeros(0, device="cuda")
    acc, nxt = verify.verify_drafts(torch.zeros(0, 50, device="cuda"), e.int(),
                                    torch.zeros(3, dtype=torch.int32, device="cuda"), e, torch.zeros(2, device="cuda"))
    assert acc.tolist() == [0, 0] and nxt.tolist() == [-1, -1]


def test_accepts_with_the_right_frequency():
    """Many independent sequences of one draft from q: the token that comes out
    (the draft or its replacement) is distributed as p.  4000 draws of 5 values:
    a frequency is within 4.5 standard deviations, sqrt(p (1 - p) / 4000)."""
    n, V = 4000, 5
    g = torch.Generator(device="cuda").manual_seed(11)
    p = torch.tensor([0.4, 0.05, 0.25, 0.2, 0.1], device="cuda")
    q = torch.tensor([0.1, 0.3, 0.3, 0.05, 0.25], device="cuda")
    z = p.log().repeat(2 * n, 1)
    tok = torch.zeros(2 * n, dtype=torch.int32, device="cuda")
    tok[1::2] = q.multinomial(n, replacement=True, generator=g).to(torch.int32)
    start = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda")
    acc, nxt = verify.verify_drafts(z, tok, start, torch.rand(2 * n, generator=g, device="cuda"),
                                    torch.rand(n, generator=g, device="cuda"), draft_probs=q.repeat(2 * n, 1))
    first = torch.where(acc > 0, tok[1::2], nxt)
    f = torch.bincount(first.long(), minlength=V).double() / n
    assert bool(((f - p.double()).abs() <= 4.5 * (p * (1 - p) / n).sqrt().double()).all())


def test_refusals():
    z, tok, start, ua, un, q = make([2, 3], 50, 1, True)
    bad = (ValueError, _lib.GptossError)
    for match, a, kw in [
        ("logits must be", (z.half(), tok, start, ua, un), {}),
        ("logits must be", (z.cpu(), tok, start, ua, un), {}),
        ("must be dense", (z.t().contiguous().t(), tok, start, ua, un), {}),
        ("tokens", (z, tok.long(), start, ua, un), {}),
        ("tokens", (z, tok[:4], start, ua, un), {}),
        ("row_start", (z, tok, start.long(), ua, un), {}),
        ("accept_draws", (z, tok, start, None, un), {}),
        ("accept_draws", (z, tok, start, ua.double(), un), {}),
        ("next_draws", (z, tok, start, ua, un[:1]), {}),
        ("draft_probs", (z, tok, start, ua, un), {"draft_probs": q[:, :40]}),
        ("temperature", (z, tok, start, ua, un), {"temperature": math.nan}),
        ("temperature", (z, tok, start, ua, un), {"temperature": math.inf}),
        ("temperature", (z, tok, start, ua, un), {"temperature": -1.0}),
    ]:
        with pytest.raises(bad, match=match):
            verify.verify_drafts(*a, **kw)


def test_one_row_has_dense_values_too():
    """Every second value of a row, or a column as a row, is refused for a single
    row as for many: the kernel reads values one after another."""
    z, tok, start, ua, un, q = make([1], 64, 2, True)
    wide, tall = torch.randn(1, 128, device="cuda"), torch.randn(64, 3, device="cuda").softmax(0)
    ok = verify.verify_drafts(z, tok, start, ua, un, draft_probs=q)
    assert ok[0].tolist() == [0]
    for view in (wide[:, ::2], tall[:, 1:2].t(), wide[:, :1].expand(1, 64)):
        with pytest.raises(ValueError, match="must be dense"):
            verify.verify_drafts(view, tok, start, ua, un)
        with pytest.raises(ValueError, match="draft_probs"):
            verify.verify_drafts(z, tok, start, ua, un, draft_probs=view)
    # what no stride of one entry says: a dense row, however it came about
    row = wide[:, :64].as_strided((1, 64), (7, 1))
    a, b = verify.verify_drafts(row, tok, start, ua, un), verify.verify_drafts(row.contiguous(), tok, start, ua, un)
    assert torch.equal(a[1], b[1])
    one = torch.zeros(2, 5, device="cuda")[:, 2:3]   # a vocabulary of one
    t2 = torch.zeros(2, dtype=torch.int32, device="cuda")
    a = verify.verify_drafts(one, t2, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), temperature=0.0)
    assert a[0].tolist() == [1] and a[1].tolist() == [0]


@pytest.mark.parametrize("temperature", [1e30, 1e46, 1e300])
def test_a_temperature_that_levels_everything(temperature):
    """Weights of 1 for every finite logit, none for -infinity."""
    V = 600
    z = torch.randn(3, V, generator=torch.Generator().manual_seed(1)).cuda()
    z[:, ::2] = -math.inf
    tok = torch.tensor([0, 7, 4], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    u = torch.tensor([0.002, 0.002, 0.5], device="cuda")  # p is 1/300
    for un in (0.0, 0.25, 0.9999):
        # token 7 stands (0.002 < 1/300), token 4 has no weight; the next is one of the odd ones, each as likely
        a, t = verify.verify_drafts(z, tok, start, u, torch.tensor([un], device="cuda"), temperature=temperature)
        assert (int(a[0]), int(t[0])) == (1, 2 * int(un * 300) + 1)


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("V,dtype", [(500003, torch.float32), (1 << 20, torch.bfloat16), (1 << 22, torch.float32)])
def test_vocabularies_beyond_what_stays_on_chip(V, dtype, probs):
    """A row's part of a CTA no longer fits shared memory: the logits are read
    twice.  (Weights in steps of 2^-40 of the largest over 2^22 values: 4e-6.)"""
    z, tok, start, ua, un, q = make([2, 3], V, 7, probs, dtype)
    check(z, tok, start, ua, un, q, 0.9)
    tok[3] = 3
    z[2, 7] = 50.0
    z[0, V - 3], z[0, 5], z[3, V - 1] = 50.0, 50.0, 50.0   # greedy: the lowest index of a tie, the last value of a row
    tok[1], tok[4] = 5, 0
    acc, nxt = verify.verify_drafts(z, tok, start, temperature=0.0)
    first = [int((row == row.max()).nonzero()[0, 0]) for row in z]
    assert first[0] == 5 and first[3] == V - 1 and first[2] != int(tok[3])
    assert acc.tolist() == [1, 0] and nxt.tolist() == [first[1], first[2]]
