"""The 8-bit KV cache: quantised as it is written (gptoss_qkv_rope_append_f8,
gptoss_kv_pages_copy_f8) and read back.  Values and codes are exact: they are
compared with the definition, computed in 64 bits from the same bf16 rows."""
import importlib
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import gpu_util as G  # noqa: E402

chunk = importlib.import_module("gpt-oss-tvm_b200.chunk")
_lib = importlib.import_module("gpt-oss-tvm_b200._lib")
D, PAGE = 64, 16
# the e4m3 values >= 0 in order, from the format: 4 exponent bits (bias 7), 3 of mantissa, 0x7F is NaN
E4M3 = np.array([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
                 for e in range(16) for m in range(8)][:127])


def definition(x):
    """bf16 rows [..., 64] (tensor) -> (value bytes, codes), by the definition in 64 bits."""
    v = x.double().cpu().numpy()
    a = np.abs(v).max(-1)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.full(a.shape, -60.0)
        for k in range(59, -61, -1):  # the smallest exponent whose reach is enough
            e[a > 448.0 * 2.0 ** k] = np.maximum(e[a > 448.0 * 2.0 ** k], k + 1)
        s = v * np.exp2(-e)[..., None]
        mag = np.minimum(np.abs(s), 448.0)
        hi = np.clip(np.searchsorted(E4M3, mag), 1, 126)
        lo = hi - 1
        down, up = mag - E4M3[lo], E4M3[hi] - mag
        near = np.where(down < up, lo, np.where(up < down, hi, np.where(lo % 2 == 0, lo, hi)))
    bits = np.where(np.signbit(v), near + 128, near).astype(np.uint8)
    nan = np.isnan(v).any(-1)
    code = np.where(nan, 255, e + 127).astype(np.uint8)
    return bits, code, nan


def same_bytes(got, want, nan):
    """Byte for byte, but for rows with a NaN, whose values say nothing."""
    g = got.view(torch.uint8).cpu().numpy()
    assert np.array_equal(g[~nan], want[~nan])


def rows_of(t, slots):
    return t.view(torch.uint8)[slots.long()]


def codes_of(s, slots):
    return s.view(torch.uint8)[slots.long() // PAGE, :, slots.long() % PAGE].cpu().numpy()


@pytest.mark.parametrize("T,hq,hkv", [(1, 64, 8), (3, 64, 8), (37, 40, 8), (130, 6, 2), (5, 3, 1), (1500, 8, 8)])
def test_rope_append(T, hq, hkv):
    g = torch.Generator(device="cuda").manual_seed(T)
    pages = -(-T // PAGE) + 2
    qkv = torch.randn(T, (hq + 2 * hkv) * D, generator=g, device="cuda").to(torch.bfloat16)
    qkv *= torch.exp2(torch.randint(-20, 20, (T, 1), generator=g, device="cuda").float()).to(torch.bfloat16)
    pos = torch.randint(0, 131072, (T,), generator=g, device="cuda").to(torch.int32)
    slots = torch.randperm(pages * PAGE, generator=g, device="cuda")[:T].to(torch.int32)
    inv = torch.tensor([150000.0 ** (-2 * i / D) for i in range(32)])
    (k, ks), (v, vs) = chunk.f8_pool(pages, hkv), chunk.f8_pool(pages, hkv)
    q = chunk.rope_append_f8(qkv, pos, slots, hq, inv, 1.3466, k, v, ks, vs)
    # the bf16 cache's append, whose rows are what is quantised
    q0 = torch.empty(T, hq, D, dtype=torch.bfloat16, device="cuda")
    k0 = torch.zeros(pages * PAGE, hkv, D, dtype=torch.bfloat16, device="cuda")
    v0 = torch.zeros_like(k0)
    G.call("gptoss_qkv_rope_append", G.P(qkv), G.P(pos), G.P(slots), T, hq, hkv, D, inv.data_ptr(), 1.3466, G.P(q0),
           G.P(k0), G.P(v0), G.S())
    assert torch.equal(q, q0)
    for t, s, t0 in ((k, ks, k0), (v, vs, v0)):
        bits, code, nan = definition(t0[slots.long()])
        same_bytes(rows_of(t, slots), bits, nan)
        assert np.array_equal(codes_of(s, slots), code)
        # nothing else was written
        rest = torch.ones(pages * PAGE, dtype=torch.bool, device="cuda")
        rest[slots.long()] = False
        assert bool((t.view(torch.uint8)[rest] == 0).all())


def special_rows():
    x = torch.zeros(16, 2, D)
    x[0, 0, 3] = 448.0                       # the top of the range, exponent 0
    x[1, 0, 3] = 450.0                       # one bf16 step above: exponent 1
    x[2, 0] = torch.linspace(-2.0, 2.0, D)
    x[3, 0, 0] = math.nan
    x[4, 0, 5] = math.inf
    x[5, 0, 5] = -math.inf
    x[6, 0, 1] = 3.0e38                      # beyond 448 * 2^60: saturates
    x[7, 0, 1] = 1e-30                       # below the smallest exponent
    x[8, 0] = 2.0 ** -133                    # the smallest subnormal bf16
    x[9, 0] = -0.0
    x[10, 0, :4] = torch.tensor([17.0, 19.0, 18.0, 1.0]) / 16  # ties to even
    x[10, 0, 4] = 448.0
    x[11, 0] = 1.0
    x[:, 1] = torch.randn(16, D, generator=torch.Generator().manual_seed(1))
    return x.to(torch.bfloat16).cuda()


def test_write_and_read_back_special_values():
    x = special_rows()
    (k, ks), (v, vs) = chunk.f8_pool(3, 2), chunk.f8_pool(3, 2)
    table = torch.tensor([[0, 0], [2, 1]], dtype=torch.int32, device="cuda")
    chunk.write_pages_f8(x, -x, k, v, ks, vs, table, 1, 5)
    j = torch.arange(5, 21, device="cuda")
    slots = table[1].long()[j // PAGE] * PAGE + j % PAGE
    for t, s, y in ((k, ks, x), (v, vs, -x)):
        bits, code, nan = definition(y)
        same_bytes(rows_of(t, slots), bits, nan)
        assert np.array_equal(codes_of(s, slots), code)
    rk, rv = chunk.read_pages_f8(k, v, ks, vs, table, 1, 5, 16)
    for got, y in ((rk, x), (rv, -x)):
        bits, code, nan = definition(y)
        want = np.where(bits < 128, 1, -1) * E4M3[np.minimum(bits & 127, 126)] * np.exp2(code.astype(float) - 127)[..., None]
        g = got.double().cpu().numpy()
        assert np.isnan(g[nan]).all() and np.array_equal(g[~nan], want[~nan])


@pytest.mark.parametrize("pos0,n", [(0, 1), (0, 16), (7, 40), (15, 2), (3, 333)])
def test_read_back_is_what_attention_sees(pos0, n):
    """Values read back are exact in bf16, at any start, in shuffled pages."""
    g = torch.Generator(device="cuda").manual_seed(n)
    x, y = (torch.randn(n, 8, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    pages = -(-(pos0 + n) // PAGE)
    (k, ks), (v, vs) = chunk.f8_pool(pages, 8), chunk.f8_pool(pages, 8)
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).reshape(1, -1)
    chunk.write_pages_f8(x, y, k, v, ks, vs, table, 0, pos0)
    rk, rv = chunk.read_pages_f8(k, v, ks, vs, table, 0, pos0, n)
    for got, src in ((rk, x), (rv, y)):
        err = (got.double() - src.double()).abs()
        # half a step of 3 mantissa bits, or of the smallest subnormal at the row's scale
        bound = torch.maximum(src.double().abs() * 2.0 ** -4,
                              torch.exp2(torch.ceil(torch.log2(src.double().abs().amax(-1, keepdim=True) / 448)) - 10))
        assert bool((err <= bound).all())
        chunk.write_pages_f8(got, got, k, v, ks, vs, table, 0, pos0)
        again, _ = chunk.read_pages_f8(k, v, ks, vs, table, 0, pos0, n)
        assert torch.equal(again, got)  # nothing is lost a second time


def test_ring_and_slots_outside_the_pool():
    (k, ks), (v, vs) = chunk.f8_pool(3, 2), chunk.f8_pool(3, 2)
    x = torch.randn(40, 2, D, device="cuda").to(torch.bfloat16)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    chunk.write_pages_f8(x, x, k, v, ks, vs, table, 0, 100)   # positions 100..139: logical pages 6, 7, 8
    rk, _ = chunk.read_pages_f8(k, v, ks, vs, table, 0, 100, 40)
    slots = torch.tensor([int(table[0, (p // PAGE) % 3]) * PAGE + p % PAGE for p in range(100, 140)], device="cuda")
    bits, code, nan = definition(x)
    same_bytes(rows_of(k, slots), bits, nan)
    assert torch.isfinite(rk).all()
    before = k.view(torch.uint8).clone()
    qkv = torch.randn(2, 6 * D, device="cuda").to(torch.bfloat16)
    chunk.rope_append_f8(qkv, torch.zeros(2, dtype=torch.int32, device="cuda"),
                         torch.tensor([-1, 48], dtype=torch.int32, device="cuda"), 2, torch.ones(32), 1.0, k, v, ks, vs)
    torch.cuda.synchronize()
    assert torch.equal(before, k.view(torch.uint8))


def test_refusals():
    (k, ks), (v, vs) = chunk.f8_pool(3, 2), chunk.f8_pool(3, 2)
    x = torch.zeros(4, 2, D, dtype=torch.bfloat16, device="cuda")
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    qkv = torch.zeros(4, 6 * D, dtype=torch.bfloat16, device="cuda")
    inv = torch.ones(32)
    bad = (ValueError, _lib.GptossError)
    for match, f in [
        ("8-bit", lambda: chunk.write_pages_f8(x, x, x, x, None, None, table, 0, 0)),
        ("rows must be", lambda: chunk.write_pages_f8(x.float(), x, k, v, ks, vs, table, 0, 0)),
        ("rows must be", lambda: chunk.write_pages_f8(x, x[:3], k, v, ks, vs, table, 0, 0)),
        ("no rows", lambda: chunk.read_pages_f8(k, v, ks, vs, table, 1, 0, 4)),
        ("no rows", lambda: chunk.read_pages_f8(k, v, ks, vs, table, 0, -1, 4)),
        ("do not fit", lambda: chunk.write_pages_f8(*(torch.zeros(49, 2, D, dtype=torch.bfloat16, device="cuda"),) * 2,
                                                    k, v, ks, vs, table, 0, 0)),
        ("scales of this pool", lambda: chunk.read_pages_f8(k, v, ks, vs[:2], table, 0, 0, 4)),
        ("page_table", lambda: chunk.read_pages_f8(k, v, ks, vs, table.long(), 0, 0, 4)),
        ("columns", lambda: chunk.rope_append_f8(qkv, i, i, 3, inv, 1.0, k, v, ks, vs)),
        ("positions", lambda: chunk.rope_append_f8(qkv, i[:3], i, 2, inv, 1.0, k, v, ks, vs)),
        ("slots", lambda: chunk.rope_append_f8(qkv, i, i.long(), 2, inv, 1.0, k, v, ks, vs)),
        ("inv_freq", lambda: chunk.rope_append_f8(qkv, i, i, 2, inv[:16], 1.0, k, v, ks, vs)),
        ("inv_freq", lambda: chunk.rope_append_f8(qkv, i, i, 2, inv.cuda(), 1.0, k, v, ks, vs)),
        ("dense CUDA", lambda: chunk.rope_append_f8(qkv[:, ::2], i, i, 2, inv, 1.0, k, v, ks, vs)),
    ]:
        with pytest.raises(bad, match=match):
            f()
    assert chunk.read_pages_f8(k, v, ks, vs, table, 0, 0, 0)[0].shape == (0, 2, D)
