"""Host logic of chunks, the 8-bit cache and speculative decoding, without a
GPU: the cache's planning, its refusals, the C entries' checks of arguments
(all made before anything is launched), draft lookup."""
import importlib

import pytest

torch = pytest.importorskip("torch")

chunk = importlib.import_module("gpt-oss-tvm_b200.chunk")
att = importlib.import_module("gpt-oss-tvm_b200.attention")
cfgm = importlib.import_module("gpt-oss-tvm_b200.config")
spec = importlib.import_module("gpt-oss-tvm_b200.speculative")
verify = importlib.import_module("gpt-oss-tvm_b200.verify")
_lib = importlib.import_module("gpt-oss-tvm_b200._lib")


def cache(max_batch=2, max_len=400, **kw):
    cfg = cfgm.GPTOssConfig(num_hidden_layers=2, num_experts=16, vocab_size=64, context_window_size=1024)
    return att.KVCache(cfg, max_batch, max_len, device="cpu", **kw)


def test_window_rings_grow_with_the_chunk():
    assert cache().window_pages == 9
    assert cache(max_chunk=1).window_pages == 9
    assert cache(max_chunk=5).window_pages == 10     # 132 keys and the page being filled
    assert cache(max_chunk=18).window_pages == 11


def test_begin_chunks_plans_every_sequence():
    c = cache(max_batch=3, max_chunk=6)
    c.begin_chunks([0, 2], [4, 6])
    assert c.positions.tolist() == [0, 1, 2, 3, 0, 1, 2, 3, 4, 5]
    assert c.q_start.tolist() == [0, 4, 10] and c.seq_rows.tolist() == [0, 2] and c.max_q == 6
    assert c.kv_len.tolist() == [4, 6]
    c.begin_chunks([2], [3])
    assert c.positions.tolist() == [6, 7, 8] and c.kv_len.tolist() == [9] and c.seq_rows.tolist() == [2]
    # the pool rows are those the page tables name
    full = [int(c.table_full_host[2, p // 16]) * 16 + p % 16 for p in (6, 7, 8)]
    assert c.slots.tolist() == full


def test_begin_chunks_refuses_what_the_ring_cannot_hold():
    c = cache(max_chunk=4)
    c.begin_chunks([0], [100])                       # nothing behind it: the ring holds it all
    with pytest.raises(ValueError, match="do not fit|does not fit"):
        c.begin_chunks([0], [80])                    # 180 positions, the window's first among them
    assert int(c.lengths[0]) == 100                  # and nothing was planned
    for n in range(30):
        c.begin_chunks([0], [4])                     # always room for max_chunk
    with pytest.raises(ValueError, match="distinct"):
        c.begin_chunks([0, 0], [1, 1])
    with pytest.raises(ValueError, match="new token"):
        c.begin_chunks([0, 1], [1, 0])
    with pytest.raises(ValueError, match="one length"):
        c.begin_chunks([0], [1, 1])
    with pytest.raises(ValueError, match="max_chunk"):
        cache(max_chunk=0)


def test_popn_of_rejected_drafts_keeps_the_window():
    c = cache(max_chunk=5)
    c.begin_chunks([0], [130])
    for _ in range(40):
        c.begin_chunks([0], [5])
        c.popn(0, 4)                                 # raises when the ring has lost the window
    assert int(c.lengths[0]) == 170


def test_8_bit_pools():
    c, b = cache(kv_dtype="float8_e4m3"), cache()
    assert c.f8 and not b.f8
    assert c.k[0].dtype == torch.float8_e4m3fn and c.k_scale[1].dtype == torch.float8_e8m0fnu
    assert c.k_scale[1].shape == (c.k[1].shape[0] // 16, 8, 16)
    assert c.memory_bytes() * 128 == b.memory_bytes() * 65
    with pytest.raises(ValueError, match="kv_dtype"):
        cache(kv_dtype="int8")


def test_8_bit_rows_and_copies_on_the_host():
    c = cache(kv_dtype="float8_e4m3", max_chunk=2)
    c.begin_forward([0], [40])
    for layer in range(2):
        rows = c.slots_for(layer).long()
        vals = torch.arange(40 * 8 * 64).reshape(40, 8, 64) % 15 - 7
        c.k[layer].view(torch.uint8)[rows] = vals.float().to(torch.float8_e4m3fn).view(torch.uint8)
        codes = (torch.arange(40)[:, None] % 5 + 125).expand(40, 8).to(torch.uint8)
        c.k_scale[layer].view(torch.uint8)[rows // 16, :, rows % 16] = codes
        want = (vals.float() * torch.exp2(torch.arange(40) % 5 - 2.0)[:, None, None]).to(torch.bfloat16)
        assert torch.equal(c.read_rows(layer, 0, 0, 40)[0], want)
    c.copy_sequence(0, 1)
    for layer in range(2):
        assert torch.equal(c.read_rows(layer, 1, 3, 37)[0], c.read_rows(layer, 0, 3, 37)[0])


def test_prompt_lookup():
    look = spec.prompt_lookup
    assert look([1, 2, 3, 4, 5, 1, 2, 3], 2) == [4, 5]
    assert look([1, 2, 3, 4, 5, 1, 2, 3], 9) == [4, 5, 1, 2, 3]
    assert look([9, 1, 2, 7, 1, 2, 8, 1, 2], 1) == [8]       # the last occurrence
    assert look([4, 4, 4], 2) == [4]
    assert look([1, 2, 3], 4) == [] and look([1], 4) == [] and look([], 4) == [] and look([1, 1], 0) == []


def test_cpu_tensors_are_refused():
    z = torch.zeros(2, 8, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    pool = torch.zeros(16, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        chunk.attend_chunks(z, pool, pool, i[None], i, torch.zeros(2, dtype=torch.int32), i, max_q=1)
    (k, ks), (v, vs) = chunk.f8_pool(1, 8, "cpu"), chunk.f8_pool(1, 8, "cpu")
    with pytest.raises(ValueError, match="CUDA"):
        chunk.rope_append_f8(torch.zeros(1, 24 * 64, dtype=torch.bfloat16), i, i, 8, torch.ones(32), 1.0, k, v, ks, vs)
    with pytest.raises(ValueError, match="CUDA"):
        chunk.read_pages_f8(k, v, ks, vs, i[None], 0, 0, 1)
    with pytest.raises(ValueError, match="CUDA"):
        verify.verify_drafts(torch.zeros(1, 5), i, torch.zeros(2, dtype=torch.int32), temperature=0.0)


def test_c_entries_check_before_they_launch():
    lib = _lib.load()
    p = 1 << 20  # an aligned address that is never used

    def rc(name, *args):
        r = getattr(lib, name)(*args)
        return r, (lib.gptoss_last_error() or b"").decode()

    base = dict(q=p, q_stride=4096, k=p, v=p, kc=None, vc=None, f8=0, pages=10, table=p, trows=1, tstride=4, rows=p,
                start=p, lens=p, N=1, T=1, max_q=1, Hq=64, Hkv=8, D=64, window=0, scale=0.125, sinks=None, ws=p,
                wsb=1 << 40, o=p, lse=None, stream=None)

    def chunk_rc(**kw):
        return rc("gptoss_attn_chunk", *{**base, **kw}.values())

    for kw, text in [(dict(D=128), "head_dim"), (dict(N=1025), "0..1024"), (dict(N=-1), "0..1024"), (dict(T=-1), "bad shape"),
                     (dict(Hq=60), "multiple of Hkv"), (dict(Hq=520), "at most 64"), (dict(q=None), "null"),
                     (dict(f8=1), "codes"), (dict(tstride=0), "page table"), (dict(pages=0), "page table"),
                     (dict(pages=1 << 27), "2^27"), (dict(max_q=0), "max_q"), (dict(scale=-1.0), "sm_scale"),
                     (dict(scale=float("nan")), "sm_scale"), (dict(q=p + 2), "aligned"), (dict(q_stride=4100), "q_stride"),
                     (dict(q_stride=64), "q_stride"), (dict(wsb=100), "workspace")]:
        r, msg = chunk_rc(**kw)
        assert r < 0 and text in msg, (kw, r, msg)
    assert chunk_rc(N=0)[0] == 0 and chunk_rc(T=0)[0] == 0
    r, msg = rc("gptoss_kv_pages_copy_f8", p, p, p, p, 4, 8, 64, p, 2, 0, 0, 33, p, p, 1, None)
    assert r < 0 and "do not fit" in msg
    r, msg = rc("gptoss_qkv_rope_append_f8", p, p, p, 4, 4, 8, 8, 32, p, 1.0, p, p, p, p, p, None)
    assert r < 0 and "head_dim" in msg
    for kw, text in [(dict(V=0), "V=0"), (dict(V=(1 << 22) + 1), "2^22"), (dict(t=-1.0), "temperature"),
                     (dict(u=None), "random numbers"), (dict(ld=4), "stride"), (dict(sb=8), "scratch"), (dict(tok=None), "null")]:
        a = {**dict(z=p, bf=0, ld=100, tok=p, start=p, T=4, N=2, V=50, t=1.0, u=p, un=p, q=None, ldq=0, s=p, sb=1 << 30,
                    acc=p, nxt=p, stream=None), **kw}
        r, msg = rc("gptoss_verify_drafts", *a.values())
        assert r < 0 and text in msg, (kw, r, msg)


def test_rows_of_dense_values():
    z = torch.zeros(4, 10)
    dense = verify._dense_rows
    assert dense(z) and dense(z[:, :7]) and dense(z[:1]) and dense(z[:0]) and dense(z[:, 3:4]) and dense(z[1:2, 3:4])
    assert not dense(z[:, ::2]) and not dense(z.t()) and not dense(z[:1].expand(4, 10))
    assert not dense(z[:1, ::2]) and not dense(z[:, 2:3].t()) and not dense(z[:1, :1].expand(1, 10))


class HostEngine:
    """An engine without a model: its target always continues with token + 1."""

    def __init__(self, **kw):
        self.device, self.max_chunk, self.max_batch_size = torch.device("cpu"), 4, 2
        self.paged_kv_cache = cache(max_chunk=4)
        self.popn, self.clear_kv_cache = self.paged_kv_cache.popn, self.paged_kv_cache.clear
        self.answer, self.error, self.resets = None, 0, 0

    def prefill(self, tokens, s):
        self.paged_kv_cache.begin_forward([s], [len(tokens)])

    def extend_batch(self, chunks, seqs):
        self.paged_kv_cache.begin_chunks(seqs, [len(c) for c in chunks])
        return None, torch.tensor([t for c in chunks for t in c], dtype=torch.int32), self.paged_kv_cache.q_start

    def verify(self, logits, ids, start, *draws, temperature):
        acc, nxt = [], []
        for a, b in zip(start.tolist(), start.tolist()[1:]):
            seq, k = ids[a:b].tolist(), 0
            while k + 1 < len(seq) and seq[k + 1] == seq[k] + 1:
                k += 1
            acc.append(k)
            nxt.append(seq[k] + 1)
        i32 = dict(dtype=torch.int32)
        return torch.tensor(acc, **i32), torch.tensor(self.answer or nxt, **i32)

    def chunk_workspace(self):
        return self

    def error_word(self):
        return torch.tensor([self.error], dtype=torch.int32)

    def reset(self):
        self.error, self.resets = 0, self.resets + 1


def test_a_speculative_step_that_fails_on_the_device_raises():
    """A next token of -1 or an error of the attention: the step raises, and texts
    and cache are as before, so that it can be taken again."""
    eng = HostEngine()
    dec = spec.SpeculativeDecoder(eng, draft_len=3, draft=lambda t, n: [t[-1] + 1, t[-1] + 2, 0][:n])
    assert dec.generate([[5, 6], [9]], 7) == [list(range(7, 14)), list(range(10, 17))]
    texts = {0: [1, 2, 3], 1: [7]}
    eng.clear_kv_cache()
    eng.prefill([1, 2], 0)
    for answer, error in (([4, -1], 0), (None, 1 << 9)):
        eng.answer, eng.error = answer, error
        with pytest.raises(RuntimeError, match="on the device"):
            dec.step(texts, {0: 9, 1: 9})
        assert texts == {0: [1, 2, 3], 1: [7]} and eng.paged_kv_cache.lengths.tolist() == [2, 0]
    eng.answer, drafted = None, dec.drafted
    assert eng.resets == 2
    dec.step(texts, {0: 9, 1: 9})
    assert texts == {0: [1, 2, 3, 4, 5, 6], 1: [7, 8, 9, 10]} and dec.drafted == drafted + 6
    assert eng.paged_kv_cache.lengths.tolist() == [5, 3]


def test_tokens_outside_the_vocabulary_never_reach_the_embedding():
    """Nor do drafts beyond what was asked for lengthen a text."""
    import types
    engm = importlib.import_module("gpt-oss-tvm_b200.engine")
    c = cache(max_chunk=4)
    planned = []
    stub = types.SimpleNamespace(max_chunk=4, config=c.config, paged_kv_cache=c, _ids=planned.append)
    for bad in ([[64]], [[1, 2], [-1]], [[3, 1 << 40]]):
        with pytest.raises(ValueError, match="vocabulary"):
            engm.Engine.extend_batch(stub, bad, list(range(len(bad))))
    assert planned == [] and c.lengths.tolist() == [0, 0]
    eng = HostEngine()
    eng.prefill([1, 2], 0)
    texts = {0: [1, 2, 3]}
    for room in (9, 2, 1):
        with pytest.raises(ValueError, match="drafts where at most"):
            spec.SpeculativeDecoder(eng, draft_len=3, draft=lambda t, n: [4] * (n + 1)).step(texts, {0: room})
    assert texts == {0: [1, 2, 3]} and eng.paged_kv_cache.lengths.tolist() == [2, 0]


def test_another_plan_ends_that_of_the_chunks():
    """forward_to="chunk" after begin_forward or a device-planned decode step has
    no chunks to attend, whatever an earlier begin_chunks left."""
    c = cache(max_chunk=4)
    for other in (lambda: c.begin_forward([0], [3]), lambda: c.begin_forward([1, 0], [1, 2]),
                  lambda: c.begin_decode_on_device(2)):
        c.begin_chunks([0, 1], [2, 1])
        assert c.q_start.tolist() == [0, 2, 3]
        other()
        assert c.q_start is None and c.seq_rows is None
    c.begin_chunks([1], [1])
    assert c.q_start.tolist() == [0, 1] and c.seq_rows.tolist() == [1]
