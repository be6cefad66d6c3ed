"""Chunks of several sequences, the 8-bit cache and speculative decoding through
KVCache, AttentionBlock, GPTOssForCausalLM and Engine.

The MoE blocks run other kernels (and activation formats) at other batch sizes,
and with random weights a difference in the last bit picks another expert, so
whole models are compared with the blocks' part of the sum switched off (weight
scales of 2^-27, no bias): what is left, the attention layers and the
unembedding, is compared with the bf16 tolerance of the attention tests, max |d|
/ max |ref| <= 2e-2.  Tokens of a chunk attend one another's keys as the 8-bit
cache holds them, a prefill its own unquantised, so 8-bit chunks are compared
with 8-bit chunks of one token."""
import importlib

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

cfgm = importlib.import_module("gpt-oss-tvm_b200.config")
engm = importlib.import_module("gpt-oss-tvm_b200.engine")
spec = importlib.import_module("gpt-oss-tvm_b200.speculative")


def config():
    return cfgm.GPTOssConfig(num_hidden_layers=2, num_experts=16, vocab_size=512, context_window_size=1024,
                             prefill_chunk_size=256)


def engine(kv_dtype, batch=3, chunk=8):
    eng = engm.Engine.random(config(), seed=5, max_batch_size=batch, max_total_seq_len=600, kv_dtype=kv_dtype,
                             max_chunk=chunk, warmup=False)
    for name, t in eng.model.named_parameters():
        if name.endswith("mlp2_weight_scales"):
            t.fill_(100)
        elif name.endswith("mlp2_bias"):
            t.zero_()
    eng.model.prepare()
    return eng


def text(n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, 512, (n,), generator=g).tolist()


def close(a, b, tol):
    d = (a.double() - b.double()).abs().max() / b.double().abs().max()
    assert float(d) <= tol, f"max |d| / max |ref| = {float(d):.3e}"


@pytest.mark.parametrize("kv_dtype", ["bfloat16", "float8_e4m3"])
def test_extend_batch_gives_the_logits_of_each_sequence(kv_dtype):
    """Uneven chunks, some behind the 128-token window's reach, against one
    token of one sequence at a time: through extend (bf16), or chunks of one."""
    prompts, new = [text(300, 1), text(5, 2), text(131, 3)], [text(5, 4), text(8, 5), text(1, 6)]
    eng = engine(kv_dtype)
    for s, p in enumerate(prompts):
        eng.paged_kv_cache.add_sequence(s)
        eng.prefill(p, s)
    logits, ids, start = eng.extend_batch(new, [0, 1, 2])
    start = start.tolist()
    assert logits.shape == (14, 512) and start == [0, 5, 13, 14]
    assert ids.tolist() == [t for n in new for t in n]
    assert eng.paged_kv_cache.lengths.tolist() == [305, 13, 132]
    for s in range(3):
        ref = engine(kv_dtype, batch=1)
        ref.prefill(prompts[s], 0)
        for i, t in enumerate(new[s]):
            row = ref.extend([t], 0) if kv_dtype == "bfloat16" else ref.extend_batch([[t]], [0])[0]
            close(logits[start[s] + i], row.reshape(-1), 2e-2)
        ref.model.release()
    eng.model.release()


def test_chunks_read_what_decode_wrote_and_the_other_way_round():
    """Decode steps and chunks of one token in turn, in 8 bits: the cache a
    chunk leaves is the one decode goes on with."""
    a, b = engine("float8_e4m3", batch=2), engine("float8_e4m3", batch=2)
    steps = [text(2, 10 + i) for i in range(6)]
    for e in (a, b):
        for s in range(2):
            e.paged_kv_cache.add_sequence(s)
            e.prefill(text(140, 30 + s), s)
    for i, t in enumerate(steps):
        la = a.decode_batch(t).reshape(2, -1)
        lb = b.extend_batch([[t[0]], [t[1]]], [0, 1])[0] if i % 2 else b.decode_batch(t).reshape(2, -1)
        close(lb, la, 2e-2)
    for layer in range(2):
        for s in range(2):
            ka, va = a.paged_kv_cache.read_rows(layer, s, 20, 126)
            kb, vb = b.paged_kv_cache.read_rows(layer, s, 20, 126)
            assert torch.equal(ka[:120], kb[:120]) and torch.equal(va[:120], vb[:120])
    a.model.release()
    b.model.release()


def test_decode_graph_on_the_8_bit_cache():
    eng = engine("float8_e4m3", batch=2)
    for s in range(2):
        eng.paged_kv_cache.add_sequence(s)
        eng.prefill(text(150, s), s)
    cache2 = engine("float8_e4m3", batch=2)
    for s in range(2):
        cache2.paged_kv_cache.add_sequence(s)
        cache2.prefill(text(150, s), s)
    g = engm.GreedyDecodeGraph(eng.model, eng.paged_kv_cache, 2, use_graph=True)
    e = engm.GreedyDecodeGraph(cache2.model, cache2.paged_kv_cache, 2, use_graph=False)
    first = torch.tensor([7, 9], device="cuda")
    g.set_tokens(first)
    e.set_tokens(first)
    for _ in range(20):
        lg, tg = g.step()
        le, te = e.step()
        assert torch.equal(lg, le) and torch.equal(tg, te)
    g.close()
    assert eng.model.model.block[0].attn.scratch.chunk().error() == 0
    eng.model.release()
    cache2.model.release()


@pytest.mark.parametrize("kv_dtype", ["bfloat16", "float8_e4m3"])
def test_greedy_speculation_follows_the_target(kv_dtype):
    """Whatever the drafts, right, wrong or none, every token that comes out is
    the target's first choice, or within the tolerance of it (the forwards of a
    step with drafts and of one without run other kernels)."""
    prompts = [text(40, 1) * 2, text(150, 2), [3]]

    def oracle_drafts(known):
        def draft(tokens, n):
            full = known[tokens[0]]
            right = full[len(tokens):len(tokens) + n]
            return [t if i % 3 else (t + (len(tokens) % 2)) % 512 for i, t in enumerate(right)]
        return draft

    plain = engine(kv_dtype)
    base = spec.SpeculativeDecoder(plain, draft_len=0).generate(prompts, 24)
    assert [len(t) for t in base] == [24, 24, 24]
    known = {p[0]: p + t for p, t in zip(prompts, base)}
    assert len(known) == 3
    for draft in (oracle_drafts(known), spec.prompt_lookup, lambda tokens, n: [511] * n):
        eng = engine(kv_dtype)
        dec = spec.SpeculativeDecoder(eng, draft_len=5, draft=draft)
        out = dec.generate(prompts, 24)
        assert [len(t) for t in out] == [24, 24, 24]
        assert 0 <= dec.accepted <= dec.drafted and dec.steps <= 24
        assert eng.paged_kv_cache.lengths.tolist() == [len(p) + 23 for p in prompts]
        for p, t in zip(prompts, out):
            plain.clear_kv_cache()
            full = p + t
            plain.paged_kv_cache.add_sequence(0)
            if len(p) > 1:
                plain.prefill(p[:-1], 0)
            for i in range(len(p) - 1, len(full) - 1):
                row = plain.extend_batch([[full[i]]], [0])[0][0]
                assert float(row.max() - row[full[i + 1]]) <= 2e-2 * float(row.abs().max())
        if draft is not spec.prompt_lookup:
            assert (dec.accepted > 20) == (draft(prompts[1], 3) != [511] * 3)
        eng.model.release()
    plain.model.release()


def test_sampled_speculation_repeats_with_its_seed():
    prompts = [text(30, 1), text(60, 2)]
    runs = []
    for seed in (1, 1, 2):
        eng = engine("float8_e4m3", batch=2)
        runs.append(spec.SpeculativeDecoder(eng, draft_len=4, temperature=0.8, seed=seed).generate(prompts, 20))
        eng.model.release()
    assert runs[0] == runs[1] and runs[0] != runs[2]
    assert all(0 <= t < 512 for r in runs for seq in r for t in seq)


def test_refusals():
    eng = engine("bfloat16", batch=2, chunk=4)
    for s in range(2):
        eng.paged_kv_cache.add_sequence(s)
    with pytest.raises(ValueError, match="max_chunk"):
        eng.extend_batch([[1] * 5], [0])
    with pytest.raises(ValueError, match="distinct"):
        eng.extend_batch([[1], [2]], [0, 0])
    with pytest.raises(ValueError, match="new token"):
        eng.extend_batch([[1], []], [0, 1])
    with pytest.raises(ValueError, match="outside the cache"):
        eng.extend_batch([[1]], [2])
    with pytest.raises(ValueError, match="max_chunk 6"):
        spec.SpeculativeDecoder(eng, draft_len=5)
    with pytest.raises(ValueError, match="prompts"):
        spec.SpeculativeDecoder(eng, draft_len=3).generate([[1], [2], [3]], 4)
    with pytest.raises(ValueError, match="needs a token"):
        spec.SpeculativeDecoder(eng, draft_len=3).generate([[1], []], 4)
    with pytest.raises(ValueError, match="kv_dtype"):
        engine("int8")
    eng.model.release()


def test_tokens_outside_the_vocabulary_are_refused():
    eng = engine("bfloat16", batch=2, chunk=4)
    for bad in ([[512]], [[1], [-1]], [[1, 2, 1 << 20]]):
        with pytest.raises(ValueError, match="vocabulary"):
            eng.extend_batch(bad, list(range(len(bad))))
    with pytest.raises(ValueError, match="vocabulary"):
        spec.SpeculativeDecoder(eng, draft_len=3, draft=lambda t, n: [512][:n]).generate([[1]], 4)
    eng.clear_kv_cache()
    logits = eng.extend_batch([[0, 511]], [0])[0]
    assert bool(torch.isfinite(logits).all())
    eng.model.release()


def test_a_chunk_forward_needs_its_own_plan():
    eng = engine("bfloat16", batch=2, chunk=4)
    eng.extend_batch([[1, 2], [3]], [0, 1])
    x = eng.model.embed(torch.tensor([4, 5, 6], device="cuda"))
    eng.paged_kv_cache.begin_forward([0], [3])
    with pytest.raises(ValueError, match="begin_chunks"):
        eng.model.chunk(x, eng.paged_kv_cache)
    eng.model.release()
