"""Measured cases of the operators that a speculative-decoding step of the engine is made of:

  attend  attention of every sequence's new tokens over the paged KV cache (bf16 or 8-bit pages)
  append  QKV split + RoPE + the keys and values quantised as they are written to 8-bit pages
  read    an 8-bit cache read back as bf16 rows
  verify  drafted tokens checked against the target's logits from given random numbers

An 8-bit page pool holds e4m3 values [rows, kv heads, 64] and one E8M0 code per row and head
[pages, kv heads, 16]: the smallest power of two that brings the row's largest magnitude to 448 or
less.  `run` gives the plain form in 32-bit torch operations, or with `own` the framework's calls.
"""
import importlib
import math

import numpy as np
import torch

own = False

HEAD = 64   # head width of the model
PAGE = 16   # tokens per cache page
VOCAB = 201088
FIX = 2.0 ** 40  # probability weights are whole multiples of 2^-40: their sums do not depend on the order


def _mod(name):
    return importlib.import_module("gpt-oss-tvm_b200." + name)


# ------------------------------------------------------------------- cases
def _attend(name, seqs, q, kv, *, ragged=False, window=0, f8=False, heads=64, kv_heads=8):
    return {"name": name, "op": "attend", "seqs": seqs, "q": q, "kv": kv, "ragged": ragged, "window": window,
            "f8": f8, "heads": heads, "kv_heads": kv_heads}


def listed():
    return [
        # one user's next token early in a chat: the smallest call, latency only
        _attend("attend 1x1 kv512", 1, 1, 512),
        # a serving batch's next tokens over an 8-bit cache
        _attend("attend 32x1 kv8192 f8", 32, 1, 8192, f8=True),
        # the target's pass over up to 4 drafts and the last token of each sequence, uneven lengths
        _attend("attend 32x5 kv8191 f8 ragged", 32, 5, 8191, ragged=True, f8=True),
        # the same on a sliding-window layer, whose pages are a ring
        _attend("attend 32x5 kv8191 window", 32, 5, 8191, ragged=True, window=128),
        # four uneven prompts at once, from an empty cache
        _attend("attend 4x1023 prompts", 4, 1023, 1023, ragged=True),
        # a chunk of a long prompt behind 30 k cached tokens
        _attend("attend 1x2048 kv32768 f8", 1, 2048, 32768, f8=True),
        # the cache write of the drafts' pass, and of a whole prefill chunk
        {"name": "append 160", "op": "append", "tokens": 160, "heads": 64, "kv_heads": 8},
        {"name": "append 8192", "op": "append", "tokens": 8192, "heads": 64, "kv_heads": 8},
        # a short context and the longest one brought back as bf16 for a prefill chunk
        {"name": "read 1000", "op": "read", "tokens": 1000, "kv_heads": 8},
        {"name": "read 131072", "op": "read", "tokens": 131072, "kv_heads": 8},
        # drafts looked up in the prompt (no draft distribution) for one user
        {"name": "verify 1x4 lookup", "op": "verify", "seqs": 1, "drafts": 4, "ragged": False, "vocab": VOCAB,
         "probs": False, "temperature": 0.7},
        # a batch whose drafts come from a small model, with its distributions
        {"name": "verify 48x5 ragged", "op": "verify", "seqs": 48, "drafts": 5, "ragged": True, "vocab": VOCAB,
         "probs": True, "temperature": 1.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "read", "verify"])
    heads, kv_heads = rng.choice([(64, 8), (64, 8), (32, 8), (40, 8), (16, 16), (32, 2)])
    if op == "append":
        return {"op": op, "tokens": _log(rng, 1, 8192), "heads": heads, "kv_heads": kv_heads}
    if op == "read":
        return {"op": op, "tokens": _log(rng, 1, 131072), "kv_heads": kv_heads}
    if op == "verify":
        return {"op": op, "seqs": _log(rng, 1, 48), "drafts": rng.randint(1, 5), "ragged": rng.random() < 0.5,
                "vocab": _log(rng, 1000, VOCAB), "probs": rng.random() < 0.5,
                "temperature": rng.choice([0.0, 0.7, 1.0])}
    seqs, q = _log(rng, 1, 64), rng.choice([rng.randint(1, 9), _log(rng, 1, 2048)])
    q = max(1, min(q, 4096 // seqs))
    kv = max(q, _log(rng, 16, max(16, min(32768, 2 ** 26 // (seqs * q), 2 ** 18 // seqs))))
    return {"op": op, "seqs": seqs, "q": q, "kv": kv, "ragged": rng.random() < 0.7,
            "window": rng.choice([0, 0, 128]), "f8": rng.random() < 0.5, "heads": heads, "kv_heads": kv_heads}


def _lengths(case):
    """(new tokens, cached + new tokens) of each sequence of an attend case."""
    n, q, kv = case["seqs"], case["q"], case["kv"]
    if not case["ragged"]:
        return [q] * n, [kv] * n
    ql = [q - (b * 7919 + 3) % max(1, (q + 1) // 2) for b in range(n)]
    kl = [max(ql[b], kv - (b * 104729 + 11) % max(1, kv // 2)) for b in range(n)]
    return ql, kl


def _rows_of(case):
    """Rows of logits (drafts and one more) of each sequence of a verify case."""
    k = case["drafts"]
    return [k + 1 - (b * 7 % (k + 1) if case["ragged"] else 0) for b in range(case["seqs"])]


# ------------------------------------------------------------------ inputs
def _quantise(x):
    """Rows [..., 64] -> e4m3 values and E8M0 codes [...]: code - 127 is the smallest exponent (in -60..60)
    with max|x| <= 448 * 2^exponent."""
    amax = x.abs().amax(-1).float()
    mant, ex = torch.frexp(amax)
    e = torch.where(mant > 0.875, ex - 8, ex - 9)  # 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e, torch.full_like(e, -60)).clamp(-60, 60)
    q = torch.ldexp(x.float(), -e.unsqueeze(-1)).to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8)


def _pool(x, pages, kv_heads):
    """A pool's 8-bit form of bf16 rows [pages * 16, kv heads, 64]."""
    q, code = _quantise(x)
    return q, code.reshape(pages, PAGE, kv_heads).transpose(1, 2).contiguous().view(torch.float8_e8m0fnu)


def _frequencies():
    f = torch.tensor([150000.0 ** (-2.0 * i / HEAD) for i in range(HEAD // 2)], dtype=torch.float32)
    return f, 0.1 * math.log(32.0) + 1.0


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    bf = dict(device=dev, dtype=torch.bfloat16)

    def normal(*shape):
        return torch.randn(*shape, generator=g, **bf)

    def order(n):
        return torch.randperm(n, generator=g, device=dev).to(torch.int32)

    st = {"op": case["op"], "case": case}
    i32 = dict(dtype=torch.int32, device=dev)
    if case["op"] == "attend":
        ql, kl = _lengths(case)
        n, hkv, w = case["seqs"], case["kv_heads"], case["window"]
        # a full layer's pages come from a shared pool in no order; a window layer's are a ring per sequence
        stride = -(-max(kl) // PAGE) if w == 0 else min(-(-max(kl) // PAGE), -(-(w + max(ql) - 1) // PAGE) + 1)
        pages = n * stride
        table = order(pages).reshape(n, stride)
        k, v = normal(pages * PAGE, hkv, HEAD), normal(pages * PAGE, hkv, HEAD)
        # keys have a few large channels, as rotated keys of a trained model do
        k *= (1.0 + 3.0 * (torch.arange(HEAD, device=dev) % 23 == 5)).to(torch.bfloat16)
        ks = vs = None
        if case["f8"]:
            (k, ks), (v, vs) = _pool(k, pages, hkv), _pool(v, pages, hkv)
        st |= {"k": k, "v": v, "ks": ks, "vs": vs, "table": table, "window": w, "max_q": max(ql), "max_kv": max(kl),
               "q": normal(sum(ql), case["heads"], HEAD), "sinks": normal(case["heads"]),
               "rows": torch.arange(n, **i32), "kv_len": torch.tensor(kl, **i32),
               "q_start": torch.tensor(np.concatenate([[0], np.cumsum(ql)]).tolist(), **i32)}
    elif case["op"] == "append":
        t, hq, hkv = case["tokens"], case["heads"], case["kv_heads"]
        pages = -(-t // PAGE) + 1
        f, conc = _frequencies()
        shape = (pages * PAGE, hkv, HEAD)
        st |= {"qkv": normal(t, (hq + 2 * hkv) * HEAD), "hq": hq, "inv_freq": f, "inv_freq_dev": f.to(dev),
               "conc": conc, "slots": order(pages * PAGE)[:t].contiguous(),
               "pos": (torch.arange(t, **i32) * 13 + int(torch.randint(0, 1000, (1,), generator=g, device=dev))) % 131072,
               "k": torch.zeros(shape, device=dev, dtype=torch.float8_e4m3fn),
               "v": torch.zeros(shape, device=dev, dtype=torch.float8_e4m3fn),
               "ks": torch.full((pages, hkv, PAGE), 127, device=dev, dtype=torch.uint8).view(torch.float8_e8m0fnu),
               "vs": torch.full((pages, hkv, PAGE), 127, device=dev, dtype=torch.uint8).view(torch.float8_e8m0fnu)}
    elif case["op"] == "read":
        n, hkv = case["tokens"], case["kv_heads"]
        pages = -(-(n + 5) // PAGE)
        (k, ks), (v, vs) = (_pool(normal(pages * PAGE, hkv, HEAD) * 2, pages, hkv) for _ in range(2))
        st |= {"k": k, "v": v, "ks": ks, "vs": vs, "n": n, "pos0": 5, "table": order(pages).reshape(1, pages)}
    else:
        rows = _rows_of(case)
        t, vocab, n = sum(rows), case["vocab"], case["seqs"]
        logits = torch.randn(t, vocab, generator=g, device=dev) * 2.5
        # the draft model agrees with the target up to noise; its tokens are drawn from its distribution
        draft = torch.softmax(logits + 0.7 * torch.randn(t, vocab, generator=g, device=dev), -1)
        tokens = torch.randint(0, vocab, (t,), generator=g, device=dev)
        if t > 1:
            # draws by the largest p / Exp(1), the token that follows each row
            drawn = (draft / torch.empty_like(draft).exponential_(1.0, generator=g)).argmax(-1)
            tokens[1:] = drawn[:-1]
            # text is mostly predictable: the target gives every drafted token some of its weight
            boost = torch.rand(t - 1, generator=g, device=dev) * 16
            logits[torch.arange(t - 1, device=dev), tokens[1:]] += boost
            draft[torch.arange(t - 1, device=dev), tokens[1:]] += 0.5
            draft /= draft.sum(-1, keepdim=True)
        st |= {"logits": logits, "tokens": tokens.to(torch.int32), "n": n, "temperature": case["temperature"],
               "draft": draft if case["probs"] else None,
               "row_start": torch.tensor(np.concatenate([[0], np.cumsum(rows)]).tolist(), **i32),
               "max_rows": max(rows),
               "accept": torch.rand(t, generator=g, device=dev), "next": torch.rand(n, generator=g, device=dev)}
    return st


# -------------------------------------------------------------- plain form
def _dequantise(k, codes, rows, kv_heads):
    """Values [..., kv heads, 64] in 32 bits of pool rows `rows`."""
    x = k[rows].float() if codes is None else k.view(torch.uint8)[rows].view(torch.float8_e4m3fn).float()
    if codes is None:
        return x
    e = codes.view(torch.uint8)[rows // PAGE, :, rows % PAGE].int() - 127
    return torch.ldexp(x, e.unsqueeze(-1))


def _plain_attend(st):
    q, kv_len, start, w = st["q"], st["kv_len"].long(), st["q_start"].long(), st["window"]
    t, hq, _ = q.shape
    hkv, dev = st["k"].shape[1], q.device
    n, stride = st["table"].shape
    mq = st["max_q"]
    span = st["max_kv"] if w == 0 else min(st["max_kv"], w + mq - 1)
    j = kv_len[:, None] - span + torch.arange(span, device=dev)  # key positions [n, span], negative: none
    jj = j.clamp(min=0)
    page = torch.gather(st["table"].long(), 1, (jj // PAGE) % stride)
    rows = page * PAGE + jj % PAGE
    k, v = (_dequantise(st[a], st[b], rows, hkv) for a, b in (("k", "ks"), ("v", "vs")))
    qlen = start[1:] - start[:-1]
    i = torch.arange(mq, device=dev)
    src = (start[:-1, None] + i).clamp(max=t - 1)                       # [n, mq]
    qq = q[src].float().reshape(n, mq, hkv, hq // hkv, HEAD).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, HEAD)
    pos = kv_len[:, None] - qlen[:, None] + i                            # [n, mq]
    see = (j[:, None, :] <= pos[:, :, None]) & (j[:, None, :] >= 0)
    if w > 0:
        see = see & (j[:, None, :] > pos[:, :, None] - w)
    s = torch.matmul(qq, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(HEAD))   # [n, hkv, g * mq, span]
    s = s.reshape(n, hkv, hq // hkv, mq, span).masked_fill_(~see[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(s.sub_(m))
    den = p.sum(-1, keepdim=True)
    lse = (m + torch.log(den)).squeeze(-1) * math.log2(math.e)
    sink = torch.exp(st["sinks"].float().reshape(1, hkv, hq // hkv, 1, 1) - m)
    o = torch.matmul(p.reshape(n, hkv, -1, span), v.permute(0, 2, 1, 3)).reshape(n, hkv, hq // hkv, mq, HEAD)
    o = o / (den + sink)
    live = (i[None, :] < qlen[:, None])
    o = o.permute(0, 3, 1, 2, 4).reshape(n, mq, hq, HEAD)[live]
    return {"o": o.to(torch.bfloat16), "lse": lse.permute(0, 3, 1, 2).reshape(n, mq, hq)[live]}


def _plain_append(st):
    t, hq, hkv = st["qkv"].shape[0], st["hq"], st["k"].shape[1]
    x = st["qkv"].reshape(t, hq + 2 * hkv, HEAD)
    ang = st["pos"].float()[:, None] * st["inv_freq_dev"][None, :]
    c, s = (torch.cos(ang) * st["conc"])[:, None, :], (torch.sin(ang) * st["conc"])[:, None, :]
    a, b = x[:, :hq + hkv, :HEAD // 2].float(), x[:, :hq + hkv, HEAD // 2:].float()
    rot = torch.cat([a * c - b * s, a * s + b * c], -1).to(torch.bfloat16)
    slots = st["slots"].long()
    for_k, for_v = _quantise(rot[:, hq:]), _quantise(x[:, hq + hkv:])
    st["k"].view(torch.uint8)[slots] = for_k[0].view(torch.uint8)
    st["v"].view(torch.uint8)[slots] = for_v[0].view(torch.uint8)
    st["ks"].view(torch.uint8)[slots // PAGE, :, slots % PAGE] = for_k[1]
    st["vs"].view(torch.uint8)[slots // PAGE, :, slots % PAGE] = for_v[1]
    return {"q": rot[:, :hq].contiguous(), "k": st["k"], "v": st["v"], "ks": st["ks"], "vs": st["vs"]}


def _plain_read(st):
    p = torch.arange(st["pos0"], st["pos0"] + st["n"], device=st["k"].device)
    rows = st["table"][0].long()[p // PAGE] * PAGE + p % PAGE
    hkv = st["k"].shape[1]
    return {a: _dequantise(st[a], st[b], rows, hkv).to(torch.bfloat16) for a, b in (("k", "ks"), ("v", "vs"))}


def _fixed(x):
    return (x * FIX).to(torch.int64)


def _plain_verify(st):
    z, start, n = st["logits"], st["row_start"].long(), st["n"]
    t, vocab = z.shape
    dev = z.device
    z = torch.where(torch.isnan(z), -math.inf, z)
    m, top = z.max(-1)
    top = (z == m[:, None]).to(torch.uint8).argmax(-1)                      # the lowest index
    row = torch.arange(t, device=dev)
    last = torch.zeros(t, dtype=torch.bool, device=dev)
    last[start[1:] - 1] = True
    follows = torch.cat([st["tokens"][1:].long(), st["tokens"].new_zeros(1).long()])  # the draft of each row
    if st["temperature"] < 1e-6:
        ok = (top == follows) & ~last
        e = p = None
    else:
        inv = 1.0 / st["temperature"]
        e = torch.exp(torch.where(z == m[:, None], 0.0, (z - m[:, None]) * inv))
        total = _fixed(e).sum(-1)
        p = e / (total.float() / FIX)[:, None]
        qx = st["draft"][row, follows] if st["draft"] is not None else torch.ones(t, device=dev)
        ok = (st["accept"] * qx < p[row, follows]) & ~last
    i = torch.arange(st["max_rows"], device=dev)
    idx = (start[:-1, None] + i).clamp(max=t - 1)
    accepted = torch.cumprod((ok[idx] & (i[None] < (start[1:] - start[:-1])[:, None])).int(), -1).sum(-1)
    at = start[:-1] + accepted                                              # the row that gives the next token
    if e is None:
        return {"accepted": accepted.int(), "next": top[at].int()}
    end = last[at]
    if st["draft"] is not None:
        r = torch.where(end[:, None], e[at], (p[at] - st["draft"][at]).clamp(min=0))
    else:
        r = torch.where((torch.arange(vocab, device=dev)[None] == follows[at][:, None]) & ~end[:, None], 0.0, e[at])
    w = _fixed(r)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, _fixed(e[at]))
    c = w.cumsum(-1)
    s = c[:, -1]
    u = torch.minimum((st["next"].double() * s.double()).floor().long(), s - 1)
    return {"accepted": accepted.int(), "next": (c <= u[:, None]).sum(-1).int()}


# --------------------------------------------------------------- one pass
def run(st):
    if not own:
        return {"attend": _plain_attend, "append": _plain_append, "read": _plain_read,
                "verify": _plain_verify}[st["op"]](st)
    if st["op"] == "attend":
        o, lse = _mod("chunk").attend_chunks(st["q"], st["k"], st["v"], st["table"], st["rows"], st["q_start"],
                                             st["kv_len"], max_q=st["max_q"], window=st["window"],
                                             sinks=st["sinks"], k_scale=st["ks"], v_scale=st["vs"], return_lse=True)
        return {"o": o, "lse": lse}
    if st["op"] == "append":
        q = _mod("chunk").rope_append_f8(st["qkv"], st["pos"], st["slots"], st["hq"], st["inv_freq"], st["conc"],
                                         st["k"], st["v"], st["ks"], st["vs"])
        return {"q": q, "k": st["k"], "v": st["v"], "ks": st["ks"], "vs": st["vs"]}
    if st["op"] == "read":
        k, v = _mod("chunk").read_pages_f8(st["k"], st["v"], st["ks"], st["vs"], st["table"], 0, st["pos0"], st["n"])
        return {"k": k, "v": v}
    accepted, nxt = _mod("verify").verify_drafts(st["logits"], st["tokens"], st["row_start"], st["accept"],
                                                 st["next"], temperature=st["temperature"], draft_probs=st["draft"])
    return {"accepted": accepted, "next": nxt}


def work(case):
    if case["op"] == "append":
        t, hq, hkv = case["tokens"], case["heads"], case["kv_heads"]
        return {"bytes": t * (2 * HEAD * (2 * hq + 2 * hkv) + 2 * hkv * (HEAD + 1) + 8), "flops": 6 * t * (hq + hkv) * HEAD}
    if case["op"] == "read":
        return {"bytes": case["tokens"] * case["kv_heads"] * 2 * (HEAD + 1 + 2 * HEAD), "flops": 0}
    if case["op"] == "verify":
        rows = sum(_rows_of(case))
        drafts = rows - case["seqs"]
        # every row of logits; of the draft distributions one value a draft, and one row a sequence at most
        per_draft = case["seqs"] * case["vocab"] * 4 if case["probs"] and case["temperature"] > 0 and drafts else 0
        return {"bytes": rows * case["vocab"] * 4 + per_draft + 16 * rows, "flops": 4 * rows * case["vocab"]}
    ql, kl = _lengths(case)
    hq, hkv, w = case["heads"], case["kv_heads"], case["window"]
    keys = sum(k if w == 0 else min(k, w + q - 1) for q, k in zip(ql, kl))
    if w == 0:
        pairs = sum(q * (k - q) + q * (q + 1) // 2 for q, k in zip(ql, kl))
    else:
        pairs = sum(sum(min(w, k - q + i + 1) for i in range(q)) for q, k in zip(ql, kl))
    row = 2 * hkv * (HEAD + 1 if case["f8"] else 2 * HEAD)
    return {"bytes": keys * row + sum(ql) * hq * (4 * HEAD + 4), "flops": 4 * HEAD * hq * pairs}


# ---------------------------------------------------------------- 64 bits
def _grid8(x):
    """x (64 bits, |x| <= 448) rounded to the nearest e4m3 value, ties to the even one."""
    e = np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6)))
    step = np.exp2(e - 3)
    return np.round(x / step) * step


def _bf16(x):
    return torch.from_numpy(x).to(torch.bfloat16).double().numpy()


def exact(case, seed):
    if case["op"] == "verify":
        return None
    st = prepare(case, seed)
    if case["op"] == "append":
        t, hq, hkv = case["tokens"], case["heads"], case["kv_heads"]
        x = st["qkv"].double().cpu().numpy().reshape(t, hq + 2 * hkv, HEAD)
        # the model's angle is the 32-bit product of position and frequency
        ang = (st["pos"].cpu().numpy().astype(np.float32)[:, None] * st["inv_freq"].numpy()[None]).astype(np.float64)
        c, s = np.cos(ang)[:, None] * st["conc"], np.sin(ang)[:, None] * st["conc"]
        lo, hi = x[:, :hq + hkv, :32], x[:, :hq + hkv, 32:]
        rot = np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)
        out, slots = {"q": rot[:, :hq]}, st["slots"].cpu().numpy()
        for name, val in (("k", _bf16(rot[:, hq:])), ("v", x[:, hq + hkv:])):
            amax = np.abs(val).max(-1)
            e = np.clip(np.ceil(np.log2(np.maximum(amax, 1e-300) / 448.0)), -60, 60)
            pool = np.zeros(st[name].shape)
            pool[slots] = _grid8(val * np.exp2(-e)[..., None])
            codes = np.ones((st["ks"].shape[0], PAGE, hkv))
            codes.reshape(-1, hkv)[slots] = np.exp2(e)
            out[name], out[name + "s"] = pool, np.ascontiguousarray(codes.transpose(0, 2, 1))
        return out
    if case["op"] == "read":
        out, table = {}, st["table"][0].cpu().numpy()
        p = np.arange(st["pos0"], st["pos0"] + st["n"])
        for a in ("k", "v"):
            val = st[a].double().reshape(-1, PAGE, case["kv_heads"], HEAD)
            val = val * st[a + "s"].double().transpose(1, 2).unsqueeze(-1)
            out[a] = val.cpu().numpy()[table[p // PAGE], p % PAGE]
        return out
    ql, kl = _lengths(case)
    hq, hkv, w = case["heads"], case["kv_heads"], case["window"]
    grp = hq // hkv
    k, v = st["k"].double(), st["v"].double()
    if case["f8"]:
        k, v = (x.reshape(-1, PAGE, hkv, HEAD) * c.double().transpose(1, 2).unsqueeze(-1)
                for x, c in ((k, st["ks"]), (v, st["vs"])))
    k, v = k.reshape(-1, PAGE, hkv, HEAD), v.reshape(-1, PAGE, hkv, HEAD)
    o = torch.empty(sum(ql), hq, HEAD, dtype=torch.float64, device="cuda")
    lse = torch.empty(sum(ql), hq, dtype=torch.float64, device="cuda")
    at, stride = 0, st["table"].shape[1]
    for b in range(case["seqs"]):
        n, length = ql[b], kl[b]
        first = max(0, length - (w + n - 1)) if w else 0
        p = torch.arange(first, length, device="cuda")
        page = st["table"][b].long()[(p // PAGE) % stride]
        kb, vb = k[page, p % PAGE], v[page, p % PAGE]
        pos = torch.arange(length - n, length, device="cuda")[:, None]
        hidden = (p[None] > pos) | ((p[None] <= pos - w) if w else (p[None] < 0))
        for h in range(hq):
            s = st["q"][at:at + n, h].double() @ kb[:, h // grp].T / 8.0
            s.masked_fill_(hidden, -math.inf)
            lg = torch.logsumexp(s, -1)
            both = torch.logaddexp(lg, st["sinks"][h].double())
            o[at:at + n, h] = torch.exp(s - both[:, None]) @ vb[:, h // grp]
            lse[at:at + n, h] = lg / math.log(2.0)
        at += n
    return {"o": o, "lse": lse}
