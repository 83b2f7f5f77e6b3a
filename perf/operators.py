"""Serving operators measured on one GPU: the 8-bit KV cache (append with QK-norm and RoPE, read-back,
decode attention), decode attention over a batch that shares a prefix, and the rules on logits.

`run` computes an operator in plain torch operations, or (with `own` set) through mllm_b200.runtime;
`exact` computes the same from the definitions in 64 bits.

Definitions
  append      per head: x * rsqrt(mean(x^2) + eps) * w for q and k (where norm weights are given), then the
              rotation of the pairs (d, d + D/2) by the given cos/sin rows.  q is rounded to bf16.  A K or V
              row (one token, one kv head) is stored as e4m3 values and one power of two 2^e, e the smallest
              integer in [-100, 120] with max|row| <= 448 * 2^e.
  read        the stored rows as bf16 (exact), zero past a sequence's length.
  decode      softmax(q K^T / sqrt(D)) V for one query per sequence over its cache rows.
  shared      the same over a bf16 cache whose sequences have their first `prefix` rows in common.
  logits      penalties, bias and mask on a row of logits; see `_plain_logits`.
"""
import math

import torch

own = False

BF16 = torch.bfloat16
FP8 = torch.float8_e4m3fn
E4M3_MAX = 448.0
E_MIN, E_MAX = -100, 120
EPS = 1e-6


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # Qwen3-8B decode step: one new token for each of 32 sequences behind 4096 cached rows
        {"name": "append_decode_32", "op": "append", "heads": 32, "kv_heads": 8, "dim": 128, "norm": True,
         "tokens": "1*32", "start": "4096*32", "block": 256},
        # Qwen3-8B prompts of different lengths joining a serving batch, packed in one call
        {"name": "append_prompts", "op": "append", "heads": 32, "kv_heads": 8, "dim": 128, "norm": True,
         "tokens": "8192,5001,2048,777", "start": "0*4", "block": 256},
        # TinyLlama geometry, one sequence just after a 512-token prompt: the latency of one small call
        {"name": "decode8_1x513", "op": "decode8", "heads": 32, "kv_heads": 4, "dim": 64, "lens": "513",
         "block": 128},
        # Qwen3-8B decode, 32 sequences of 4096 rows
        {"name": "decode8_32x4096", "op": "decode8", "heads": 32, "kv_heads": 8, "dim": 128,
         "lens": "4096*32", "block": 256},
        # Qwen3-14B decode of 64 ragged requests, 256 .. 32768 rows each
        {"name": "decode8_ragged_64", "op": "decode8", "heads": 40, "kv_heads": 8, "dim": 128,
         "lens": "ragged:64:256:32768:14", "block": 256},
        # a second chunk of a prompt needs the first chunk's rows back: two short sequences
        {"name": "read8_2x300", "op": "read8", "kv_heads": 8, "dim": 128, "lens": "300,129", "rows": 300,
         "block": 128},
        # eight 2048-row prompts of a batch read back for their next chunk (some shorter)
        {"name": "read8_8x2048", "op": "read8", "kv_heads": 8, "dim": 128,
         "lens": "2048,2048,1999,2048,1,1024,2048,700", "rows": 2048, "block": 256},
        # TinyLlama geometry, eight requests behind a 512-token system prompt
        {"name": "shared_8x512", "op": "shared", "heads": 32, "kv_heads": 4, "dim": 64, "prefix": 512,
         "suffix": "ragged:8:1:64:3", "block": 128},
        # Qwen3-8B, 32 requests behind an 8192-token prompt (a document, few-shot examples)
        {"name": "shared_32x8192", "op": "shared", "heads": 32, "kv_heads": 8, "dim": 128, "prefix": 8192,
         "suffix": "ragged:32:1:512:5", "block": 256},
        # Qwen3-14B, 64 requests behind a 32768-token prompt that ends inside a page
        {"name": "shared_64x32700", "op": "shared", "heads": 40, "kv_heads": 8, "dim": 128, "prefix": 32700,
         "suffix": "ragged:64:64:2048:7", "block": 256},
        # one chat request: Qwen3 vocabulary, fp32 logits, a short history and a few biases, no grammar
        {"name": "logits_1", "op": "logits", "rows": 1, "vocab": 151936, "bf16": False, "history": "200",
         "bias": 8, "mask": False},
        # 64 requests with long histories under a grammar
        {"name": "logits_64", "op": "logits", "rows": 64, "vocab": 151936, "bf16": False,
         "history": "ragged:64:0:5000:9", "bias": 40, "mask": True},
    ]


_HEADS = [(32, 8, 128), (40, 8, 128), (32, 4, 64), (8, 2, 128), (10, 2, 128), (5, 1, 128), (4, 4, 64)]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "append", "decode8", "decode8", "decode8", "read8", "shared", "shared", "shared",
                     "logits", "logits"])
    H, Hkv, D = rng.choice(_HEADS)
    block = rng.choice([128, 256, 384])
    if op == "append":
        n = _log_int(rng, 1, 64)
        most = max(1, 16000 // n)
        kind = rng.choice(["one", "many"])
        tokens = [1 if kind == "one" else _log_int(rng, 1, most) for _ in range(n)]
        start = [0 if rng.random() < 0.3 else _log_int(rng, 1, 4096) for _ in range(n)]
        return {"op": op, "heads": H, "kv_heads": Hkv, "dim": D, "norm": rng.random() < 0.7,
                "tokens": ",".join(map(str, tokens)), "start": ",".join(map(str, start)), "block": block}
    if op == "decode8":
        n = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, min(32768, 1000000 // n))
        return {"op": op, "heads": H, "kv_heads": Hkv, "dim": D, "block": block,
                "lens": f"ragged:{n}:{_log_int(rng, 1, hi)}:{hi}:{rng.randrange(1 << 20)}"}
    if op == "read8":
        n = _log_int(rng, 1, 16)
        lens = [_log_int(rng, 1, max(1, 16000 // n)) for _ in range(n)]
        return {"op": op, "kv_heads": Hkv, "dim": D, "block": block, "lens": ",".join(map(str, lens)),
                "rows": max(lens) + rng.randrange(0, 20)}
    if op == "shared":
        n = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, min(2048, 65000 // n))
        return {"op": op, "heads": H, "kv_heads": Hkv, "dim": D, "block": block, "prefix": _log_int(rng, 1, 32700),
                "suffix": f"ragged:{n}:{_log_int(rng, 1, hi)}:{hi}:{rng.randrange(1 << 20)}"}
    n = _log_int(rng, 1, 64)
    return {"op": op, "rows": n, "vocab": _log_int(rng, 1000, 151936), "bf16": rng.random() < 0.5,
            "history": f"ragged:{n}:0:{_log_int(rng, 1, 5000)}:{rng.randrange(1 << 20)}",
            "bias": rng.randrange(0, 41), "mask": rng.random() < 0.6}


def _ints(text):
    """'3,4,5', '7*32' or 'ragged:n:lo:hi:seed' -> a list of whole numbers."""
    if text.startswith("ragged:"):
        n, lo, hi, seed = map(int, text.split(":")[1:])
        g = torch.Generator().manual_seed(seed)
        return torch.randint(lo, hi + 1, (n,), generator=g).tolist()
    out = []
    for part in text.split(","):
        v, _, k = part.partition("*")
        out += [int(v)] * (int(k) if k else 1)
    return out


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *size):
    return torch.randn(*size, device="cuda", generator=g)


# ------------------------------------------------------------------------------------------------
# pages
# ------------------------------------------------------------------------------------------------
def _page_order(lens, block):
    """Blocks of each sequence when all of them grow together, one block at a time."""
    need = [-(-n // block) for n in lens]
    blocks = [[] for _ in lens]
    nxt = 0
    for i in range(max(need + [0])):
        for b, k in enumerate(need):
            if i < k:
                blocks[b].append(nxt)
                nxt += 1
    return blocks, nxt


def _table(blocks):
    width = max(1, max(len(x) for x in blocks))
    return torch.tensor([x + [0] * (width - len(x)) for x in blocks], dtype=torch.int32, device="cuda")


def _pool8(g, blocks, Hkv, block, D):
    """Random e4m3 rows with their largest element near 448, as quantised rows have, and exponents around
    that of unit-variance keys (or values, which vary more from row to row)."""
    pool = torch.empty((blocks, Hkv, block, D), dtype=FP8, device="cuda")
    for i in range(0, blocks, 256):
        j = min(blocks, i + 256)
        pool[i:j] = (_randn(g, j - i, Hkv, block, D) * 110).clamp_(-E4M3_MAX, E4M3_MAX).to(FP8)
    return pool


def _exps(g, blocks, Hkv, block, lo, hi):
    return torch.randint(127 + lo, 127 + hi + 1, (blocks, Hkv, block), device="cuda", generator=g).to(torch.uint8)


def _cache8(st, lens):
    """The framework's cache object holding the state's pools."""
    from mllm_b200 import runtime as rt
    nb, Hkv, block, D = st["kp"].shape
    blocks = st["blocks"]
    c = rt.PagedKVCache8(nb, Hkv, D, block_size=block, max_seqs=len(lens), max_blocks_per_seq=st["table"].shape[1])
    for i in range(max(len(x) for x in blocks)):
        for b, x in enumerate(blocks):
            if i < len(x):
                c.reserve(b, (i + 1) * block)
    c.set_lengths(lens)
    c.k_pool, c.v_pool, c.k_exp, c.v_exp = st["kp"], st["vp"], st["ke"], st["ve"]
    c.block_table.copy_(st["table"])
    return c


def prepare(case, seed):
    return {"append": _prep_append, "decode8": _prep_decode8, "read8": _prep_read8, "shared": _prep_shared,
            "logits": _prep_logits}[case["op"]](case, _gen(seed))


def _prep_append(case, g):
    H, Hkv, D, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    tokens, start = _ints(case["tokens"]), _ints(case["start"])
    T = sum(tokens)
    ends = [s + n for s, n in zip(start, tokens)]
    qkv = _randn(g, T, (H + 2 * Hkv) * D).bfloat16()
    pos = torch.cat([torch.arange(s, e, dtype=torch.float64) for s, e in zip(start, ends)]).cuda()
    inv = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    ang = torch.cat([pos[:, None] * inv] * 2, 1)
    blocks, nb = _page_order(ends, block)
    cu = [0]
    for n in tokens:
        cu.append(cu[-1] + n)
    st = {"op": "append", "q": qkv[:, : H * D].view(T, H, D), "k": qkv[:, H * D:(H + Hkv) * D].view(T, Hkv, D),
          "v": qkv[:, (H + Hkv) * D:].view(T, Hkv, D), "cos": ang.cos().float(), "sin": ang.sin().float(),
          "qn": None, "kn": None, "blocks": blocks, "table": _table(blocks),
          "cu": torch.tensor(cu, dtype=torch.int32, device="cuda"),
          "start": torch.tensor(start, dtype=torch.int32, device="cuda"),
          "lens": torch.tensor(ends, dtype=torch.int32, device="cuda"), "rows": max(tokens)}
    if case["norm"]:
        st["qn"] = (1 + 0.1 * _randn(g, D)).bfloat16()
        st["kn"] = (1 + 0.1 * _randn(g, D)).bfloat16()
    seq = torch.cat([torch.full((n,), b, dtype=torch.int64) for b, n in enumerate(tokens)]).cuda()
    st["seq"], st["slot"] = seq, pos.long()
    st["kp"], st["vp"] = _pool8(g, nb, Hkv, block, D), _pool8(g, nb, Hkv, block, D)
    st["ke"], st["ve"] = _exps(g, nb, Hkv, block, -8, -6), _exps(g, nb, Hkv, block, -9, -5)
    if own:
        st["cache"] = _cache8(st, ends)
    return st


def _prep_decode8(case, g):
    H, Hkv, D, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    lens = _ints(case["lens"])
    blocks, nb = _page_order(lens, block)
    st = {"op": "decode8", "q": (1.5 * _randn(g, len(lens), H, D)).bfloat16(), "blocks": blocks,
          "table": _table(blocks), "host_lens": lens, "max_len": max(lens),
          "kp": _pool8(g, nb, Hkv, block, D), "vp": _pool8(g, nb, Hkv, block, D),
          "ke": _exps(g, nb, Hkv, block, -8, -6), "ve": _exps(g, nb, Hkv, block, -9, -5)}
    if own:
        st["cache"] = _cache8(st, lens)
    return st


def _prep_read8(case, g):
    Hkv, D, block = case["kv_heads"], case["dim"], case["block"]
    lens = _ints(case["lens"])
    blocks, nb = _page_order(lens, block)
    st = {"op": "read8", "blocks": blocks, "table": _table(blocks), "rows": case["rows"],
          "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
          "kp": _pool8(g, nb, Hkv, block, D), "vp": _pool8(g, nb, Hkv, block, D),
          "ke": _exps(g, nb, Hkv, block, -8, -6), "ve": _exps(g, nb, Hkv, block, -9, -5)}
    if own:
        st["cache"] = _cache8(st, lens)
    return st


def _shared_blocks(prefix, lens, block):
    """Sequence 0 holds the prefix; the others take its full blocks and a copy of its last, partial one;
    then every sequence gets blocks for its own rows, in order."""
    full, part = prefix // block, prefix % block
    blocks = [list(range(full + (part > 0)))]
    nxt = len(blocks[0])
    copies = []
    for b in range(1, len(lens)):
        blocks.append(list(range(full)))
        if part:
            copies.append((full, nxt))
            blocks[b].append(nxt)
            nxt += 1
    for b, n in enumerate(lens):
        while len(blocks[b]) * block < n:
            blocks[b].append(nxt)
            nxt += 1
    return blocks, nxt, copies


def _prep_shared(case, g):
    H, Hkv, D, block, P = case["heads"], case["kv_heads"], case["dim"], case["block"], case["prefix"]
    lens = [P + s for s in _ints(case["suffix"])]
    blocks, nb, copies = _shared_blocks(P, lens, block)
    kp = _randn(g, nb, Hkv, block, D).bfloat16()
    vp = _randn(g, nb, Hkv, block, D).bfloat16()
    for src, dst in copies:
        kp[dst, :, : P % block] = kp[src, :, : P % block]
        vp[dst, :, : P % block] = vp[src, :, : P % block]
    st = {"op": "shared", "q": (1.5 * _randn(g, len(lens), H, D)).bfloat16(), "kp": kp, "vp": vp,
          "table": _table(blocks), "host_lens": lens, "max_len": max(lens), "prefix": P}
    if own:
        from mllm_b200 import runtime as rt
        c = rt.PagedKVCache(nb, Hkv, D, block_size=block, max_seqs=len(lens), max_blocks_per_seq=st["table"].shape[1])
        c.reserve(0, P)
        for b in range(1, len(lens)):
            c.fork(0, b, P)
        c.set_lengths(lens)
        c.k_pool, c.v_pool = kp, vp
        c.block_table.copy_(st["table"])
        st["cache"] = c
    return st


def _prep_logits(case, g):
    B, V, nb = case["rows"], case["vocab"], case["bias"]
    lens = _ints(case["history"])
    n = max(lens + [1])
    x = 3 * _randn(g, B, V)
    # generated text repeats itself: half of the history comes from a small set of tokens
    few = torch.randint(0, V, (B, 50), device="cuda", generator=g)
    pick = torch.randint(0, 50, (B, n), device="cuda", generator=g)
    hist = torch.where(torch.rand(B, n, device="cuda", generator=g) < 0.5,
                       torch.randint(0, V, (B, n), device="cuda", generator=g), few.gather(1, pick))
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st = {"op": "logits", "hist": hist, "hist_lens": lens, "out_start": lens // 3,
          "rep": 1 + 0.5 * torch.rand(B, device="cuda", generator=g),
          "pres": 0.5 * torch.rand(B, device="cuda", generator=g),
          "freq": 0.25 * torch.rand(B, device="cuda", generator=g), "mask": None,
          "bias_ids": None, "bias_vals": None, "bias_lens": None}
    if nb:
        st["bias_ids"] = torch.randint(0, V, (B, nb), device="cuda", generator=g)
        st["bias_ids"][:, 0] = hist[:, 0]                       # a bias on a token that was seen
        st["bias_vals"] = torch.randint(-40, 41, (B, nb), device="cuda", generator=g) / 8.0
        st["bias_lens"] = torch.randint(0, nb + 1, (B,), device="cuda", generator=g).int()
    if case["mask"]:
        # a grammar allows a share of the vocabulary that differs from row to row
        allow = torch.rand(B, V, device="cuda", generator=g) < torch.rand(B, 1, device="cuda", generator=g)
        x = torch.where(~allow & (torch.rand(B, V, device="cuda", generator=g) < 1e-3), float("nan"), x)
        bits = torch.nn.functional.pad(allow, (0, -V % 32)).view(B, -1, 32).long()
        words = (bits << torch.arange(32, device="cuda")).sum(-1)
        st["mask"] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()
    st["x"] = x.bfloat16() if case["bf16"] else x
    return st


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


def _own_append(st):
    from mllm_b200 import runtime as rt
    q = rt.qkv_epilogue_kv8(st["q"], st["k"], st["v"], st["cache"], st["cu"], st["start"],
                            rope_table=(st["cos"], st["sin"]), q_norm_weight=st["qn"], k_norm_weight=st["kn"], eps=EPS)
    k, v = rt.kv8_read(st["cache"], st["lens"], st["rows"], first=st["start"])
    return q, k, v


def _own_decode8(st):
    from mllm_b200 import runtime as rt
    return rt.decode_attention(st["q"], st["cache"], st["kp"].shape[1], max_kv_len=st["max_len"])


def _own_read8(st):
    from mllm_b200 import runtime as rt
    return rt.kv8_read(st["cache"], st["lens"], st["rows"])


def _own_shared(st):
    from mllm_b200 import runtime as rt
    return rt.decode_attention_shared(st["q"], st["cache"], st["kp"].shape[1], st["prefix"],
                                      max_kv_len=st["max_len"])


def _own_logits(st):
    from mllm_b200 import runtime as rt
    return rt.apply_logit_rules(st["x"], history=st["hist"], history_lens=st["hist_lens"],
                                output_start=st["out_start"], repetition=st["rep"], presence=st["pres"],
                                frequency=st["freq"], bias_ids=st["bias_ids"], bias_values=st["bias_vals"],
                                bias_lens=st["bias_lens"], allowed=st["mask"])


def _quantise(y):
    """fp32 rows -> (e4m3 values, exponent bytes)."""
    amax = y.abs().amax(-1)
    m, x = torch.frexp(amax)                                    # amax = m 2^x, 0.5 <= m < 1
    e = torch.where(m <= 0.875, x - 9, x - 8).clamp(E_MIN, E_MAX)
    return torch.ldexp(y, -e[..., None]).to(FP8), (e + 127).to(torch.uint8)


def _dequantise(values, exps):
    return torch.ldexp(values.float(), (exps.int() - 127)[..., None])


def _plain_append(st):
    def norm_rope(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        h = x.shape[-1] // 2
        turned = torch.cat([-x[..., h:], x[..., :h]], -1)
        return x * st["cos"][:, None] + turned * st["sin"][:, None]
    q = norm_rope(st["q"], st["qn"]).bfloat16()
    block = st["kp"].shape[2]
    blk, row = st["table"][st["seq"], st["slot"] // block].long(), st["slot"] % block
    n, Hkv, D = st["table"].shape[0], st["kp"].shape[1], st["kp"].shape[3]
    at = torch.arange(len(st["seq"]), device="cuda") - st["cu"][st["seq"]].long()
    outs = []
    for x, w, pool, exps in ((st["k"], st["kn"], "kp", "ke"), (st["v"], None, "vp", "ve")):
        y = norm_rope(x, w) if pool == "kp" else x.float()
        v8, e8 = _quantise(y)
        st[pool].view(torch.uint8)[blk, :, row] = v8.view(torch.uint8)
        st[exps][blk, :, row] = e8
        back = torch.zeros((n, st["rows"], Hkv, D), dtype=BF16, device="cuda")
        back[st["seq"], at] = _dequantise(st[pool].view(torch.uint8)[blk, :, row].view(FP8), st[exps][blk, :, row]).bfloat16()
        outs.append(back.transpose(1, 2).contiguous())
    return q, outs[0], outs[1]


def _rows(pool, table, b, first, last):
    """Cache rows first .. last - 1 of sequence b, [Hkv, rows, ...]."""
    block = pool.shape[2]
    blks = table[b, first // block: -(-last // block)].long()
    x = pool.view(torch.uint8)[blks].view(pool.dtype) if pool.dtype == FP8 else pool[blks]
    x = x.transpose(0, 1).flatten(1, 2)
    off = first // block * block
    return x[:, first - off: last - off]


def _rows8(st, which, b, first, last):
    return _dequantise(_rows(st[which + "p"], st["table"], b, first, last),
                       _rows(st[which + "e"].unsqueeze(-1), st["table"], b, first, last).squeeze(-1))


def _plain_read8(st):
    outs = []
    for which in ("k", "v"):
        _, Hkv, block, D = st[which + "p"].shape
        out = torch.zeros((st["table"].shape[0], Hkv, st["rows"], D), dtype=BF16, device="cuda")
        for b, x in enumerate(st["blocks"]):
            n = min(len(x) * block, st["rows"])
            keep = (torch.arange(n, device="cuda") < st["lens"][b])[None, :, None]
            out[b, :, :n] = torch.where(keep, _rows8(st, which, b, 0, n), 0.0).bfloat16()
        outs.append(out)
    return tuple(outs)


def _attend(q, k, v):
    """q [Hkv, n, D], k and v [Hkv, L, D], fp32 -> [Hkv, n, D]."""
    s = q @ k.transpose(1, 2) / math.sqrt(q.shape[-1])
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return (p @ v) / p.sum(-1, keepdim=True)


def _plain_decode8(st):
    q = st["q"].float()
    B, H, D = q.shape
    Hkv = st["kp"].shape[1]
    out = torch.empty((B, 1, H * D), dtype=BF16, device="cuda")
    for b, n in enumerate(st["host_lens"]):
        o = _attend(q[b].view(Hkv, H // Hkv, D), _rows8(st, "k", b, 0, n), _rows8(st, "v", b, 0, n))
        out[b, 0] = o.reshape(-1).bfloat16()
    return out


def _plain_shared(st):
    """The prefix once for all rows of the batch, every sequence's own rows, joined by their maxima and sums."""
    q = st["q"].float()
    B, H, D = q.shape
    Hkv, P = st["kp"].shape[1], st["prefix"]
    R = H // Hkv
    qg = q.view(B, Hkv, R, D).transpose(0, 1).reshape(Hkv, B * R, D)

    def part(qq, k, v):
        s = qq @ k.float().transpose(1, 2) / math.sqrt(D)
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - m)
        return m, p.sum(-1, keepdim=True), p @ v.float()
    m0, l0, o0 = (x.view(Hkv, B, R, -1) for x in part(qg, _rows(st["kp"], st["table"], 0, 0, P),
                                                      _rows(st["vp"], st["table"], 0, 0, P)))
    out = torch.empty((B, 1, H * D), dtype=BF16, device="cuda")
    for b, n in enumerate(st["host_lens"]):
        m1, l1, o1 = part(q[b].view(Hkv, R, D), _rows(st["kp"], st["table"], b, P, n), _rows(st["vp"], st["table"], b, P, n))
        m = torch.maximum(m0[:, b], m1)
        w0, w1 = torch.exp(m0[:, b] - m), torch.exp(m1 - m)
        out[b, 0] = ((o0[:, b] * w0 + o1 * w1) / (l0[:, b] * w0 + l1 * w1)).reshape(-1).bfloat16()
    return out


def _plain_logits(st):
    """A token that occurs in the history: x / r (x >= 0) or x * r (x < 0).  Then minus frequency times its count
    among the generated tokens (from output_start on), minus presence if that count is not zero, plus its biases;
    -inf where the mask forbids the token."""
    x = st["x"].float()
    B, V = x.shape
    at = torch.arange(st["hist"].shape[1], device="cuda")
    valid = at < st["hist_lens"][:, None]
    made = valid & (at >= st["out_start"][:, None])
    seen = torch.zeros((B, V), device="cuda").scatter_add_(1, st["hist"], valid.float()) > 0
    count = torch.zeros((B, V), device="cuda").scatter_add_(1, st["hist"], made.float())
    r = st["rep"][:, None]
    x = torch.where(seen, torch.where(x < 0, x * r, x / r), x)
    x = x - count * st["freq"][:, None] - (count > 0) * st["pres"][:, None]
    if st["bias_ids"] is not None:
        use = torch.arange(st["bias_ids"].shape[1], device="cuda") < st["bias_lens"][:, None]
        x = x + torch.zeros((B, V), device="cuda").scatter_add_(1, st["bias_ids"], torch.where(use, st["bias_vals"], 0.0))
    if st["mask"] is not None:
        v = torch.arange(V, device="cuda")
        x = torch.where((st["mask"][:, v // 32] >> (v % 32)) & 1 == 1, x, float("-inf"))
    return x.to(st["x"].dtype)


_PLAIN = {"append": _plain_append, "decode8": _plain_decode8, "read8": _plain_read8, "shared": _plain_shared,
          "logits": _plain_logits}
_OWN = {"append": _own_append, "decode8": _own_decode8, "read8": _own_read8, "shared": _own_shared,
        "logits": _own_logits}


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "logits":
        B, V, n = case["rows"], case["vocab"], sum(_ints(case["history"]))
        return {"bytes": B * V * 2 * (2 if case["bf16"] else 4) + case["mask"] * B * V // 8 + 8 * n
                + 12 * B * case["bias"], "flops": B * V + 4 * n}
    Hkv, D = case["kv_heads"], case["dim"]
    if op == "read8":
        lens = _ints(case["lens"])
        return {"bytes": 2 * Hkv * (sum(lens) * (D + 1) + len(lens) * case["rows"] * D * 2),
                "flops": 2 * Hkv * sum(lens) * D}
    H = case["heads"]
    if op == "append":
        tokens = _ints(case["tokens"])
        T, n = sum(tokens), len(tokens)
        return {"bytes": T * (2 * H * D * 2 + 2 * Hkv * D * 2 + 2 * Hkv * (D + 1) + 8 * D)
                + n * max(tokens) * 2 * Hkv * D * 2, "flops": T * D * (10 * (H + Hkv) + 3 * Hkv)}
    if op == "decode8":
        lens = _ints(case["lens"])
        return {"bytes": 2 * Hkv * (D + 1) * sum(lens) + 4 * len(lens) * H * D, "flops": 4 * H * D * sum(lens)}
    suffix, P = _ints(case["suffix"]), case["prefix"]
    return {"bytes": 4 * Hkv * D * (P + sum(suffix)) + 4 * len(suffix) * H * D,
            "flops": 4 * H * D * (P * len(suffix) + sum(suffix))}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    before, own = own, False                    # plain inputs are enough here
    try:
        st = prepare(case, seed)
    finally:
        own = before
    return _EXACT[case["op"]](st, case)


def _e4m3_64(x):
    """Nearest e4m3 value of a 64-bit number of magnitude at most 448, ties to the even mantissa."""
    ax = x.abs().clamp_min(1e-300)
    step = torch.exp2((torch.floor(torch.log2(ax))).clamp_min(-6.0) - 3)
    return torch.round(x / step) * step


def _exact_append(st, case):
    c, s = st["cos"].double(), st["sin"].double()

    def head(x, w):                             # x [T, D], 64 bits
        if w is not None:
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()
        lo, hi = x.chunk(2, -1)
        h = lo.shape[-1]
        return torch.cat([lo * c[:, :h] - hi * s[:, :h], hi * c[:, h:] + lo * s[:, h:]], -1)

    def stored(y):
        scale = torch.exp2(torch.ceil(torch.log2(y.abs().amax(-1, keepdim=True).clamp_min(1e-300) / 448))
                           .clamp(E_MIN, E_MAX))
        return _e4m3_64(y / scale) * scale
    q = torch.stack([head(st["q"][:, h].double(), st["qn"]) for h in range(case["heads"])], 1)
    tokens = _ints(case["tokens"])
    k = torch.zeros((len(tokens), case["kv_heads"], max(tokens), case["dim"]), dtype=torch.float64, device="cuda")
    v = torch.zeros_like(k)
    for h in range(case["kv_heads"]):
        kk, vv = stored(head(st["k"][:, h].double(), st["kn"])), stored(st["v"][:, h].double())
        t = 0
        for b, n in enumerate(tokens):
            k[b, h, :n], v[b, h, :n] = kk[t:t + n], vv[t:t + n]
            t += n
    return q, k, v


def _seq64(st, which, b, n, g=None):
    """Rows 0 .. n - 1 of sequence b as 64-bit numbers, block by block."""
    pool = st[which + "p"]
    parts = []
    for i in range(-(-n // pool.shape[2])):
        blk = int(st["host_table"][b][i])
        x = pool[blk].double()
        if which + "e" in st:
            x = x * torch.exp2(st[which + "e"][blk].double() - 127).unsqueeze(-1)
        parts.append(x)
    return torch.cat(parts, 1)[:, :n]


def _exact_read8(st, case):
    st["host_table"] = st["table"].tolist()
    outs = []
    for which in ("k", "v"):
        lens = _ints(case["lens"])
        out = torch.zeros((len(lens), case["kv_heads"], case["rows"], case["dim"]), dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            out[b, :, :n] = _seq64(st, which, b, n)
        outs.append(out)
    return tuple(outs)


def _exact_decode(st, case):
    st["host_table"] = st["table"].tolist()
    q = st["q"].double()
    B, H, D = q.shape
    R = H // case["kv_heads"]
    out = torch.empty((B, 1, H * D), dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["host_lens"]):
        k, v = _seq64(st, "k", b, n), _seq64(st, "v", b, n)
        w = torch.softmax(torch.einsum("grd,gtd->grt", q[b].view(-1, R, D), k) * D ** -0.5, -1)
        out[b, 0] = torch.einsum("grt,gtd->grd", w, v).reshape(-1)
    return out


def _exact_logits(st, case):
    x = st["x"].double()
    B, V = x.shape
    n = st["hist_lens"].tolist()
    first = st["out_start"].tolist()
    for b in range(B):
        h = st["hist"][b, :n[b]]
        seen, made = torch.unique(h), torch.bincount(h[first[b]:], minlength=V)
        r = st["rep"][b].double()
        x[b, seen] = torch.where(x[b, seen] < 0, x[b, seen] * r, x[b, seen] / r)
        x[b] -= made * st["freq"][b].double() + (made > 0) * st["pres"][b].double()
        if st["bias_ids"] is not None:
            m = int(st["bias_lens"][b])
            x[b] += torch.bincount(st["bias_ids"][b, :m], weights=st["bias_vals"][b, :m].double(), minlength=V)
        if st["mask"] is not None:
            words = st["mask"][b].long() & 0xFFFFFFFF
            allow = (words[:, None] >> torch.arange(32, device="cuda")) & 1
            x[b, allow.flatten()[:V] == 0] = float("-inf")
    return x


_EXACT = {"append": _exact_append, "decode8": _exact_decode, "read8": _exact_read8, "shared": _exact_decode,
          "logits": _exact_logits}
