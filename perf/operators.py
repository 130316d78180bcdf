"""The paged key-value cache operators, measured: cases, plain forms, 64-bit values.

Five operators stand between the q|k|v projection of a decode or prefill step
and its output projection:

  norm_rope   per-head RMS norm of queries and keys and the position rotation
  fused       the same, with the keys and values written to the paged cache
  roundtrip   keys and values written to a Q8_0 cache (quantised as written),
              then the sequences read back as values
  gather      positions of a paged cache read back in a given order
  attention   one query token per sequence over its pages

A case is a dict of sizes.  ``run`` computes it from elementary torch
operations, or with ``own`` set through the ``tir`` package.  Every size that a
kernel sees follows from the case alone (lengths, positions); the values and
the order of the pages follow from the seed.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "q8_0": torch.int8}
_ES = {"f32": 4.0, "f16": 2.0, "bf16": 2.0, "q8_0": 34.0 / 32.0}
EPS = 1e-5
BASE = 10000.0


def _tir():
    pkg = os.path.join(_ROOT, "tensor-inference-runtime_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import tir
    return tir


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _case(op, dtype, cache, seqs, new, ctx, heads, page, lens="same", pairs="adjacent", norm=True, pad=0, window=0):
    """seqs sequences, each appending `new` tokens (attention: one query); ctx:
    positions held afterwards (the longest, where lens is "ragged")."""
    q_heads, kv_heads, dim = heads
    return {"op": op, "dtype": dtype, "cache": cache, "seqs": seqs, "new": new, "ctx": ctx, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "lens": lens, "pairs": pairs, "norm": norm, "pad": pad,
            "window": window}


_TINY = (32, 4, 64)    # the heads of the runtime's own TinyLlama shape
_WIDE = (32, 8, 128)   # a wider model: four query heads per key-value head


def listed():
    c = {
        # one sequence decoding: the smallest call, all latency
        "norm_rope_one_f32": _case("norm_rope", "f32", "f32", 1, 1, 145, _TINY, 16),
        # the runtime's prefill workload: 16 prompts of 512 tokens
        "norm_rope_prefill_f32": _case("norm_rope", "f32", "f32", 16, 512, 512, _TINY, 16),
        # 64 sequences decoding, two of the batch's rows idle
        "fused_decode64_bf16": _case("fused", "bf16", "bf16", 64, 1, 47, _WIDE, 16, pairs="halves", pad=2),
        # ragged prompts joining a batch, an odd token count
        "fused_prefill_f16": _case("fused", "f16", "f16", 7, 587, 587, _WIDE, 16, pairs="halves"),
        # 64 sequences decoding into a quantised cache, then moved out whole
        "roundtrip_decode64_q8": _case("roundtrip", "f32", "q8_0", 64, 1, 130, _TINY, 16),
        # prompts quantised as they are written, read back in 16 bits
        "roundtrip_prefill_q8": _case("roundtrip", "bf16", "q8_0", 8, 1024, 1024, _WIDE, 16),
        # one long sequence moved out of the runtime's f32 cache
        "gather_long_f32": _case("gather", "f32", "f32", 1, 1, 2047, _TINY, 16),
        # the default decode workload's last step: 16 + 128 positions
        "attn_one_f32": _case("attention", "f32", "f32", 1, 1, 144, _TINY, 16),
        # the batched workload's last step in the runtime's own cache type
        "attn_batch64_f32": _case("attention", "f32", "f32", 64, 1, 256, _TINY, 16),
        # the long-context workload, quantised, 32 sequences of different length
        "attn_ragged_q8": _case("attention", "f32", "q8_0", 32, 1, 8191, _TINY, 16, lens="ragged"),
        # one very long document
        "attn_long_one_bf16": _case("attention", "bf16", "bf16", 1, 1, 131071, _WIDE, 64),
        # a full serving batch of different lengths
        "attn_ragged64_bf16": _case("attention", "bf16", "bf16", 64, 1, 8192, _WIDE, 16, lens="ragged"),
    }
    return [{"name": n, **v} for n, v in c.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "fused", "roundtrip", "gather", "attention", "attention", "attention"])
    dim = rng.choice([64, 64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8, 12])
    heads = (kv_heads * group, kv_heads, dim)
    page = rng.choice([1, 7, 16, 16, 32, 64, 100])
    dtype = rng.choice(["f32", "f32", "f16", "bf16"])
    cache = rng.choice([dtype, "q8_0"]) if dtype != "f32" else rng.choice(["f32", "f16", "bf16", "q8_0"])
    pairs = rng.choice(["adjacent", "halves"])
    if op == "attention":
        room = int((1 << 29) / max(2.0, _ES[cache]))  # cached keys: what the largest listed case may hold
        ctx = _log_int(rng, 1, 131072)
        ctx = max(1, min(ctx, room // (kv_heads * dim)))
        seqs = max(1, min(_log_int(rng, 1, 200), room // (kv_heads * dim * ctx)))
        window = rng.choice([0, 0, 0, max(1, ctx // 3)])
        return _case(op, dtype, cache, seqs, 1, ctx, heads, page, lens=rng.choice(["same", "ragged"]), window=window)
    decode = rng.random() < 0.4
    seqs = _log_int(rng, 1, 256) if decode else rng.randint(1, 12)
    new = 1 if decode else _log_int(rng, 2, 700)
    ctx = new + (rng.randint(0, 60) if decode else rng.choice([0, 0, 33]))
    pad = min(rng.choice([0, 0, 3]), seqs * new - 1)
    if op == "gather":
        new, ctx = 1, _log_int(rng, 1, 2000)
        seqs = max(1, min(seqs, 8192 // ctx))
    if op in ("roundtrip",):
        cache = "q8_0"
    if op == "fused" and cache == "q8_0":
        cache = dtype
    return _case(op, dtype, cache, seqs, new, ctx, heads, page, pairs=pairs, norm=rng.random() < 0.8, pad=pad)


def _lens(case):
    """Positions held by each sequence after the step; from the case alone."""
    n, ctx = case["seqs"], case["ctx"]
    if case["lens"] == "same":
        return [ctx] * n
    r = random.Random(n * 1000003 + ctx)
    out = [r.randint(1, ctx) for _ in range(n)]
    out[0] = ctx
    if n > 3:
        out[n // 2] = 0  # a finished sequence whose row is still in the batch
    return out


def _tokens(case):
    """(sequence, position) of the step's new tokens; -1 in the padded rows."""
    seq, pos = [], []
    for s in range(case["seqs"]):
        for i in range(case["new"]):
            seq.append(s)
            pos.append(case["ctx"] - case["new"] + i)
    for i in range(case["pad"]):  # idle rows of a padded batch, inside it
        pos[len(pos) - 1 - 2 * i if len(pos) > 2 * i + 1 else 0] = -1
    return seq, pos


def _held(case):
    """(sequence, position) of every position held."""
    n, ctx = case["seqs"], case["ctx"]
    return [s for s in range(n) for _ in range(ctx)], list(range(ctx)) * n


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dev, op = "cuda", case["op"]
    dt, ct = _DT[case["dtype"]], _DT[case["cache"]]
    qh, kh, d, ps, n = case["q_heads"], case["kv_heads"], case["dim"], case["page"], case["seqs"]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    # channels of different size, as projections have them
    k_chan = torch.exp(0.5 * normal(kh, d))
    s = {"case": dict(case)}
    if op != "norm_rope":
        pages = -(-case["ctx"] // ps)
        total = n * pages + 3
        order = torch.randperm(total, device=dev, generator=g)[:n * pages]
        s["table"] = order.to(torch.int32).reshape(n, pages).contiguous()
        shape = (total, ps, kh, d)
        if case["cache"] == "q8_0":
            for x in "kv":
                s[x + "_pool"] = torch.randint(-127, 128, shape, device=dev, generator=g, dtype=torch.int8)
                s[x + "_scale"] = ((0.5 + torch.rand(total, ps, kh, d // 32, device=dev, generator=g)) / 64).half()
        else:
            s["k_pool"] = (normal(*shape) * k_chan).to(ct)
            s["v_pool"] = normal(*shape).to(ct)
    if op == "attention":
        s["q"] = (normal(n, qh, d) * 1.5).to(dt)
        s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device=dev)
        s["out"] = torch.zeros(n, qh, d, dtype=dt, device=dev)
    elif op == "gather":
        seq, pos = _held(case)
        s["back_seq"], s["back_pos"] = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (seq, pos))
    else:
        seq, pos = _tokens(case)
        t = len(seq)
        s["seq"], s["pos"] = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (seq, pos))
        s["live"] = torch.tensor([i for i, x in enumerate(pos) if x >= 0], dtype=torch.int64, device=dev)
        # one row of the projection per token: q | k | v
        s["qkv"] = normal(t, (qh + 2 * kh) * d)
        s["qkv"][:, qh * d:(qh + kh) * d] *= k_chan.reshape(-1)
        s["qkv"] = s["qkv"].to(dt)
        s["q_w"], s["k_w"] = 1 + 0.1 * normal(d), 1 + 0.1 * normal(d)
        n_pos, half = case["ctx"], d // 2
        freq = np.float32(BASE) ** (-2.0 * np.arange(half, dtype=np.float32) / np.float32(d))
        ang = np.arange(n_pos, dtype=np.float32)[:, None] * freq.astype(np.float32)[None, :]
        table = np.stack([np.cos(ang.astype(np.float64)), np.sin(ang.astype(np.float64))], -1).astype(np.float32)
        s["rope"] = torch.from_numpy(np.ascontiguousarray(table)).to(dev)
        s["q_out"] = torch.zeros(t, qh, d, dtype=dt, device=dev)
        s["k_out"] = torch.zeros(t, kh, d, dtype=dt, device=dev)
        if op == "roundtrip":
            seq, pos = _held(case)
            s["back_seq"], s["back_pos"] = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (seq, pos))
    if op in ("gather", "roundtrip"):
        m = s["back_seq"].numel()
        s["k_back"] = torch.zeros(m, kh, d, dtype=dt, device=dev)
        s["v_back"] = torch.zeros(m, kh, d, dtype=dt, device=dev)
    if own:
        tir = _tir()
        if op != "norm_rope":
            s["kv"] = tir.KVPages(s["k_pool"], s["v_pool"], s["table"], s.get("k_scale"), s.get("v_scale"))
        if op == "attention":
            b = tir.paged_attention_workspace(s["kv"], n, qh, max_len=case["ctx"], window=case["window"])
            s["workspace"] = torch.empty(b, dtype=torch.uint8, device=dev)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _split(s):
    c = s["case"]
    qh, kh, d = c["q_heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].view(-1, qh + 2 * kh, d)
    return x[:, :qh], x[:, qh:qh + kh], x[:, qh + kh:]


def _rotate(x, cs, pairs):
    """x [t, h, d]; cs [t, d/2, 2]: (cos, sin) of each pair's angle."""
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    if pairs == "adjacent":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], -1).reshape(x.shape)
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _norm_rope(x, w, s, norm):
    x = x.float()
    if norm:
        x = x * w / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    return _rotate(x, s["rope"][s["pos"].long().clamp(min=0)], s["case"]["pairs"])


def _slots(s, seq, pos):
    ps = s["case"]["page"]
    pos = pos.long()
    return s["table"][seq.long(), pos // ps].long(), pos % ps


def _store(s, k, v):
    """Writes rows k, v (f32) to the cache at the new tokens' slots."""
    seq, pos = s["seq"], s["pos"]
    if s["case"]["pad"]:
        live = s["live"]
        seq, pos, k, v = seq[live], pos[live], k[live], v[live]
    at = _slots(s, seq, pos)
    for x, pool in ((k, "k"), (v, "v")):
        if s["case"]["cache"] != "q8_0":
            s[pool + "_pool"][at] = x.to(s[pool + "_pool"].dtype)
            continue
        b = x.reshape(*x.shape[:-1], -1, 32)
        a = b.abs()
        top = a.amax(-1, keepdim=True)
        # the last of the block's largest magnitudes gives the scale its sign
        last = torch.where(a == top, torch.arange(32, device=x.device), -1).amax(-1, keepdim=True)
        scale = b.gather(-1, last) / 127.0
        r = torch.where(scale == 0, 0.0, b / scale)
        whole = r.trunc()
        r = whole + torch.where((r - whole).abs() >= 0.5, r.sign(), 0.0)  # halves away from zero
        s[pool + "_pool"][at] = r.clamp(-128, 127).to(torch.int8).reshape(x.shape)
        s[pool + "_scale"][at] = scale.squeeze(-1).half()


def _load(s, at):
    out = []
    for x in "kv":
        y = s[x + "_pool"][at].float()
        if s["case"]["cache"] == "q8_0":
            y = (y.reshape(*y.shape[:-1], -1, 32) * s[x + "_scale"][at].float()[..., None]).reshape(y.shape)
        out.append(y)
    return out


def _run_plain(s):
    c = s["case"]
    op, dt = c["op"], _DT[c["dtype"]]
    if op in ("norm_rope", "fused"):
        q, k, v = _split(s)
        q, k = _norm_rope(q, s["q_w"], s, c["norm"]), _norm_rope(k, s["k_w"], s, c["norm"])
        live = (s["pos"] >= 0)[:, None, None]
        s["q_out"].copy_(torch.where(live, q.to(dt), s["q_out"]))
        if op == "norm_rope":
            s["k_out"].copy_(torch.where(live, k.to(dt), s["k_out"]))
            return s["q_out"], s["k_out"]
        _store(s, k, v.float())
        return s["q_out"], s["k_pool"], s["v_pool"]
    if op in ("roundtrip", "gather"):
        if op == "roundtrip":
            _, k, v = _split(s)
            _store(s, k.float(), v.float())
        k, v = _load(s, _slots(s, s["back_seq"], s["back_pos"]))
        s["k_back"].copy_(k)
        s["v_back"].copy_(v)
        return s["k_back"], s["v_back"]
    n, qh, kh, d, ctx = c["seqs"], c["q_heads"], c["kv_heads"], c["dim"], c["ctx"]
    where = torch.arange(ctx, device="cuda")
    k, v = _load(s, (s["table"].long()[:, where // c["page"]], (where % c["page"])[None, :].expand(n, -1)))
    q = s["q"].float().reshape(n, kh, qh // kh, d)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(d)      # [n, kh, group, ctx]
    lens = s["lens"].long()[:, None]
    seen = where[None] < lens
    if c["window"]:
        seen = seen & (where[None] >= lens - c["window"])
    x = torch.where(seen[:, None, None], x, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == float("-inf"), 0.0, top))
    o = torch.matmul(p, v.permute(0, 2, 1, 3)) / p.sum(-1, keepdim=True)
    s["out"].copy_(torch.where((lens > 0)[..., None], o.reshape(n, qh, d), 0.0))
    return s["out"]


def _run_own(s):
    tir = _tir()
    c = s["case"]
    op = c["op"]
    if op == "attention":
        tir.paged_attention(s["q"], s["kv"], s["lens"], s["out"], max_len=c["ctx"], window=c["window"],
                            workspace=s["workspace"])
        return s["out"]
    if op == "gather":
        tir.kv_gather(s["kv"], s["k_back"], s["v_back"], s["back_seq"], s["back_pos"])
        return s["k_back"], s["v_back"]
    q, k, v = _split(s)
    if op == "roundtrip":
        tir.kv_append(s["kv"], k, v, s["seq"], s["pos"])
        tir.kv_gather(s["kv"], s["k_back"], s["v_back"], s["back_seq"], s["back_pos"])
        return s["k_back"], s["v_back"]
    w = {"q_weight": s["q_w"], "k_weight": s["k_w"]} if c["norm"] else {}
    if op == "norm_rope":
        tir.qk_norm_rope(q, k, s["q_out"], s["k_out"], s["pos"], s["rope"], eps=EPS, pairs=c["pairs"], **w)
        return s["q_out"], s["k_out"]
    tir.qk_norm_rope_append(q, k, v, s["q_out"], s["kv"], s["seq"], s["pos"], s["rope"], eps=EPS, pairs=c["pairs"], **w)
    return s["q_out"], s["k_pool"], s["v_pool"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    qh, kh, d = case["q_heads"], case["kv_heads"], case["dim"]
    es, cs = _ES[case["dtype"]], _ES[case["cache"]]
    op = case["op"]
    if op == "attention":
        n, keys = case["seqs"], sum(min(x, case["window"] or x) for x in _lens(case))
        pages = sum(-(-x // case["page"]) for x in _lens(case))
        return {"bytes": keys * kh * d * 2 * cs + 2 * n * qh * d * es + 4 * n + 4 * pages,
                "flops": 4.0 * keys * qh * d}
    held = case["seqs"] * case["ctx"]
    back = held * kh * d * 2 * (cs + es) + 8 * held
    if op == "gather":
        return {"bytes": back, "flops": 0}
    t = case["seqs"] * case["new"] - case["pad"]
    if op == "roundtrip":
        return {"bytes": back + t * kh * d * 2 * (es + cs) + 8 * t, "flops": 4.0 * t * kh * d}
    table = min(t, case["ctx"]) * d * 4 if case["new"] > 1 else d * 4
    if op == "norm_rope":
        return {"bytes": t * (qh + kh) * d * 2 * es + 4 * t + table, "flops": 7.0 * t * (qh + kh) * d}
    return {"bytes": t * (qh + 2 * kh) * d * es + t * qh * d * es + t * kh * d * 2 * cs + 8 * t + table,
            "flops": 7.0 * t * (qh + kh) * d}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_head(x, w, rope, pos, case):
    """One head vector per row of x [t, h, d], float64."""
    d = case["dim"]
    if case["norm"]:
        ms = torch.einsum("thd,thd->th", x, x) / d
        x = torch.einsum("thd,d,th->thd", x, w, (ms + EPS) ** -0.5)
    cos, sin = rope[pos][..., 0], rope[pos][..., 1]
    i = torch.arange(d // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if case["pairs"] == "adjacent" else (i, i + d // 2)
    y = torch.empty_like(x)
    y[..., a] = torch.einsum("thi,ti->thi", x[..., a], cos) - torch.einsum("thi,ti->thi", x[..., b], sin)
    y[..., b] = torch.einsum("thi,ti->thi", x[..., a], sin) + torch.einsum("thi,ti->thi", x[..., b], cos)
    return y


def _exact_q8(x):
    """Values that Q8_0 blocks of x stand for.  The format fixes two roundings:
    the block's step is max / 127 in 32 bits, the quotient is a 32-bit one."""
    b = x.reshape(-1, 32)
    at = 31 - torch.argmax(b.abs().flip(-1), -1)
    step = (b[torch.arange(b.shape[0], device=x.device), at] / 127).float().double()[:, None]
    r = torch.where(step == 0, torch.zeros_like(b), b / step).float().double()
    q = torch.sign(r) * torch.floor(r.abs() + 0.5)
    return (q.clamp(-128, 127) * step.half().double()).reshape(x.shape)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op, qh, kh, d, ps = case["op"], case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    pools = {}
    if op != "norm_rope":
        for x in "kv":
            y = s.pop(x + "_pool").double()
            if case["cache"] == "q8_0":
                y = y * torch.repeat_interleave(s.pop(x + "_scale").double(), 32, -1)
            pools[x] = y.reshape(-1, kh, d)  # one row per slot
        table = s["table"].long()

        def slot(seq, pos):
            return table[seq, pos // ps] * ps + pos % ps
    if op == "attention":
        out = torch.zeros(case["seqs"], qh, d, dtype=torch.float64, device="cuda")
        for r, n in enumerate(_lens(case)):
            if n == 0:
                continue
            first = max(0, n - case["window"]) if case["window"] else 0
            at = slot(r, torch.arange(first, n, device="cuda"))
            q = s["q"][r].double().reshape(kh, qh // kh, d)
            x = torch.einsum("hgd,nhd->hgn", q, pools["k"][at]) * d ** -0.5
            p = torch.softmax(x, -1)
            out[r] = torch.einsum("hgn,nhd->hgd", p, pools["v"][at]).reshape(qh, d)
        return out
    if op in ("norm_rope", "fused", "roundtrip"):
        seq, pos = s["seq"].long(), s["pos"].long()
        live = torch.nonzero(pos >= 0).reshape(-1)
        rows = s["qkv"].double().reshape(-1, qh + 2 * kh, d)[live]
        rope = s["rope"].double()
        q, k, v = rows[:, :qh], rows[:, qh:qh + kh], rows[:, qh + kh:]
    if op in ("norm_rope", "fused"):
        q_out, k_out = s["q_out"].double(), s["k_out"].double()
        q_out[live] = _exact_head(q, s["q_w"].double(), rope, pos[live], case)
        k = _exact_head(k, s["k_w"].double(), rope, pos[live], case)
        if op == "norm_rope":
            k_out[live] = k
            return q_out, k_out
        at = slot(seq[live], pos[live])
        pools["k"][at], pools["v"][at] = k, v
        return [q_out] + [pools[x].reshape(-1, ps, kh, d) for x in "kv"]
    if op == "roundtrip":
        at = slot(seq[live], pos[live])
        pools["k"][at], pools["v"][at] = _exact_q8(k), _exact_q8(v)
    at = slot(s["back_seq"].long(), s["back_pos"].long())
    return pools["k"][at], pools["v"][at]
