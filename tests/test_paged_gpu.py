"""Paged cache operators on the GPU against plain 64-bit implementations.

Tolerances.  u(t) = torch.finfo(t).eps / 2 is the most a rounding to type t is
off, relative to the value.
* norm and rotation: f32 inside.  The sum of squares is off by at most
  (8 + log2(dim / 8)) u32 relative (a chain of 8 and a tree), half of that after
  the square root; division, root, product, quotient and eps add 5 u32; the
  rotation's two products and sum 2 u32: at most 14 u32 (|x cos| + |y sin|), then
  one rounding to the output's type.
* cache writes in f32, f16 or bf16 are the one rounding; Q8_0 writes are
  activated_q8's blocks, bit for bit; read-back is exact, then one rounding.
* attention: rel-L2 of f32 outputs 1e-5, the bar of tir_attention's test; 16-bit
  outputs add their rounding, u(t) relative per element and so at most u(t) in
  rel-L2.  Per element: a score's error e (natural units) multiplies its weight by
  exp(e), numerator and denominator alike, so an output moves by at most
  2 max(e) sum p |v|.  e <= (2 (dim / 8) + 4) 2^-23 scale sum |q k| (a chain of
  dim / 8 tensor-core additions, each off by two steps of the f32 sum at most, and
  operands kept to 22 bits) + 2^-20 (exponential, weights kept to 20 bits or more),
  and the chain over the keys adds n / 8 * 2^-23 + 2^-20 of sum p |v|."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

BAD = float("nan")


def dtype(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "q8_0": torch.int8}[name]


def u(torch, t):
    return torch.finfo(t).eps / 2


def cache(torch, tirlib, kind, rows, max_len, kv_heads, dim, page, seed=0, order="page,pos,head", spare=3, fill=True):
    """A cache with every sequence's pages scattered over the pool; unused slots
    hold NaN (Q8_0: NaN steps).  Returns (kv, values f64 [rows, cap, 2, kv_heads,
    dim], poison(lens, window))."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = max(1, -(-max_len // page))
    total = rows * pages + spare
    perm = torch.randperm(total, device="cuda", generator=g)[:rows * pages].to(torch.int32).reshape(rows, pages)
    table = torch.full((rows, pages + 2), -1, dtype=torch.int32, device="cuda")  # rows longer than what is used
    table[:, :pages] = perm
    table = table[:, :pages]
    axes = {"page": total, "pos": page, "head": kv_heads}
    names = order.split(",")
    back = [names.index(x) for x in ("page", "pos", "head")] + [3]

    def pool(last, dt):
        return torch.empty(*[axes[n] for n in names], last, dtype=dt, device="cuda").permute(*back)

    t = dtype(torch, kind)
    ks = vs = None
    k, v = pool(dim, t), pool(dim, t)
    if kind == "q8_0":
        ks, vs = pool(dim // 32, torch.float16), pool(dim // 32, torch.float16)
        for x, s in ((k, ks), (v, vs)):
            x.copy_(torch.randint(-127, 128, x.shape, device="cuda", generator=g, dtype=torch.int8))
            s.copy_(((0.5 + torch.rand(s.shape, device="cuda", generator=g)) / 64))
    else:
        chan = torch.exp(0.5 * torch.randn(kv_heads, dim, device="cuda", generator=g))
        k.copy_(torch.randn(k.shape, device="cuda", generator=g) * chan)
        v.copy_(torch.randn(v.shape, device="cuda", generator=g))
    kv = tirlib.KVPages(k, v, table, ks, vs)

    def values():
        out = []
        for x, s in ((k, ks), (v, vs)):
            y = x.double()
            if s is not None:
                y = y * s.double().repeat_interleave(32, -1)
            y = y[table.long().reshape(-1).clamp(0, total - 1)]
            out.append(y.reshape(rows, pages * page, kv_heads, dim))
        return torch.stack(out, 2)

    def poison(lens, window=0):
        """NaN wherever no row of these lengths may look."""
        seen = torch.zeros(total, page, dtype=torch.bool, device="cuda")
        for r, n in enumerate(lens):
            first = max(0, n - window) if window else 0
            for p in range(first // page, -(-n // page)):
                a, b = max(first - p * page, 0), min(n - p * page, page)
                seen[perm[r, p].long(), a:b] = True
        for x in ((ks, vs) if kind == "q8_0" else (k, v)):
            x[~seen] = BAD

    return kv, values, poison


def attention_ref(torch, q, vals, lens, scale, window):
    """float64 outputs, sum p |v| and max |score terms| per (row, head, :)."""
    rows, qh, dim = q.shape
    kh = vals.shape[3]
    out = torch.zeros(rows, qh, dim, dtype=torch.float64, device="cuda")
    mass, big = torch.zeros_like(out), torch.zeros(rows, qh, 1, dtype=torch.float64, device="cuda")
    for r, n in enumerate(lens):
        if n == 0:
            continue
        first = max(0, n - window) if window else 0
        K, V = vals[r, first:n, 0], vals[r, first:n, 1]
        for h in range(qh):
            g = h // (qh // kh)
            x = (K[:, g] @ q[r, h].double()) * scale
            p = torch.softmax(x, 0)
            out[r, h] = p @ V[:, g]
            mass[r, h] = p @ V[:, g].abs()
            big[r, h] = (K[:, g].abs() @ q[r, h].double().abs()).max() * scale
    return out, mass, big


def check_attention(torch, got, ref, mass, big, dim, n):
    t = got.dtype
    ut = u(torch, t) if t != torch.float32 else 2.0 ** -24
    e = (2 * dim / 8 + 4) * 2.0 ** -23 * big + 2.0 ** -20
    bound = (2 * e + n / 8 * 2.0 ** -23 + 2.0 ** -20) * mass + ut * ref.abs() + 2.0 ** -25
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), float((err / bound).max())
    rel = float((got.double() - ref).norm() / ref.norm().clamp(min=1e-30))
    assert rel < 1e-5 + (ut if t != torch.float32 else 0.0), rel


PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f32", "q8_0"), ("f16", "f16"), ("bf16", "bf16"),
         ("f16", "q8_0"), ("bf16", "q8_0")]
EDGES = [0, 1, 2, 7, 15, 16, 17, 31, 33, 63, 64, 65, 127, 130, 257, 0, 300]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("act,kind", PAIRS)
def test_attention_types_and_edges(cuda, tirlib, act, kind, dim):
    """Every type pair and head size, lengths around the tile and page borders,
    empty rows, NaN wherever a row must not look."""
    torch = cuda
    lens = EDGES
    kv, values, poison = cache(torch, tirlib, kind, len(lens), max(lens), 2, dim, 16, seed=dim)
    q = (1.5 * torch.randn(len(lens), 8, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(1))).to(dtype(torch, act))
    vals = values()
    poison(lens)
    out = torch.full((len(lens) + 2, 8, dim), 7.0, dtype=q.dtype, device="cuda")
    tirlib.paged_attention(q, kv, torch.tensor(lens, dtype=torch.int32, device="cuda"), out[:len(lens)])
    assert (out[len(lens):] == 7.0).all()  # rows behind the last sequence
    assert (out[[i for i, n in enumerate(lens) if n == 0]] == 0).all()
    ref = attention_ref(torch, q, vals, lens, 1 / math.sqrt(dim), 0)
    check_attention(torch, out[:len(lens)], *ref, dim, max(lens))
    tirlib.ops_check()


@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (3, 3), (7, 1), (8, 1), (9, 1), (16, 1), (17, 1), (10, 2), (40, 8), (71, 1)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "q8_0"])
def test_attention_head_groups(cuda, tirlib, kind, q_heads, kv_heads):
    torch = cuda
    lens = [5, 100, 0, 211]
    kv, values, poison = cache(torch, tirlib, kind, 4, 211, kv_heads, 64, 16, seed=q_heads)
    act = "f32" if kind != "bf16" else "bf16"
    q = torch.randn(4, q_heads, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(dtype(torch, act))
    vals = values()
    poison(lens)
    out = torch.empty_like(q)
    tirlib.paged_attention(q, kv, torch.tensor(lens, dtype=torch.int32, device="cuda"), out)
    check_attention(torch, out, *attention_ref(torch, q, vals, lens, 0.125, 0), 64, 211)


@pytest.mark.parametrize("page", [1, 3, 7, 16, 100, 256])
@pytest.mark.parametrize("order", ["page,pos,head", "page,head,pos", "head,page,pos"])
@pytest.mark.parametrize("act,kind", [("f32", "f32"), ("bf16", "bf16"), ("f32", "q8_0")])
def test_attention_pages_and_layouts(cuda, tirlib, act, kind, order, page):
    """Page sizes that end inside a tile, pools in other orders, q and out as
    parts of wider rows, another scale."""
    torch = cuda
    lens = [page, page + 1, max(page - 1, 1), 190]
    kv, values, poison = cache(torch, tirlib, kind, 4, max(lens), 3, 128, page, seed=page, order=order)
    t = dtype(torch, act)
    wide = torch.randn(4, 18, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(t)
    q = wide[:, 6:12]
    outs = torch.full((4, 9, 128), 3.0, dtype=t, device="cuda")
    vals = values()
    poison(lens)
    tirlib.paged_attention(q, kv, torch.tensor(lens, dtype=torch.int32, device="cuda"), outs[:, 2:8], scale=0.2)
    assert (outs[:, :2] == 3.0).all() and (outs[:, 8:] == 3.0).all()
    check_attention(torch, outs[:, 2:8], *attention_ref(torch, q, vals, lens, 0.2, 0), 128, max(lens))


@pytest.mark.parametrize("act,kind,dim", [("f32", "f32", 64), ("bf16", "bf16", 128), ("f32", "q8_0", 64), ("f16", "q8_0", 128)])
def test_attention_many_rows(cuda, tirlib, act, kind, dim):
    """More rows than the GPU holds CTAs, short and long, a third of them empty; the
    table longer than the lengths."""
    torch = cuda
    rows = 450
    lens = [(37 * i) % 300 if i % 3 else 0 for i in range(rows)]
    lens[7] = 1900
    kv, values, poison = cache(torch, tirlib, kind, rows, 1900, 1, dim, 32, seed=dim)
    q = torch.randn(rows, 3, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(4)).to(dtype(torch, act))
    vals = values()
    poison(lens)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref = attention_ref(torch, q, vals, lens, 1 / math.sqrt(dim), 0)
    for max_len in (0, 1900):
        out = torch.full_like(q, BAD)
        tirlib.paged_attention(q, kv, n, out, max_len=max_len)
        check_attention(torch, out, *ref, dim, 1900)
        assert (out[n == 0] == 0).all()


@pytest.mark.parametrize("window", [1, 5, 16, 100, 4000])
@pytest.mark.parametrize("act,kind", [("f32", "f32"), ("f16", "f16"), ("f32", "q8_0")])
def test_attention_window(cuda, tirlib, act, kind, window):
    torch = cuda
    lens = [0, 1, 5, 16, 17, 99, 101, 1500]
    kv, values, poison = cache(torch, tirlib, kind, len(lens), 1500, 2, 64, 16, seed=window)
    q = torch.randn(len(lens), 8, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(4)).to(dtype(torch, act))
    vals = values()
    poison(lens, window)
    out = torch.empty_like(q)
    tirlib.paged_attention(q, kv, torch.tensor(lens, dtype=torch.int32, device="cuda"), out, window=window)
    check_attention(torch, out, *attention_ref(torch, q, vals, lens, 0.125, window), 64, 1500)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("act,kind", PAIRS)
def test_attention_long_rows_split_and_joined(cuda, tirlib, act, kind, dim):
    """Few long rows of unequal length: their parts are joined; the same bits
    every time, and the same values whatever max_len says."""
    torch = cuda
    lens = [9001, 1, 0, 4097]
    kv, values, poison = cache(torch, tirlib, kind, 4, 9001, 1, dim, 16, seed=dim + 1)
    q = (2 * torch.randn(4, 5, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(5))).to(dtype(torch, act))
    vals = values()
    poison(lens)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref = attention_ref(torch, q, vals, lens, 1 / math.sqrt(dim), 0)
    first = None
    for max_len in (0, 9001, 1):
        out = torch.full_like(q, BAD)
        tirlib.paged_attention(q, kv, n, out, max_len=max_len)
        check_attention(torch, out, *ref, dim, 9001)
        again = torch.full_like(q, BAD)
        tirlib.paged_attention(q, kv, n, again, max_len=max_len)
        assert torch.equal(out, again)
        first = out if first is None else first


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "q8_0"])
def test_attention_extreme_scores(cuda, tirlib, kind):
    """One key far above the others late in a row, a rising row, equal scores,
    scores of the type's lowest values: weights stay finite and sum to one."""
    torch = cuda
    dim, n = 64, 700
    kv, values, _ = cache(torch, tirlib, kind, 4, n, 1, dim, 16, seed=9)
    q = torch.zeros(4, 4, dim, device="cuda")
    q[:, :, 0] = torch.tensor([1.0, 30.0, -30.0, 1000.0], device="cuda")
    flat = kv.k[kv.table.long().reshape(-1)].reshape(4, -1, 1, dim).clone()
    if kind == "q8_0":
        steps = kv.k_scale[kv.table.long().reshape(-1)].reshape(4, -1, 1, dim // 32).clone()
        steps[:] = 1.0
        flat[:] = 0
        flat[0, 650, 0, 0] = 127
        flat[1, :, 0, 0] = (torch.arange(flat.shape[1], device="cuda") // 8 - 60).clamp(-127, 127).to(torch.int8)
        flat[3, :, 0, 0] = -127
        kv.k_scale[kv.table.long().reshape(-1)] = steps.reshape(-1, 16, 1, dim // 32)
    else:
        flat[:] = 0
        flat[0, 650, 0, 0] = 1000.0
        flat[1, :, 0, 0] = torch.arange(flat.shape[1], device="cuda").to(flat.dtype)
        flat[3, :, 0, 0] = -60000.0 if kind == "f16" else -1e30
    kv.k[kv.table.long().reshape(-1)] = flat.reshape(-1, 16, 1, dim)
    out = torch.full((4, 4, dim), BAD, device="cuda")
    lens = [n, n, n, n]
    tirlib.paged_attention(q, kv, torch.tensor(lens, dtype=torch.int32, device="cuda"), out)
    ref, mass, _ = attention_ref(torch, q, values(), lens, 0.125, 0)
    assert torch.isfinite(out).all()
    # the scores are single products: off by their own rounding (2 u32 of up to
    # 1e5 natural units only where another key leads by as much), so rows whose
    # weights are one-hot or equal are compared closely, the rising one by 1e-2
    for r, tol in ((0, 1e-4), (2, 1e-4), (3, 1e-4)):
        assert ((out[r].double() - ref[r]).abs() <= tol * mass[r] + 1e-6).all(), r
    assert ((out[1].double() - ref[1]).abs() <= 1e-2 * mass[1] + 1e-6).all()


def test_attention_large_values_of_small_steps(cuda, tirlib):
    """Q8_0 values whose steps differ by many powers of two within a row."""
    torch = cuda
    for low, high in ((-20, -14), (-14, 0), (0, 15)):
        kv, values, _ = cache(torch, tirlib, "q8_0", 2, 400, 2, 64, 16, seed=low + 40)
        g = torch.Generator("cuda").manual_seed(6)
        kv.v_scale.copy_(torch.exp2(low + (high - low) * torch.rand(kv.v_scale.shape, device="cuda", generator=g)))
        q = torch.randn(2, 8, 64, device="cuda", generator=g)
        out = torch.empty_like(q)
        tirlib.paged_attention(q, kv, torch.tensor([400, 333], dtype=torch.int32, device="cuda"), out)
        ref = attention_ref(torch, q, values(), [400, 333], 0.125, 0)
        rel = float((out.double() - ref[0]).norm() / ref[0].norm())
        assert rel < 1e-5, (low, rel)


def test_attention_offsets_past_32_bits(cuda, tirlib):
    """A pool of more than 2^32 elements, pages at both its ends."""
    torch = cuda
    total = (1 << 32) // (16 * 2 * 64) + 64
    k = torch.empty(total, 16, 2, 64, dtype=torch.int8, device="cuda")
    v = torch.empty_like(k)
    ks = torch.empty(total, 16, 2, 2, dtype=torch.float16, device="cuda")
    vs = torch.empty_like(ks)
    pages = [total - 1, 0, total - 2, 5]
    g = torch.Generator("cuda").manual_seed(8)
    for p in pages:
        for x, s in ((k, ks), (v, vs)):
            x[p] = torch.randint(-127, 128, (16, 2, 64), device="cuda", generator=g, dtype=torch.int8)
            s[p] = 1 / 64
    table = torch.tensor([pages[:2], pages[2:]], dtype=torch.int32, device="cuda")
    kv = tirlib.KVPages(k, v, table, ks, vs)
    new = torch.randn(2, 2, 64, device="cuda", generator=g)
    seq = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([3, 30], dtype=torch.int32, device="cuda")
    tirlib.kv_append(kv, new, 2 * new, seq, pos)
    back_k, back_v = torch.empty_like(new), torch.empty_like(new)
    tirlib.kv_gather(kv, back_k, back_v, seq, pos)
    # half a step of a block whose largest value is below 5: 5 / 127 / 2, and the step's own rounding
    assert ((back_k - new).abs() <= new.abs().max() / 127 * 0.51).all()
    assert ((back_v - 2 * new).abs() <= 2 * new.abs().max() / 127 * 0.51).all()
    q = torch.randn(2, 4, 64, device="cuda", generator=g)
    out = torch.empty_like(q)
    tirlib.paged_attention(q, kv, torch.tensor([32, 31], dtype=torch.int32, device="cuda"), out)
    at = torch.tensor(pages, device="cuda")
    vals = torch.stack([x[at].double() * s[at].double().repeat_interleave(32, -1) for x, s in ((k, ks), (v, vs))], 3)
    vals = vals.reshape(2, 32, 2, 2, 64).permute(0, 1, 3, 2, 4)
    check_attention(torch, out, *attention_ref(torch, q, vals, [32, 31], 0.125, 0), 64, 32)
    tirlib.ops_check()


def test_bad_indices_are_reported_once_and_skipped(cuda, tirlib):
    torch = cuda
    kv, values, _ = cache(torch, tirlib, "f32", 2, 64, 2, 64, 16, seed=10)
    keep = kv.table.clone()
    q = torch.randn(2, 4, 64, device="cuda")
    out = torch.empty_like(q)
    lens = torch.tensor([64, 64], dtype=torch.int32, device="cuda")

    def reported(part):
        with pytest.raises(tirlib.TirError) as e:
            tirlib.ops_check()
        assert e.value.name == "INVALID_ARG" and part in e.value.message
        tirlib.ops_check()  # once

    for bad in (-1, 1 << 30):
        kv.table[1, 2] = bad
        tirlib.paged_attention(q, kv, lens, out)
        reported("page id")
        assert torch.isfinite(out).all()
        ref = attention_ref(torch, q, values(), [64, 64], 0.125, 0)
        assert (out[0].double() - ref[0][0]).abs().max() < 1e-4  # the other row is untouched
        kv.table.copy_(keep)
    tirlib.paged_attention(q, kv, torch.tensor([65, -1], dtype=torch.int32, device="cuda"), out)
    reported("length")
    assert (out[1] == 0).all()
    before = kv.k.clone(), kv.v.clone()
    rows = torch.randn(4, 2, 64, device="cuda")
    seqs = torch.tensor([2, -1, 0, 1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([0, 0, 64, 1 << 30], dtype=torch.int32, device="cuda")
    tirlib.kv_append(kv, rows, rows, seqs, pos)
    reported("position")
    assert torch.equal(kv.k, before[0]) and torch.equal(kv.v, before[1])
    back = torch.full_like(rows, 5.0)
    tirlib.kv_gather(kv, back, back.clone(), seqs, pos)
    reported("position")
    assert (back == 5.0).all()
    rope = torch.from_numpy(tirlib.rope_table(1e4, 64, 8)).cuda()
    q_out, k_out = torch.full_like(q, 5.0), torch.full((2, 2, 64), 5.0, device="cuda")
    tirlib.qk_norm_rope(q, rows[:2], q_out, k_out, torch.tensor([8, 7], dtype=torch.int32, device="cuda"), rope)
    reported("position")
    assert (q_out[0] == 5.0).all() and (k_out[0] == 5.0).all() and (q_out[1] != 5.0).any()


# ---------------------------------------------------------------------------
# norm, rotation, cache write, read-back
# ---------------------------------------------------------------------------
def norm_rope_ref(torch, x, w, table, pos, pairs, eps):
    """float64 result and |x cos| + |y sin| of every element."""
    x = x.double()
    if w is not None:
        x = x * w.double() / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    y, mass = x.clone(), x.abs()
    if table is not None:
        half = table.shape[1]
        i = torch.arange(half, device=x.device)
        a, b = (2 * i, 2 * i + 1) if pairs == "adjacent" else (i, i + half)
        c, s = (table[pos.long().clamp(min=0)][..., j].double()[:, None] for j in (0, 1))
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
        mass = mass.clone()
        mass[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
        mass[..., b] = (x[..., a] * s).abs() + (x[..., b] * c).abs()
    return y, mass


def near(torch, got, ref, mass):
    ut = 0.0 if got.dtype == torch.float32 else u(torch, got.dtype)
    tiny = {torch.float16: 2.0 ** -25}.get(got.dtype, 0.0)  # half a step of f16 below its normal range
    err = (got.double() - ref).abs()
    bound = 14 * 2.0 ** -24 * mass * (1 + ut) + ut * ref.abs() + tiny + 1e-37
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rot", [(1, 32, 4, 64, 64), (5, 3, 3, 64, 32), (129, 8, 1, 128, 128),
                                                             (33, 5, 5, 128, 16), (17, 4, 2, 256, 256), (3, 1, 1, 256, 80)])
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
def test_qk_norm_rope(cuda, tirlib, act, pairs, tokens, q_heads, kv_heads, dim, rot):
    torch = cuda
    t = dtype(torch, act)
    g = torch.Generator("cuda").manual_seed(tokens + dim)
    # q and k as parts of one q|k|v row, values far from one
    row = (3 * torch.randn(tokens, q_heads + 2 * kv_heads, dim, device="cuda", generator=g)).to(t)
    row[0, 0] *= 0.001
    q, k = row[:, :q_heads], row[:, q_heads:q_heads + kv_heads]
    wq, wk = (1 + 0.1 * torch.randn(dim, device="cuda", generator=g) for _ in range(2))
    table = torch.from_numpy(tirlib.rope_table(10000.0, rot, 700)).cuda()
    pos = torch.randint(0, 700, (tokens,), device="cuda", generator=g).to(torch.int32)
    if tokens > 2:
        pos[1] = -1
    live = pos >= 0
    for a, b, rope in ((wq, wk, table), (None, wk, table), (wq, wk, None), (None, None, table)):
        q_out = torch.full((tokens, q_heads + 1, dim), 9.0, dtype=t, device="cuda")
        k_out = torch.full((tokens, kv_heads, dim), 9.0, dtype=t, device="cuda")
        tirlib.qk_norm_rope(q, k, q_out[:, 1:], k_out, pos, rope, a, b, eps=1e-6, pairs=pairs)
        assert (q_out[:, 0] == 9.0).all() and (q_out[~live] == 9.0).all() and (k_out[~live] == 9.0).all()
        for x, w, out in ((q, a, q_out[:, 1:]), (k, b, k_out)):
            ref, mass = norm_rope_ref(torch, x, w, rope, pos, pairs, 1e-6)
            near(torch, out[live], ref[live], mass[live])
    # in place: the same bits
    q2, k2 = q.clone(), k.clone()
    tirlib.qk_norm_rope(q2, k2, q2, k2, pos, table, wq, wk, eps=1e-6, pairs=pairs)
    q3, k3 = torch.empty_like(q2), torch.empty_like(k2)
    tirlib.qk_norm_rope(q, k, q3, k3, pos, table, wq, wk, eps=1e-6, pairs=pairs)
    assert torch.equal(q2[live], q3[live]) and torch.equal(k2[live], k3[live])
    assert torch.equal(q2[~live], q[~live]) and torch.equal(k2[~live], k[~live])
    tirlib.ops_check()


@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rot,pairs", [(1300, 13, 3, 64, 64, "adjacent"), (1300, 13, 3, 64, 32, "halves"),
                                                                   (901, 9, 5, 128, 48, "halves"), (600, 7, 2, 256, 256, "adjacent")])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
def test_qk_norm_rope_many_tokens(cuda, tirlib, act, tokens, q_heads, kv_heads, dim, rot, pairs):
    """Enough heads that a lane group takes four of a kind, the last group fewer."""
    torch = cuda
    t = dtype(torch, act)
    g = torch.Generator("cuda").manual_seed(tokens + dim)
    row = (3 * torch.randn(tokens, q_heads + kv_heads, dim, device="cuda", generator=g)).to(t)
    q, k = row[:, :q_heads], row[:, q_heads:]
    wq, wk = (1 + 0.1 * torch.randn(dim, device="cuda", generator=g) for _ in range(2))
    table = torch.from_numpy(tirlib.rope_table(10000.0, rot, 700)).cuda()
    pos = torch.randint(0, 700, (tokens,), device="cuda", generator=g).to(torch.int32)
    pos[::17] = -1
    live = pos >= 0
    q_out, k_out = torch.full((tokens, q_heads, dim), 9.0, dtype=t, device="cuda"), torch.full((tokens, kv_heads, dim), 9.0, dtype=t, device="cuda")
    tirlib.qk_norm_rope(q, k, q_out, k_out, pos, table, wq, wk, eps=1e-6, pairs=pairs)
    assert (q_out[~live] == 9.0).all() and (k_out[~live] == 9.0).all()
    for x, w, out in ((q, wq, q_out), (k, wk, k_out)):
        ref, mass = norm_rope_ref(torch, x, w, table, pos, pairs, 1e-6)
        near(torch, out[live], ref[live], mass[live])
    tirlib.ops_check()


def test_qk_norm_rope_without_positions_or_rotation(cuda, tirlib):
    torch = cuda
    q, k = torch.randn(7, 4, 64, device="cuda"), torch.randn(7, 2, 64, device="cuda")
    w = 1 + 0.1 * torch.randn(64, device="cuda")
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    tirlib.qk_norm_rope(q, k, q_out, k_out, None, None, w, w)
    for x, out in ((q, q_out), (k, k_out)):
        near(torch, out, *norm_rope_ref(torch, x, w, None, None, "adjacent", 1e-5))
    tirlib.qk_norm_rope(q, k, q_out, k_out, None)  # nothing to do but copy
    assert torch.equal(q, q_out) and torch.equal(k, k_out)


def test_norm_of_tiny_and_huge_heads(cuda, tirlib):
    """Sums of squares that leave f32 only where the 64-bit result does, too, and
    heads of zeros (eps alone under the root)."""
    torch = cuda
    x = torch.randn(6, 1, 64, device="cuda")
    x[0] = 0
    x[1] *= 1e-18
    x[2] *= 1e15
    x[3] *= 1e-4
    w = torch.ones(64, device="cuda")
    out, k_out = torch.empty_like(x), torch.empty_like(x)
    tirlib.qk_norm_rope(x, x, out, k_out, None, None, w, w, eps=1e-5)
    near(torch, out, *norm_rope_ref(torch, x, w, None, None, "adjacent", 1e-5))
    assert (out[0] == 0).all()


def test_qk_norm_rope_is_the_runtimes_own_rope(cuda, tirlib):
    """Rotation alone, f32, adjacent pairs: bit for bit tir_rope at that position."""
    torch = cuda
    table = torch.from_numpy(tirlib.rope_table(10000.0, 64, 2048)).cuda()
    for pos in (0, 1, 143, 2047):
        q, k = torch.randn(1, 32, 64, device="cuda"), torch.randn(1, 4, 64, device="cuda")
        a, b = q.clone(), k.clone()
        tirlib.rope(a, 2048, b, 256, tirlib.rope_angles(10000.0, pos, 64), 64)
        tirlib.qk_norm_rope(q, k, q, k, torch.tensor([pos], dtype=torch.int32, device="cuda"), table)
        assert torch.equal(a, q) and torch.equal(b, k)


def q8_blocks(orc, x):
    """activated_q8 of f32 rows: (int8 quants like x, f16 steps)."""
    flat = np.ascontiguousarray(x, np.float32).reshape(-1)
    b = orc.activated_q8(flat).reshape(-1, 34)
    return b[:, 2:].copy().view(np.int8).reshape(x.shape), b[:, :2].copy().view(np.float16).reshape(*x.shape[:-1], x.shape[-1] // 32)


@pytest.mark.parametrize("order", ["page,pos,head", "page,head,pos"])
@pytest.mark.parametrize("act,kind", [(a, c) for a in ("f32", "f16", "bf16") for c in ("f32", "f16", "bf16", "q8_0")])
@pytest.mark.parametrize("dim,page,kv_heads", [(64, 16, 4), (128, 7, 3), (256, 1, 1)])
def test_append_and_gather(cuda, tirlib, orc, act, kind, dim, page, kv_heads, order):
    """Written slots hold the rounded or quantised rows, every other slot its old
    content; read-back gives them in any order, repeats included."""
    torch = cuda
    t, ct = dtype(torch, act), dtype(torch, kind)
    rows, n = 5, 60
    kv, _, _ = cache(torch, tirlib, kind, rows, n, kv_heads, dim, page, seed=dim, order=order)
    g = torch.Generator("cuda").manual_seed(dim + page)
    slots = torch.randperm(rows * n, device="cuda", generator=g)[:83]
    seq, pos = (slots // n).to(torch.int32), (slots % n).to(torch.int32)
    pos[7] = -1
    live = pos >= 0
    x = (2 * torch.randn(83, 2 * kv_heads + 1, dim, device="cuda", generator=g)).to(t)
    x[3] = 0
    x[4, :, 5], x[4, :, 9] = 100.0, -100.0   # equal magnitudes: the later one's sign
    x[5] *= 1e-4
    k, v = x[:, 1:1 + kv_heads], x[:, 1 + kv_heads:]
    before = [y.clone() if y is not None else None for y in (kv.k, kv.v, kv.k_scale, kv.v_scale)]
    tirlib.kv_append(kv, k, v, seq, pos)
    at = (kv.table[seq[live].long(), pos[live].long() // page].long(), pos[live].long() % page)
    for pool, steps, old, old_steps, rows_in in ((kv.k, kv.k_scale, before[0], before[2], k),
                                                 (kv.v, kv.v_scale, before[1], before[3], v)):
        if kind == "q8_0":
            quants, d = q8_blocks(orc, rows_in[live].float().cpu().numpy())
            old[at] = torch.from_numpy(quants).cuda()
            old_steps[at] = torch.from_numpy(d).cuda()
            assert torch.equal(steps.contiguous().view(torch.int16), old_steps.contiguous().view(torch.int16))
        else:
            old[at] = rows_in[live].float().to(ct)
        assert torch.equal(pool, old)
    pick = torch.randint(0, 83, (200,), device="cuda", generator=g)
    bs, bp = seq[pick].contiguous(), pos[pick].contiguous()
    wide = torch.full((200, 2 * kv_heads + 1, dim), 4.0, dtype=t, device="cuda")
    tirlib.kv_gather(kv, wide[:, :kv_heads], wide[:, kv_heads + 1:], bs, bp)
    ok = bp >= 0
    assert (wide[:, kv_heads] == 4.0).all() and (wide[~ok] == 4.0).all()
    where = (kv.table[bs[ok].long(), bp[ok].long() // page].long(), bp[ok].long() % page)
    for pool, steps, out in ((kv.k, kv.k_scale, wide[:, :kv_heads]), (kv.v, kv.v_scale, wide[:, kv_heads + 1:])):
        y = pool[where].float()
        if kind == "q8_0":
            y = (y.reshape(*y.shape[:-1], -1, 32) * steps[where].float()[..., None]).reshape(y.shape)
        assert torch.equal(out[ok], y.to(t))
    tirlib.ops_check()


@pytest.mark.parametrize("act,kind", [("f32", "q8_0"), ("bf16", "q8_0"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("dim,kv_heads", [(64, 3), (128, 5), (256, 2)])
def test_append_and_gather_many_tokens(cuda, tirlib, orc, act, kind, dim, kv_heads):
    """Enough heads that a lane group takes four of a kind; Q8_0 blocks bit for bit."""
    torch = cuda
    t, ct = dtype(torch, act), dtype(torch, kind)
    rows, n, page = 8, 520, 16
    kv, _, _ = cache(torch, tirlib, kind, rows, n, kv_heads, dim, page, seed=dim)
    g = torch.Generator("cuda").manual_seed(dim)
    count = 4000
    slots = torch.randperm(rows * n, device="cuda", generator=g)[:count]
    seq, pos = (slots // n).to(torch.int32), (slots % n).to(torch.int32)
    pos[::29] = -1
    live = pos >= 0
    x = (2 * torch.randn(count, 2 * kv_heads, dim, device="cuda", generator=g)).to(t)
    x[5] = 0
    k, v = x[:, :kv_heads], x[:, kv_heads:]
    old = [kv.k.clone(), kv.v.clone()]
    tirlib.kv_append(kv, k, v, seq, pos)
    at = (kv.table[seq[live].long(), pos[live].long() // page].long(), pos[live].long() % page)
    for pool, steps, before, rows_in in ((kv.k, kv.k_scale, old[0], k), (kv.v, kv.v_scale, old[1], v)):
        if kind == "q8_0":
            quants, d = q8_blocks(orc, rows_in[live].float().cpu().numpy())
            before[at] = torch.from_numpy(quants).cuda()
            assert torch.equal(steps[at].view(torch.int16), torch.from_numpy(d).cuda().view(torch.int16))
        else:
            before[at] = rows_in[live].float().to(ct)
        assert torch.equal(pool, before)
    out = torch.full((2, count, kv_heads, dim), 4.0, dtype=t, device="cuda")
    tirlib.kv_gather(kv, out[0], out[1], seq, pos)
    assert (out[:, ~live] == 4.0).all()
    for pool, steps, got in ((kv.k, kv.k_scale, out[0]), (kv.v, kv.v_scale, out[1])):
        y = pool[at].float()
        if kind == "q8_0":
            y = (y.reshape(*y.shape[:-1], -1, 32) * steps[at].float()[..., None]).reshape(y.shape)
        assert torch.equal(got[live], y.to(t))
    tirlib.ops_check()


def test_q8_values_next_to_a_half_step(cuda, tirlib, orc):
    """Quotients within a few units of the last place of a half, and exact halves:
    the quants are the divided ones, halves away from zero."""
    torch = cuda
    g = torch.Generator("cuda").manual_seed(77)
    top = 1 + torch.rand(512, 1, 1, device="cuda", generator=g)
    x = (torch.randint(-126, 126, (512, 1, 64), device="cuda", generator=g) + 0.5) * (top / 127)
    x = torch.nextafter(x, x + torch.randint(-2, 3, x.shape, device="cuda", generator=g))
    x[..., ::32] = top                      # sets the step
    x[256:, :, 7] = 63.5 * 2
    x[256:, :, 32:] = torch.arange(32, device="cuda") + 0.5
    x[256:, :, 63] = 127.0                  # step 1: exact halves
    kv, _, _ = cache(torch, tirlib, "q8_0", 1, 512, 1, 64, 16, seed=2)
    pos = torch.arange(512, dtype=torch.int32, device="cuda")
    seq = torch.zeros_like(pos)
    tirlib.kv_append(kv, x, -x, seq, pos)
    at = (kv.table[0, pos.long() // 16].long(), pos.long() % 16)
    for pool, y in ((kv.k, x), (kv.v, -x)):
        assert torch.equal(pool[at], torch.from_numpy(q8_blocks(orc, y.cpu().numpy())[0]).cuda())


def test_q8_blocks_with_infinities_and_nan_stay_apart(cuda, tirlib, orc):
    """A NaN or infinity spoils its own block of 32 values only, as activated_q8's."""
    torch = cuda
    kv, _, _ = cache(torch, tirlib, "q8_0", 1, 16, 1, 128, 16, seed=3)
    x = torch.randn(4, 1, 128, device="cuda")
    x[0, 0, 40], x[1, 0, 70], x[2, 0, 127], x[3, 0, 0] = BAD, float("inf"), float("-inf"), 3e38
    pos = torch.arange(4, dtype=torch.int32, device="cuda")
    seq = torch.zeros(4, dtype=torch.int32, device="cuda")
    tirlib.kv_append(kv, x, x, seq, pos)
    k, v = torch.empty_like(x), torch.empty_like(x)
    tirlib.kv_gather(kv, k, v, seq, pos)
    quants, d = q8_blocks(orc, x.cpu().numpy())
    with np.errstate(invalid="ignore"):  # 0 * inf: the blocks that are spoilt
        want = torch.from_numpy((quants.reshape(4, 4, 32).astype(np.float32) * d.reshape(4, 4, 1).astype(np.float32))).cuda()
    for got in (k, v):
        got = got.reshape(4, 4, 32)
        assert torch.equal(torch.isfinite(got), torch.isfinite(want))
        fine = torch.isfinite(want)
        assert torch.equal(got[fine], want[fine])
        assert int((~fine).any(-1).sum()) == 4


@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("act,kind", [("f32", "f32"), ("f32", "q8_0"), ("bf16", "bf16"), ("f16", "q8_0")])
def test_fused_is_norm_rope_then_append(cuda, tirlib, act, kind, pairs):
    """The fused pass writes what the two separate ones write, from a key that has
    not been rounded to the activations' type in between."""
    torch = cuda
    t = dtype(torch, act)
    g = torch.Generator("cuda").manual_seed(12)
    kv, _, _ = cache(torch, tirlib, kind, 6, 50, 2, 128, 16, seed=1)
    tok = 40
    slots = torch.randperm(6 * 50, device="cuda", generator=g)[:tok]
    seq, pos = (slots // 50).to(torch.int32), (slots % 50).to(torch.int32)
    pos[3] = pos[39] = -1
    x = torch.randn(tok, 10, 128, device="cuda", generator=g).to(t)
    q, k, v = x[:, :6], x[:, 6:8], x[:, 8:]
    w = 1 + 0.1 * torch.randn(2, 128, device="cuda", generator=g)
    table = torch.from_numpy(tirlib.rope_table(10000.0, 128, 50)).cuda()
    q_out, q_two = torch.full((2, tok, 6, 128), 2.0, dtype=t, device="cuda")
    tirlib.qk_norm_rope_append(q, k, v, q_out, kv, seq, pos, table, w[0].contiguous(), w[1].contiguous(), pairs=pairs)
    got = [y.clone() if y is not None else None for y in (kv.k, kv.v, kv.k_scale, kv.v_scale)]
    k32 = torch.empty(tok, 2, 128, device="cuda")
    tirlib.qk_norm_rope(q, k, q_two, torch.empty_like(k), pos, table, w[0].contiguous(), w[1].contiguous(), pairs=pairs)
    tirlib.qk_norm_rope(q.float(), k.float(), torch.empty(tok, 6, 128, device="cuda"), k32, pos, table, w[0].contiguous(),
                        w[1].contiguous(), pairs=pairs)
    tirlib.kv_append(kv, k32, v.float(), seq, pos)
    assert torch.equal(q_out, q_two)
    for a, b in zip(got, (kv.k, kv.v, kv.k_scale, kv.v_scale)):
        assert a is None or torch.equal(a, b)


@pytest.mark.parametrize("dim,rot", [(64, 64), (64, 16), (64, 48), (128, 32), (128, 112), (256, 256), (256, 80)])
@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("tokens,q_heads,kv_heads", [(19, 3, 2), (2500, 7, 5)])
def test_fused_rotates_part_of_a_head(cuda, tirlib, tokens, q_heads, kv_heads, kind, dim, rot):
    """Rotations of part of the head, with few tokens (a head a group of lanes) and
    many (four, the last group not full): the cache holds the same bits as after
    the separate passes, quantised blocks included."""
    torch = cuda
    g = torch.Generator("cuda").manual_seed(dim + rot)
    kv, _, _ = cache(torch, tirlib, kind, 4, 640, kv_heads, dim, 16, seed=1)
    slots = torch.randperm(4 * 640, device="cuda", generator=g)[:tokens]
    seq, pos = (slots // 640).to(torch.int32), (slots % 640).to(torch.int32)
    q = torch.randn(tokens, q_heads, dim, device="cuda", generator=g)
    k, v = torch.randn(2, tokens, kv_heads, dim, device="cuda", generator=g)
    w = 1 + 0.1 * torch.randn(2, dim, device="cuda", generator=g)
    table = torch.from_numpy(tirlib.rope_table(10000.0, rot, 640)).cuda()
    q_out, q_two = torch.zeros(2, tokens, q_heads, dim, device="cuda")
    tirlib.qk_norm_rope_append(q, k, v, q_out, kv, seq, pos, table, w[0].contiguous(), w[1].contiguous(), pairs="halves")
    pools = [y for y in (kv.k, kv.v, kv.k_scale, kv.v_scale) if y is not None]
    got = [y.clone() for y in pools]
    for y in pools:
        y.zero_()
    k_two = torch.empty_like(k)
    tirlib.qk_norm_rope(q, k, q_two, k_two, pos, table, w[0].contiguous(), w[1].contiguous(), pairs="halves")
    tirlib.kv_append(kv, k_two, v, seq, pos)
    assert torch.equal(q_out, q_two)
    page, at = kv.table[seq.long(), (pos // 16).long()].long(), (pos % 16).long()
    for a, b in zip(got, pools):
        assert torch.equal(a[page, at], b[page, at])
    tirlib.ops_check()


# ---------------------------------------------------------------------------
# together, as a serving loop uses them
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("act,kind", [("f32", "f32"), ("f32", "q8_0"), ("bf16", "bf16")])
def test_prompts_then_decode_steps(cuda, tirlib, act, kind):
    """Ragged prompts, then decode steps of a batch in which one sequence is idle
    and another joins late: every step's attention against a 64-bit softmax over
    the values the cache holds, and those against the step's own rows."""
    torch = cuda
    t = dtype(torch, act)
    g = torch.Generator("cuda").manual_seed(20)
    rows, qh, kh, dim, page, cap = 4, 8, 2, 64, 16, 96
    kv, values, _ = cache(torch, tirlib, kind, rows, cap, kh, dim, page, seed=21)
    for x in (kv.k_scale, kv.v_scale) if kind == "q8_0" else (kv.k, kv.v):
        x.fill_(BAD)
    table = torch.from_numpy(tirlib.rope_table(10000.0, dim, cap)).cuda()
    w = (1 + 0.1 * torch.randn(2, dim, device="cuda", generator=g))
    wq, wk = w[0].contiguous(), w[1].contiguous()
    held = [0] * rows
    truth = torch.zeros(rows, cap, 2, kh, dim, dtype=torch.float64, device="cuda")
    out = torch.empty(rows, qh, dim, dtype=t, device="cuda")
    ws = torch.empty(tirlib.paged_attention_workspace(kv, rows, qh, cap), dtype=torch.uint8, device="cuda")
    for step in range(20):
        new = [37, 1, 0, 16] if step == 0 else [1, 1, 21 if step == 5 else int(step > 5), int(step % 3 != 0)]
        seq = [s for s in range(rows) for _ in range(new[s])]
        pos = [held[s] + i for s in range(rows) for i in range(new[s])]
        held = [a + b for a, b in zip(held, new)]
        n = len(seq)
        sd, pd = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seq, pos))
        x = torch.randn(n, qh + 2 * kh, dim, device="cuda", generator=g).to(t)
        q_out = torch.empty(n, qh, dim, dtype=t, device="cuda")
        tirlib.qk_norm_rope_append(x[:, :qh], x[:, qh:qh + kh], x[:, qh + kh:], q_out, kv, sd, pd, table, wq, wk)
        truth[sd.long(), pd.long(), 0] = norm_rope_ref(torch, x[:, qh:qh + kh], wk, table, pd, "adjacent", 1e-5)[0]
        truth[sd.long(), pd.long(), 1] = x[:, qh + kh:].double()
        last = [max([i for i in range(n) if seq[i] == s], default=0) for s in range(rows)]
        q = q_out[last].contiguous()
        tirlib.paged_attention(q, kv, torch.tensor(held, dtype=torch.int32, device="cuda"), out, max_len=cap, workspace=ws)
        vals = values()
        check_attention(torch, out, *attention_ref(torch, q, vals, held, 0.125, 0), dim, cap)
        for s in range(rows):
            a, b = vals[s, :held[s]], truth[s, :held[s]]
            if kind == "q8_0":  # half a step of the block, and the step's f16 rounding on 127 of them
                tol = b.reshape(*b.shape[:-1], dim // 32, 32).abs().amax(-1).repeat_interleave(32, -1) / 127 * (0.5 + 127 * 2.0 ** -11 + 1e-3)
            else:
                tol = (u(torch, t) if act != "f32" else 0.0) * b.abs() + 16 * 2.0 ** -24 * b.abs().amax(-1, keepdim=True)
            assert ((a - b).abs() <= tol).all()
    tirlib.ops_check()


def test_captured_step_replays_on_new_lengths(cuda, tirlib):
    """Append and attention captured into a graph: replays read lengths, positions
    and pages anew; two graphs share one workspace one after the other."""
    torch = cuda
    kv, values, _ = cache(torch, tirlib, "q8_0", 3, 2000, 2, 64, 16, seed=30)
    g = torch.Generator("cuda").manual_seed(31)
    x = torch.randn(3, 12, 64, device="cuda", generator=g)
    q, k, v = x[:, :8], x[:, 8:10], x[:, 10:]
    q_out, out = torch.empty(2, 3, 8, 64, device="cuda")
    pos = torch.tensor([5, 900, 0], dtype=torch.int32, device="cuda")
    lens = pos + 1
    table = torch.from_numpy(tirlib.rope_table(10000.0, 64, 2000)).cuda()
    ws = torch.empty(tirlib.paged_attention_workspace(kv, 3, 8, 2000), dtype=torch.uint8, device="cuda")

    def step():
        tirlib.qk_norm_rope_append(q, k, v, q_out, kv, None, pos, table)
        tirlib.paged_attention(q_out, kv, lens, out, max_len=2000, workspace=ws)

    step()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append(graph)
    for i, (p, n) in enumerate((([5, 900, 0], [6, 901, 1]), ([1999, 17, 64], [2000, 18, 0]), ([3, 1500, 7], [0, 1501, 8]))):
        pos.copy_(torch.tensor(p))
        lens.copy_(torch.tensor(n))
        x.copy_(torch.randn(3, 12, 64, device="cuda", generator=g))
        out.fill_(BAD)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        check_attention(torch, out, *attention_ref(torch, q_out, values(), n, 0.125, 0), 64, 2000)
    tirlib.ops_check()


@pytest.mark.parametrize("rows,ctx", [(2, 150), (40, 150), (2, 3000)])
@pytest.mark.parametrize("captured", [False, True])
def test_calls_see_what_was_written_just_before(cuda, tirlib, captured, rows, ctx):
    """New keys, table and lengths, written by the kernels right before on the same stream
    and, in a graph, on another one joined to it: the same bits as with waits between."""
    torch = cuda
    g = torch.Generator("cuda").manual_seed(rows + ctx)
    kv, _, _ = cache(torch, tirlib, "bf16", rows, ctx, 2, 64, 16, seed=1)
    other = torch.cuda.Stream()
    states = []
    for i in range(4):
        table = torch.randperm(kv.table.numel(), device="cuda", generator=g).to(torch.int32).reshape(kv.table.shape)
        lens = torch.randint(1, ctx + 1, (rows,), device="cuda", generator=g).to(torch.int32)
        x = torch.randn(rows, 12, 64, device="cuda", generator=g).bfloat16()
        states.append((table, lens, x))
    rope = torch.from_numpy(tirlib.rope_table(10000.0, 64, ctx)).cuda()
    lens, pos, q = torch.zeros(2, rows, dtype=torch.int32, device="cuda").unbind() + (torch.zeros(rows, 8, 64, dtype=torch.bfloat16, device="cuda"),)
    seq = torch.arange(rows, dtype=torch.int32, device="cuda")
    ws = torch.empty(max(16, tirlib.paged_attention_workspace(kv, rows, 8, ctx)), dtype=torch.uint8, device="cuda")
    outs = torch.zeros(2, 24, rows, 8, 64, dtype=torch.bfloat16, device="cuda")

    def step(i, out, wait, fork):
        table, new, x = states[i % 4]
        if fork:
            other.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(other):
                lens.copy_(new)
            torch.cuda.current_stream().wait_stream(other)
        else:
            lens.copy_(new)
        kv.table.copy_(table)
        torch.sub(lens, 1, out=pos)
        wait()
        tirlib.qk_norm_rope_append(x[:, :8], x[:, 8:10], x[:, 10:], q, kv, seq, pos, rope)
        wait()
        tirlib.paged_attention(q, kv, lens, out, max_len=ctx, workspace=ws)
        wait()

    before = kv.k.clone(), kv.v.clone()
    for i in range(24):
        step(i, outs[0, i], torch.cuda.synchronize, False)
    kv.k.copy_(before[0])
    kv.v.copy_(before[1])
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for i in range(24):
                step(i, outs[1, i], lambda: None, i % 2 == 1)
        graph.replay()
    else:
        for i in range(24):
            step(i, outs[1, i], lambda: None, False)
    assert torch.equal(outs[0], outs[1])
    tirlib.ops_check()


@pytest.mark.parametrize("before", ["copy", "set", "upload", "event", "nothing"])
def test_a_graph_of_one_call_behind_any_node(cuda, tirlib, before):
    """What stands before a call in a graph may be a copy, a memory set, an upload, another
    stream's work or nothing: the call waits for it."""
    torch = cuda
    kv, _, _ = cache(torch, tirlib, "f32", 3, 700, 2, 64, 16, seed=1)
    q = torch.randn(3, 8, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    want = torch.tensor([700, 1, 333], dtype=torch.int32)
    if before == "set":
        want.zero_()
    host = want.pin_memory()
    lens, new, out, ref = want.cuda(), want.cuda(), torch.ones_like(q), torch.empty_like(q)
    ws = torch.empty(max(16, tirlib.paged_attention_workspace(kv, 3, 8, 700)), dtype=torch.uint8, device="cuda")
    tirlib.paged_attention(q, kv, lens, ref, max_len=700, workspace=ws)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        if before == "copy":
            lens.copy_(new)
        elif before == "set":
            lens.zero_()
        elif before == "upload":
            lens.copy_(host, non_blocking=True)
        elif before == "event":
            other.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(other):
                torch.add(new, 0, out=lens)
            torch.cuda.current_stream().wait_stream(other)
        tirlib.paged_attention(q, kv, lens, out, max_len=700, workspace=ws)
    for _ in range(3):
        if before != "nothing":
            lens.fill_(5)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
    tirlib.ops_check()


def test_more_blocks_of_tokens_than_one_dimension_of_a_grid(cuda, tirlib):
    """140001 tokens of one head of 256: 35001 blocks."""
    torch = cuda
    n, dim, page = 140001, 256, 64
    g = torch.Generator("cuda").manual_seed(5)
    q, k = torch.randn(2, n, 1, dim, device="cuda", generator=g).bfloat16()
    w = 1 + 0.1 * torch.randn(dim, device="cuda", generator=g)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    tirlib.qk_norm_rope(q, k, q_out, k_out, pos, None, w, w, eps=1e-6)
    for x, out in ((q, q_out), (k, k_out)):
        ref, mass = norm_rope_ref(torch, x, w, None, pos, "halves", 1e-6)
        near(torch, out, ref, mass)
    pages = -(-n // page)
    pool = torch.zeros(2, pages, page, 1, dim, dtype=torch.bfloat16, device="cuda")
    table = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).reshape(1, pages)
    kv = tirlib.KVPages(pool[0], pool[1], table)
    seq = torch.zeros(n, dtype=torch.int32, device="cuda")
    tirlib.kv_append(kv, k_out, q_out, seq, pos)
    back = torch.zeros(2, n, 1, dim, dtype=torch.bfloat16, device="cuda")
    tirlib.kv_gather(kv, back[0], back[1], seq, pos)
    assert torch.equal(back[0], k_out) and torch.equal(back[1], q_out)
    tirlib.ops_check()


def test_streams_run_side_by_side(cuda, tirlib):
    """Two streams, each with its own cache and workspace, many calls in flight."""
    torch = cuda
    jobs = []
    for seed in (40, 41):
        kv, values, _ = cache(torch, tirlib, "bf16", 2, 3000, 2, 128, 16, seed=seed)
        q = torch.randn(2, 8, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(torch.bfloat16)
        lens = torch.tensor([3000, 1200 + seed], dtype=torch.int32, device="cuda")
        ws = torch.empty(tirlib.paged_attention_workspace(kv, 2, 8, 3000), dtype=torch.uint8, device="cuda")
        jobs.append((torch.cuda.Stream(), kv, q, lens, torch.empty_like(q), ws, values, [3000, 1200 + seed]))
    torch.cuda.synchronize()
    for _ in range(50):
        for s, kv, q, lens, out, ws, _, _ in jobs:
            tirlib.paged_attention(q, kv, lens, out, max_len=3000, workspace=ws, stream=s)
    torch.cuda.synchronize()
    for s, kv, q, lens, out, ws, values, n in jobs:
        check_attention(torch, out, *attention_ref(torch, q, values(), n, 1 / math.sqrt(128), 0), 128, 3000)


def test_bindings_check_shapes_types_and_workspace(cuda, tirlib):
    torch = cuda
    kv, _, _ = cache(torch, tirlib, "f32", 2, 64, 2, 64, 16)
    q = torch.zeros(2, 4, 64, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    bad = [dict(q=q[..., :32]), dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)), dict(out=q[:1]),
           dict(out=torch.zeros(2, 4, 64)), dict(out=q.half()), dict(seq_lens=lens.long()), dict(seq_lens=lens[:1]),
           dict(seq_lens=lens.cpu()), dict(q=torch.zeros(3, 4, 64, device="cuda"), out=torch.zeros(3, 4, 64, device="cuda"),
                                           seq_lens=torch.ones(3, dtype=torch.int32, device="cuda"))]
    for kw in bad:
        a = dict(q=q, kv=kv, seq_lens=lens, out=torch.empty_like(q))
        a.update(kw)
        with pytest.raises(tirlib.TirError) as e:
            tirlib.paged_attention(**a)
        assert e.value.name == "INVALID_ARG"
    big, _, _ = cache(torch, tirlib, "f32", 1, 20000, 1, 64, 16)
    need = tirlib.paged_attention_workspace(big, 1, 4)
    one = torch.zeros(1, 4, 64, device="cuda")
    if need:
        with pytest.raises(tirlib.TirError) as e:
            tirlib.paged_attention(one, big, lens[:1], torch.empty_like(one),
                                   workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
        assert e.value.name == "INVALID_ARG" and "workspace" in e.value.message
    with pytest.raises(tirlib.TirError):
        tirlib.kv_append(kv, q[:, :2], q[:1, :2], None, lens)
    with pytest.raises(tirlib.TirError):
        tirlib.qk_norm_rope(q, q[:, :2], q, q[:, :2], lens, rope=torch.zeros(4, 32, 2, device="cuda").half())
    torch.cuda.synchronize()
