"""What the paged cache operators promise, where it is easiest to break: quotients at the edge
of a half step, weights far below a row's largest, pages outside the pool, infinities inside
a row, reports of several streams,
workspaces sized once.  Tolerances as in test_paged_gpu.py, whose helpers these tests use."""
import math
import threading

import numpy as np
import pytest

from test_paged_gpu import attention_ref, cache, check_attention, dtype, q8_blocks

pytestmark = pytest.mark.gpu


def half_step_blocks():
    """f32 rows of two Q8_0 blocks whose steps are 2^-10 to 2^10 of either sign: every quotient
    n + 1/2 and the three f32 values on either side of it, n = 0 to 126, of either sign."""
    x = np.arange(127, dtype=np.float32) + np.float32(0.5)
    near = [x]
    for way in (0.0, 200.0):
        y = x
        for _ in range(3):
            y = np.nextafter(y, np.float32(way), dtype=np.float32)
            near.append(y)
    near = np.concatenate(near)
    near = np.concatenate([near, -near])
    near = np.concatenate([near, np.zeros(-near.size % 31, np.float32)]).reshape(-1, 31)
    blocks = [np.concatenate([np.full((near.shape[0], 1), sign * 127.0, np.float32), near], 1) * np.float32(2.0 ** k)
              for k in range(-10, 11) for sign in (1, -1)]
    return np.concatenate(blocks).reshape(-1, 1, 64)


@pytest.mark.parametrize("entry", ["kv_append", "qk_norm_rope_append"])
def test_q8_quotients_next_to_every_half(cuda, tirlib, orc, entry):
    """Steps that are powers of two: quotients land exactly on a half and on the f32 values
    next to it, also below one half, where f32's step changes.  Bit for bit activated_q8's."""
    torch = cuda
    rows = half_step_blocks()
    n = rows.shape[0]
    kv, _, _ = cache(torch, tirlib, "q8_0", 1, n, 1, 64, 16, seed=2)
    x = torch.from_numpy(rows).cuda()
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    seq = torch.zeros_like(pos)
    if entry == "kv_append":
        tirlib.kv_append(kv, x, -x, seq, pos)
    else:
        q = torch.zeros_like(x)
        tirlib.qk_norm_rope_append(q, x, -x, torch.empty_like(q), kv, seq, pos)
    at = (kv.table[0, pos.long() // 16].long(), pos.long() % 16)
    for pool, steps, y in ((kv.k, kv.k_scale, rows), (kv.v, kv.v_scale, -rows)):
        quants, d = q8_blocks(orc, y)
        assert torch.equal(pool[at], torch.from_numpy(quants).cuda())
        assert torch.equal(steps[at], torch.from_numpy(d).cuda())
    tirlib.ops_check()


def write_rows(torch, tirlib, kv, k, v):
    """k, v [positions, kv_heads, dim] f32 into row 0 of the cache."""
    pos = torch.arange(k.shape[0], dtype=torch.int32, device="cuda")
    tirlib.kv_append(kv, k.contiguous(), v.contiguous(), torch.zeros_like(pos), pos)


FAR = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "q8_0"), ("f16", "q8_0"), ("bf16", "q8_0")]


@pytest.mark.parametrize("lead", [12.0, 16.0, 21.0, 25.0])
@pytest.mark.parametrize("where", [100, 15000])
@pytest.mark.parametrize("act,kind", FAR)
def test_weights_far_below_a_leading_key(cuda, tirlib, act, kind, where, lead):
    """One key leads a long row by many natural units; its value is zero, so the output is
    what the small weights make of the others' values, all of one sign.  Undivided
    (max_len 1) and divided."""
    torch = cuda
    n, dim = 20000, 64
    g = torch.Generator("cuda").manual_seed(int(lead) + where)
    kv, values, _ = cache(torch, tirlib, kind, 1, n, 1, dim, 16, seed=3)
    k = 0.1 * torch.randn(n, 1, dim, device="cuda", generator=g)
    k[:, 0, 0] = 0.0
    k[where] = 0.0
    k[where, 0, 0] = 8.0
    v = 1024 * (0.5 + torch.rand(n, 1, dim, device="cuda", generator=g))  # f16 outputs stay above its smallest normal value
    v[where] = 0.0
    write_rows(torch, tirlib, kv, k, v)
    q = torch.randn(1, 4, dim, device="cuda", generator=g)
    q[..., 0] = lead / 8.0 / 0.125
    q = q.to(dtype(torch, act))
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    ref = attention_ref(torch, q, values(), [n], 0.125, 0)
    for max_len in (1, n):
        out = torch.empty_like(q)
        tirlib.paged_attention(q, kv, lens, out, max_len=max_len)
        check_attention(torch, out, *ref, dim, n)
    tirlib.ops_check()


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("differ", ["blocks", "positions"])
def test_q8_values_of_very_different_steps(cuda, tirlib, act, differ):
    """Q8_0 values whose steps differ by up to 2^24: between the blocks of a head, and between
    positions of which those of large steps have next to no weight.  Every element against
    its own values' size."""
    torch = cuda
    n, dim = 700, 64
    g = torch.Generator("cuda").manual_seed(5)
    kv, values, _ = cache(torch, tirlib, "q8_0", 1, n, 2, dim, 16, seed=4)
    q = torch.randn(1, 8, dim, device="cuda", generator=g)
    kv.v_scale.copy_(torch.exp2(-14.0 + torch.rand(kv.v_scale.shape, device="cuda", generator=g)))
    if differ == "blocks":
        kv.v_scale[..., 0] *= 2.0 ** 22
    else:
        big = kv.table[0, ::5].long()
        kv.v_scale[big] *= 2.0 ** 22
        q[..., 0] = 40.0
        kv.k[..., 0] = 40
        kv.k[big, ..., 0] = -120
        kv.k_scale[..., 0] = 2.0 ** -5
    q = q.to(dtype(torch, act))
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    ref, mass, big_score = attention_ref(torch, q, values(), [n], 0.125, 0)
    for max_len in (1, n):
        out = torch.empty_like(q)
        tirlib.paged_attention(q, kv, lens, out, max_len=max_len)
        tiny = 2.0 ** -25 if act == "f16" else 0.0  # half a step of f16 below its normal range
        ut = torch.finfo(dtype(torch, act)).eps / 2
        e = (2 * dim / 8 + 4) * 2.0 ** -23 * big_score + 2.0 ** -20
        bound = (2 * e + n / 8 * 2.0 ** -23 + 2.0 ** -20) * mass + ut * ref.abs() + tiny
        err = (out.double() - ref).abs()
        assert (err <= bound).all(), float((err / bound).max())
    tirlib.ops_check()


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_q8_keys_with_one_large_channel(cuda, tirlib, act, dim):
    """Every block of keys has one channel far above the others, which sets its step, and the
    query looks away from it: the small quants carry the scores."""
    torch = cuda
    n = 500
    g = torch.Generator("cuda").manual_seed(6)
    kv, values, _ = cache(torch, tirlib, "q8_0", 1, n, 1, dim, 16, seed=7)
    kv.k.copy_(torch.randint(-3, 4, kv.k.shape, device="cuda", generator=g, dtype=torch.int8))
    kv.k[..., ::32] = 127
    kv.k_scale.fill_(1.0)
    q = (0.5 + torch.rand(1, 8, dim, device="cuda", generator=g)).to(dtype(torch, act))
    q[..., ::32] = 0
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    tirlib.paged_attention(q, kv, lens, out)
    check_attention(torch, out, *attention_ref(torch, q, values(), [n], 1 / math.sqrt(dim), 0), dim, n)


def attention_over(torch, q, vals, seen, scale):
    """float64 outputs of row 0 over the positions of the mask `seen`; zeros for none."""
    rows, qh, dim = q.shape
    out = torch.zeros(rows, qh, dim, dtype=torch.float64, device="cuda")
    mass, big = torch.zeros_like(out), torch.zeros(rows, qh, 1, dtype=torch.float64, device="cuda")
    for r in range(rows):
        if not seen[r].any():
            continue
        K, V = vals[r, :, 0][seen[r]], vals[r, :, 1][seen[r]]
        for h in range(qh):
            kh = h // (qh // K.shape[1])
            x = (K[:, kh] @ q[r, h].double()) * scale
            p = torch.softmax(x, 0)
            out[r, h], mass[r, h] = p @ V[:, kh], p @ V[:, kh].abs()
            big[r, h] = (K[:, kh].abs() @ q[r, h].double().abs()).max() * scale
    return out, mass, big


@pytest.mark.parametrize("act,kind", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "q8_0")])
@pytest.mark.parametrize("dim", [64, 128])
def test_positions_on_a_bad_page_take_no_part(cuda, tirlib, act, kind, dim):
    """Pages outside the pool, at the start, inside and at the end of a row, and a row of
    nothing else: the softmax is over the other positions, and zeros where there are none."""
    torch = cuda
    n, page, rows = 2100, 7, 4
    kv, values, _ = cache(torch, tirlib, kind, rows, n, 1, dim, page, seed=8)
    vals = values()
    seen = torch.ones(rows, vals.shape[1], dtype=torch.bool, device="cuda")
    seen[:, n:] = False
    bad = {0: [0, 1, 5, 40, 41, 42, 43, 44, 45, 200, 299], 1: list(range(kv.table.shape[1])), 2: list(range(1, kv.table.shape[1]))}
    for r, pages in bad.items():
        for i, p in enumerate(pages):
            kv.table[r, p] = (-1, 1 << 30, -(1 << 31), kv.k.shape[0])[i % 4]
            seen[r, p * page:(p + 1) * page] = False
    q = torch.randn(rows, 4, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(9)).to(dtype(torch, act))
    lens = torch.full((rows,), n, dtype=torch.int32, device="cuda")
    ref = attention_over(torch, q, vals, seen, 1 / math.sqrt(dim))
    for max_len in (1, n):
        out = torch.full_like(q, 3.0)
        tirlib.paged_attention(q, kv, lens, out, max_len=max_len)
        check_attention(torch, out, *ref, dim, n)
        assert (out[1] == 0).all()
        with pytest.raises(tirlib.TirError) as e:
            tirlib.ops_check()
        assert e.value.name == "INVALID_ARG" and "page id" in e.value.message
    tirlib.ops_check()


@pytest.mark.parametrize("act,kind", FAR)
@pytest.mark.parametrize("max_len", [1, 0])
def test_nan_and_infinity_inside_a_row(cuda, tirlib, act, kind, max_len):
    """A NaN in a key, or a NaN or infinity in a value, makes the heads that read it
    non-finite; a key of score -inf has no weight or makes its head non-finite, one of
    +inf makes it non-finite; the other row and the other key-value head are as they were."""
    torch = cuda
    n, dim, inf = 3000, 64, float("inf")
    kv, values, _ = cache(torch, tirlib, kind, 2, n, 2, dim, 16, seed=11)
    q = torch.randn(2, 4, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(12))
    q[..., 5] = 1.0 + q[..., 5].abs()
    q = q.to(dtype(torch, act))
    lens = torch.tensor([n, n], dtype=torch.int32, device="cuda")
    clean = torch.empty_like(q)
    tirlib.paged_attention(q, kv, lens, clean, max_len=max_len)
    pos = 1234
    page, slot = int(kv.table[0, pos // 16]), pos % 16
    q8 = kind == "q8_0"
    pools = (kv.k_scale, kv.v_scale) if q8 else (kv.k, kv.v)
    for what, x in (("k", float("nan")), ("k", inf), ("k", -inf), ("v", float("nan")), ("v", inf), ("v", -inf)):
        pool = pools[what == "v"]
        c = 0 if q8 else 5
        old = pool[page, slot, 0, c].clone()
        pool[page, slot, 0, c] = x
        score = 0.0
        if what == "k" and x == x:  # sign of the score
            score = x if not q8 else None
        out = torch.empty_like(q)
        tirlib.paged_attention(q, kv, lens, out, max_len=max_len)
        assert torch.equal(out[1], clean[1]) and torch.equal(out[0, 2:], clean[0, 2:]), (what, x)
        if what == "v":
            d = slice(0, 32) if q8 else 5
            assert not torch.isfinite(out[0, :2, d]).any(), (what, x)
        elif x != x or score == inf:
            assert not torch.isfinite(out[0, :2]).any(), (what, x)
        else:
            pool[page, slot, 0, c] = old
            seen = torch.ones(2, values().shape[1], dtype=torch.bool, device="cuda")
            seen[:, n:] = False
            seen[0, pos] = False
            ref = attention_over(torch, q, values(), seen, 0.125)
            for h in range(2):
                if torch.isfinite(out[0, h]).all():
                    check_attention(torch, out[:1, h:h + 1], *(y[:1, h:h + 1] for y in ref), dim, n)
        pool[page, slot, 0, c] = old
    pools[0][kv.table[0].long(), :, 0, 0 if q8 else 5] = -inf
    out = torch.empty_like(q)
    tirlib.paged_attention(q, kv, lens, out, max_len=max_len)
    assert not torch.isfinite(out[0, :2]).any() and torch.equal(out[1], clean[1]) and torch.equal(out[0, 2:], clean[0, 2:])
    tirlib.ops_check()


def test_reports_of_another_stream_are_not_lost(cuda, tirlib):
    """A bad page, some work, then a bad length on one stream while another is being checked:
    both are reported, wherever the second falls in a check of the first."""
    torch = cuda
    kv, _, _ = cache(torch, tirlib, "f32", 1, 64, 1, 64, 16, seed=13)
    q = torch.randn(1, 4, 64, device="cuda")
    out, x = torch.empty_like(q), torch.zeros(200000, device="cuda")
    bad = tirlib.KVPages(kv.k, kv.v, torch.full_like(kv.table, -1))
    one, long = (torch.tensor([n], dtype=torch.int32, device="cuda") for n in (1, 65))
    busy, checked = torch.cuda.Stream(), torch.cuda.Stream()
    tirlib.paged_attention(q, kv, one, out)
    tirlib.ops_check()
    lost = 0
    for work in range(0, 80, 4):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            tirlib.paged_attention(q, bad, one, out)
            for _ in range(work):
                x.add_(1)
            tirlib.paged_attention(q, kv, long, out)
        for _ in range(20):
            with torch.cuda.stream(busy):
                graph.replay()
            told, last = "", False
            while True:
                done = busy.query()
                try:
                    tirlib.ops_check(checked)
                except tirlib.TirError as e:
                    assert e.name == "INVALID_ARG"
                    told += e.message
                if last:
                    break
                last = done  # one more check after all is done
            lost += "page id" not in told or "length" not in told
    assert lost == 0


def test_checks_and_calls_from_several_threads(cuda, tirlib):
    """Two threads check streams of their own while a third calls operators on both, a bad
    page among them now and then: all come to an end, and the bad pages are reported."""
    torch = cuda
    kv, _, _ = cache(torch, tirlib, "f32", 2, 64, 1, 64, 16, seed=18)
    bad = tirlib.KVPages(kv.k, kv.v, torch.full_like(kv.table, -1))
    q, lens = torch.randn(2, 4, 64, device="cuda"), torch.tensor([64, 3], dtype=torch.int32, device="cuda")
    outs = torch.empty(2, *q.shape, device="cuda")
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    told, failed, done = [], [], threading.Event()

    def check(stream):
        while True:
            last = done.is_set()
            try:
                tirlib.ops_check(stream)
            except tirlib.TirError as e:
                (told if e.name == "INVALID_ARG" and "page id" in e.message else failed).append(str(e))
            if last:
                return

    threads = [threading.Thread(target=check, args=(s,)) for s in streams]
    for t in threads:
        t.start()
    for i in range(400):
        for s, out in zip(streams, outs):
            tirlib.paged_attention(q, bad if i % 50 == 7 else kv, lens, out, stream=s)
    torch.cuda.synchronize()
    done.set()
    for t in threads:
        t.join(timeout=60)
        assert not t.is_alive()
    assert told and not failed


@pytest.mark.parametrize("kind,q_heads,kv_heads,dim", [("bf16", 32, 8, 128), ("f32", 32, 4, 64), ("q8_0", 8, 1, 256), ("f16", 71, 1, 64)])
def test_workspace_of_the_largest_sizes_serves_smaller_ones(cuda, tirlib, kind, q_heads, kv_heads, dim):
    """The bytes needed never shrink with more rows, a longer max_len or a wider window."""
    torch = cuda
    rows, ctx = 300, 8192
    t = dtype(torch, kind)
    pool = torch.zeros(2, 4, 16, kv_heads, dim, dtype=t, device="cuda")
    scale = torch.ones(2, 4, 16, kv_heads, dim // 32, dtype=torch.float16, device="cuda") if kind == "q8_0" else (None, None)
    kv = tirlib.KVPages(pool[0], pool[1], torch.zeros(rows, ctx // 16, dtype=torch.int32, device="cuda"), scale[0], scale[1])
    act = torch.float32 if kind in ("f32", "q8_0") else t
    q = torch.zeros(rows, q_heads, dim, dtype=act, device="cuda")
    out = torch.empty_like(q)
    lens = torch.full((rows,), 100, dtype=torch.int32, device="cuda")
    ws = torch.empty(tirlib.paged_attention_workspace(kv, rows, q_heads, ctx), dtype=torch.uint8, device="cuda")
    sizes = lambda n, m, w: tirlib.paged_attention_workspace(kv, n, q_heads, m, w)
    for a, b in zip((1, 2, 3, 7, 20, 64, 100, 150, 200, 256), (2, 3, 7, 20, 64, 100, 150, 200, 256, 300)):
        for m in (1, 100, 2048, ctx):
            assert sizes(a, m, 0) <= sizes(b, m, 0)
            assert sizes(a, m, 0) <= sizes(a, ctx, 0) <= ws.numel()
            assert sizes(a, ctx, m) <= sizes(a, ctx, 0)
        for m in (1, 2048, ctx):
            tirlib.paged_attention(q[:a], kv, lens, out[:a], max_len=m, workspace=ws)
    torch.cuda.synchronize()
    tirlib.ops_check()


@pytest.mark.parametrize("act,kind,dim", [("f32", "f32", 64), ("bf16", "bf16", 128), ("f32", "q8_0", 64)])
def test_divided_rows_agree_whatever_max_len_says(cuda, tirlib, act, kind, dim):
    """The number of parts changes an output by no more than the two roundings' bounds, and
    the same call gives the same bits; max_len does divide the rows."""
    torch = cuda
    lens = [9001, 1, 0, 4097]
    kv, values, _ = cache(torch, tirlib, kind, 4, 9001, 1, dim, 16, seed=14)
    q = torch.randn(4, 5, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(15)).to(dtype(torch, act))
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    assert tirlib.paged_attention_workspace(kv, 4, 5) > 0 and tirlib.paged_attention_workspace(kv, 4, 5, 9001) > 0
    assert tirlib.paged_attention_workspace(kv, 4, 5, 1) == 0
    outs = []
    for max_len in (0, 9001, 1, 3000):
        pair = torch.empty(2, *q.shape, dtype=q.dtype, device="cuda")
        for o in pair:
            tirlib.paged_attention(q, kv, n, o, max_len=max_len)
        assert torch.equal(pair[0], pair[1])
        outs.append(pair[0].double())
    ref, mass, big = attention_ref(torch, q, values(), lens, 1 / math.sqrt(dim), 0)
    ut = torch.finfo(q.dtype).eps / 2
    e = (2 * dim / 8 + 4) * 2.0 ** -23 * big + 2.0 ** -20
    bound = 2 * ((2 * e + 9001 / 8 * 2.0 ** -23 + 2.0 ** -20) * mass + ut * ref.abs() + 2.0 ** -25)
    for o in outs[1:]:
        assert ((o - outs[0]).abs() <= bound).all()


def test_too_small_a_workspace_is_refused(cuda, tirlib):
    torch = cuda
    kv, _, _ = cache(torch, tirlib, "f32", 1, 20000, 1, 64, 16)
    need = tirlib.paged_attention_workspace(kv, 1, 4)
    assert need > 0
    q, lens = torch.zeros(1, 4, 64, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(tirlib.TirError) as e:
        tirlib.paged_attention(q, kv, lens, torch.empty_like(q), workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
    assert e.value.name == "INVALID_ARG" and "workspace" in e.value.message


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_heads,kv_heads", [(9, 1), (17, 1), (24, 2), (71, 1)])
@pytest.mark.parametrize("act,kind", [("f16", "f16"), ("f32", "f16"), ("bf16", "q8_0"), ("f32", "q8_0"), ("f32", "bf16")])
def test_large_head_groups(cuda, tirlib, act, kind, q_heads, kv_heads, dim):
    """More than eight query heads on a key-value head, in every type whose weights have parts
    of their own place; short rows, one over many tiles, a window."""
    torch = cuda
    lens = [5, 100, 0, 1211]
    kv, values, poison = cache(torch, tirlib, kind, 4, 1211, kv_heads, dim, 16, seed=q_heads)
    q = torch.randn(4, q_heads, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(19)).to(dtype(torch, act))
    vals = values()
    poison(lens)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for window in (0, 333):
        out = torch.empty_like(q)
        tirlib.paged_attention(q, kv, n, out, window=window)
        check_attention(torch, out, *attention_ref(torch, q, vals, lens, 1 / math.sqrt(dim), window), dim, 1211)
    tirlib.ops_check()


def test_another_stream_without_a_workspace(cuda, tirlib):
    """Rows that are not divided need none; a call that would divide them is refused there,
    and takes its workspace from torch on the current stream."""
    torch = cuda
    kv, values, _ = cache(torch, tirlib, "f32", 64, 256, 4, 64, 16, seed=16)
    q = torch.randn(64, 32, 64, device="cuda")
    lens = torch.full((64,), 256, dtype=torch.int32, device="cuda")
    out, other = torch.empty_like(q), torch.cuda.Stream()
    torch.cuda.synchronize()
    tirlib.paged_attention(q, kv, lens, out, max_len=256, stream=other)
    torch.cuda.synchronize()
    check_attention(torch, out, *attention_ref(torch, q, values(), [256] * 64, 0.125, 0), 64, 256)
    kv, values, _ = cache(torch, tirlib, "f32", 1, 20000, 1, 64, 16, seed=17)
    q, lens = q[:1, :4], lens[:1] * 70
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    with pytest.raises(tirlib.TirError) as e:
        tirlib.paged_attention(q, kv, lens, out, stream=other)
    assert e.value.name == "INVALID_ARG" and "workspace" in e.value.message
    tirlib.paged_attention(q, kv, lens, out, stream=torch.cuda.current_stream())
    check_attention(torch, out, *attention_ref(torch, q, values(), [17920], 0.125, 0), 64, 17920)
