"""What the paged cache operators promise, where it is easiest to break: quotients at the edge
of a half step.  Tolerances as in test_paged_gpu.py, whose helpers these tests use."""
import numpy as np
import pytest

from test_paged_gpu import cache, q8_blocks

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
