"""Descriptions, lengths and shapes at the edge of what append and attention take, on the GPU; beside test_gpu_attention.py."""
import pytest
import torch

import ojas_engine_b200 as ob
from ojas_engine_b200 import tp
from attn_helpers import TORCH, Batch, attention_bound, buf, check, rope_bound, rope_exact

pytestmark = pytest.mark.gpu
F32, F16, BF16 = ob.F32, ob.F16, ob.BF16
HALVES, INTER = ob.ROPE_HALF, ob.ROPE_INTERLEAVED


def randn(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---------------------------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("layout", [HALVES, INTER])
@pytest.mark.parametrize("xt,ct,qt", [(F32, F16, F32), (BF16, BF16, BF16)])
@pytest.mark.parametrize("dim,rot,hq,hk", [(64, 64, 4, 2), (64, 8, 9, 1), (64, 24, 3, 3), (256, 256, 8, 1), (256, 64, 5, 5), (256, 40, 16, 4)])
def test_append_head_sizes(gpu, layout, xt, ct, qt, dim, rot, hq, hk):
    """Heads of 64 and 256, rotated in part: four pairs at a time, their angles read two by two."""
    b = Batch([3, 1, 20], [3, 50, 90], kv_heads=hk, dim=dim, page=16, cache=ct, seed=rot).upload(gpu)
    x = randn(dim + rot, b.M, hq + 2 * hk, dim, dtype=TORCH[xt])
    xd, qo = x.cuda(), torch.zeros(b.M, hq, dim, dtype=TORCH[qt]).cuda()
    base, size, rope, freq = buf(xd), dim * xd.element_size(), ob.Rope(gpu, rot), ob.rope_frequencies(rot)
    q, k, v = (ob.Buf(base.ptr + n * size, base.nbytes - n * size) for n in (0, hq, hq + hk))
    torch.cuda.synchronize()
    gpu.kv_append(b.kv, b.seqs, k, v, b.M, rope=rope, layout=layout, x_type=xt, x_stride=(hq + 2 * hk) * dim, q=q, q_out=buf(qo), q_heads=hq, q_type=qt)
    gpu.sync()
    kc, vc = (b.view(b.dev[n].cpu()) for n in ("k", "v"))
    for i, (n, total) in enumerate(zip(b.rows, b.lens)):
        t0, pos = int(b.cu[i]), torch.arange(total - n, total)
        rows = x[t0 : t0 + n]
        at = (b.table[i].long()[pos // b.page], pos % b.page)
        for got, part, t in ((qo[t0 : t0 + n], rows[:, :hq], qt), (kc[at], rows[:, hq : hq + hk], ct)):
            want = rope_exact(part, pos, freq, layout)
            check(got, want, rope_bound(part, want, rot, layout, 1.0, t))
        assert torch.equal(vc[at], rows[:, hq + hk :].to(TORCH[ct]))


# ------------------------------------------------------------------------------------------ rows outside the call
@pytest.mark.parametrize("shift,cut", [(0, 2), (0, 5), (0, 6), (-1, 0), (-4, 0)])
@pytest.mark.parametrize("rows,max_rows", [([3, 2, 5], 5), ([40, 30, 5], 40), ([1] * 140 + [5], 5), ([1] * 140 + [5], 600)])
def test_rows_outside_the_call_are_reported(gpu, rows, max_rows, shift, cut):
    """Offsets that lead behind the call's last row (``cut`` rows, the last sequence wholly among them from five on) or in front of its
    first: an error from either call; the rows inside are stored and attended at the places their sequences give them.  Row tiles
    of every sequence (max_rows near the rows) and tiles counted over the sequences."""
    b = Batch(rows, [n + 20 for n in rows], kv_heads=1, dim=64, seed=3, max_rows=max_rows)
    q, total = randn(1, b.M, 4, 64), b.M
    want, weight, vmax = b.attention_exact(q, 4)
    bound = attention_bound(want, weight, vmax, 64, max(b.lens), F32, F16, 2)
    b.cu += shift
    b.upload(gpu)
    m = total + shift - cut                                    # rows of the call: those of q from -shift on
    inside = slice(-shift, -shift + m)
    qd, out = q[inside].contiguous().cuda(), torch.full((m + 3, 4, 64), 77.0).cuda()
    torch.cuda.synchronize()
    gpu.attention(b.kv, b.seqs, buf(qd), buf(out), m, 4)
    with pytest.raises(ob.OjasB200Error) as e:
        gpu.sync()
    assert e.value.code == -5 and "batch" in str(e.value)
    torch.cuda.synchronize()
    check(out[:m], want[inside], bound[inside])
    assert (out[m:] == 77).all()
    x, before = randn(2, m, 64).cuda(), b.dev["k"].clone()
    torch.cuda.synchronize()
    gpu.kv_append(b.kv, b.seqs, buf(x), buf(x), m)
    with pytest.raises(ob.OjasB200Error) as e:
        gpu.sync()
    assert e.value.code == -5 and "batch" in str(e.value)
    torch.cuda.synchronize()
    t, stored, old = 0, b.view(b.dev["k"].cpu()), b.view(before.cpu())
    for i, (n, length) in enumerate(zip(b.rows, b.lens)):
        for p in range(length - n, length):
            row, at = t + shift, (b.table[i, p // b.page], p % b.page)
            t += 1
            kept = row < 0 or row >= m or int(b.cu[i]) < 0     # (a sequence that begins in front of the call is not stored)
            assert torch.equal(stored[at][0], old[at][0] if kept else x[row].half().cpu()), (i, p)
            old[at] = stored[at]
    assert torch.equal(stored.nan_to_num(nan=9.0), old.nan_to_num(nan=9.0))


def test_a_batch_with_nothing_wrong_is_not_reported(gpu):
    """Empty sequences at both ends, rows behind the last one, fewer rows than the call has."""
    b = Batch([0, 3, 0, 1, 0], [0, 40, 7, 9, 0], kv_heads=1, dim=64, seed=3, extra_rows=4, max_rows=300).upload(gpu)
    q = randn(1, b.M, 4, 64).cuda()
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    gpu.attention(b.kv, b.seqs, buf(q), buf(out), b.M, 4)
    gpu.kv_append(b.kv, b.seqs, buf(q), buf(q), b.M, x_stride=256)
    gpu.sync()


def test_a_wrong_batch_and_a_lost_wait_are_both_named(gpu):
    """One status word for two errors: the message says both, and after each alone only that one."""
    b = Batch([1], [20], kv_heads=1, dim=64, seed=3).upload(gpu)
    b.dev["table"][0, 0] = b.pages
    q = randn(1, 1, 4, 64).cuda()
    out, y = torch.empty_like(q), gpu.alloc(64)
    group = tp.TpGroup(gpu, 1, 0, 64, lambda blob: [blob])
    group.set_wait_us(2000)
    torch.cuda.synchronize()
    for batch, wait in ((True, True), (True, False), (False, True)):
        if batch:
            gpu.attention(b.kv, b.seqs, buf(q), buf(out), 1, 4)
        if wait:
            group.join(group.COL, y, 64)                      # nothing was pushed: its wait ends by itself
        with pytest.raises(ob.OjasB200Error) as e:
            gpu.sync()
        assert ("batch" in str(e.value)) == batch and ("bounded wait" in str(e.value)) == wait
    group.close()
    gpu.free(y)
