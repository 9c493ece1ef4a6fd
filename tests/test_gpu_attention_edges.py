"""Descriptions, lengths and shapes at the edge of what append and attention take, on the GPU; beside test_gpu_attention.py."""
import decimal
import math

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


# -------------------------------------------------------------------------------------------------------------- rotation
PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


def turns_128(rot, base):
    """Turns per position of each pair, base^(-2i / rot) / 2 pi, as integers over 2^128, formed in 60 digits."""
    with decimal.localcontext(prec=60):
        ln = decimal.Decimal(base).ln()
        return [int((-2 * i * ln / rot).exp() / (2 * PI) * 2**128) for i in range(rot // 2)]


@pytest.mark.parametrize("base", [10000, 500000])
@pytest.mark.parametrize("near", [0, 131072, 2**24 + 1, -(10**9), 2**31 - 2001, -(2**31)])
def test_angles_at_every_position(gpu, base, near):
    """Angles within 2e-9 radians: seen where a sine or a cosine is below 2^-8, whose own rounding (sincospi, one correction, one
    product: four steps of 2^-23 relative at most) then stays below 2e-9 too."""
    rot, n = 128, 2001
    pos = torch.arange(near, near + n, dtype=torch.int64)
    x = torch.zeros(n, 1, rot)
    x[..., : rot // 2] = 1.0
    xd, pd, rope = x.cuda(), pos.to(torch.int32).cuda(), ob.Rope(gpu, rot, base=float(base))
    torch.cuda.synchronize()
    gpu.rope_rows(rope, buf(xd), buf(xd), buf(pd), n, 1, rot)
    gpu.sync()
    got = xd.cpu().double()[:, 0]
    turns, whole = turns_128(rot, base), 2**128
    frac = torch.tensor([[((p * t + whole // 2) % whole - whole // 2) / whole for t in turns] for p in pos.tolist()], dtype=torch.float64)
    worst = 0.0
    for value, want in ((got[:, : rot // 2], torch.cos(2 * math.pi * frac)), (got[:, rot // 2 :], torch.sin(2 * math.pi * frac))):
        small = want.abs() < 2.0**-8
        assert near == 0 or small.sum() > 100
        worst = max(worst, ((value - want).abs() - 4 * 2.0**-23 * want.abs())[small].max().item())
        assert ((value - want).abs() <= 2e-9 + 4 * 2.0**-23).all()
    assert worst <= 2e-9, worst


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


@pytest.mark.parametrize("dim,q_heads", [(64, 8), (128, 32), (256, 16)])
def test_one_short_sequence_joins_in_one_launch(gpu, dim, q_heads):
    """A B200 places the clusters that the splits of a short sequence make: no workspace, no second launch."""
    b = Batch([1], [900], kv_heads=q_heads // 4, dim=dim, seed=3).upload(gpu)
    assert gpu.attention_workspace_bytes(b.kv, b.seqs, 1, q_heads) == 0
    q = randn(1, 1, q_heads, dim)
    qd, out, before = q.cuda(), torch.empty(1, q_heads, dim).cuda(), gpu.launch_count
    torch.cuda.synchronize()
    gpu.attention(b.kv, b.seqs, buf(qd), buf(out), 1, q_heads)
    gpu.sync()
    assert gpu.launch_count == before + 1
    want, weight, vmax = b.attention_exact(q, q_heads)
    check(out, want, attention_bound(want, weight, vmax, dim, 900, F32, F16, 2))
