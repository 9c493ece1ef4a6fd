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


# ------------------------------------------------------------------------------------------------------- long loops, splits
def exact_on_gpu(b, q, hq, causal=True, window=0):
    """Batch.attention_exact by the GPU's 64-bit units, for sizes that take the host too long: out and the scores' sizes."""
    d, group = b.dim, hq // b.hk
    out, weight = (torch.zeros(b.M, hq, n, dtype=torch.float64) for n in (d, 1))
    for i, (n, total) in enumerate(zip(b.rows, b.lens)):
        t0, key = int(b.cu[i]), torch.arange(total).cuda()
        pos = torch.arange(total - n, total).cuda()[:, None]
        seen = (key <= pos) & (key > pos - (window or total)) if causal else (key >= 0).expand(n, total)
        for h in range(b.hk):
            k, v = b.k_rows[i][:, h].cuda().double(), b.v_rows[i][:, h].cuda().double()
            for j in range(h * group, (h + 1) * group):
                x = q[t0 : t0 + n, j].cuda().double()
                s = (x @ k.T * d**-0.5).masked_fill_(~seen, -math.inf)
                out[t0 : t0 + n, j] = (torch.softmax(s, -1) @ v).cpu()
                weight[t0 : t0 + n, j] = (x.abs() @ k.abs().T * d**-0.5).masked_fill_(~seen, 0.0).amax(-1, keepdim=True).cpu()
    return out, weight


def attend(gpu, b, q, hq, act, window=0, causal=True):
    qd = q.to(TORCH[act]).cuda()
    out = torch.full_like(qd, 77.0)
    torch.cuda.synchronize()
    gpu.attention(b.kv, b.seqs, buf(qd), buf(out), b.M, hq, act_type=act, window=window, causal=causal)
    gpu.sync()
    return out


def splits(gpu, b, hq, act, window=0):
    """In how many parts the keys of a call that joins through its workspace are split (1: it needs none)."""
    need = gpu.attention_workspace_bytes(b.kv, b.seqs, b.M, hq, act, window)
    return max(1, need // (b.M * hq * (8 + 4 * b.dim)))


FLUSH = 512                                                    # keys after which f32 results are added to rounded sums


@pytest.mark.parametrize("dim,tokens,heads,split", [(64, 200, 8, False), (128, 200, 8, False), (256, 200, 8, True), (256, 288, 8, False), (64, 160, 4, True),
                                                    (128, 160, 4, True), (256, 160, 4, True), (64, 30, 1, True), (128, 30, 1, True), (256, 30, 1, True)])
def test_sums_of_many_keys_keep_f32_precision(gpu, dim, tokens, heads, split):
    """f32 activations, 12 000 keys of nearly equal weight, values between 1 and 2: everything the accumulator loses has one sign.
    Between two roundings into the sums it takes 512 keys: 2 * 512 / 16 instructions that cut up to 2^-23 of what has grown so far, half of
    the whole on average, so 32 steps of 2^-23; then one rounded addition per 512 keys and per split; the rest as in attention_bound, with
    scores small enough not to matter.  (Without the sums: 1500 instructions, 750 steps at most, 280 on average.)"""
    group, keys = 8, 12000
    b = Batch([tokens], [keys], kv_heads=heads, dim=dim, page=64, seed=dim)
    b.v_rows[0] = (1 + torch.rand(keys, heads, dim, generator=b.g)).half()
    b.put(b.v, 0, 0, b.v_rows[0])
    b.upload(gpu)
    n = splits(gpu, b, heads * group, F32)
    assert (n > 1) == split and (tokens == 30 or keys / n > 3 * FLUSH + 128)         # three flushes at least in one CTA
    q = randn(1, tokens, heads * group, dim) * 0.01
    want, weight = exact_on_gpu(b, q, heads * group)
    steps = 32 + keys / FLUSH + n + 16
    rel = 2 * (weight * ((dim / 16 + 4) * 2.0**-23 + 2 * 2.0**-22 + 2.0**-22) + 2.0**-21) + 2 * 2.0**-22 + steps * 2.0**-23
    check(attend(gpu, b, q, heads * group, F32), want, 2 * rel + 2.0**-24 * want)


@pytest.mark.parametrize("act,cache", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens,heads", [(200, 8), (160, 2)])
def test_a_maximum_that_grows_along_the_keys(gpu, act, cache, dim, tokens, heads):
    """Keys that grow all along a sequence of 4000: maxima rise in most blocks, before and after results were added to the sums."""
    group, keys = 8, 4000
    b = Batch([tokens], [keys], kv_heads=heads, dim=dim, page=32, cache=cache, seed=dim + tokens)
    b.k_rows[0] = (b.k_rows[0].float() * torch.linspace(0.02, 3, keys)[:, None, None]).to(TORCH[cache])
    b.put(b.k, 0, 0, b.k_rows[0])
    b.upload(gpu)
    q = randn(1, tokens, heads * group, dim).to(TORCH[act])
    want, weight = exact_on_gpu(b, q, heads * group)
    vmax = b.v_rows[0].double().abs().max()
    check(attend(gpu, b, q, heads * group, act), want, attention_bound(want, weight, vmax, dim, keys, act, cache, 2 if act == F32 else 1))


@pytest.mark.parametrize("act,cache", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("dim,rows,lens,heads,group,window", [
    (64, [2500], [2500], 8, 4, 0), (128, [2200], [3001], 4, 4, 0), (256, [1500], [2000], 4, 4, 0),               # prompts, keys not split
    (64, [900, 1, 70], [3300, 2047, 1000], 2, 7, 0), (128, [300, 5], [4100, 4000], 1, 8, 0), (256, [40, 200], [5000, 999], 2, 2, 0),
    (64, [3000], [3000], 4, 2, 500), (128, [1000, 1000], [1000, 2500], 4, 4, 777), (256, [700], [1700], 2, 4, 64),
    (64, [1, 1, 1], [6000, 1, 2049], 2, 8, 0), (128, [1, 3], [9000, 500], 1, 4, 0), (256, [1, 2], [7000, 65], 2, 4, 0), (128, [4], [5000], 2, 3, 1000)])
def test_every_key_counts_once(gpu, act, cache, dim, rows, lens, heads, group, window):
    """Value j is the unit vector of j modulo dim: an element of the result is the weight of every dim-th key, and is off by a
    relative error only.  One key too many or too few among the some tens of an element is beyond any rounding."""
    b = Batch(rows, lens, kv_heads=heads, dim=dim, page=16, cache=cache, seed=dim + len(rows))
    for i, n in enumerate(lens):
        b.v_rows[i] = torch.eye(dim).repeat((n + dim - 1) // dim, 1)[:n, None].expand(n, heads, dim).to(TORCH[cache]).contiguous()
        b.put(b.v, i, 0, b.v_rows[i])
    b.upload(gpu)
    q = (randn(1, b.M, heads * group, dim) * 0.3).to(TORCH[act])
    want, weight = exact_on_gpu(b, q, heads * group, window=window)
    bound = attention_bound(want, weight, want, dim, max(lens), act, cache, 2 if act == F32 else 1)
    check(attend(gpu, b, q, heads * group, act, window=window), want, bound)


@pytest.mark.parametrize("act,cache", [(F32, F16), (BF16, BF16)])
@pytest.mark.parametrize("dim,rows,group", [(64, [1, 3, 1], 4), (64, [2, 1, 1], 14), (128, [1, 1, 2], 8), (256, [1, 2, 1], 4), (256, [3, 1, 1], 5)])
def test_few_rows_joined_through_the_workspace(gpu, act, cache, dim, rows, group):
    """More splits than a cluster has, planned for lengths far beyond the actual ones: long, short and single-block sequences."""
    b = Batch(rows, [6000, 700, 9], kv_heads=1, dim=dim, cache=cache, seed=dim, max_len=500000).upload(gpu)
    assert splits(gpu, b, group, act) > 16
    q = randn(2, b.M, group, dim).to(TORCH[act])
    want, weight, vmax = b.attention_exact(q, group)
    check(attend(gpu, b, q, group, act), want, attention_bound(want, weight, vmax, dim, 6000, act, cache, 2 if act == F32 else 1))


@pytest.mark.parametrize("rows,max_len", [(1, 500000), (60, 9000)])
def test_two_streams_with_a_workspace_each(gpu, rows, max_len):
    """Two contexts on streams of their own, splits that join through scratch, different queries: neither sees the other's."""
    b = Batch([rows, rows], [9000, 4000], kv_heads=2, dim=128, seed=5, max_len=max_len).upload(gpu)
    qs = [randn(seed, b.M, 8, 128) for seed in (3, 4)]
    exact = [b.attention_exact(q, 8) for q in qs]
    others, on_gpu = [ob.B200Gpu(0) for _ in qs], [q.cuda() for q in qs]
    outs = [torch.empty(b.M, 8, 128).cuda() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for o, q, out in zip(others, on_gpu, outs):
            assert o.attention_workspace_bytes(b.kv, b.seqs, b.M, 8) > 0
            o.attention(b.kv, b.seqs, buf(q), buf(out), b.M, 8)
    for o, out, (want, weight, vmax) in zip(others, outs, exact):
        o.sync()
        check(out, want, attention_bound(want, weight, vmax, 128, 9000, F32, F16, 2))
        o.close()


@pytest.mark.parametrize("rows,max_len", [(1, 500000), (60, 9000)])
def test_two_graphs_share_a_workspace_in_turn(gpu, rows, max_len):
    b = Batch([rows, rows], [5000, 300], kv_heads=2, dim=128, seed=5, max_len=max_len).upload(gpu)
    assert gpu.attention_workspace_bytes(b.kv, b.seqs, b.M, 8) > 0
    qs = [randn(seed, b.M, 8, 128) for seed in (3, 4)]
    on_gpu, outs = [q.cuda() for q in qs], [torch.empty(b.M, 8, 128).cuda() for _ in qs]
    torch.cuda.synchronize()
    gpu.attention(b.kv, b.seqs, buf(on_gpu[0]), buf(outs[0]), b.M, 8)
    gpu.sync()
    graphs = []
    for q, out in zip(on_gpu, outs):
        gpu.graph_begin()
        gpu.attention(b.kv, b.seqs, buf(q), buf(out), b.M, 8)
        graphs.append(gpu.graph_end())
    first = None
    for _ in range(5):
        for gr in graphs:
            gpu.graph_launch(gr)
        gpu.sync()
        first = first or [o.clone() for o in outs]
        assert all(torch.equal(a, o) for a, o in zip(first, outs))
    for q, out in zip(qs, outs):
        want, weight, vmax = b.attention_exact(q, 8)
        check(out, want, attention_bound(want, weight, vmax, 128, 5000, F32, F16, 2))
    for gr in graphs:
        gpu.graph_destroy(gr)


@pytest.mark.parametrize("act,cache", [(F32, F16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("dim,rows", [(128, 1), (64, 5), (256, 2), (128, 60), (64, 300), (256, 100)])
@pytest.mark.parametrize("scale", [0.0, -0.11, 1.5])
def test_scales_of_any_sign(gpu, act, cache, dim, rows, scale):
    b = Batch([rows, 1], [rows + 130, 77], kv_heads=2, dim=dim, cache=cache, seed=dim + rows).upload(gpu)
    q = randn(1, b.M, 8, dim).to(TORCH[act])
    qd, out = q.cuda(), torch.empty(b.M, 8, dim, dtype=TORCH[act]).cuda()
    torch.cuda.synchronize()
    gpu.attention(b.kv, b.seqs, buf(qd), buf(out), b.M, 8, act_type=act, scale=scale)
    gpu.sync()
    want, weight, vmax = b.attention_exact(q, 8, scale=scale)
    check(out, want, attention_bound(want, weight, vmax, dim, max(b.lens), act, cache, 2 if act == F32 else 1))


@pytest.mark.parametrize("rows,act", [(1, F32), (100, F16)])
def test_a_length_of_31_bits_is_reported(gpu, rows, act):
    """Longer than max_len may be, with a table that would hold it: no key of it is read, the rows give zeros."""
    b = Batch([rows], [rows], kv_heads=1, dim=64, page=16, seed=3)
    b.lens, b.stride, b.table = [2**31 - 1], 2**27, torch.full((1, 2**27), -1, dtype=torch.int32)
    b.upload(gpu)
    q = randn(1, rows, 4, 64, dtype=TORCH[act]).cuda()
    out = torch.full_like(q, 77.0)
    torch.cuda.synchronize()
    gpu.attention(b.kv, b.seqs, buf(q), buf(out), rows, 4, act_type=act, window=16)
    with pytest.raises(ob.OjasB200Error) as e:
        gpu.sync()
    assert e.value.code == -5 and "batch" in str(e.value)
    torch.cuda.synchronize()
    assert (out == 0).all()


@pytest.mark.parametrize("act,cache", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,lens,heads,group", [([2], [2534], 3, 17), ([8, 8], [1355, 410], 2, 9), ([20, 1], [3000, 100], 1, 5), ([120], [5000], 1, 1), ([130, 30], [4000, 3999], 1, 2)])
def test_one_tile_split_along_the_keys(gpu, act, cache, dim, rows, lens, heads, group):
    """Between what the kernel for few rows takes and two tiles of 128 rows, with the keys split: unnormalized f32 sums leave the
    kernel whatever the activations are."""
    b = Batch(rows, lens, kv_heads=heads, dim=dim, page=192 if len(rows) == 1 else 32, nhd=len(rows) == 1, cache=cache, seed=dim).upload(gpu)
    assert splits(gpu, b, heads * group, act) > 1
    q = randn(1, b.M, heads * group, dim).to(TORCH[act])
    want, weight, vmax = b.attention_exact(q, heads * group)
    check(attend(gpu, b, q, heads * group, act), want, attention_bound(want, weight, vmax, dim, max(lens), act, cache, 2 if act == F32 else 1))
