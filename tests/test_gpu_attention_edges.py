"""Descriptions, lengths and shapes at the edge of what append and attention take, on the GPU; beside test_gpu_attention.py."""
import pytest
import torch

import ojas_engine_b200 as ob
from attn_helpers import TORCH, Batch, buf, check, rope_bound, rope_exact

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
