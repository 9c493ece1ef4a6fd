"""Batches over a paged cache for the tests of rotary positions, the append and attention, and their plain forms in 64 bits."""
import math

import numpy as np
import torch

import ojas_engine_b200 as ob

TORCH = {ob.F32: torch.float32, ob.F16: torch.float16, ob.BF16: torch.bfloat16}
HALF = {ob.F32: 2.0 ** -24, ob.F16: 2.0 ** -11, ob.BF16: 2.0 ** -8}      # half a step of each type, relative


def buf(t: torch.Tensor) -> ob.Buf:
    return ob.Buf(t.data_ptr(), t.untyped_storage().nbytes() - t.storage_offset() * t.element_size())


class Batch:
    """Sequences with ``rows[b]`` new rows, ``lens[b]`` tokens long with them, in a cache of shuffled pages.  Everything the
    cache holds outside the sequences is NaN, and page-table entries past a sequence's last page are -1."""

    def __init__(self, rows, lens, kv_heads=2, dim=128, page=16, cache=ob.F16, nhd=False, seed=0, extra_rows=0, max_rows=None, max_len=None, spare=2):
        self.rows, self.lens, self.hk, self.dim, self.page, self.cache = list(rows), list(lens), kv_heads, dim, page, cache
        self.g = torch.Generator().manual_seed(seed)
        used = [(n + page - 1) // page for n in lens]
        self.pages, self.stride = sum(used) + spare, max(max(used), 1)
        order = torch.randperm(self.pages, generator=self.g)[: sum(used)].tolist()
        table = torch.full((len(lens), self.stride), -1, dtype=torch.int32)
        for b, n in enumerate(used):
            table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.cu = torch.tensor([0] + list(rows)).cumsum(0).to(torch.int32)
        self.M = int(self.cu[-1]) + extra_rows
        self.k_rows = [torch.randn(n, kv_heads, dim, generator=self.g).to(TORCH[cache]) for n in lens]
        self.v_rows = [torch.randn(n, kv_heads, dim, generator=self.g).to(TORCH[cache]) for n in lens]
        self.nhd, self.table = nhd, table
        self.shape = (self.pages, page, kv_heads, dim) if nhd else (self.pages, kv_heads, page, dim)
        self.k, self.v = (torch.full(self.shape, math.nan, dtype=TORCH[cache]) for _ in range(2))
        for b in range(len(lens)):
            self.put(self.k, b, 0, self.k_rows[b])
            self.put(self.v, b, 0, self.v_rows[b])
        self.max_rows, self.max_len = max_rows or max(max(rows), 1), max_len or max(max(lens), 1)

    def view(self, cache):                                   # [pages, page, heads, dim]
        return cache if self.nhd else cache.transpose(1, 2)

    def put(self, cache, b, first, rows):
        at = torch.arange(first, first + len(rows))
        if len(rows):
            self.view(cache)[self.table[b].long()[at // self.page], at % self.page] = rows.to(cache.dtype)

    def upload(self, gpu):
        self.dev = {n: getattr(self, n).cuda() for n in ("k", "v", "cu", "table")}
        self.dev["len"] = torch.tensor(self.lens, dtype=torch.int32).cuda()
        strides = dict(page_stride=self.page * self.hk * self.dim, head_stride=self.dim, token_stride=self.hk * self.dim) if self.nhd else {}
        self.kv = ob.KvCache(gpu, self.cache, buf(self.dev["k"]), buf(self.dev["v"]), self.pages, self.page, self.hk, self.dim, **strides)
        self.seqs = ob.Seqs(buf(self.dev["cu"]), buf(self.dev["len"]), buf(self.dev["table"]), len(self.lens), self.stride, self.max_rows, self.max_len)
        return self

    def attention_exact(self, q, hq, scale=None, causal=True, window=0, fill=None):
        """out [M, hq, dim] and the elementwise bound of an f32 evaluation with exact inputs, both in 64 bits.  Rows of no
        sequence hold ``fill``."""
        d, group = self.dim, hq // self.hk
        scale = d ** -0.5 if scale is None else scale
        out = torch.full((self.M, hq, d), 0.0 if fill is None else fill, dtype=torch.float64)
        weight, vmax = torch.zeros(self.M, hq, 1, dtype=torch.float64), torch.zeros(self.M, hq, 1, dtype=torch.float64)
        for b, (n, total) in enumerate(zip(self.rows, self.lens)):
            t0 = int(self.cu[b])
            pos, key = torch.arange(total - n, total)[:, None], torch.arange(total)
            seen = (key <= pos) if causal else (key >= 0).expand(n, total)
            if window:
                seen = seen & (key > pos - window)
            k = self.k_rows[b].double().repeat_interleave(group, 1).transpose(0, 1)
            v = self.v_rows[b].double().repeat_interleave(group, 1).transpose(0, 1)
            x = q[t0 : t0 + n].double().transpose(0, 1)
            s = (x @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)) if total else s
            tot = p.sum(-1, keepdim=True)
            out[t0 : t0 + n] = ((p @ v) / tot.clamp(min=1e-300)).transpose(0, 1)
            size = (x.abs() @ k.abs().transpose(1, 2) * abs(scale)).masked_fill(~seen, 0.0)
            if total:
                weight[t0 : t0 + n] = size.amax(-1, keepdim=True).transpose(0, 1)
                vmax[t0 : t0 + n] = v.abs().amax((1, 2))[None, :, None]
        return out, weight, vmax


def attention_bound(out, weight, vmax, dim, keys, act, cache, p_terms):
    """How far an element may be off, from the roundings an evaluation makes (first order, worst case):
    a score s = sum q k over dim products, accumulated in f32 over dim / 16 instructions, a step of 2^-23 each (the tensor
    cores cut), with q in two terms of the cache's type when it is f32; exp2 and its argument: 2^-21 and 2^-22 |s|; a
    probability in p_terms terms; dim-independent accumulation over the keys, 16 per instruction, 2^-23 each; the
    final division and the rounding to the activations' type."""
    q_off = 0.0 if act != ob.F32 else 2 * HALF[cache] ** 2
    ds = weight * ((dim / 16 + 4) * 2.0 ** -23 + q_off + 2.0 ** -22) + 2.0 ** -21
    rel = 2 * ds + HALF[cache] ** p_terms * (2 if p_terms == 2 else 1) + (keys / 16 + 16) * 2.0 ** -23
    return rel * vmax + HALF[act] * (out.abs() + rel * vmax) + 1e-30


def rope_exact(x, pos, freq, layout, magnitude=1.0):
    """x [tokens, heads, dim] turned in 64 bits: the rotation as complex numbers."""
    rot = 2 * len(freq)
    x = x.double()
    angle = torch.as_tensor(freq, dtype=torch.float64)[None, None] * pos.double()[:, None, None]
    a, b = (x[..., : rot // 2], x[..., rot // 2 : rot]) if layout == ob.ROPE_HALF else (x[..., 0:rot:2], x[..., 1:rot:2])
    u, v = magnitude * (a * angle.cos() - b * angle.sin()), magnitude * (b * angle.cos() + a * angle.sin())
    y = x.clone()
    if layout == ob.ROPE_HALF:
        y[..., : rot // 2], y[..., rot // 2 : rot] = u, v
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = u, v
    return y


def rope_bound(x, y, rot, layout, magnitude, out_type):
    """An f32 rotation: the angle within 2^-23 (its rounding to 24 bits of at most pi) + 2^-22 for sine and cosine, two
    products and a sum; then the output's type."""
    x = x.double().abs()
    a, b = (x[..., : rot // 2], x[..., rot // 2 : rot]) if layout == ob.ROPE_HALF else (x[..., 0:rot:2], x[..., 1:rot:2])
    size = (a + b) * magnitude * (math.pi * 2.0 ** -24 + 2.0 ** -22 + 4 * 2.0 ** -24)
    e = torch.zeros_like(x)
    if layout == ob.ROPE_HALF:
        e[..., : rot // 2], e[..., rot // 2 : rot] = size, size
    else:
        e[..., 0:rot:2], e[..., 1:rot:2] = size, size
    tiny = {ob.F32: 0.0, ob.F16: 2.0 ** -25, ob.BF16: 0.0}[out_type]          # half a step of f16's subnormals
    return e + HALF[out_type] * (y.abs() + e) + tiny + 1e-37


def check(got, want, bound, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: {int((~torch.isfinite(got)).sum())} values are not finite"
    over = ((got - want).abs() / bound).max().item()
    assert over <= 1.0, f"{what}: {over:.2f} times the bound"
    return over
