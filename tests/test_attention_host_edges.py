"""Host side of rotary positions, the paged cache and attention at its edges (no GPU); beside test_attention_host.py."""
import ctypes as C

import numpy as np
import pytest

import ojas_engine_b200 as ob
from ojas_engine_b200 import runtime


@pytest.mark.parametrize("kw", [dict(factor=5e-324), dict(factor=1e-308, freq_factors=[1e-3] * 32)])
def test_frequencies_beyond_a_double_are_refused(kw):
    with pytest.raises(ob.OjasB200Error, match="frequenc"):
        ob.rope_frequencies(64, **kw)


def test_a_factor_that_no_pair_is_divided_by():
    """By parts, every pair turns more than beta_fast times (the slowest 4096 * 0.13 / 2 pi = 87): all keep their frequency, however
    far the divided one would lie beyond a double."""
    got = ob.rope_frequencies(64, factor=1e-308, freq_factors=[1e-3] * 32, orig_len=4096)
    assert np.allclose(got, ob.rope_frequencies(64, freq_factors=[1e-3] * 32), rtol=1e-15, atol=0)


class FakeLibrary:
    """The calls a B200Gpu makes of the library around attention, recorded; device memory is numbers."""

    def __init__(self, workspace=4096, context=0x1000):
        self.calls, self.live, self.workspace, self.context, self.next = [], {}, workspace, context, 0x100000

    def ojas_b200_create(self, device, stream, out):
        out._obj.value = self.context
        return 0

    def ojas_b200_destroy(self, ctx):
        self.calls.append("destroy")

    def ojas_b200_sync(self, ctx):
        self.calls.append("sync")
        return 0

    def ojas_b200_alloc(self, ctx, nbytes, out):
        self.next += 0x10000
        self.live[self.next] = nbytes
        out._obj.value = self.next
        return 0

    def ojas_b200_free(self, ctx, ptr):
        self.calls.append("free")
        del self.live[ptr.value]
        return 0

    def ojas_b200_last_error(self, ctx):
        return b""

    def ojas_b200_kv_create(self, *args):
        args[-1]._obj.value = 0x2000
        return 0

    def ojas_b200_kv_destroy(self, h):
        pass

    def ojas_b200_attention_workspace_bytes(self, *args):
        return self.workspace

    def ojas_b200_attention(self, *args):
        self.calls.append(("attention", args[-1]))
        return 0


def fake_gpu(monkeypatch, **kw):
    fake = FakeLibrary(**kw)
    monkeypatch.setattr(runtime._lib, "load", lambda: fake)
    return fake, ob.B200Gpu(0)


def fake_call(gpu, seqs=None, m=1):
    kv = ob.KvCache(gpu, ob.F16, ob.Buf(4096, 1 << 30), ob.Buf(4096, 1 << 30), 4, 16, 2, 128)
    seqs = seqs or ob.Seqs(ob.Buf(0, 8), ob.Buf(0, 4), ob.Buf(0, 16), 1, 4, m, 60)
    gpu.attention(kv, seqs, ob.Buf(0, 1 << 20), ob.Buf(0, 1 << 20), m, 4)
    return seqs


def test_closing_frees_the_scratch(monkeypatch):
    """Scratch a context grew through belongs to it: freed once its work has ended, before the context itself."""
    fake, gpu = fake_gpu(monkeypatch)
    fake_call(gpu)
    fake.workspace = 100000
    fake_call(gpu, m=2)
    assert len(fake.live) == 2                                 # a captured graph may use the first
    gpu.close()
    assert not fake.live
    assert fake.calls[-4:] == ["sync", "free", "free", "destroy"]
    gpu.close()                                                # twice: nothing more
    assert fake.calls.count("destroy") == 1


def test_closing_an_unused_context_does_not_wait(monkeypatch):
    fake, gpu = fake_gpu(monkeypatch)
    gpu.close()
    assert fake.calls == ["destroy"]


def test_closing_after_an_error_still_frees(monkeypatch):
    fake, gpu = fake_gpu(monkeypatch)
    fake_call(gpu)
    fake.ojas_b200_sync = lambda ctx: -5
    gpu.close()
    assert not fake.live and fake.calls[-1] == "destroy"


def test_the_workspace_is_asked_for_by_the_context_in_use(monkeypatch):
    """A Seqs outlives its context and a new one gets the old one's address: what the old one needed says nothing about the new one."""
    fake, gpu = fake_gpu(monkeypatch)
    seqs = fake_call(gpu)
    gpu.close()
    fake, gpu = fake_gpu(monkeypatch, workspace=1 << 20)
    fake_call(gpu, seqs)
    assert fake.calls[-1] == ("attention", 1 << 20)


def test_the_workspace_is_asked_for_once_per_shape(monkeypatch):
    fake, gpu = fake_gpu(monkeypatch)
    asked = []
    fake.ojas_b200_attention_workspace_bytes = lambda *args: asked.append(args) or 4096
    seqs = fake_call(gpu)
    fake_call(gpu, seqs)
    assert len(asked) == 1
    fake_call(gpu, seqs, m=2)
    assert len(asked) == 2


@pytest.mark.parametrize("scale,ok", [(0.0, True), (-0.5, True), (2.3e38, True), (2.4e38, False), (-3e38, False)])
def test_a_scale_stays_finite_in_powers_of_two(scale, ok):
    """Scores are formed in powers of two: the scale times log2(e) has to be a number, or equal scores of 0 were not."""
    seqs = runtime._lib.SeqsStruct(256, 512, 1024, 3, 8, 4, 100)
    rc = runtime._lib.load().ojas_b200_attention_check(ob.F16, 16, 2, 128, ob.F32, 8, 1024, 0, 4096, 0, scale, 1, 0, C.byref(seqs), 12, None, 0)
    assert rc == (0 if ok else -1)


def test_a_mix_over_the_index_goes_in_as_factors():
    """The other scaling by parts, linear in the pair's index between the indices where a pair turns beta_fast and beta_slow times:
    given as factors, which are f32 (half a step, 2^-24 relative at most)."""
    rot, base, orig, factor, fast, slow = 128, 10000.0, 4096, 8.0, 32.0, 1.0
    f = base ** (-2 * np.arange(rot // 2) / rot)
    index = [rot * np.log(orig / (2 * np.pi * turns)) / (2 * np.log(base)) for turns in (fast, slow)]
    keep = 1 - np.clip((np.arange(rot // 2) - np.floor(index[0])) / (np.ceil(index[1]) - np.floor(index[0])), 0, 1)
    want = f * keep + f / factor * (1 - keep)
    assert np.allclose(ob.rope_frequencies(rot, base, freq_factors=1 / (keep + (1 - keep) / factor)), want, rtol=2.0**-24, atol=0)
    turns = ob.rope_frequencies(rot, base, factor=factor, orig_len=orig, beta_fast=fast, beta_slow=slow)
    assert 0.4 < (turns / want).min() < 0.5                     # the two forms are not the same
