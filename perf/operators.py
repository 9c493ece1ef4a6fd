"""What is measured of the operators between a layer's projections: rotary positions, appending keys and values to a
paged cache with the rotation applied on the way, and attention of new tokens over that cache.

A case describes a batch of sequences; its lengths follow from the case alone, its values from the seed.  ``run`` is one
pass: in the plain form elementary torch operations, with ``own`` the calls a program makes of the library.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 30}          # the element types' GGUF codes


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    attn = dict(op="attention", layout="hnd", window=0, ragged=1)
    return [
        # rotating the query and key heads of eight decoded tokens, far into long contexts: the smallest call
        dict(name="rope_decode", op="rope", tokens=8, heads=40, fused=48, dim=128, rot=128, pairs="half", act="f32", out="f32", scaled=0, far=131072),
        # the same for a prompt's chunk: 64 query and 8 key heads, half of each head rotated, frequencies scaled by parts
        dict(name="rope_chunk", op="rope", tokens=2048, heads=72, fused=80, dim=128, rot=64, pairs="interleaved", act="f32", out="f32", scaled=1, far=32768),
        # one new token for each of 64 sequences, straight from the fused projection's rows into the cache
        dict(name="append_decode", op="append", seqs=64, rows=1, len=4096, ragged=1, q_heads=32, kv_heads=8, dim=128, page=16, layout="hnd", pairs="half",
             rot=128, scaled=0, act="f32", cache="f16", q_out="f32"),
        # prompts' chunks of different lengths, interleaved pairs, scaled frequencies, a cache whose pages hold token after token
        dict(name="append_chunk", op="append", seqs=5, rows=1500, len=9000, ragged=1, q_heads=64, kv_heads=8, dim=128, page=32, layout="nhd",
             pairs="interleaved", rot=128, scaled=1, act="f32", cache="bf16", q_out="bf16"),
        # one short sequence, one token: latency is all
        dict(attn, name="decode_one", seqs=1, rows=1, len=777, q_heads=32, kv_heads=8, dim=128, page=16, act="f32", cache="f16"),
        # a serving batch, one token each, lengths from a few tokens to thousands
        dict(attn, name="decode_batch", seqs=64, rows=1, len=8192, q_heads=64, kv_heads=8, dim=128, page=64, act="f32", cache="f16"),
        # two very long sequences: the work has to be split along them
        dict(attn, name="decode_long", seqs=2, rows=1, len=131000, q_heads=32, kv_heads=8, dim=128, page=128, act="bf16", cache="bf16", layout="nhd"),
        # heads of 256, eight query heads to a key head, several tokens checked at once
        dict(attn, name="decode_wide", seqs=16, rows=2, len=6000, q_heads=16, kv_heads=2, dim=256, page=16, act="f32", cache="f16"),
        # a few drafted tokens per sequence, seven query heads to a key head
        dict(attn, name="verify", seqs=8, rows=5, len=5000, q_heads=28, kv_heads=4, dim=128, page=16, act="bf16", cache="bf16"),
        # a whole prompt
        dict(attn, name="prefill", seqs=1, rows=8192, len=8192, q_heads=32, kv_heads=8, dim=128, page=64, act="f16", cache="f16"),
        # a chunk of a prompt behind a long beginning, between one-token sequences, activations as the projections give them
        dict(attn, name="chunk", seqs=4, rows=1000, len=12000, q_heads=32, kv_heads=8, dim=128, page=16, act="f32", cache="f16", layout="nhd", ragged=2),
        # prompts under a sliding window, heads of 64
        dict(attn, name="window", seqs=3, rows=4000, len=5000, q_heads=16, kv_heads=8, dim=64, page=32, act="bf16", cache="bf16", window=1024),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    while True:
        op = rng.choice(["rope", "append", "attention", "attention", "attention"])
        dim = rng.choice([64, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8, 8])
        group = rng.choice([1, 2, 3, 4, 5, 7, 8, 8])
        pairs, scaled = rng.choice(["half", "interleaved"]), rng.randint(0, 1)
        rot = rng.choice([dim, dim // 2])
        act, cache = rng.choice([("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
        if op == "rope":
            tokens = _log(rng, 1, 6000)
            heads = kv * (group + 1)
            if tokens * heads * dim > 36_000_000:
                continue
            return dict(op=op, tokens=tokens, heads=heads, fused=heads + kv, dim=dim, rot=rot, pairs=pairs, act=rng.choice(["f32", act]), out=act, scaled=scaled,
                        far=_log(rng, 4096, 1 << 20))
        seqs, layout, page = _log(rng, 1, 64), rng.choice(["hnd", "nhd"]), rng.choice([16, 32, 48, 64, 128, 256])
        if op == "append":
            rows, length = _log(rng, 1, 2000), _log(rng, 2000, 30000)
            if seqs * rows * (kv * (group + 2)) * dim > 60_000_000 or seqs * length * kv * dim > 200_000_000:
                continue
            return dict(op=op, seqs=seqs, rows=rows, len=length, ragged=rng.randint(0, 1), q_heads=kv * group, kv_heads=kv, dim=dim, page=page, layout=layout,
                        pairs=pairs, rot=rot, scaled=scaled, act="f32", cache=cache, q_out=act)
        rows = 1 if rng.random() < 0.5 else _log(rng, 2, 4000)
        length = max(rows, _log(rng, 1, 100000))
        if dim == 256 and rows * group > 64:      # wide heads are drawn for decoding and checking
            continue
        case = dict(op=op, seqs=seqs, rows=rows, len=length, q_heads=kv * group, kv_heads=kv, dim=dim, page=page, act=act, cache=cache, layout=layout,
                    ragged=rng.randint(0, 2) if rows > 1 else rng.randint(0, 1), window=rng.choice([0, 0, 0, 128, 1000]))
        if seqs * length * kv * dim > 250_000_000 or seqs * rows * length * kv * group > 1_000_000_000 or work(case)["flops"] > 2.5e11:
            continue
        return case


def lengths(case):
    """New rows and cache lengths of the sequences.  ragged = 0: all alike; 1: spread between a small part and the whole;
    2: the same, but every second sequence has one new row."""
    n, rows, length = case["seqs"], case["rows"], case["len"]
    part = [1.0 if not case["ragged"] or i == 0 else 0.02 + 0.98 * ((i * 0.6180339887) % 1.0) for i in range(n)]
    new = [max(1, int(rows * p)) for p in part]
    if case["ragged"] == 2:
        new = [1 if i % 2 else r for i, r in enumerate(new)]
    return new, [max(r, int(length * p)) for r, p in zip(new, part)]


def visible(case):
    """(pairs of row and key that attention has to look at, keys that some row sees)."""
    pairs = keys = 0
    w = case["window"]
    for n, length in zip(*lengths(case)):
        first = length - n + 1                                    # keys that the first new row sees, without a window
        if w and length > w:
            short = max(0, min(n, w - first))                     # rows that see fewer than w keys
            pairs += short * first + short * (short - 1) // 2 + (n - short) * w
            keys += min(length, n - 1 + w)
        else:
            pairs += n * first + n * (n - 1) // 2
            keys += length
    return pairs, keys


def work(case):
    size = {k: DT[case[k]].itemsize for k in ("act", "out", "cache", "q_out") if k in case}
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": n * (size["act"] + size["out"]) + 4 * case["tokens"], "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    total = sum(lengths(case)[0])
    q, kv = total * case["q_heads"] * case["dim"], total * case["kv_heads"] * case["dim"]
    if case["op"] == "append":
        return {"bytes": (q + 2 * kv) * size["act"] + q * size["q_out"] + 2 * kv * size["cache"], "flops": 3 * total * (case["q_heads"] + case["kv_heads"]) * case["rot"]}
    pairs, keys = visible(case)
    return {"bytes": 2 * q * size["act"] + 2 * keys * case["kv_heads"] * case["dim"] * size["cache"], "flops": 4 * pairs * case["q_heads"] * case["dim"]}


def frequencies(case):
    """Radians per position of each pair, in 64 bits: base^(-2i/rot); scaled: divided by 8 where a pair turns less than once
    within 4096 positions, kept where it turns more than 32 times, mixed between; and the magnitude of rotated values."""
    f = 10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])
    if not case["scaled"]:
        return f, 1.0
    keep = ((4096 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
    return f * keep + f / 8 * (1 - keep), 0.1 * math.log(8.0) + 1.0


# ---------------------------------------------------------------------------------------------------------------- state
def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32 if dtype == torch.float32 else torch.float16).to(dtype)

    s = dict(case)
    if case["op"] != "attention":
        freq, s["mag"] = frequencies(case)
        s["freq"] = freq.cuda()
    if case["op"] == "rope":
        s["x"] = randn(case["tokens"], case["fused"], case["dim"], dtype=DT[case["act"]])          # the rotated heads lead each fused row
        s["pos"] = torch.randint(0, case["far"], (case["tokens"],), generator=g, device="cuda", dtype=torch.int32)
        s["y"] = torch.empty(case["tokens"], case["heads"], case["dim"], device="cuda", dtype=DT[case["out"]])
    else:
        new, length = lengths(case)
        page, hk, d = case["page"], case["kv_heads"], case["dim"]
        per = (max(length) + page - 1) // page                    # entries of a sequence's row in the page table
        used = [(n + page - 1) // page for n in length]
        pages = sum(used) + 3
        order = torch.randperm(pages, generator=g, device="cuda")[: sum(used)].to(torch.int32)
        row = torch.repeat_interleave(torch.arange(len(used)), torch.tensor(used))
        at = torch.arange(sum(used)) - torch.repeat_interleave(torch.tensor(used).cumsum(0) - torch.tensor(used), torch.tensor(used))
        s["table"] = torch.full((len(used), per), -1, device="cuda", dtype=torch.int32)
        s["table"][row.cuda(), at.cuda()] = order
        s["cu"] = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
        s["len_"] = torch.tensor(length, dtype=torch.int32).cuda()
        s["max_rows"], s["max_len"], s["tokens"] = max(new), max(length), sum(new)
        shape = (pages, hk, page, d) if case["layout"] == "hnd" else (pages, page, hk, d)
        s["k_cache"], s["v_cache"] = randn(*shape, dtype=DT[case["cache"]]), randn(*shape, dtype=DT[case["cache"]])
        if case["op"] == "append":
            s["qkv"] = randn(s["tokens"], case["q_heads"] + 2 * hk, d, dtype=DT[case["act"]])
            s["q_to"] = torch.empty(s["tokens"], case["q_heads"], d, device="cuda", dtype=DT[case["q_out"]])
        else:
            s["q"] = randn(s["tokens"], case["q_heads"], d, dtype=DT[case["act"]]) * 1.5
            s["out"] = torch.empty(s["tokens"], case["q_heads"], d, device="cuda", dtype=DT[case["act"]])
    if own:
        _handles(case, s)
    return s


_gpu = None


def _handles(case, s):
    """The library's context (one per process, on torch's stream), and what a program keeps per layer: rotation, cache, batch."""
    global _gpu
    import ojas_engine_b200 as ob
    if _gpu is None:
        _gpu = ob.B200Gpu(torch.cuda.current_device(), stream=torch.cuda.current_stream().cuda_stream or 1)   # 1: the legacy default stream
    s["gpu"] = _gpu

    def buf(t):
        return ob.Buf(t.data_ptr(), t.numel() * t.element_size())

    if case["op"] != "attention":
        more = dict(factor=8.0, orig_len=4096, beta_fast=32.0, beta_slow=1.0, magnitude=s["mag"]) if case["scaled"] else {}
        s["rope"] = ob.Rope(_gpu, case["rot"], base=10000.0, **more)
        s["pairs_"] = ob.ROPE_HALF if case["pairs"] == "half" else ob.ROPE_INTERLEAVED
    if case["op"] == "rope":
        s["x_"], s["pos_"], s["y_"] = buf(s["x"]), buf(s["pos"]), buf(s["y"])
        return
    page, hk, d = case["page"], case["kv_heads"], case["dim"]
    stride = dict(page_stride=page * hk * d, head_stride=page * d, token_stride=d) if case["layout"] == "hnd" else dict(page_stride=page * hk * d, head_stride=d, token_stride=hk * d)
    s["kv"] = ob.KvCache(_gpu, CODE[case["cache"]], buf(s["k_cache"]), buf(s["v_cache"]), s["k_cache"].shape[0], page, hk, d, **stride)
    s["seqs_"] = ob.Seqs(buf(s["cu"]), buf(s["len_"]), buf(s["table"]), case["seqs"], s["table"].shape[1], s["max_rows"], s["max_len"])
    if case["op"] == "append":
        b = buf(s["qkv"])
        w = d * s["qkv"].element_size()
        s["q_"], s["k_"], s["v_"] = (ob.Buf(b.ptr + w * n, b.nbytes - w * n) for n in (0, case["q_heads"], case["q_heads"] + hk))
        s["q_to_"] = buf(s["q_to"])
    else:
        s["q_"], s["out_"] = buf(s["q"]), buf(s["out"])


# ----------------------------------------------------------------------------------------------------------- plain form
def rotated(x, pos, s):
    """x [tokens, heads, dim] in 32 bits, rotated; angles in 64 bits."""
    rot = s["rot"]
    angle = pos.double()[:, None, None] * s["freq"]
    cos, sin = angle.cos().float() * s["mag"], angle.sin().float() * s["mag"]
    if s["pairs"] == "half":
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def places(s):
    """Sequence and position of each new row."""
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n, output_size=s["tokens"])
    return seq, torch.arange(s["tokens"], device="cuda") - s["cu"].long()[seq] + (s["len_"].long() - n)[seq]


def run(s):
    if own:
        return _run_own(s)
    d = s["dim"]
    if s["op"] == "rope":
        s["y"].copy_(rotated(s["x"][:, : s["heads"]].float(), s["pos"], s))
        return s["y"]
    seq, pos = places(s)
    if s["op"] == "append":
        hq, hk = s["q_heads"], s["kv_heads"]
        page, slot = s["table"].long()[seq, pos // s["page"]], pos % s["page"]
        x = s["qkv"].float()
        turned = rotated(x[:, : hq + hk], pos, s)
        for cache, rows in ((s["k_cache"], turned[:, hq:]), (s["v_cache"], x[:, hq + hk :])):
            view = cache.transpose(1, 2) if s["layout"] == "hnd" else cache
            view[page, slot] = rows.to(cache.dtype)
        s["q_to"].copy_(turned[:, :hq])
        return s["q_to"], s["k_cache"], s["v_cache"]
    # attention: the batch padded to its longest sequence
    n_seqs, hk, hq = s["seqs"], s["kv_heads"], s["q_heads"]
    at = torch.arange(s["tokens"], device="cuda") - s["cu"].long()[seq]
    q = torch.zeros(n_seqs, s["max_rows"], hk, hq // hk, d, device="cuda")
    q[seq, at] = s["q"].float().view(s["tokens"], hk, hq // hk, d)
    where = torch.zeros(n_seqs, s["max_rows"], device="cuda", dtype=torch.long)
    where[seq, at] = pos

    def gather(cache):                                            # [sequence, head, key, dim]
        x = cache[s["table"].clamp(min=0).long()]
        x = x.transpose(2, 3) if s["layout"] == "hnd" else x
        return x.flatten(1, 2)[:, : s["max_len"]].float().transpose(1, 2)

    key = torch.arange(s["max_len"], device="cuda")
    seen = (key <= where[..., None]) & (key < s["len_"][:, None, None])
    if s["window"]:
        seen &= key > where[..., None] - s["window"]
    k, v = gather(s["k_cache"]), gather(s["v_cache"])
    v = v * (key < s["len_"][:, None])[:, None, :, None]
    scores = torch.matmul(q.permute(0, 2, 3, 1, 4).flatten(2, 3), k.transpose(2, 3)).unflatten(2, (hq // hk, s["max_rows"])) / math.sqrt(d)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (hq // hk, s["max_rows"])) / total.clamp(min=1e-38)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4)[seq, at].flatten(1, 2))
    return s["out"]


def _run_own(s):
    gpu, c = s["gpu"], CODE
    if s["op"] == "rope":
        gpu.rope_rows(s["rope"], s["x_"], s["y_"], s["pos_"], s["tokens"], s["heads"], s["dim"], layout=s["pairs_"], x_type=c[s["act"]], y_type=c[s["out"]],
                      x_stride=s["fused"] * s["dim"])
        return s["y"]
    if s["op"] == "append":
        stride = (s["q_heads"] + 2 * s["kv_heads"]) * s["dim"]
        gpu.kv_append(s["kv"], s["seqs_"], s["k_"], s["v_"], s["tokens"], rope=s["rope"], layout=s["pairs_"], x_type=c[s["act"]], x_stride=stride,
                      q=s["q_"], q_out=s["q_to_"], q_heads=s["q_heads"], q_type=c[s["q_out"]])
        return s["q_to"], s["k_cache"], s["v_cache"]
    gpu.attention(s["kv"], s["seqs_"], s["q_"], s["out_"], s["tokens"], s["q_heads"], act_type=c[s["act"]], window=s["window"])
    return s["out"]


# ------------------------------------------------------------------------------------------------- definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)

    def turn(x, pos):                                             # [tokens, heads, dim]: each pair as a complex number
        rot = case["rot"]
        head = x.double()[..., :rot]
        z = torch.complex(head[..., : rot // 2], head[..., rot // 2 :]) if case["pairs"] == "half" else torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous())
        z = z * torch.polar(torch.full_like(s["freq"], s["mag"]), s["freq"] * pos.double()[:, None])[:, None]
        head = torch.cat([z.real, z.imag], -1) if case["pairs"] == "half" else torch.view_as_real(z).flatten(-2)
        return torch.cat([head, x.double()[..., rot:]], -1)

    if case["op"] == "rope":
        return turn(s["x"][:, : case["heads"]], s["pos"])
    new, length = lengths(case)
    hk, hq, d, page = case["kv_heads"], case["q_heads"], case["dim"], case["page"]
    hnd = case["layout"] == "hnd"
    if case["op"] == "append":
        q_to, kc, vc, t0 = [], s["k_cache"].double(), s["v_cache"].double(), 0
        for b, (n, total) in enumerate(zip(new, length)):
            x = s["qkv"][t0 : t0 + n]
            pos = torch.arange(total - n, total, device="cuda")
            q_to.append(turn(x[:, :hq], pos))
            to = s["table"][b].long()[pos // page] * page + pos % page
            for cache, rows in ((kc, turn(x[:, hq : hq + hk], pos)), (vc, x[:, hq + hk :].double())):
                if hnd:
                    cache[to // page, :, to % page] = rows
                else:
                    cache.view(-1, hk, d)[to] = rows
            t0 += n
        return torch.cat(q_to), kc, vc
    out, t0, w = torch.zeros(s["tokens"], hq, d, device="cuda", dtype=torch.float64), 0, case["window"]
    for b, (n, total) in enumerate(zip(new, length)):
        ids = s["table"][b, : (total + page - 1) // page].long()
        pos, key = torch.arange(total - n, total, device="cuda")[:, None], torch.arange(total, device="cuda")
        hidden = (key > pos) | (key <= pos - w) if w else key > pos
        for h in range(hk):
            k, v = ((c[ids, h] if hnd else c[ids, :, h]).reshape(-1, d)[:total].double() for c in (s["k_cache"], s["v_cache"]))
            for i in range(h * (hq // hk), (h + 1) * (hq // hk)):
                z = (s["q"][t0 : t0 + n, i].double() @ k.T * d ** -0.5).masked_fill(hidden, -math.inf)
                out[t0 : t0 + n, i] = torch.softmax(z, -1) @ v
        t0 += n
    return out
