"""What the decoder-block operators are measured on.

Four operators that sit between the quantized linears of a served decoder:

* ``norm``: residual addition + RMSNorm, 8-bit codes with one scale per row;
* ``rope``: rotary positions with several axes, alone or with the rotated k
  and v written into a paged key-value cache;
* ``packed``: attention over whole prompts, packed sequences, grouped heads;
* ``paged``: attention of one new token per sequence over the paged cache.

``run`` computes them in plain torch operations in 32 bits, or, with ``own``
set, through ``qi_b200.kernels``.
"""

import math

import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # a decode step's norm of one token, in front of an FP8 linear
        {"name": "norm one token fp8", "op": "norm", "rows": 1, "dim": 4096, "fmt": "fp8", "residual": True},
        # a short prompt at the action expert's width, in front of an INT8 linear
        {"name": "norm action rows int8", "op": "norm", "rows": 777, "dim": 1024, "fmt": "int8", "residual": True},
        # the norm of a whole batch of prompts
        {"name": "norm prompt fp8", "op": "norm", "rows": 16384, "dim": 8192, "fmt": "fp8", "residual": True},
        # one decode step of 64 sequences: rotate q, write k and v to the cache
        {"name": "rope decode store bf16", "op": "rope", "rows": 64, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "sections": "64", "shared": True, "interleaved": False, "cache": "bf16", "page": 16},
        # the DiT's video tokens: (frame, height, width) axes, even/odd pairs
        {"name": "rope video 3 axes", "op": "rope", "rows": 3120, "heads": 24, "kv_heads": 24, "head_dim": 128,
         "sections": "22,21,21", "shared": False, "interleaved": True, "cache": "none", "page": 0},
        # a long prompt of text and images written to an 8-bit cache
        {"name": "rope prompt store fp8", "op": "rope", "rows": 16384, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "sections": "16,24,24", "shared": True, "interleaved": False, "cache": "fp8", "page": 64},
        # a batch of short prompts of very different lengths
        {"name": "packed ragged prompts", "op": "packed", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "q_lens": "1,17,600,128,33,257,5,411,64,129,300,2,95,511,256,31", "k_lens": "", "causal": True},
        # new chunks of prompts over keys that are there already
        {"name": "packed chunks after prefix", "op": "packed", "heads": 16, "kv_heads": 2, "head_dim": 64,
         "q_lens": "512,512,300,1000", "k_lens": "4608,8192,300,2777", "causal": True},
        # one long prompt, the repository's 24 heads of 128 over 8 key heads
        {"name": "packed long prompt", "op": "packed", "heads": 24, "kv_heads": 8, "head_dim": 128,
         "q_lens": "16384", "k_lens": "", "causal": True},
        # one sequence, short context: latency
        {"name": "paged one sequence", "op": "paged", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16,
         "cache": "bf16", "lens": "1000"},
        # a batch of 64 sequences of mixed lengths
        {"name": "paged ragged batch bf16", "op": "paged", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16,
         "cache": "bf16", "lens": ",".join(str(1 + (i * 2654435761 >> 7) % 8192) for i in range(64))},
        # long contexts in an 8-bit cache
        {"name": "paged long fp8", "op": "paged", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "cache": "fp8", "lens": "65536,50001,32768,65535,777,60000,44444,16384"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _lens(text):
    return [int(t) for t in text.split(",")] if text else []


def draw(rng):
    op = rng.choice(("norm", "rope", "packed", "paged"))
    if op == "norm":
        return {"op": op, "rows": _log_int(rng, 1, 16384), "dim": 8 * _log_int(rng, 64, 1024),
                "fmt": rng.choice(("fp8", "int8")), "residual": rng.random() < 0.75}
    group, kv_heads = rng.choice((1, 2, 3, 4, 6, 8)), rng.choice((1, 2, 4, 8))
    if op == "rope":
        half = rng.choice((32, 64))
        a = rng.randint(1, half - 2)
        b = rng.randint(1, half - a - 1)
        sections = rng.choice((str(half), "%d,%d,%d" % (a, b, half - a - b)))
        return {"op": op, "rows": _log_int(rng, 1, 16384), "heads": min(32, group * kv_heads) // kv_heads * kv_heads,
                "kv_heads": kv_heads, "head_dim": 2 * half, "sections": sections, "shared": rng.random() < 0.5,
                "interleaved": rng.random() < 0.5, "cache": rng.choice(("none", "bf16", "fp8")),
                "page": rng.choice((16, 32, 64))}
    head_dim = rng.choice((64, 128))
    if op == "packed":
        group = rng.choice((1, 2, 3, 4))
        n = _log_int(rng, 1, 24)
        most = _log_int(rng, 16, 4096 // n)
        q = [rng.randint(1, most) for _ in range(n)]
        prefix = rng.random() < 0.4
        k = [v + rng.randint(0, 2 * most) for v in q] if prefix else []
        return {"op": op, "heads": group * kv_heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "q_lens": ",".join(map(str, q)), "k_lens": ",".join(map(str, k)), "causal": rng.random() < 0.8}
    n = _log_int(rng, 1, 64)
    most = _log_int(rng, 16, 160000 // n)
    return {"op": op, "heads": group * kv_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": rng.choice((16, 32, 64)), "cache": rng.choice(("bf16", "fp8")),
            "lens": ",".join(str(rng.randint(max(1, most // 8), most)) for _ in range(n))}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


class State:
    """What a user's program holds before the call."""

    def __init__(self, **kw):
        self.__dict__.update(kw)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _cu(lens):
    return torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)


def _frequencies(case):
    """Per pair: the angle of one step of its axis (radians, 64 bits) and the axis."""
    sections = _lens(case["sections"])
    total = sum(sections)
    freq, axis = [], []
    for a, n in enumerate(sections):
        for i in range(n):
            step = len(freq) / total if case["shared"] else i / n
            freq.append(10000.0 ** -step)
            axis.append(a)
    return freq, axis


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    bf16 = torch.bfloat16
    if op == "norm":
        rows, dim = case["rows"], case["dim"]
        channels = 1 + 4 * (torch.rand(dim, generator=g, device=DEV) < 0.01)  # a few channels run hot
        x = (_randn(g, rows, dim) * channels).to(bf16)
        y = (_randn(g, rows, dim) * 0.5).to(bf16) if case["residual"] else None
        weight = (1 + 0.1 * _randn(g, dim)).to(bf16)
        return State(case=case, x=x, y=y, weight=weight, x_out=torch.empty_like(x) if case["residual"] else None)
    hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if op == "rope":
        rows = case["rows"]
        qkv = _randn(g, rows, (hq + 2 * hk) * d).to(bf16)  # what the fused q/k/v linear writes
        axes = len(_lens(case["sections"]))
        if axes == 1:
            start = int(torch.randint(0, 100000, (1,), generator=g, device=DEV))
            positions = torch.arange(start, start + rows, device=DEV, dtype=torch.int32)[None]
        else:  # frames of 12 x 10 patches
            t = torch.arange(rows, device=DEV, dtype=torch.int32) + int(torch.randint(0, 5000, (1,), generator=g, device=DEV))
            positions = torch.stack([t // 120, t % 120 // 10, t % 10])[:axes]
        freq, axis = _frequencies(case)
        s = State(case=case, q=qkv[:, :hq * d], k=qkv[:, hq * d:(hq + hk) * d], v=qkv[:, (hq + hk) * d:],
                  positions=positions.contiguous(), freq=torch.tensor(freq, dtype=torch.float64, device=DEV),
                  axis=torch.tensor(axis, dtype=torch.int32, device=DEV), slots=None, k_scale=None, v_scale=None)
        if case["cache"] != "none":
            page = case["page"]
            pages = -(-rows // page) + 3
            s.slots = torch.randperm(pages * page, generator=g, device=DEV)[:rows]
            kind = bf16 if case["cache"] == "bf16" else torch.uint8
            s.k_cache = torch.zeros(pages, page, hk, d, dtype=kind, device=DEV)
            s.v_cache = torch.zeros(pages, page, hk, d, dtype=kind, device=DEV)
            if case["cache"] == "fp8":
                s.k_scale = 0.02 + 0.01 * torch.rand(hk, generator=g, device=DEV)
                s.v_scale = 0.02 + 0.01 * torch.rand(hk, generator=g, device=DEV)
        return s
    if op == "packed":
        ql = _lens(case["q_lens"])
        kl = _lens(case["k_lens"]) or ql
        if case["k_lens"]:
            q = _randn(g, sum(ql), hq * d).to(bf16)
            kv = _randn(g, sum(kl), 2 * hk * d).to(bf16)
            k, v = kv[:, :hk * d], kv[:, hk * d:]
        else:
            qkv = _randn(g, sum(ql), (hq + 2 * hk) * d).to(bf16)
            q, k, v = qkv[:, :hq * d], qkv[:, hq * d:(hq + hk) * d], qkv[:, (hq + hk) * d:]
        row = torch.cat([b * max(ql) + torch.arange(n) for b, n in enumerate(ql)]).to(DEV)
        return State(case=case, q=q, k=k, v=v, cu_q=_cu(ql), cu_k=_cu(kl), q_len=torch.tensor(ql, device=DEV),
                     k_len=torch.tensor(kl, device=DEV), longest=(max(ql), max(kl)), row=row)
    lens, page = _lens(case["lens"]), case["page"]
    need = [-(-n // page) for n in lens]
    total = sum(need) + 5
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    q = _randn(g, len(lens), hq * d).to(bf16)
    cache = [_randn(g, total, page, hk, d) for _ in range(2)]
    k_scale = v_scale = None
    if case["cache"] == "fp8":
        k_scale, v_scale = (0.02 + 0.01 * torch.rand(hk, generator=g, device=DEV) for _ in range(2))
        cache = [(c / s[:, None]).to(torch.float8_e4m3fn).view(torch.uint8) for c, s in zip(cache, (k_scale, v_scale))]
    else:
        cache = [c.to(bf16) for c in cache]
    return State(case=case, q=q, k_cache=cache[0], v_cache=cache[1], pages=table,
                 lens=torch.tensor(lens, dtype=torch.int32, device=DEV), longest=max(lens), k_scale=k_scale,
                 v_scale=v_scale)


# ---------------------------------------------------------------------------
# the operators, plainly, in 32 bits
# ---------------------------------------------------------------------------


def _to_e4m3(v):
    return v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _plain_norm(s):
    if s.y is None:
        h = s.x
    else:
        h = (s.x.float() + s.y.float()).to(torch.bfloat16)
        s.x_out.copy_(h)
    f = h.float()
    v = f * torch.rsqrt((f * f).mean(1, keepdim=True) + 1e-6) * s.weight.float()
    amax = v.abs().amax(1)
    if s.case["fmt"] == "fp8":
        scale = (amax / 448.0).clamp_min(1e-12)
        return _to_e4m3(v / scale[:, None]), scale, s.x_out
    scale = (amax / 127.0).clamp_min(1e-10)
    return (v / scale[:, None]).round().clamp(-127, 127).to(torch.bfloat16), scale, s.x_out


def _rotate(x, heads, cos, sin, interleaved):
    rows = x.shape[0]
    x = x.float().view(rows, heads, -1)
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
    else:
        a, b = x.chunk(2, -1)
    ra, rb = a * cos - b * sin, a * sin + b * cos
    out = torch.stack([ra, rb], -1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    return out.view(rows, -1)


def _plain_rope(s):
    c = s.case
    angle = s.positions.double()[s.axis.long()].t() * s.freq  # far positions: 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _rotate(s.q, c["heads"], cos, sin, c["interleaved"]).to(torch.bfloat16)
    k = _rotate(s.k, c["kv_heads"], cos, sin, c["interleaved"])
    if c["cache"] == "none":
        return q, k.to(torch.bfloat16)
    shape = (-1, c["kv_heads"], c["head_dim"])
    k, v = k.view(shape), s.v.float().view(shape)
    kc, vc = s.k_cache.view(shape), s.v_cache.view(shape)
    if c["cache"] == "bf16":
        kc[s.slots], vc[s.slots] = k.to(torch.bfloat16), v.to(torch.bfloat16)
        return q, s.k_cache, s.v_cache
    kc[s.slots] = _to_e4m3(k / s.k_scale[:, None]).view(torch.uint8)
    vc[s.slots] = _to_e4m3(v / s.v_scale[:, None]).view(torch.uint8)
    return q, s.k_cache.view(torch.float8_e4m3fn), s.v_cache.view(torch.float8_e4m3fn)


def _softmax_(scores, visible):
    """Softmax over the last axis of the visible scores; a row without any gives zeros."""
    scores.masked_fill_(~visible, -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    return scores.div_(scores.sum(-1, keepdim=True).clamp_min(1e-30))


def _plain_packed(s):
    c = s.case
    hk, d = c["kv_heads"], c["head_dim"]
    n, (lq, lk) = s.q_len.numel(), s.longest
    at_q = (s.cu_q[:-1, None] + torch.arange(lq, device=DEV)).clamp_max(s.q.shape[0] - 1)
    at_k = (s.cu_k[:-1, None] + torch.arange(lk, device=DEV)).clamp_max(s.k.shape[0] - 1)
    q = s.q[at_q].float().view(n, lq, hk, -1, d).permute(0, 2, 3, 1, 4)          # [n, hk, group, lq, d]
    k = s.k[at_k].float().view(n, lk, hk, 1, d).permute(0, 2, 3, 4, 1)           # [n, hk, 1, d, lk]
    v = s.v[at_k].float().view(n, lk, hk, 1, d).permute(0, 2, 3, 1, 4)           # [n, hk, 1, lk, d]
    i, j = torch.arange(lq, device=DEV)[:, None], torch.arange(lk, device=DEV)
    visible = (j < s.k_len[:, None, None]).expand(n, lq, lk)
    if c["causal"]:
        visible = visible & (j <= i + (s.k_len - s.q_len)[:, None, None])
    p = _softmax_((q * d ** -0.5) @ k, visible[:, None, None])
    o = (p @ v).permute(0, 3, 1, 2, 4).reshape(n * lq, -1)
    return o[s.row].to(torch.bfloat16)


def _plain_paged(s):
    c = s.case
    hk, d = c["kv_heads"], c["head_dim"]
    n = s.lens.numel()
    k, v = s.k_cache[s.pages.long()], s.v_cache[s.pages.long()]                   # [n, pages, page, hk, d]
    if c["cache"] == "fp8":
        k = k.view(torch.float8_e4m3fn).float() * s.k_scale[:, None]
        v = v.view(torch.float8_e4m3fn).float() * s.v_scale[:, None]
    k = k.float().view(n, -1, hk, d).permute(0, 2, 3, 1)
    v = v.float().view(n, -1, hk, d).permute(0, 2, 1, 3)
    q = s.q.float().view(n, hk, -1, d)
    visible = torch.arange(k.shape[-1], device=DEV) < s.lens[:, None]
    p = _softmax_((q * d ** -0.5) @ k, visible[:, None, None])
    return (p @ v).reshape(n, -1).to(torch.bfloat16)


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------


def _own(s):
    from qi_b200 import _lib, kernels

    c = s.case
    if c["op"] == "norm":
        kind = _lib.KIND_FP8_E4M3 if c["fmt"] == "fp8" else _lib.KIND_INT8
        codes, scale = kernels.rms_norm_quant(kind, s.x, s.weight, s.y, eps=1e-6, x_out=s.x_out)
        codes = codes.view(torch.float8_e4m3fn) if c["fmt"] == "fp8" else codes.to(torch.bfloat16)
        return codes, scale, s.x_out
    if c["op"] == "rope":
        if c["cache"] == "none":
            return kernels.rope_axes(s.q, s.k, s.positions, s.freq, s.axis, c["head_dim"],
                                     interleaved=c["interleaved"])
        q = kernels.rope_axes_store(s.q, s.k, s.v, s.positions, s.freq, s.axis, c["head_dim"], s.k_cache,
                                    s.v_cache, s.slots, interleaved=c["interleaved"], k_scale=s.k_scale, v_scale=s.v_scale)
        if c["cache"] == "bf16":
            return q, s.k_cache, s.v_cache
        return q, s.k_cache.view(torch.float8_e4m3fn), s.v_cache.view(torch.float8_e4m3fn)
    if c["op"] == "packed":
        return kernels.attention_packed(s.q, s.k, s.v, s.cu_q, s.cu_k, c["heads"], c["kv_heads"], causal=c["causal"])
    return kernels.attention_paged(s.q, s.k_cache, s.v_cache, s.pages, s.lens, k_scale=s.k_scale, v_scale=s.v_scale)


_PLAIN = {"norm": _plain_norm, "rope": _plain_rope, "packed": _plain_packed, "paged": _plain_paged}


def run(state):
    return _own(state) if own else _PLAIN[state.case["op"]](state)


# ---------------------------------------------------------------------------
# the least work, and the results in 64 bits
# ---------------------------------------------------------------------------


def _visible_pairs(case):
    ql = _lens(case["q_lens"])
    kl = _lens(case["k_lens"]) or ql
    if not case["causal"]:
        return sum(a * b for a, b in zip(ql, kl))
    pairs = 0
    for a, b in zip(ql, kl):
        last, first = b, b - a + 1  # keys that the last and the first query see
        skip = max(0, 1 - first)    # queries in front of every key
        pairs += (a - skip) * (last + max(1, first)) // 2
    return pairs


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["dim"]
        return {"bytes": n * (7 if case["residual"] else 3) + 4 * case["rows"] + 2 * case["dim"], "flops": 6 * n}
    hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    size = 1 if case.get("cache") == "fp8" else 2
    if case["op"] == "rope":
        per = 4 * hq * d + (4 * hk * d if case["cache"] == "none" else 2 * hk * d * (2 + size) + 8)
        return {"bytes": case["rows"] * (per + 4 * len(_lens(case["sections"]))), "flops": case["rows"] * (hq + hk) * d * 3}
    if case["op"] == "packed":
        ql = _lens(case["q_lens"])
        kl = _lens(case["k_lens"]) or ql
        return {"bytes": 4 * sum(ql) * hq * d + 4 * sum(kl) * hk * d, "flops": 4 * d * hq * _visible_pairs(case)}
    lens = _lens(case["lens"])
    pages = sum(-(-n // case["page"]) for n in lens)
    return {"bytes": 2 * sum(lens) * hk * d * size + 4 * len(lens) * hq * d + 4 * pages, "flops": 4 * d * hq * sum(lens)}


def _e4m3_64(v):
    """The nearest E4M3 value, ties to even, in 64 bits."""
    v = v.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def _exact_norm(s):
    h = s.x.double()
    if s.y is not None:
        h = (h + s.y.double()).to(torch.bfloat16).double()
    v = s.weight.double() * h / torch.sqrt(h.square().sum(1, keepdim=True) / h.shape[1] + 1e-6)
    top = v.abs().max(1).values
    stored = None if s.y is None else h
    if s.case["fmt"] == "fp8":
        scale = torch.clamp(top / 448, min=1e-12)
        return _e4m3_64(v / scale[:, None]), scale, stored
    scale = torch.clamp(top / 127, min=1e-10)
    return torch.round(v / scale[:, None]), scale, stored


def _exact_rope(s):
    c = s.case
    d, half = c["head_dim"], c["head_dim"] // 2
    turn = torch.stack([s.positions[int(a)].double() * f for f, a in zip(s.freq, s.axis)], 1)
    spin = torch.polar(torch.ones_like(turn), turn)

    def rotated(x, heads):
        x = x.double().reshape(x.shape[0], heads, d)
        pairs = x.reshape(x.shape[0], heads, half, 2) if c["interleaved"] else x.reshape(x.shape[0], heads, 2, half).transpose(2, 3)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * spin[:, None])
        return (z if c["interleaved"] else z.transpose(2, 3)).reshape(x.shape[0], heads, d)

    q, k = rotated(s.q, c["heads"]).flatten(1), rotated(s.k, c["kv_heads"])
    if c["cache"] == "none":
        return q, k.flatten(1)
    out = []
    for x, scale, cache in ((k, s.k_scale, s.k_cache), (s.v.double().reshape(k.shape), s.v_scale, s.v_cache)):
        if c["cache"] == "fp8":
            x = _e4m3_64(x / scale.double()[:, None])
        whole = torch.zeros(cache.shape, dtype=torch.float64, device=DEV)
        whole.view(-1, *x.shape[1:]).index_copy_(0, s.slots, x)
        out.append(whole)
    return q, out[0], out[1]


def _attend_64(q, k, v, first):
    """q [a, d], k, v [b, d]: query i sees the keys up to first + i (all, where first is None)."""
    scores = q @ k.t() / math.sqrt(q.shape[1])
    if first is not None:
        i = torch.arange(q.shape[0], device=DEV)[:, None]
        scores = torch.where(torch.arange(k.shape[0], device=DEV) > first + i, -math.inf, scores)
    p = torch.softmax(scores, 1)
    return torch.nan_to_num(p) @ v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    if case["op"] == "rope":
        return _exact_rope(s)
    hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEV)
    if case["op"] == "packed":
        cq, ck = s.cu_q.tolist(), s.cu_k.tolist()
        for b in range(len(cq) - 1):
            rows, keys = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
            first = (ck[b + 1] - ck[b]) - (cq[b + 1] - cq[b]) if case["causal"] else None
            for h in range(hq):
                g = h * hk // hq
                out[rows, h * d:(h + 1) * d] = _attend_64(s.q[rows, h * d:(h + 1) * d].double(),
                                                          s.k[keys, g * d:(g + 1) * d].double(),
                                                          s.v[keys, g * d:(g + 1) * d].double(), first)
        return out
    for b, n in enumerate(_lens(case["lens"])):
        at = torch.arange(n, device=DEV)
        page, off = s.pages[b, at // case["page"]].long(), at % case["page"]
        k, v = s.k_cache[page, off], s.v_cache[page, off]                        # [n, hk, d]
        if case["cache"] == "fp8":
            k = k.view(torch.float8_e4m3fn).double() * s.k_scale.double()[:, None]
            v = v.view(torch.float8_e4m3fn).double() * s.v_scale.double()[:, None]
        for g in range(hk):
            heads = slice(g * (hq // hk) * d, (g + 1) * (hq // hk) * d)
            out[b, heads] = _attend_64(s.q[b, heads].double().view(-1, d), k[:, g].double(), v[:, g].double(), None).flatten()
    return out
