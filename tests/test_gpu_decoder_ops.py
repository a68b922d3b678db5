"""GPU: the decoder-block operators against plain 64-bit implementations.

Tolerances, from the roundings each kernel makes (half a step relative to the
value: bf16 2^-8, fp16 2^-11, E4M3 2^-4 of a normal value):

* ``rms_norm_quant``: v / s carries fp32 errors only.  The sum of squares adds
  at most 64 terms in a row per thread and 10 levels of a tree, so its relative
  error is below 74 * 2^-24; square root, two divisions and three products add
  a few 2^-24 more: 2^-17 in all covers it.  A code is then at most half a
  step plus 2^-17 |v / s| away from the exact v / s.
* ``rope_axes``: the turn is reduced in 64 bits, cos and sin are off by less
  than 2^-21 in all, so a rotated element by (|x| + |y|) 2^-20 plus the
  rounding of the output's type.
* attention: probabilities round once (bf16 2^-8, fp16 2^-11 in an E4M3
  cache), the output once (2^-8).  With A = sum_j p_j |v_j| the result is off
  by at most r_p A + 2^-8 |o|, plus the scores' fp32 errors: (D + 16) 2^-24
  times the largest scale * sum |q| |k|, twice (numerator and sum), times A.
  Second-order terms are below 1 % of that.
"""

import math

import pytest
import torch

from qi_b200 import _lib, kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    _lib.load()
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()
    st = _lib.device_status(clear=True)
    assert st[0] == 0, f"device status word: {st}"


def gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def randn(g, *shape, mul=1.0):
    return (torch.randn(*shape, generator=g) * mul).to(BF).to(DEV)


def e4m3_value(codes):
    return codes.view(torch.float8_e4m3fn).double()


def e4m3_half_step(v):
    """Half the distance of E4M3 values around |v| (64 bits)."""
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 4)


# ---------------------------------------------------------------------------
# rms_norm_quant
# ---------------------------------------------------------------------------


def check_norm(kind, x, w, y, eps, q, s, h, xn=None):
    hd = h.double()
    v = hd * w.double() / torch.sqrt(hd.square().mean(1, keepdim=True) + eps)
    if xn is not None:
        assert ((xn.double() - v).abs() <= v.abs() * (2.0 ** -8 + 2.0 ** -17)).all()
    if kind == _lib.KIND_BF16:
        return
    top = 127.0 if kind == _lib.KIND_INT8 else 448.0
    want = (v.abs().amax(1) / top).clamp_min(1e-10 if kind == _lib.KIND_INT8 else 1e-12)
    assert ((s.double() - want).abs() <= want * 2.0 ** -17).all()
    t = v / want[:, None]
    got = q.double() if kind == _lib.KIND_INT8 else e4m3_value(q)
    half = torch.full_like(t, 0.5) if kind == _lib.KIND_INT8 else e4m3_half_step(t)
    assert ((got - t).abs() <= half + t.abs() * 2.0 ** -17).all()


@pytest.mark.parametrize("kind", [_lib.KIND_INT8, _lib.KIND_FP8_E4M3, _lib.KIND_BF16])
@pytest.mark.parametrize("M,D,residual", [
    (1, 4096, True), (1, 8, False), (3, 520, True), (777, 1024, True), (300, 1000, False), (5, 16384, True),
    (257, 8192, True), (260, 16384, False), (64, 2056, True), (1024, 264, True),
])
def test_rms_norm_quant(kind, M, D, residual):
    g = gen(M * 31 + D)
    x, w = randn(g, M, D, mul=3.0), randn(g, D)
    y = randn(g, M, D) if residual else None
    h = (x.float() + y.float()).to(BF) if residual else x.clone()
    xn = torch.empty_like(x)
    x0 = x.clone()
    x_out = torch.empty_like(x) if residual else None
    q, s = K.rms_norm_quant(kind, x, w, y, eps=1e-5, x_out=x_out, xn=xn)
    assert torch.equal(x, x0)
    if residual:
        assert torch.equal(x_out, h)
    check_norm(kind, x, w, y, 1e-5, q, s, h, xn)
    q2, s2 = K.rms_norm_quant(kind, x, w, y, eps=1e-5, xn=xn if kind == _lib.KIND_BF16 else None)  # in place
    if residual:
        assert torch.equal(x, h)
    if kind != _lib.KIND_BF16:
        assert torch.equal(q, q2) and torch.equal(s, s2)


@pytest.mark.parametrize("kind", [_lib.KIND_INT8, _lib.KIND_FP8_E4M3])
@pytest.mark.parametrize("mul", [1e-9, 0.03, 1.0, 300.0])
def test_rms_norm_quant_codes_are_those_of_exact_arithmetic(kind, mul):
    """Where the scale is not its floor, v / s is top h w / max|h w| whatever the norm is, a quotient of values that
    fp32 holds exactly, and its codes are those of the fp64 quotient.  Rounding it to fp32 first cannot move it onto a
    code's border: with n, d < 2^16 the significands of h w and of the maximum, a quotient that is not on a border is
    1 / (254 n) > 2^-24 of itself or more from one for INT8, 1 / (7 n) or 1 / (31 d) for E4M3."""
    g = gen(int(mul * 1000) + kind)
    M, D = 400, 2048
    x, w = randn(g, M, D, mul=mul), randn(g, D)
    q, s = K.rms_norm_quant(kind, x, w, eps=0.0)
    t = (x.double() * w.double()).cpu()  # powers of two are exact there; the device's pow is not
    top = 127.0 if kind == _lib.KIND_INT8 else 448.0
    v = t * top / t.abs().amax(1, keepdim=True)
    if kind == _lib.KIND_INT8:
        assert torch.equal(q.cpu().double(), v.round())
    else:
        # fp64 -> E4M3 by hand: 8 steps to a binade, ties to even
        step = 2.0 ** (torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))).clamp(-6, 8) - 3)
        got = e4m3_value(q.cpu())
        assert torch.equal(got, torch.round(v / step) * step)
        assert torch.equal(torch.signbit(got), torch.signbit(v))


def test_rms_norm_quant_strided_rows():
    g = gen(4)
    M, D = 50, 640
    wide, yw, ow = randn(g, M, 3 * D), randn(g, M, D + 8), torch.zeros(M + 2, D + 16, dtype=BF, device=DEV)
    x, y, w = wide[:, D:2 * D], yw[:, 8:], randn(g, D)
    q, s = K.rms_norm_quant(_lib.KIND_INT8, x, w, y, x_out=ow[1:-1, :D])
    want = K.rms_norm_quant(_lib.KIND_INT8, x.contiguous(), w, y.contiguous(), x_out=torch.empty(M, D, dtype=BF, device=DEV))
    assert torch.equal(q, want[0]) and torch.equal(s, want[1])
    assert torch.equal(ow[1:-1, :D], (x.float() + y.float()).to(BF))
    assert ow[0].abs().sum() == 0 and ow[-1].abs().sum() == 0 and ow[:, D:].abs().sum() == 0


@pytest.mark.parametrize("kind", [_lib.KIND_INT8, _lib.KIND_FP8_E4M3])
def test_rms_norm_quant_zero_and_non_finite_rows(kind):
    x = torch.ones(5, 64, dtype=BF, device=DEV)
    x[1] = 0
    x[2, 7] = float("inf")
    x[3, 9] = float("nan")
    w = torch.full((64,), 2.0, dtype=BF, device=DEV)
    q, s = K.rms_norm_quant(kind, x, w)
    assert s[1].item() == pytest.approx(1e-10 if kind == _lib.KIND_INT8 else 1e-12)
    assert (q[1] == 0).all()
    assert torch.isnan(s[2]) and torch.isnan(s[3])
    assert torch.isfinite(s[[0, 4]]).all() and torch.equal(q[0], q[4])


@pytest.mark.parametrize("kind", [_lib.KIND_INT8, _lib.KIND_FP8_E4M3])
@pytest.mark.parametrize("M,D", [(3, 64), (5, 4096), (300, 8192)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_rms_norm_quant_non_finite_weight(kind, M, D, what):
    """An infinity or a NaN in the weight is in a value of every row: no row has a scale."""
    g = gen(M + D)
    x, w = randn(g, M, D), randn(g, D)
    x[0] = 0
    w[D - 3] = what
    xn = torch.empty_like(x)
    q, s = K.rms_norm_quant(kind, x, w, xn=xn)
    assert torch.isnan(s).all()
    assert not torch.isfinite(xn[1:, D - 3]).any()


@pytest.mark.parametrize("kind", [_lib.KIND_INT8, _lib.KIND_FP8_E4M3])
def test_rms_norm_quant_rows_beyond_fp32(kind):
    """Finite rows whose sum of squares passes fp32's range have no scale; rows in front of it have theirs."""
    x = torch.full((3, 512), 1e17, dtype=BF, device=DEV)
    x[1] = 2e18  # 512 * 4e36 > 3.4e38
    w = torch.full((512,), 0.5, dtype=BF, device=DEV)
    q, s = K.rms_norm_quant(kind, x, w)
    assert torch.isnan(s[1]) and torch.isfinite(s[[0, 2]]).all()
    keep = torch.tensor([0, 2], device=DEV)
    check_norm(kind, None, w, None, 1e-6, q[keep], s[keep], x[keep])


# ---------------------------------------------------------------------------
# rope_axes
# ---------------------------------------------------------------------------


def rotate_ref(x, heads, D, positions, freqs, axes, interleaved):
    """(rotated fp64 [M, heads, D], |x| + |y| of each element's pair)."""
    M, P = x.shape[0], freqs.numel()
    xd = x.double().reshape(M, heads, D)
    ang = positions.double()[axes.long()].t() * freqs
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    out, mag = xd.clone(), torch.zeros_like(xd)
    ia = torch.arange(P, device=x.device) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else P)
    a, b = xd[..., ia], xd[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return out, mag


@pytest.mark.parametrize("M,hq,hk,D,sections,shared,interleaved,idx", [
    (1, 32, 8, 128, (64,), True, False, torch.int32),
    (3120, 24, 24, 128, (22, 21, 21), False, True, torch.int64),
    (77, 5, 1, 64, (10, 11, 11), True, False, torch.int32),
    (2500, 4, 2, 64, (16,), False, True, torch.int64),      # half of the head rotates
    (13, 3, 3, 80, (8, 8, 8), True, False, torch.int32),    # 48 of 80 elements
    (9, 2, 1, 512, (256,), True, True, torch.int32),
    (6, 1, 2, 16, (8,), True, False, torch.int32),
    (2600, 1, 1, 16, (8,), True, True, torch.int64),
])
def test_rope_axes(M, hq, hk, D, sections, shared, interleaved, idx):
    g = gen(M + D)
    qkv = randn(g, M, (hq + 2 * hk) * D)
    q, k = qkv[:, :hq * D], qkv[:, hq * D:(hq + hk) * D]
    freqs, axes = K.rope_axes_frequencies(sections, shared=shared, device=DEV)
    positions = torch.randint(-5, 1 << 20, (len(sections), M), generator=g).to(idx).to(DEV)
    positions[:, 0] = (1 << 31) - 1  # the farthest position
    oq, ok = K.rope_axes(q, k, positions, freqs, axes, D, interleaved=interleaved)
    # the turn of position 2^31 is exact to 2^-53 relative: 2^-24 of a turn
    for x, o, h in ((q, oq, hq), (k, ok, hk)):
        want, mag = rotate_ref(x, h, D, positions, freqs, axes, interleaved)
        assert ((o.double().view(M, h, D) - want).abs() <= mag * 2.0 ** -20 + want.abs() * 2.0 ** -8).all()
    before = qkv.clone()
    K.rope_axes(q, k, positions, freqs, axes, D, interleaved=interleaved, out_q=q, out_k=k)  # in place
    assert torch.equal(q, oq) and torch.equal(k, ok)
    assert torch.equal(qkv[:, (hq + hk) * D:], before[:, (hq + hk) * D:])
    only, none = K.rope_axes(before[:, :hq * D], None, positions, freqs, axes, D, interleaved=interleaved)
    assert none is None and torch.equal(only, oq)


def test_rope_axes_matches_the_dit_table():
    """The repository's 3-axis video table (fp32 cos / sin) gives the same rotation to the table's own fp32 error."""
    from qi_b200.dit import CFG5, rope_apply, rope_tables

    spec = CFG5.experts[0]
    g = gen(3)
    q = randn(g, spec.tokens, 2 * 128)
    t = torch.arange(spec.tokens, device=DEV, dtype=torch.int32)
    positions = torch.stack([t // 120, t % 120 // 10, t % 10]).contiguous()
    freqs, axes = K.rope_axes_frequencies((22, 21, 21), device=DEV)
    o, _ = K.rope_axes(q, None, positions, freqs, axes, 128)
    want = rope_apply(q[None], rope_tables(CFG5, spec, DEV), 2)[0]
    # both round the same value to bf16: at most one step (2 x 2^-8) where fp32 errors straddle a border
    assert ((o.float() - want.float()).abs() <= want.float().abs() * 2.0 ** -7 + 2.0 ** -18).all()


@pytest.mark.parametrize("kind", ["bf16", "fp8", "fp8_one_scale"])
@pytest.mark.parametrize("M,hq,hk,D,page,layout", [
    (1, 8, 2, 128, 16, "token"), (50, 4, 4, 64, 7, "head"), (333, 6, 1, 128, 64, "joint"), (2400, 2, 2, 128, 1, "token"),
])
def test_rope_axes_store(kind, M, hq, hk, D, page, layout):
    g = gen(M * 3 + D)
    qkv = randn(g, M, (hq + 2 * hk) * D)
    q, k, v = qkv[:, :hq * D], qkv[:, hq * D:(hq + hk) * D], qkv[:, (hq + hk) * D:]
    freqs, axes = K.rope_axes_frequencies((D // 2,), shared=True, device=DEV)
    positions = torch.randint(0, 5000, (M,), generator=g).to(DEV)
    pages = -(-M // page) + 2
    dt = BF if kind == "bf16" else torch.uint8
    if layout == "token":
        kc, vc = (torch.full((pages, page, hk, D), 3, dtype=dt, device=DEV) for _ in range(2))
    elif layout == "head":
        kc, vc = (torch.full((pages, hk, page, D), 3, dtype=dt, device=DEV).transpose(1, 2) for _ in range(2))
    else:
        both = torch.full((pages, 2, page, hk, D), 3, dtype=dt, device=DEV)
        kc, vc = both[:, 0], both[:, 1]
    n_scale = 1 if kind == "fp8_one_scale" else hk
    ks, vs = (None, None) if kind == "bf16" else (0.01 + 0.02 * torch.rand(2, n_scale, generator=g).to(DEV))
    slots = torch.randperm(pages * page, generator=g)[:M].to(DEV)
    slots[::5] = -1  # padding rows
    ok = torch.zeros(M, hk * D, dtype=BF, device=DEV)
    oq = K.rope_axes_store(q, k, v, positions, freqs, axes, D, kc, vc, slots, interleaved=False, k_scale=ks, v_scale=vs,
                           out_k=ok)
    want_q, want_k = K.rope_axes(q, k, positions, freqs, axes, D, interleaved=False)
    assert torch.equal(oq, want_q) and torch.equal(ok, want_k)
    kr, mag = rotate_ref(k, hk, D, positions[None], freqs, axes, False)
    live = slots >= 0
    at = slots[live].long()
    for x, m, c, sc in ((kr, mag, kc, ks), (v.double().reshape(M, hk, D), torch.zeros_like(mag), vc, vs)):
        got = c[at // page, at % page]
        if kind == "bf16":
            assert ((got.double() - x[live]).abs() <= m[live] * 2.0 ** -20 + x[live].abs() * 2.0 ** -8).all()
        else:
            s = sc.double().expand(hk)[None, :, None]
            t = (x[live] / s).clamp(-448, 448)
            tol = e4m3_half_step(t) + m[live] / s * 2.0 ** -19 + t.abs() * 2.0 ** -22
            assert ((e4m3_value(got.contiguous()) - t).abs() <= tol).all()
        rest = torch.ones(pages * page, dtype=torch.bool, device=DEV)
        rest[at] = False
        r = rest.nonzero()[:, 0]
        assert (c[r // page, r % page] == 3).all()  # every other slot as it was


def test_rope_axes_store_codes_of_every_value():
    """E4M3 codes are the rounded fp32 quotient's for every bf16 value, zeros' signs, infinities and NaN included, and
    for scales from fp32's least to its largest magnitudes (one per key head)."""
    scales = torch.tensor([1e-41, 1e-38, 3e-25, 1e-12, 0.0137, 0.3, 1.0, 3.0, 448.0, 7e23, 3e24, 3e38], device=DEV)
    hk, D = scales.numel(), 128
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF).to(DEV).view(512, 1, D)
    v = every.expand(512, hk, D).reshape(512, hk * D).contiguous()
    kc, vc = (torch.zeros(16, 32, hk, D, dtype=torch.uint8, device=DEV) for _ in range(2))
    freqs, axes = K.rope_axes_frequencies((D // 2,), shared=True, device=DEV)
    K.rope_axes_store(torch.zeros(512, D, dtype=BF, device=DEV), torch.zeros_like(v), v, torch.zeros(512, dtype=torch.int32, device=DEV),
                      freqs, axes, D, kc, vc, torch.arange(512, device=DEV), interleaved=False, k_scale=scales, v_scale=scales)
    quotient = v.float().view(512, hk, D) / scales[:, None]
    want = quotient.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    got, nan = vc.view(512, hk, D), quotient.isnan()
    assert torch.equal(got[~nan], want[~nan])
    assert ((got[nan] & 0x7f) == 0x7f).all()
    assert (kc == 0).all()


def test_rope_axes_store_index_and_code_types():
    """int32 slots and a float8_e4m3fn cache give what int64 slots and a uint8 cache give."""
    g = gen(2)
    M, hk, D = 37, 2, 64
    x = randn(g, M, 3 * hk * D)
    q, k, v = x.split(hk * D, 1)
    freqs, axes = K.rope_axes_frequencies((32,), device=DEV)
    pos = torch.arange(M, device=DEV)
    slots = torch.randperm(64, generator=g)[:M].to(DEV)
    s = torch.full((1,), 0.02, device=DEV)
    out = []
    for dt, idx in ((torch.uint8, torch.int64), (torch.float8_e4m3fn, torch.int32)):
        kc, vc = (torch.zeros(8, 8, hk, D, dtype=torch.uint8, device=DEV).view(dt) for _ in range(2))
        K.rope_axes_store(q, k, v, pos.to(idx), freqs, axes, D, kc, vc, slots.to(idx), k_scale=s, v_scale=s)
        table, n = torch.arange(8, dtype=torch.int32, device=DEV)[None], torch.tensor([60], dtype=torch.int32, device=DEV)
        out.append((kc.view(torch.uint8), vc.view(torch.uint8),
                    K.attention_paged(q[:1], kc, vc, table, n, k_scale=s, v_scale=s)))
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_rope_axes_store_reports_slots_outside_the_cache():
    g = gen(1)
    x = randn(g, 4, 3 * 64)
    freqs, axes = K.rope_axes_frequencies((32,), device=DEV)
    kc, vc = (torch.zeros(2, 4, 1, 64, dtype=BF, device=DEV) for _ in range(2))
    slots = torch.tensor([0, 8, 3, 1 << 40], device=DEV)
    pos = torch.arange(4, device=DEV)
    K.rope_axes_store(x[:, :64], x[:, 64:128], x[:, 128:], pos, freqs, axes, 64, kc, vc, slots)
    with pytest.raises(_lib.QiB200DeviceError, match="out of range"):
        _lib.raise_on_device_error()
    assert _lib.device_status()[0] == 0
    assert torch.equal(vc.view(8, 64)[[0, 3]], x[[0, 2], 128:])
    assert vc.view(8, 64)[[1, 2, 4, 5, 6, 7]].abs().sum() == 0
    K.rope_axes(x[:, :64], None, pos, freqs, torch.full_like(axes, 1), 64)  # an axis that positions do not have
    with pytest.raises(_lib.QiB200DeviceError, match="out of range"):
        _lib.raise_on_device_error()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


def attend_ref(q, k, v, first, scale, r_p):
    """fp64 attention of q [a, D] on k, v [b, D]: (o, tolerance, lse); ``first``: query i sees keys <= first + i."""
    a, b = q.shape[0], k.shape[0]
    if b == 0:
        z = torch.zeros_like(q, dtype=torch.float64)
        return z, z, torch.full((a,), -math.inf, dtype=torch.float64, device=q.device)
    q, k, v = q.double(), k.double(), v.double()
    s = scale * q @ k.t()
    if first is not None:
        i, j = torch.arange(a, device=q.device)[:, None], torch.arange(b, device=q.device)
        s = s.masked_fill(j > first + i, -math.inf)
    top = s.amax(1, keepdim=True).clamp_min(-1e300)
    e = torch.exp(s - top)
    l = e.sum(1, keepdim=True)
    p = torch.where(l > 0, e / l.clamp_min(1e-300), 0.0)
    o, A = p @ v, p @ v.abs()
    D = q.shape[1]
    sabs = (scale * (q.abs() @ k.abs().t())).amax(1, keepdim=True)
    tol = 1.01 * (r_p * A + 2.0 ** -8 * o.abs() + 2 * (D + 16) * 2.0 ** -24 * sabs * A) + 1e-30
    return o, tol, (top + l.log())[:, 0]


def packed_ref(q, k, v, ql, kl, hq, hk, D, causal, scale):
    o, tol = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    lse = torch.zeros(q.shape[0], hq, dtype=torch.float64, device=DEV)
    i = j = 0
    for a, b in zip(ql, kl):
        for h in range(hq):
            g = h // (hq // hk)
            c = slice(h * D, (h + 1) * D)
            o[i:i + a, c], tol[i:i + a, c], lse[i:i + a, h] = attend_ref(
                q[i:i + a, c], k[j:j + b, g * D:(g + 1) * D], v[j:j + b, g * D:(g + 1) * D],
                b - a if causal else None, scale, 2.0 ** -8)
        i, j = i + a, j + b
    return o, tol, lse


def cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)


def close_lse(got, want):
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin].double(), want[~fin])
    assert ((got.double() - want)[fin].abs() <= 1e-5 * (1 + want[fin].abs())).all()


PACKED = [
    # q lengths, k lengths (None: the same), heads, kv_heads, D, causal
    ([1], None, 1, 1, 128, True),
    ([128], None, 2, 1, 128, True),
    ([129], None, 1, 1, 64, False),
    ([256], None, 3, 1, 128, True),
    ([300, 1, 17, 128, 0, 257, 2], None, 4, 2, 128, True),
    ([300, 1, 17, 128, 0, 257, 2], None, 3, 3, 64, True),
    ([64, 200], [700, 513], 8, 2, 64, True),        # chunks after a prefix
    ([64, 200], [700, 513], 6, 2, 128, False),
    ([300, 5, 130], [100, 0, 129], 2, 2, 128, True),  # queries in front of every key; no keys at all
    ([300, 5, 130], [100, 0, 129], 2, 1, 64, False),
    ([1000], None, 24, 8, 128, True),
    ([1, 1, 1, 1], [1, 129, 1000, 16], 4, 1, 128, True),
    ([3] * 70, None, 2, 1, 64, True),               # more sequences than a warp has lanes
    ([40, 700] * 40, None, 2, 2, 128, True),
    ([129], [9000], 2, 2, 128, True),               # few items over many keys: cut over the SMs and joined
    ([700, 3, 0, 200], [20000, 1500, 700, 0], 6, 2, 64, True),
    ([260, 40], [3000, 2500], 3, 1, 128, False),
    ([2200, 300], [2200, 100], 16, 16, 128, True),  # cut, with query blocks that see no key
    ([1] * 700 + [3000] + [130] * 500, None, 4, 1, 64, True),  # over 1024 sequences, one of them long
    ([300] + [260] * 40, [300] + [0] * 40, 40, 40, 64, True),  # many items without keys behind some with
    ([300] + [260] * 40 + [129], [300] + [0] * 40 + [129], 24, 4, 128, False),
]


@pytest.mark.parametrize("ql,kl,hq,hk,D,causal", PACKED)
def test_attention_packed(ql, kl, hq, hk, D, causal):
    g = gen(sum(ql) + D + hq)
    kl = kl or ql
    q, k, v = randn(g, sum(ql), hq * D), randn(g, sum(kl), hk * D), randn(g, sum(kl), hk * D)
    lse = torch.full((sum(ql), hq), 7.0, device=DEV)
    o = K.attention_packed(q, k, v, cu(ql), cu(kl), hq, hk, causal=causal, lse=lse)
    want, tol, wl = packed_ref(q, k, v, ql, kl, hq, hk, D, causal, D ** -0.5)
    assert ((o.double() - want).abs() <= tol).all(), ((o.double() - want).abs() / tol).max().item()
    close_lse(lse, wl)
    assert torch.equal(o, K.attention_packed(q, k, v, cu(ql), cu(kl), hq, hk, causal=causal))


@pytest.mark.parametrize("mul,scale", [(8.0, None), (1.0, 3.0), (0.02, 1e-3)])
def test_attention_packed_growing_maxima(mul, scale):
    """Large logits, with keys that grow towards the front, so that the running maximum moves in every step."""
    g = gen(11)
    n, hq, D = 1500, 2, 128
    q, v = randn(g, n, hq * D), randn(g, n, hq * D)
    k = (torch.randn(n, hq * D, generator=g) * torch.linspace(mul, 0.1 * mul, n)[:, None]).to(BF).to(DEV)
    o = K.attention_packed(q, k, v, cu([n]), cu([n]), hq, hq, scale=scale)
    want, tol, _ = packed_ref(q, k, v, [n], [n], hq, hq, D, True, scale or D ** -0.5)
    assert ((o.double() - want).abs() <= tol).all()


def test_attention_packed_strided_and_rows_left_alone():
    """Slices of one fused projection with padding rows behind the last sequence that hold NaN, a neighbour whose
    values are NaN, and an output whose other rows and columns keep their contents."""
    g = gen(12)
    ql, hq, hk, D = [150, 37], 4, 2, 64
    T = sum(ql)
    qkv = randn(g, T + 9, (hq + 2 * hk) * D + 8)
    qkv[T:] = float("nan")
    q, k, v = qkv[:, :hq * D], qkv[:, hq * D:(hq + hk) * D], qkv[:, (hq + hk) * D:(hq + 2 * hk) * D]
    big = torch.full((T + 9, hq * D + 16), 5.0, dtype=BF, device=DEV)
    lse = torch.full((T + 9, hq), 5.0, device=DEV)
    K.attention_packed(q, k, v, cu(ql), cu(ql), hq, hk, out=big[:, 8:8 + hq * D], lse=lse)
    want, tol, _ = packed_ref(q[:T], k[:T], v[:T], ql, ql, hq, hk, D, True, D ** -0.5)
    assert ((big[:T, 8:8 + hq * D].double() - want).abs() <= tol).all()
    assert (big[T:] == 5).all() and (big[:, :8] == 5).all() and (big[:, 8 + hq * D:] == 5).all() and (lse[T:] == 5).all()
    poisoned = qkv.clone()
    poisoned[150:T] = float("nan")  # the second sequence
    p = K.attention_packed(poisoned[:, :hq * D], poisoned[:, hq * D:(hq + hk) * D],
                           poisoned[:, (hq + hk) * D:(hq + 2 * hk) * D], cu(ql), cu(ql), hq, hk)
    assert torch.equal(p[:150], big[:150, 8:8 + hq * D]) and torch.isnan(p[150:T]).all()


@pytest.mark.parametrize("ql,kl,hq,hk,D", [
    ([300, 40], None, 2, 1, 128),        # pairs of heads
    ([300, 40], None, 3, 3, 64),         # one head, two query tiles
    ([129], [9000], 2, 2, 128),          # cut over the SMs and joined
    ([130, 77], [6000, 5100], 4, 2, 64),
])
def test_attention_packed_later_keys_do_not_reach_a_query(ql, kl, hq, hk, D):
    """Infinities and NaN in keys and values that causality hides: a query in front of them is as without them, one
    behind them has them in their columns (a value) or in all (a key)."""
    kl = kl or ql
    g = gen(sum(kl) + D)
    q, k, v = randn(g, sum(ql), hq * D), randn(g, sum(kl), hk * D), randn(g, sum(kl), hk * D)
    lq, lk = ql[0], kl[0]
    bad_v, bad_k, columns = lk - 70, lk - 25, (5, D - 3)  # keys of the first sequence
    zeroed = v.clone()
    zeroed[bad_v, list(columns)] = 0
    want, tol, wl = packed_ref(q, k, zeroed, ql, kl, hq, hk, D, True, D ** -0.5)
    v[bad_v, columns[0]], v[bad_v, columns[1]] = float("nan"), float("inf")
    clean = k.clone()
    k[bad_k] = float("nan")
    lse = torch.empty(sum(ql), hq, device=DEV)
    o = K.attention_packed(q, k, v, cu(ql), cu(kl), hq, hk, lse=lse)
    after_v, after_k = bad_v - (lk - lq), bad_k - (lk - lq)  # the first queries that see them
    hit = torch.zeros(sum(ql), hq, D, dtype=torch.bool, device=DEV)
    for h in range(hq // hk):  # the value's columns belong to key head 0
        hit[after_v:lq, h, list(columns)] = True
    hit[after_k:lq] = True
    hit = hit.view(sum(ql), hq * D)
    assert not torch.isfinite(o[hit]).any() and torch.isnan(o[after_k:lq]).all()
    assert ((o.double() - want).abs() <= tol)[~hit].all()
    close_lse(torch.cat([lse[:after_k], lse[lq:]]), torch.cat([wl[:after_k], wl[lq:]]))
    # the same without the key: only the value's columns are lost
    o = K.attention_packed(q, clean, v, cu(ql), cu(kl), hq, hk)
    hit = hit.view(sum(ql), hq, D)
    hit[after_k:lq] = hit[after_v]
    hit = hit.view(sum(ql), hq * D)
    assert not torch.isfinite(o[hit]).any() and ((o.double() - want).abs() <= tol)[~hit].all()


@pytest.mark.parametrize("ql,kl", [([40, 300], [40, 300]), ([129], [9000])])
def test_attention_packed_nan_queries_and_keys(ql, kl):
    """A NaN in a query is in its row's output and lse, a NaN in a key in those of every query that sees it, whole
    items and cut ones alike; no other row changes."""
    g = gen(sum(kl))
    hq, hk, D = 2, 1, 128
    q, k, v = randn(g, sum(ql), hq * D), randn(g, sum(kl), hk * D), randn(g, sum(kl), hk * D)
    lse, lse0 = (torch.empty(sum(ql), hq, device=DEV) for _ in range(2))
    plain = K.attention_packed(q, k, v, cu(ql), cu(kl), hq, hk, lse=lse0)
    q[20, 3] = float("nan")  # head 0
    k[kl[0] - 10, 7] = float("nan")
    o = K.attention_packed(q, k, v, cu(ql), cu(kl), hq, hk, lse=lse)
    hit = torch.zeros(sum(ql), hq, dtype=torch.bool, device=DEV)
    hit[20, 0] = True
    hit[ql[0] - 10:ql[0]] = True
    o, plain = o.view(-1, hq, D), plain.view(-1, hq, D)
    assert torch.isnan(o[hit]).all() and torch.isnan(lse[hit]).all()
    assert torch.equal(o[~hit], plain[~hit]) and torch.equal(lse[~hit], lse0[~hit])


@pytest.mark.parametrize("ql,kl,hq,hk,D", [
    ([300], [100], 2, 1, 128),           # pairs of heads: tokens 128 to 199 share a tile with some that see keys
    ([300], [100], 1, 1, 64),            # one head, two query tiles
    ([300, 70], [100, 0], 3, 3, 128),
    ([1500, 2000], [1400, 1990], 4, 2, 128),  # the steps cut evenly over the SMs
    ([1500, 2000], [1400, 1990], 3, 1, 64),
])
def test_attention_packed_queries_without_a_key_give_zeros(ql, kl, hq, hk, D):
    """Queries in front of every key give zeros (lse -inf) whatever the keys and values hold; behind them, only those
    that see an infinity or a NaN have it."""
    g = gen(sum(ql) + hq + D)
    q, k, v = randn(g, sum(ql), hq * D), randn(g, sum(kl), hk * D), randn(g, sum(kl), hk * D)
    lq, lk = ql[0], kl[0]
    want, tol, wl = packed_ref(q, k, v, ql, kl, hq, hk, D, True, D ** -0.5)
    v[lk - 2], v[lk - 1], k[lk - 1, ::3] = float("nan"), float("inf"), float("nan")
    lse = torch.empty(sum(ql), hq, device=DEV)
    o = K.attention_packed(q, k, v, cu(ql), cu(kl), hq, hk, lse=lse)
    first = 0
    for a, b in zip(ql, kl):
        none = slice(first, first + max(0, a - b))
        assert (o[none] == 0).all() and (lse[none] == -math.inf).all()
        first += a
    hit = torch.zeros(sum(ql), dtype=torch.bool, device=DEV)
    hit[lq - 2:lq] = True
    assert torch.isnan(o[hit]).all()
    assert ((o.double() - want).abs() <= tol)[~hit].all()
    hit[lq - 2] = False  # it sees a value only
    close_lse(lse[~hit], wl[~hit])


@pytest.mark.parametrize("ql,front,back,hq,hk,D", [
    ([50, 70], 0, 9, 4, 2, 128), ([300], 5, 0, 3, 3, 64), ([129], 700, 900, 2, 1, 128), ([1500, 0, 40], 1, 3, 4, 4, 64),
    ([], 0, 33, 2, 2, 128),
])
def test_attention_packed_rows_outside_of_a_new_output_are_zeros(ql, front, back, hq, hk, D):
    """A padded batch: rows that belong to no sequence are zeros in an output that the call allocates, whatever its
    memory held, and stay as they were in a given one and in lse."""
    g = gen(sum(ql) + front + hq)
    n = sum(ql)
    q, k, v = (randn(g, front + n + back, h * D) for h in (hq, hk, hk))
    for t in (q, k, v):
        t[:front], t[front + n:] = float("nan"), float("nan")
    c = (cu(ql) + front).to(torch.int32)
    given, lse = torch.full_like(q, 4), torch.full((q.shape[0], hq), 4.0, device=DEV)
    K.attention_packed(q, k, v, c, c, hq, hk, out=given, lse=lse)
    used = torch.full_like(q, float("nan"))  # its memory is the next output's
    at = used.data_ptr()
    del used
    o = K.attention_packed(q, k, v, c, c, hq, hk)
    assert o.data_ptr() == at
    rest = torch.ones(q.shape[0], dtype=torch.bool, device=DEV)
    rest[front:front + n] = False
    assert (o[rest] == 0).all() and (given[rest] == 4).all() and (lse[rest] == 4).all()
    assert torch.equal(o[~rest], given[~rest]) and torch.isfinite(o).all()


def test_attention_packed_looks_at_rows_again_for_longer_than_its_waits():
    """Rows whose outputs are computed once more (a value behind them holds a NaN) over a sequence so long that this
    takes longer than a wait may: the waits of the CTA's next item do not give up.  Without a workspace nothing is cut,
    so two items come one after the other."""
    g = gen(31)
    hq, D, lq, lk = 300, 64, 129, 400_000
    q, k, v = randn(g, lq, hq * D), randn(g, lk, D), randn(g, lk, D)
    v[lk - 60] = float("nan")  # queries 0 to 68 do not see it
    o = torch.empty_like(q)
    c, ck = cu([lq]), cu([lk])
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    _lib.check("qi_b200_attention_packed", _lib.load().qi_b200_attention_packed(
        q.data_ptr(), hq * D, k.data_ptr(), D, v.data_ptr(), D, o.data_ptr(), hq * D, None, c.data_ptr(), ck.data_ptr(), 1,
        lq, lk, hq, 1, D, 1, 0.5, None, 0, torch.cuda.current_stream().cuda_stream))
    end.record()
    torch.cuda.synchronize()
    _lib.raise_on_device_error()
    assert start.elapsed_time(end) > 2000  # the limit of a wait: else the test does not show what it is for
    v[lk - 60] = 0
    assert torch.isfinite(o[:69]).all() and torch.isnan(o[69:]).all()
    for h in (0, 148, 299):
        want, tol, _ = attend_ref(q[:69, h * D:(h + 1) * D], k[:lk - 60], v[:lk - 60], lk - lq, 0.5, 2.0 ** -8)
        # fp32 sums of 100,000 terms to a chain, each addition off by 2^-24 of the sum so far: 0.006 of sum p|v| and
        # of the sum of p at worst; tol holds at least 2^-8 sum p|v|, so the first is below 1.6 tol
        tol = 2.6 * tol + 0.006 * want.abs()
        assert ((o[:69, h * D:(h + 1) * D].double() - want).abs() <= tol).all()


def test_attention_packed_nothing_to_do():
    q = torch.zeros(0, 128, dtype=BF, device=DEV)
    assert K.attention_packed(q, q, q, cu([]), cu([]), 1, 1).shape == (0, 128)
    q = torch.ones(3, 128, dtype=BF, device=DEV)
    o = torch.full_like(q, 2)
    K.attention_packed(q, q, q, cu([]), cu([]), 1, 1, out=o)
    assert (o == 2).all()
    e = torch.zeros(0, 128, dtype=BF, device=DEV)
    K.attention_packed(q, e, e, cu([3]), cu([0]), 1, 1, out=o)
    assert (o == 0).all()


def make_cache(g, lens, page, hk, D, kind, layout, spare=3):
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(need + [1]) + 1), -7, dtype=torch.int32)  # unused entries are never read
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (total, page, hk, D) if layout == "token" else (total, hk, page, D)
    caches = [torch.randn(*shape, generator=g).to(DEV) for _ in range(2)]
    scales = (None, None)
    if kind == "fp8":
        scales = tuple((0.005 + 0.02 * torch.rand(hk, generator=g)).to(DEV) for _ in range(2))
        caches = [(c * 50).to(torch.float8_e4m3fn).view(torch.uint8) for c in caches]
    else:
        caches = [c.to(BF) for c in caches]
    if layout != "token":
        caches = [c.transpose(1, 2) for c in caches]
    return table.to(DEV), caches[0], caches[1], scales


def paged_ref(q, kc, vc, table, lens, ks, vs, scale, kind):
    page, hk, D = kc.shape[1], kc.shape[2], kc.shape[3]
    hq = q.shape[1] // D
    o, tol = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    lse = torch.zeros(q.shape[0], hq, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        t = torch.arange(n, device=DEV)
        k, v = (c[table[b, t // page].long(), t % page] for c in (kc, vc))
        if kind == "fp8":
            k = e4m3_value(k.contiguous()) * ks.double()[:, None]
            v = e4m3_value(v.contiguous()) * vs.double()[:, None]
        for h in range(hq):
            g = h // (hq // hk)
            c = slice(h * D, (h + 1) * D)
            o[b:b + 1, c], tol[b:b + 1, c], lse[b:b + 1, h] = attend_ref(
                q[b:b + 1, c], k[:, g], v[:, g], None, scale, 2.0 ** -11 if kind == "fp8" else 2.0 ** -8)
    return o, tol, lse


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,hq,hk,page,layout", [
    ([1], 1, 1, 16, "token"),
    ([1000], 32, 8, 16, "token"),
    ([0, 1, 16, 17, 63, 64, 65, 0], 8, 2, 16, "token"),
    ([5000, 3, 777], 24, 1, 64, "head"),      # more than 16 query heads per key head
    ([300, 200], 12, 1, 24, "token"),         # 9 to 16 heads; pages that end inside a block
    ([129, 40], 6, 3, 1, "head"),
    ([2049] * 5 + [0] + [31] * 3, 16, 4, 128, "head"),
    ([20000, 1], 4, 2, 32, "token"),          # split over many SMs
    ([37] * 300, 4, 4, 16, "token"),          # many short sequences
    ([0, 0], 2, 1, 16, "token"),
    ([4000, 1, 0, 2500, 77], 8, 8, 16, "token"),   # all key heads in one item
    ([3000, 900] * 3, 24, 12, 48, "token"),        # four key heads per item, pages of any size
    ([9000, 5555, 777, 2048], 16, 8, 64, "token"),  # ranges that begin anywhere in a page
    ([4100, 61, 3333], 4, 4, 32, "token"),
])
def test_attention_paged(kind, D, lens, hq, hk, page, layout):
    g = gen(sum(lens) + D + hq)
    table, kc, vc, (ks, vs) = make_cache(g, lens, page, hk, D, kind, layout)
    q = randn(g, len(lens), hq * D)
    lse = torch.zeros(len(lens), hq, device=DEV)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = K.attention_paged(q, kc, vc, table, n, k_scale=ks, v_scale=vs, lse=lse)
    want, tol, wl = paged_ref(q, kc, vc, table, lens, ks, vs, D ** -0.5, kind)
    assert ((o.double() - want).abs() <= tol).all(), ((o.double() - want).abs() / tol).max().item()
    close_lse(lse, wl)
    assert torch.equal(o, K.attention_paged(q, kc, vc, table, n, k_scale=ks, v_scale=vs))  # deterministic


def test_attention_paged_large_queries_fp8():
    """q far outside fp16's range: the row's power of two keeps it inside."""
    g = gen(5)
    table, kc, vc, (ks, vs) = make_cache(g, [100], 16, 1, 128, "fp8", "token")
    q = randn(g, 1, 2 * 128, mul=1e8)
    o = K.attention_paged(q, kc, vc, table, torch.tensor([100], dtype=torch.int32, device=DEV), k_scale=ks, v_scale=vs,
                          scale=1e-9)
    want, tol, _ = paged_ref(q, kc, vc, table, [100], ks, vs, 1e-9, "fp8")
    assert ((o.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("outlier", [0, 12, 17, 22, 26])
@pytest.mark.parametrize("mul,scale", [(1.0, None), (1e-30, 1e29), (1e36, 1e-37)])
def test_attention_paged_queries_of_many_magnitudes_fp8(outlier, mul, scale):
    """A column of q that is 2^outlier times the others, where the keys are zero: the scores are those of the other
    columns.  In fp16 the row's largest element lies in its last binade, [2^15, 2^16), and half a step of its smallest
    numbers is 2^-25: an element is off by 2^-40 of the largest at most where 2^-11 of itself is not more; bf16's 8 bits
    fit where it is above 2^-14, so the rest is exact."""
    g = gen(outlier + int(mul < 1))
    lens = [700, 64]
    table, kc, vc, (ks, vs) = make_cache(g, lens, 16, 2, 128, "fp8", "token")
    q = randn(g, 2, 4 * 128)
    q = (q.double() * (mul if outlier == 0 or mul <= 1 else mul * 2.0 ** -outlier)).to(BF)
    q[:, 5::128] = (q[:, 6::128].double() * 2.0 ** outlier).to(BF)
    if mul > 1 and outlier:
        scale = scale * 2.0 ** outlier
    if outlier:
        kc[..., 5] = 0
    scale = scale or 128 ** -0.5
    o = K.attention_paged(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=DEV), k_scale=ks, v_scale=vs,
                          scale=scale)
    want, tol, _ = paged_ref(q, kc, vc, table, lens, ks, vs, scale, "fp8")
    most = (e4m3_value(kc.contiguous()).abs() * ks.double()[:, None]).nan_to_num().sum(-1).max()
    top = q.double().abs().max()
    values = e4m3_value(vc.contiguous()).abs().max() * vs.max()
    tol = tol + 2 * 2.0 ** -40 * top * most * scale * values
    assert torch.isfinite(o).all()
    assert ((o.double() - want).abs() <= tol).all(), ((o.double() - want).abs() / tol).max().item()


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("lens,hq,hk,D,page", [
    ([20000], 4, 1, 128, 16),              # one sequence over many SMs
    ([9000, 33, 6000] + [700] * 40, 8, 4, 64, 64),
    ([500] * 300, 12, 1, 128, 32),         # whole sequences in one range, 9 to 16 heads
])
@pytest.mark.parametrize("nats,spread", [(3, 0.3), (12, 0.3), (15, 0.0), (16.9, 0.0), (17.5, 0.3), (19, 0.3), (20, 0.0), (30, 0.0)])
def test_attention_paged_sinks(kind, lens, hq, hk, D, page, nats, spread):
    """A token that outweighs all others and whose value is zero: the output is made of the others' small
    probabilities.  Over an E4M3 cache they are fp16 above a base 2^-15 of the largest: half a step is 2^-11 of the value
    or 2^-25 2^-15, whichever is more, so a probability is off by 2^-40 at most where it is below fp16's normal range."""
    g = gen(sum(lens) + D + int(nats * 10))
    n = [-(-m // page) for m in lens]
    sign = (torch.randint(0, 2, (hk, D), generator=g) * 2 - 1).float()
    q = sign.repeat_interleave(hq // hk, 0).reshape(1, -1).expand(len(lens), -1).to(BF).to(DEV).contiguous()
    # rest: scores of standard deviation ``spread`` nats below the sink's
    scale = nats / D
    kc = torch.randn(sum(n), page, hk, D, generator=g) * (spread / (scale * D ** 0.5))
    vc = torch.randn(sum(n), page, hk, D, generator=g)
    table = torch.zeros(len(lens), max(n), dtype=torch.int32)
    at = 0
    for b, m in enumerate(n):
        table[b, :m] = torch.arange(at, at + m)
        at += m
    for b, m in enumerate(lens):
        t = int(torch.randint(0, m, (1,), generator=g))
        kc[table[b, t // page], t % page] = sign
        vc[table[b, t // page], t % page] = 0
    kc, vc, table = kc.to(DEV), vc.to(DEV), table.to(DEV)
    kw = {}
    if kind == "fp8":
        kc, vc = (c.to(torch.float8_e4m3fn).view(torch.uint8) for c in (kc, vc))
        kw = {"k_scale": torch.ones(hk, device=DEV), "v_scale": torch.ones(hk, device=DEV)}
    else:
        kc, vc = kc.to(BF), vc.to(BF)
    lse = torch.empty(len(lens), hq, device=DEV)
    o = K.attention_paged(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=DEV), scale=scale, lse=lse, **kw)
    some = [0, 1, 2, len(lens) - 1] if len(lens) > 3 else range(len(lens))  # sequences that are looked at
    want, tol, wl = paged_ref(q[some], kc, vc, table[some], [lens[b] for b in some], kw.get("k_scale"), kw.get("v_scale"),
                              scale, kind)
    if kind == "fp8":
        top = e4m3_value(vc).abs().max()
        tol = tol + torch.tensor([[lens[b]] for b in some], device=DEV) * 2.0 ** -40 * top
    assert ((o[some].double() - want).abs() <= tol).all(), ((o[some].double() - want).abs() / tol).max().item()
    close_lse(lse[some], wl)


@pytest.mark.parametrize("lens", [[40, 300] * 60, [20000, 33]])
@pytest.mark.parametrize("v_scale", [1e-37, 1e-20, 1e20, 2e36])
def test_attention_paged_value_scales_of_many_magnitudes(lens, v_scale):
    """Items inside one range and items that are cut and joined: outputs lie inside bf16's range, and no sum on the way
    leaves fp32's."""
    g = gen(len(lens))
    table, kc, vc, (ks, _) = make_cache(g, lens, 16, 2, 64, "fp8", "token")
    vs = torch.tensor([v_scale, v_scale / 3], device=DEV)
    q = randn(g, len(lens), 4 * 64)
    o = K.attention_paged(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=DEV), k_scale=ks, v_scale=vs)
    some = [0, 1, len(lens) - 1]
    want, tol, _ = paged_ref(q[some], kc, vc, table[some], [lens[b] for b in some], ks, vs, 64 ** -0.5, "fp8")
    tol = tol - 1e-30 + 2.0 ** -134  # half a step of bf16's smallest numbers in place of the reference's floor
    assert ((o[some].double() - want).abs() <= tol).all(), ((o[some].double() - want).abs() / tol).max().item()


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_attention_paged_garbage_behind_the_length(kind):
    """Slots behind a sequence's last token hold NaN (bf16 and E4M3 have one): the result does not see them."""
    g = gen(6)
    lens = [5, 70]
    table, kc, vc, (ks, vs) = make_cache(g, lens, 16, 2, 64, kind, "token")
    q = randn(g, 2, 4 * 64)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = K.attention_paged(q, kc, vc, table, n, k_scale=ks, v_scale=vs)
    nan = float("nan") if kind == "bf16" else 0x7F
    for b, m in enumerate(lens):
        last = table[b, (m - 1) // 16].long()
        kc[last, (m - 1) % 16 + 1:] = nan
        vc[last, (m - 1) % 16 + 1:] = nan
    assert torch.equal(o, K.attention_paged(q, kc, vc, table, n, k_scale=ks, v_scale=vs))


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("lens", [[40] * 300, [5000, 33]])
def test_attention_paged_nan_queries_and_keys(kind, lens):
    """A NaN in a query head is in that head's output and lse, a NaN in a cached key in those of its sequence's heads,
    items inside one range and items cut by ranges alike; no other row changes."""
    g = gen(sum(lens))
    hq, hk, D, page = 4, 2, 128, 16
    q = randn(g, len(lens), hq * D)
    n = [-(-m // page) for m in lens]
    kc, vc = (randn(g, sum(n) * page * hk, D).view(sum(n), page, hk, D) for _ in range(2))
    kw = {}
    if kind == "fp8":
        kc, vc = (c.to(torch.float8_e4m3fn) for c in (kc, vc))
        kw = {"k_scale": torch.ones(1, device=DEV), "v_scale": torch.ones(1, device=DEV)}
    pages = torch.zeros(len(lens), max(n), dtype=torch.int32)
    at = 0
    for i, c in enumerate(n):
        pages[i, :c] = torch.arange(at, at + c)
        at += c
    pages, lengths = pages.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    lse, lse0 = (torch.empty(len(lens), hq, device=DEV) for _ in range(2))
    plain = K.attention_paged(q, kc, vc, pages, lengths, lse=lse0, **kw)
    q[0, 2 * D + 5] = float("nan")  # sequence 0, head 2
    kc[n[0], 3, 1, 9] = float("nan")  # sequence 1, key head 1: heads 2 and 3
    o = K.attention_paged(q, kc, vc, pages, lengths, lse=lse, **kw)
    hit = torch.zeros(len(lens), hq, dtype=torch.bool, device=DEV)
    hit[0, 2] = True
    hit[1, 2:] = True
    o, plain = o.view(-1, hq, D), plain.view(-1, hq, D)
    assert torch.isnan(o[hit]).all() and torch.isnan(lse[hit]).all()
    assert torch.equal(o[~hit], plain[~hit]) and torch.equal(lse[~hit], lse0[~hit])


def test_attention_paged_bad_pages_and_lengths_are_left_out():
    g = gen(7)
    lens = [64, 48]
    table, kc, vc, _ = make_cache(g, lens, 16, 1, 128, "bf16", "token")
    q = randn(g, 2, 2 * 128)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    bad = table.clone()
    bad[0, 1], bad[0, 3] = -1, 10 ** 6
    o = K.attention_paged(q, kc, vc, bad, n)
    with pytest.raises(_lib.QiB200DeviceError, match="out of range"):
        _lib.raise_on_device_error()
    keep = table.clone()
    keep[0, 1] = table[0, 2]
    want = K.attention_paged(q, kc, vc, keep, torch.tensor([32, 48], dtype=torch.int32, device=DEV))
    # the same 32 keys in another grouping: both within half a step of bf16 (and of its P) of the exact result
    assert ((o.float() - want.float()).abs() <= 2.0 ** -5).all()
    assert torch.equal(o[1], want[1])
    long = torch.tensor([64, 10 ** 9], dtype=torch.int32, device=DEV)  # behind the table: cut to its 5 columns
    full = torch.cat([table, table[:, :0]], 1)
    full[:, 3:] = full[:, :1]
    o2 = K.attention_paged(q, kc, vc, full, long)
    with pytest.raises(_lib.QiB200DeviceError, match="out of range"):
        _lib.raise_on_device_error()
    cut = torch.tensor([64, 16 * full.shape[1]], dtype=torch.int32, device=DEV)
    assert torch.equal(o2, K.attention_paged(q, kc, vc, full, cut))
    _lib.raise_on_device_error()


def test_attention_paged_negative_lengths_are_reported():
    g = gen(8)
    table, kc, vc, _ = make_cache(g, [40, 40, 40], 16, 1, 64, "bf16", "token")
    q = randn(g, 3, 2 * 64)
    lse = torch.full((3, 2), 3.0, device=DEV)
    lengths = lambda *n: torch.tensor(n, dtype=torch.int32, device=DEV)
    o = K.attention_paged(q, kc, vc, table, lengths(40, -1, -(1 << 31)), lse=lse)
    with pytest.raises(_lib.QiB200DeviceError, match="out of range"):
        _lib.raise_on_device_error()
    assert (o[1:] == 0).all() and (lse[1:] == -math.inf).all()
    assert torch.equal(o, K.attention_paged(q, kc, vc, table, lengths(40, 0, 0)))
    _lib.raise_on_device_error()


# ---------------------------------------------------------------------------
# streams, graphs, refusals, and all of them together
# ---------------------------------------------------------------------------


def test_side_stream_and_graph_replay():
    """All operators captured twice into graphs with their own workspaces, replayed on two streams at once with new
    inputs, give the eager results."""
    g = gen(8)
    lens, hq, hk, D = [700, 3000], 8, 2, 128
    table, kc, vc, _ = make_cache(g, lens, 16, hk, D, "bf16", "token")
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    freqs, axes = K.rope_axes_frequencies((D // 2,), shared=True, device=DEV)
    w = randn(g, hq * D)
    pos = torch.arange(2, device=DEV)
    c = cu([1, 1])

    def chain(x):
        q8, s8 = K.rms_norm_quant(_lib.KIND_FP8_E4M3, x, w)
        q, _ = K.rope_axes(x, None, pos, freqs, axes, D)
        a = K.attention_paged(q, kc, vc, table, n)
        return a, q8, s8, K.attention_packed(a, a[:, :hk * D], a[:, hk * D:2 * hk * D], c, c, hq, hk)

    xs = [randn(g, 2, hq * D) for _ in range(4)]
    want = [chain(x) for x in xs]
    graphs, ins, outs = [], [], []
    for i in range(2):
        x = xs[i].clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = chain(x)
        graphs.append(graph), ins.append(x), outs.append(o)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for base in (0, 2):
        for i in range(2):
            ins[i].copy_(xs[base + i])
        torch.cuda.synchronize()
        for rep in range(3):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            for a, b in zip(outs[i], want[base + i]):
                assert torch.equal(a, b)
    with torch.cuda.stream(streams[0]):
        got = chain(xs[3])
    streams[0].synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[3]))


def test_offsets_beyond_32_bits():
    """Rows and cache pages more than 2^32 elements behind the first give what the same values give close together."""
    g = gen(77)
    free = torch.cuda.mem_get_info()[0]
    if free < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    M, hq, hk, D = 4200, 2, 1, 128
    wide = torch.empty(M, 1 << 20, dtype=BF, device=DEV)  # 8.8 GB
    near = {n: randn(g, M, h * D) for n, h in (("q", hq), ("k", hk), ("v", hk), ("y", hq))}
    far, at = {}, 8
    for n, x in near.items():
        far[n] = wide[:, at:at + x.size(1)]
        far[n].copy_(x)
        at += x.size(1)
    w = randn(g, 1, hq * D)[0]
    out = wide[:, 1 << 19:(1 << 19) + hq * D]
    codes, scales = K.rms_norm_quant(_lib.KIND_FP8_E4M3, far["q"], w, far["y"], x_out=out)
    stream = near["q"].clone()
    want = K.rms_norm_quant(_lib.KIND_FP8_E4M3, stream, w, near["y"])
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1]) and torch.equal(out, stream)
    freqs, axes = K.rope_axes_frequencies((D // 2,), shared=True, device=DEV)
    pos = torch.arange(M, dtype=torch.int32, device=DEV)
    want = K.rope_axes(near["q"], near["k"], pos, freqs, axes, D)
    K.rope_axes(far["q"], far["k"], pos, freqs, axes, D, out_q=far["q"], out_k=far["k"])
    assert torch.equal(far["q"], want[0]) and torch.equal(far["k"], want[1])
    n = cu([M - 300, 300])
    K.attention_packed(far["q"], far["k"], far["v"], n, n, hq, hk, out=out)
    assert torch.equal(out, K.attention_packed(*want, near["v"], n, n, hq, hk))
    del wide, far, out
    # 100 tokens in the last pages of a cache, against the same pages alone
    pages, page, hk = (1 << 16) + 3, 64, 8
    cache = torch.empty(pages, 2, page, hk, D, dtype=torch.uint8, device=DEV)  # 8.6 GB
    few = torch.zeros(3, 2, page, hk, D, dtype=torch.uint8, device=DEV)
    cache[-3:] = 0
    k, v, q = randn(g, 100, hk * D), randn(g, 100, hk * D), randn(g, 100, hk * D)
    s = torch.ones(1, device=DEV)
    slots = torch.randperm(3 * page, generator=g)[:100].to(DEV)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([3 * page], dtype=torch.int32, device=DEV)
    got = []
    for c, first in ((cache, pages - 3), (few, 0)):
        K.rope_axes_store(q, k, v, pos[:100], freqs, axes, D, c[:, 0], c[:, 1], slots + first * page, k_scale=s, v_scale=s)
        got.append(K.attention_paged(q[:1], c[:, 0], c[:, 1], table + first, lengths, k_scale=s, v_scale=s))
    assert torch.equal(cache[-3:], few) and torch.equal(got[0], got[1])
    _lib.raise_on_device_error()


def test_refusals():
    x = torch.zeros(4, 256, dtype=BF, device=DEV)
    w = torch.ones(256, dtype=BF, device=DEV)
    bad = [
        lambda: K.rms_norm_quant(_lib.KIND_INT8, x.float(), w),
        lambda: K.rms_norm_quant(_lib.KIND_INT8, x[:, :250], w[:250]),
        lambda: K.rms_norm_quant(_lib.KIND_INT8, x[:, 1:249], w[:248]),
        lambda: K.rms_norm_quant(_lib.KIND_INT8, x, w[:128]),
        lambda: K.rms_norm_quant(_lib.KIND_INT8, x, w, x[:3]),
        lambda: K.rms_norm_quant(_lib.KIND_INT8, x, w, x_out=x),
        lambda: K.rms_norm_quant(_lib.KIND_BF16, x, w),
        lambda: K.rms_norm_quant(7, x, w),
        lambda: K.rms_norm_quant(_lib.KIND_INT8, x.cpu(), w),
        lambda: K.rms_norm_quant(_lib.KIND_INT8, x, w, q=torch.zeros(4, 256, dtype=torch.uint8, device=DEV)),
        lambda: K.rms_norm_quant(_lib.KIND_INT8, torch.zeros(1, 16392, dtype=BF, device=DEV),
                                 torch.zeros(16392, dtype=BF, device=DEV)),
    ]
    f, a = K.rope_axes_frequencies((64,), device=DEV)
    pos = torch.zeros(4, dtype=torch.int32, device=DEV)
    kc = torch.zeros(2, 4, 1, 128, dtype=BF, device=DEV)
    k1 = x[:, :128]
    slots = torch.arange(4, device=DEV)
    bad += [
        lambda: K.rope_axes_frequencies((8, 0), device=DEV),
        lambda: K.rope_axes(x, None, pos[:3], f, a, 128),
        lambda: K.rope_axes(x, None, pos.float(), f, a, 128),
        lambda: K.rope_axes(x, None, pos, f.float(), a, 128),
        lambda: K.rope_axes(x, None, pos, f[:60], a[:60], 128),
        lambda: K.rope_axes(x, None, pos, f, a, 64),       # 64 pairs do not fit a head of 64
        lambda: K.rope_axes(x, None, pos, f, a, 96),       # 256 columns are no whole number of heads
        lambda: K.rope_axes_store(x, k1, k1, pos, f, a, 128, kc, kc[:1], slots),
        lambda: K.rope_axes_store(x, k1, None, pos, f, a, 128, kc, kc, slots),
        lambda: K.rope_axes_store(x, k1, k1, pos, f, a, 128, kc, kc, slots[:3]),
        lambda: K.rope_axes_store(x, x, x, pos, f, a, 128, kc, kc, slots),
        lambda: K.rope_axes_store(x, k1, k1, pos, f, a, 128, kc.to(torch.uint8), kc.to(torch.uint8), slots),
        lambda: K.rope_axes_store(x, k1, k1, pos, f, a, 128, kc, kc, slots, k_scale=torch.ones(1, device=DEV)),
        lambda: K.rope_axes_store(x, k1, k1, pos, f, a, 128, kc.half(), kc.half(), slots),
    ]
    c = cu([4])
    bad += [
        lambda: K.attention_packed(x, x, x, c, c, 4, 3),
        lambda: K.attention_packed(x, x, x, c, c, 2, 1),
        lambda: K.attention_packed(x, x, x, c, c, 1, 1),   # head dim 256
        lambda: K.attention_packed(x, x, x[:3], c, c, 2, 2),
        lambda: K.attention_packed(x, x, x, c.long(), c.long(), 2, 2),
        lambda: K.attention_packed(x, x, x, c, cu([2, 2]), 2, 2),
        lambda: K.attention_packed(x, x, x, c, c, 2, 2, scale=0.0),
        lambda: K.attention_packed(x, x, x, c, c, 2, 2, scale=float("nan")),
        lambda: K.attention_packed(x, x, x, c, c, 2, 2, lse=torch.zeros(4, 3, device=DEV)),
        lambda: K.attention_packed(x, x, x, c, c, 2, 2, out=torch.zeros(3, 256, dtype=BF, device=DEV)),
    ]
    t, n = torch.zeros(4, 2, dtype=torch.int32, device=DEV), torch.ones(4, dtype=torch.int32, device=DEV)
    bad += [
        lambda: K.attention_paged(x, kc, kc, t[:3], n),
        lambda: K.attention_paged(x, kc, kc, t.long(), n),
        lambda: K.attention_paged(x, kc, kc, t, n[:3]),
        lambda: K.attention_paged(x, kc, kc, t, n.long()),
        lambda: K.attention_paged(x, kc[..., :96], kc[..., :96], t, n),
        lambda: K.attention_paged(x, kc[..., 4:68], kc[..., 4:68], t, n),
        lambda: K.attention_paged(x, kc, kc, t, n, v_scale=torch.ones(1, device=DEV)),
        lambda: K.attention_paged(x, kc.view(torch.uint8), kc.view(torch.uint8), t, n),
        lambda: K.attention_paged(x, kc[:0], kc[:0], t, n),
        lambda: K.attention_paged(x, kc, kc, t, n, scale=-1.0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, _lib.QiB200Error)):
            call()
            print("not refused:", i)


def test_decoder_block_prompt_then_tokens():
    """The operators as they are used: prompts through norm -> INT8 q/k/v linear -> rotary + cache -> packed attention
    -> INT8 output linear with residual, then three single tokens through the paged path.  Every step is checked against
    its 64-bit form on the framework's own inputs of that step, and the paged result against packed attention over the
    whole sequence."""
    g = gen(9)
    hid, hq, hk, D, page = 512, 8, 2, 64, 16
    lens = [75, 130, 1]
    width = (hq + 2 * hk) * D

    def int8_weight(n, k):
        w = torch.randint(-127, 128, (n, k), generator=g).to(torch.int8).to(DEV)
        return w, torch.full((n,), 0.7 / 127 / k ** 0.5, device=DEV)

    wqkv, sqkv = int8_weight(width, hid)
    wo, so = int8_weight(hid, hq * D)
    norm = randn(g, hid, mul=0.1) + 1
    freqs, axes = K.rope_axes_frequencies((8, 12, 12), shared=True, device=DEV)
    pages = sum(-(-(n + 3) // page) for n in lens)
    kc, vc = (torch.zeros(pages, page, hk, D, dtype=BF, device=DEV) for _ in range(2))
    table = torch.zeros(len(lens), 10, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        m = -(-(n + 3) // page)
        table[b, :m] = torch.arange(at, at + m)
        at += m

    def layer(x, y, pos, slots):
        q8, s8 = K.rms_norm_quant(_lib.KIND_INT8, x, norm, y)
        check_norm(_lib.KIND_INT8, None, norm, None, 1e-6, q8, s8, x)
        qkv = K.gemm(_lib.KIND_INT8, q8, wqkv, s8, sqkv)
        q, k, v = qkv[:, :hq * D], qkv[:, hq * D:(hq + hk) * D], qkv[:, (hq + hk) * D:]
        K.rope_axes_store(q, k, v, pos, freqs, axes, D, kc, vc, slots, interleaved=False, out_q=q, out_k=k)
        return q, k, v

    x = randn(g, sum(lens), hid)
    y = randn(g, sum(lens), hid)
    pos = torch.cat([torch.arange(n) for n in lens]).expand(3, -1).contiguous().to(DEV)
    seq = torch.cat([torch.full((n,), b) for b, n in enumerate(lens)])
    slot = lambda b, t: table[b, t // page].long() * page + t % page
    q, k, v = layer(x, y, pos, slot(seq, pos[0].cpu()).to(DEV))
    c = cu(lens)
    o = K.attention_packed(q, k, v, c, c, hq, hk)
    want, tol, _ = packed_ref(q, k, v, lens, lens, hq, hk, D, True, D ** -0.5)
    assert ((o.double() - want).abs() <= tol).all()
    y = K.int8_linear(o, wo, so)
    history = [(list(torch.split(k, lens)), list(torch.split(v, lens)))]
    ks, vs = history[0]
    last = c[1:].long() - 1
    xt, yt = x[last].contiguous(), y[last].contiguous()
    for step in range(3):
        now = torch.tensor([n + step for n in lens])
        q, k, v = layer(xt, yt, now.expand(3, -1).contiguous().to(DEV), slot(torch.arange(3), now).to(DEV))
        n = (now + 1).to(torch.int32).to(DEV)
        o = K.attention_paged(q, kc, vc, table.to(DEV), n)
        ks = [torch.cat([a, k[b:b + 1]]) for b, a in enumerate(ks)]
        vs = [torch.cat([a, v[b:b + 1]]) for b, a in enumerate(vs)]
        total = [a.shape[0] for a in ks]
        want, tol, _ = packed_ref(q, torch.cat(ks), torch.cat(vs), [1] * 3, total, hq, hk, D, True, D ** -0.5)
        assert ((o.double() - want).abs() <= tol).all()
        same = K.attention_packed(q, torch.cat(ks), torch.cat(vs), cu([1] * 3), cu(total), hq, hk)
        assert ((same.double() - want).abs() <= tol).all()
        yt = K.int8_linear(o, wo, so)


# ---------------------------------------------------------------------------
# tracing
# ---------------------------------------------------------------------------


def test_operators_pass_torchs_checks():
    """torch's own checks of every form: what the schema does not declare written is not, results alias nothing that is
    not declared, and the traced shapes are the real ones."""
    g = gen(21)
    M, hq, hk, D, page = 12, 4, 2, 64, 4
    x, w = randn(g, M, hq * D), randn(g, hq * D)
    k, v = randn(g, M, hk * D), randn(g, M, hk * D)
    freqs, axes = K.rope_axes_frequencies((D // 2,), device=DEV)
    pos, slots = torch.arange(M, device=DEV), torch.arange(M, device=DEV)
    kc, vc = (randn(g, 3 * page, hk * D).view(3, page, hk, D) for _ in range(2))
    c = cu([5, 7])
    table, n = torch.tensor([[2, 0, 1]] * M, dtype=torch.int32, device=DEV), torch.full((M,), 9, dtype=torch.int32, device=DEV)
    new = lambda t: torch.empty_like(t)
    q8, s8 = torch.empty(M, hq * D, dtype=torch.int8, device=DEV), torch.empty(M, device=DEV)
    lse = torch.empty(M, hq, device=DEV)
    ops = torch.ops.qi_b200
    K.rms_norm_quant(_lib.KIND_INT8, x, w)  # registers the operators
    rope, store = (x, k, pos, freqs, axes, D, False), (x, k, v, pos, freqs, axes, D, kc, vc, slots, False, None, None)
    packed, paged = (x, k, v, c, c, hq, hk, True, None), (x, kc, vc, table, n, None, None, None)
    for op, args in [
        (ops.rms_norm_quant.fresh, (0, x, w, None, 1e-6, None, new(x))),
        (ops.rms_norm_quant.fresh, (1, x, w, k.repeat(1, 2), 1e-6, new(x), None)),
        (ops.rms_norm_quant.out, (0, x, w, None, 1e-6, None, q8, s8, None)),
        (ops.rms_norm_quant.default, (0, x, w, None, 1e-6, None, q8, None, None)),
        (ops.rope_axes.fresh, rope), (ops.rope_axes.out, rope + (new(x), new(k))),
        (ops.rope_axes.default, rope + (new(x), None)),
        (ops.rope_axes_store.fresh, store + (None,)), (ops.rope_axes_store.out, store + (new(x), new(k))),
        (ops.rope_axes_store.default, store + (new(x), None)),
        (ops.attention_packed.fresh, packed + (lse,)), (ops.attention_packed.out, packed + (new(x), None)),
        (ops.attention_packed.default, packed + (new(x), None)),
        (ops.attention_paged.fresh, paged + (lse,)), (ops.attention_paged.out, paged + (new(x), None)),
        (ops.attention_paged.default, paged + (new(x), None)),
    ]:
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("dynamic", [False, True])
def test_operators_in_a_compiled_function(dynamic):
    """A decoder step traced as one graph (no breaks) gives the eager step's results, caches and residual stream."""
    g = gen(22)
    hq, hk, D, page = 4, 2, 64, 16
    w = randn(g, hq * D)
    wq = randn(g, hq * D, (hq + 2 * hk) * D, mul=0.05)
    freqs, axes = K.rope_axes_frequencies((D // 2,), device=DEV)

    def step(x, y, kc, vc, pos, slots, c, table, n):
        xn = torch.empty_like(x)
        q8, s8 = K.rms_norm_quant(_lib.KIND_FP8_E4M3, x, w, y, xn=xn)
        q, k, v = (xn @ wq).split([hq * D, hk * D, hk * D], 1)
        q2, k2 = K.rope_axes(q, k, pos, freqs, axes, D)
        K.rope_axes_store(q, k, v, pos, freqs, axes, D, kc, vc, slots, out_q=q, out_k=k)
        a = K.attention_packed(q, k, v, c, c, hq, hk)
        b = K.attention_paged(q, kc, vc, table, n)
        return q8, s8, q2, k2, a, b + a

    compiled = torch.compile(step, backend="aot_eager", fullgraph=True, dynamic=dynamic)
    for T in (40, 56):
        x, y = randn(g, T, hq * D), randn(g, T, hq * D)
        pages = -(-T // page)
        state = [randn(g, pages * page, hk * D).view(pages, page, hk, D) for _ in range(2)]
        pos = torch.arange(T, device=DEV)
        rest = (pos, torch.randperm(pages * page, generator=g)[:T].to(DEV), cu([T - 9, 9]),
                torch.randint(0, pages, (T, pages), generator=g).to(torch.int32).to(DEV),
                torch.randint(1, T, (T,), generator=g).to(torch.int32).to(DEV))
        runs = []
        for fn in (compiled, step):
            mine = [t.clone() for t in (x, y, *state)]
            out = fn(*mine, *rest)
            runs.append([*out, *mine])
        for i, (a, b) in enumerate(zip(*runs)):
            assert torch.equal(a, b), i
