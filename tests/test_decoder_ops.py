"""The decoder-block operators on CPU: what they refuse (the checks of types,
shapes and strides run before the tensors' device is asked for, so CPU tensors
reach them), the C ABI's own checks, and the index arithmetic of the two
attention kernels' work splits, restated here."""

import ctypes
import random

import pytest
import torch

from qi_b200 import _lib, build, kernels as K

BF = torch.bfloat16
I8, FP8, BF16 = _lib.KIND_INT8, _lib.KIND_FP8_E4M3, _lib.KIND_BF16


@pytest.fixture(scope="module", autouse=True)
def _libraries():
    build.build()
    build.build_torch_ops()


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


X = z(4, 256)
W = z(256)
F, A = torch.zeros(64, dtype=torch.float64), torch.zeros(64, dtype=torch.int32)
POS, SLOTS = z(4, dtype=torch.int32), z(4, dtype=torch.int64)
KC, K1 = z(2, 4, 1, 128), X[:, :128]
U8 = z(2, 4, 1, 128, dtype=torch.uint8)
S1 = torch.ones(1)
CU = torch.tensor([0, 4], dtype=torch.int32)
PT, LEN = z(4, 2, dtype=torch.int32), z(4, dtype=torch.int32)


def store(q=X, k=K1, v=K1, kc=KC, vc=KC, slots=SLOTS, D=128, **kw):
    return K.rope_axes_store(q, k, v, POS, F, A, D, kc, vc, slots, **kw)


def packed(q=X, k=X, v=X, cu_q=CU, cu_k=CU, heads=2, kv_heads=2, **kw):
    return K.attention_packed(q, k, v, cu_q, cu_k, heads, kv_heads, **kw)


def paged(q=X, kc=KC, vc=KC, pages=PT, lengths=LEN, **kw):
    return K.attention_paged(q, kc, vc, pages, lengths, **kw)


REFUSED = [
    (lambda: K.rms_norm_quant(9, X, W), "unknown kind"),
    (lambda: K.rms_norm_quant(I8, X.float(), W), "x must be a 2-D bfloat16"),
    (lambda: K.rms_norm_quant(I8, X[0], W), "x must be 2-D"),
    (lambda: K.rms_norm_quant(I8, X[:, :250], W[:250]), "D % 8"),
    (lambda: K.rms_norm_quant(I8, z(1, 16392), z(16392)), "D <= 16384"),
    (lambda: K.rms_norm_quant(I8, X[:, 1:249], W[:248]), "16-byte aligned rows"),
    (lambda: K.rms_norm_quant(I8, X[:1].expand(4, 256), W), "do not overlap"),
    (lambda: K.rms_norm_quant(I8, X.t().contiguous().t(), W), "unit column stride"),
    (lambda: K.rms_norm_quant(I8, X, W[:128]), "weight must be"),
    (lambda: K.rms_norm_quant(I8, X, W.float()), "weight must be"),
    (lambda: K.rms_norm_quant(I8, X, W, X[:3]), "y must be"),
    (lambda: K.rms_norm_quant(I8, X, W, x_out=X), "x_out needs y"),
    (lambda: K.rms_norm_quant(I8, X, W, X, x_out=X[:3]), "x_out must be"),
    (lambda: K.rms_norm_quant(I8, X, W, eps=-1.0), "eps"),
    (lambda: K.rms_norm_quant(I8, X, W, q=z(4, 256, dtype=torch.uint8)), "q must be"),
    (lambda: K.rms_norm_quant(FP8, X, W, q=z(4, 256, dtype=torch.int8)), "q must be"),
    (lambda: K.rms_norm_quant(FP8, X, W, s=torch.zeros(3)), "s must be"),
    (lambda: K.rms_norm_quant(BF16, X, W), "writes xn only"),
    (lambda: K.rms_norm_quant(BF16, X, W, xn=X, s=torch.zeros(4)), "writes xn only"),
    (lambda: K.rms_norm_quant(I8, X, W, xn=X[:3]), "xn must be"),
    (lambda: K.rms_norm_quant(I8, X, W), "x must be a CUDA tensor"),
    (lambda: K.rope_axes_frequencies((), device="cpu"), "sections"),
    (lambda: K.rope_axes_frequencies((8, 0), device="cpu"), "sections"),
    (lambda: K.rope_axes(X, None, POS[:3], F, A, 128), "positions must be"),
    (lambda: K.rope_axes(X, None, POS.float(), F, A, 128), "int32 or int64"),
    (lambda: K.rope_axes(X, None, z(0, 4, dtype=torch.int32), F, A, 128), "positions must be"),
    (lambda: K.rope_axes(X, None, POS, F.float(), A, 128), "freqs must be"),
    (lambda: K.rope_axes(X, None, POS, F, A.long(), 128), "axes must be"),
    (lambda: K.rope_axes(X, None, POS, F[:60], A[:60], 128), "multiple of 8 pairs"),
    (lambda: K.rope_axes(X, None, POS, F, A, 64), "at most 32"),
    (lambda: K.rope_axes(X, None, POS, F, A, 96), "q must be"),
    (lambda: K.rope_axes(X, None, POS, F, A, 100), "head_dim"),
    (lambda: K.rope_axes(X, X[:, :64], POS, F, A, 128), "k must be"),
    (lambda: K.rope_axes(X, None, POS, F, A, 128, out_k=X), "out_k needs k"),
    (lambda: K.rope_axes(X, None, POS, F, A, 128, out_q=X[:3]), "out_q must be"),
    (lambda: K.rope_axes(X, K1, POS, F, A, 128), "q must be a CUDA tensor"),
    (lambda: store(v=None), "needs k, v and slots"),
    (lambda: store(vc=KC[:1]), "both caches alike"),
    (lambda: store(slots=SLOTS[:3]), "slots must be"),
    (lambda: store(slots=SLOTS.float()), "int32 or int64"),
    (lambda: store(k=X, v=X), "must hold 2 heads"),
    (lambda: store(kc=KC.half(), vc=KC.half()), "the cache must be"),
    (lambda: store(kc=U8, vc=U8), "needs k_scale"),
    (lambda: store(kc=U8, vc=U8, k_scale=S1, v_scale=torch.ones(2)), "v_scale must be"),
    (lambda: store(k_scale=S1), "belongs to an E4M3 cache"),
    (lambda: store(kc=KC[:0], vc=KC[:0]), "at least one token"),
    (lambda: store(), "q must be a CUDA tensor"),
    (lambda: store(kc=U8, vc=U8, k_scale=S1, v_scale=S1), "q must be a CUDA tensor"),
    (lambda: packed(heads=4, kv_heads=3), "evenly"),
    (lambda: packed(heads=3), "q must be"),
    (lambda: packed(heads=1, kv_heads=1), "head_dim must be 64 or 128"),
    (lambda: packed(kv_heads=1), "k must be"),
    (lambda: packed(v=X[:3]), "v must be"),
    (lambda: packed(cu_q=CU.long()), "cu_q must be"),
    (lambda: packed(cu_k=torch.zeros(3, dtype=torch.int32)), "cu_k must be"),
    (lambda: packed(cu_q=CU[:0], cu_k=CU[:0]), "one value more"),
    (lambda: packed(scale=0.0), "scale"),
    (lambda: packed(scale=float("nan")), "scale"),
    (lambda: packed(scale=float("inf")), "scale"),
    (lambda: packed(lse=torch.zeros(4, 3)), "lse must be"),
    (lambda: packed(out=X[:3]), "out must be"),
    (lambda: packed(), "q must be a CUDA tensor"),
    (lambda: paged(pages=PT[:3]), "pages must be"),
    (lambda: paged(pages=PT.long()), "pages must be"),
    (lambda: paged(pages=PT[:1].expand(4, 2)), "pages must be"),
    (lambda: paged(lengths=LEN[:3]), "lengths must be"),
    (lambda: paged(lengths=LEN.long()), "lengths must be"),
    (lambda: paged(kc=KC[0], vc=KC[0]), "k_cache must be"),
    (lambda: paged(kc=KC[..., :96], vc=KC[..., :96]), "q must be"),
    (lambda: paged(kc=KC[..., 4:68], vc=KC[..., 4:68]), "16-byte aligned heads"),
    (lambda: paged(v_scale=S1), "belongs to an E4M3 cache"),
    (lambda: paged(kc=U8, vc=U8, k_scale=S1), "needs v_scale"),
    (lambda: paged(q=z(4, 192), kc=z(2, 4, 2, 64), vc=z(2, 4, 2, 64)), "evenly"),
    (lambda: paged(scale=-1.0), "scale"),
    (lambda: paged(), "q must be a CUDA tensor"),
]


@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_refused(i):
    call, message = REFUSED[i]
    with pytest.raises(ValueError) as e:
        call()
    assert message in str(e.value), str(e.value)


def test_frequencies():
    f, a = K.rope_axes_frequencies((2, 3), theta=100.0, device="cpu")
    assert a.tolist() == [0, 0, 1, 1, 1]
    assert f.tolist() == pytest.approx([1.0, 0.1, 1.0, 100 ** (-1 / 3), 100 ** (-2 / 3)], rel=1e-15)
    f, a = K.rope_axes_frequencies((2, 3), theta=100.0, shared=True, device="cpu")
    assert f.tolist() == pytest.approx([100 ** (-i / 5) for i in range(5)], rel=1e-15)


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: for machines without a device")
def test_c_abi_refuses_before_it_touches_the_device():
    """Every bad argument of the C entries is answered without a CUDA call (there is no device here)."""
    lib = _lib.load()
    p = 0x1000  # a 16-byte aligned address that is never read
    norm = lambda kind=I8, x=p, ldx=64, y=None, ldy=0, h=None, ldh=0, w=p, q=p, s=p, xn=None, M=2, D=64, eps=1e-6: \
        lib.qi_b200_rms_norm_quant(kind, x, ldx, y, ldy, h, ldh, w, q, s, xn, M, D, eps, None)
    assert norm(M=0) == _lib.OK
    assert norm(M=-1) == norm(D=60) == norm(D=16392, ldx=16392) == norm(ldx=56) == norm(ldx=68) == _lib.ESHAPE
    assert norm(kind=5) == norm(x=None) == norm(q=None) == norm(y=p, ldy=64) == norm(kind=BF16) == _lib.EINVAL
    assert norm(x=p + 8) == norm(q=p + 4) == norm(w=p + 2) == _lib.EALIGN
    assert norm() == _lib.ECUDA  # nothing left to refuse: the device is asked for

    c = _lib.PagedCache(k=p, v=p, pages=4, page_size=16)
    c.page_stride[:] = (2048, 2048)
    c.slot_stride[:] = (128, 128)
    c.head_stride[:] = (128, 128)
    ref = ctypes.byref
    rope = lambda q=p, ldq=128, k=p, v=p, pos=p, pairs=64, M=2, heads=1, kv=1, D=128, cache=c, slots=p: \
        lib.qi_b200_rope_axes(q, ldq, k, 128, v, 128, p, 128, None, 0, pos, 0, p, p, pairs, 1, 0, M, heads, kv, D,
                              None if cache is None else ref(cache), slots, 0, None)
    assert rope(M=0) == _lib.OK
    assert rope(pairs=60) == rope(pairs=72) == rope(D=120) == rope(heads=0) == rope(ldq=120) == _lib.ESHAPE
    assert rope(pos=None) == rope(v=None) == rope(slots=None) == rope(cache=None) == _lib.EINVAL
    assert rope(q=p + 8) == rope(v=p + 8) == _lib.EALIGN
    assert rope() == _lib.ECUDA
    for field, value, status in (("k", None, _lib.EINVAL), ("page_size", 0, _lib.ESHAPE), ("pages", -1, _lib.ESHAPE),
                                 ("v", p + 8, _lib.EALIGN), ("fp8", 1, _lib.EINVAL)):
        old = getattr(c, field)
        setattr(c, field, value)
        assert rope() == status, field
        setattr(c, field, old)
    c.slot_stride[1] = 100
    assert rope() == _lib.EALIGN
    c.slot_stride[1] = 128

    packed_ = lambda q=p, k=p, ldq=256, n=1, tq=4, heads=2, kv=1, D=128, scale=1.0, cu=p, ws=None: \
        lib.qi_b200_attention_packed(q, ldq, k, 128, p, 128, p, 256, None, cu, p, n, tq, 4, heads, kv, D, 1, scale,
                                     ws, 1 << 30, None)
    assert packed_(n=0) == packed_(tq=0) == _lib.OK
    assert packed_(D=96) == packed_(heads=3, kv=2) == packed_(ldq=128) == packed_(ldq=260) == _lib.ESHAPE
    assert packed_(q=None) == packed_(k=None) == packed_(cu=None) == packed_(scale=0.0) == _lib.EINVAL
    assert packed_(scale=float("nan")) == packed_(scale=float("inf")) == _lib.EINVAL
    assert packed_(tq=0x3fffffff) == _lib.ETOOBIG
    assert packed_(k=p + 8) == packed_(ws=p + 8) == _lib.EALIGN
    size = ref(ctypes.c_size_t())
    assert lib.qi_b200_attention_packed_workspace_bytes(1, 4, 4, 3, 2, 128, size) == _lib.ESHAPE
    assert lib.qi_b200_attention_packed_workspace_bytes(1, 4, 4, 2, 2, 96, size) == _lib.ESHAPE
    assert lib.qi_b200_attention_packed_workspace_bytes(1, 4, 4, 2, 2, 128, None) == _lib.EINVAL
    assert packed_() == _lib.ECUDA

    paged_ = lambda q=p, B=2, heads=2, kv=1, D=128, mp=4, ld=4, ws=p, scale=1.0, nb=1 << 30: \
        lib.qi_b200_attention_paged(q, 256, ref(c), p, ld, mp, p, p, 256, None, B, heads, kv, D, scale, ws, nb, None)
    assert paged_(B=0) == _lib.OK
    assert paged_(D=32) == paged_(B=65536) == paged_(heads=3, kv=2) == paged_(ld=3) == _lib.ESHAPE
    assert paged_(q=None) == paged_(ws=None) == paged_(scale=-1.0) == paged_(scale=float("inf")) == _lib.EINVAL
    assert paged_(q=p + 8) == paged_(ws=p + 8) == _lib.EALIGN
    assert paged_(mp=1 << 28, ld=1 << 28) == _lib.ETOOBIG  # lengths of 2^32 tokens
    assert paged_() == _lib.ECUDA
    assert lib.qi_b200_attention_paged_workspace_bytes(1, 96, ref(ctypes.c_size_t())) == _lib.ESHAPE
    assert lib.qi_b200_attention_paged_workspace_bytes(1, 128, None) == _lib.EINVAL


def test_device_error_names_bad_indexes():
    e = _lib.QiB200DeviceError((2, 0x800, 1, 7))
    assert "out of range" in str(e) and "timed out" not in str(e)
    assert "timed out" in str(_lib.QiB200DeviceError((1, 0x800, 1, 7)))


@pytest.mark.parametrize("seed", range(6))
def test_paged_ranges_cover_every_unit_once(seed):
    """The cut of T units into min(T, CTAs) ranges: none empty, the owner formula names the range of every unit, and
    an item's ranges are consecutive, its first part the only one that may lie at a range's end."""
    rng = random.Random(seed)
    ctas = rng.choice((1, 3, 148))
    items = [rng.randint(1, rng.choice((2, 40, 900))) for _ in range(rng.randint(1, 50))]
    T = sum(items)
    G = min(T, ctas)
    lo = [c * T // G for c in range(G + 1)]
    assert lo[0] == 0 and lo[G] == T and all(a < b for a, b in zip(lo, lo[1:]))
    owner = lambda u: ((u + 1) * G - 1) // T
    for u in range(T):
        assert lo[owner(u)] <= u < lo[owner(u) + 1]
    u0 = 0
    used = set()
    for n in items:
        c0, c1 = owner(u0), owner(u0 + n - 1)
        if c0 != c1:
            for c in range(c0, c1 + 1):  # workspace place of each part: 1 where the item begins, 0 where it goes on
                place = (c, 1 if lo[c] <= u0 else 0)
                assert (place[1] == 1) == (c == c0)
                assert place not in used
                used.add(place)
        u0 += n


@pytest.mark.parametrize("seed", range(6))
def test_packed_items_are_taken_once_longest_first(seed):
    """The order of the packed attention's items (level by level, sequences in chunks of 32, back and forth over the
    CTAs): every (sequence, query block, head item) is taken by exactly one CTA, and a CTA's levels descend."""
    rng = random.Random(seed)
    lens = [rng.choice((0, 1, 128, 129, rng.randint(1, 3000))) for _ in range(rng.choice((1, 5, 33, 70)))]
    rows, heads, G = rng.choice((128, 256)), rng.choice((1, 3, 8)), rng.choice((1, 7, 148))
    blocks = [-(-n // rows) for n in lens]
    seen = []

    def walk(cta):
        level, chunk, base, rnd = max(blocks) - 1, 0, 0, 0
        active = lambda: [b for b in range(chunk, min(chunk + 32, len(lens))) if blocks[b] > level]
        while level >= 0:
            target = rnd * G + (G - 1 - cta if rnd & 1 else cta)
            while target >= base + len(active()) * heads:
                base += len(active()) * heads
                chunk += 32
                if chunk >= len(lens):
                    chunk, level = 0, level - 1
                    if level < 0:
                        return
            rnd += 1
            i = target - base
            yield active()[i // heads], level, i % heads

    for cta in range(G):
        mine = list(walk(cta))
        assert [m[1] for m in mine] == sorted((m[1] for m in mine), reverse=True)
        seen += mine
    assert sorted(seen) == sorted((b, l, h) for b in range(len(lens)) for l in range(blocks[b]) for h in range(heads))


# ---------------------------------------------------------------------------
# tracing: results from shapes alone, and schemas that say what is written
# ---------------------------------------------------------------------------

OPS = ("rms_norm_quant", "rope_axes", "rope_axes_store", "attention_packed", "attention_paged")


def decoder_calls(dev):
    """(call, [(shape, dtype)] of its results) for every form of every operator; ``dev`` makes the tensors."""
    e = lambda *shape, dtype=BF: torch.empty(*shape, dtype=dtype, device=dev)
    i32, i64, f32 = torch.int32, torch.int64, torch.float32
    x, w, f, a = e(4, 256), e(256), e(64, dtype=torch.float64), e(64, dtype=i32)
    qkv = e(4, 512)
    q, k, v = qkv.split([256, 128, 128], 1)
    pos, slots = e(4, dtype=i32), e(4, dtype=i64)
    kc, k8 = e(2, 4, 1, 128), e(2, 4, 1, 128, dtype=torch.uint8)
    s1, cu, table, n = e(1, dtype=f32), e(2, dtype=i32), e(4, 2, dtype=i32), e(4, dtype=i32)
    q8, s, lse = e(4, 256, dtype=torch.int8), e(4, dtype=f32), e(4, 2, dtype=f32)
    row, kv = ((4, 256), BF), ((4, 128), BF)
    i8, u8, sc = ((4, 256), torch.int8), ((4, 256), torch.uint8), ((4,), f32)
    rope = lambda k=k, **kw: K.rope_axes(q, k, pos, f, a, 128, **kw)
    store = lambda c=kc, **kw: K.rope_axes_store(q, k, v, pos, f, a, 128, c, c, slots, **kw)
    packed = lambda **kw: K.attention_packed(q, k, v, cu, cu, 2, 1, **kw)
    paged = lambda c=kc, **kw: K.attention_paged(q, c, c, table, n, **kw)
    fp8 = dict(c=k8, k_scale=s1, v_scale=s1)
    return [
        (lambda: K.rms_norm_quant(I8, x, w), [i8, sc]),
        (lambda: K.rms_norm_quant(FP8, x, w, q, x_out=e(4, 256)), [u8, sc]),
        (lambda: K.rms_norm_quant(I8, x, w, q), [i8, sc]),
        (lambda: K.rms_norm_quant(I8, x, w, q, q=q8), [i8, sc]),
        (lambda: K.rms_norm_quant(I8, x, w, s=s, xn=e(4, 256)), [i8, sc]),
        (lambda: K.rms_norm_quant(I8, x, w, q=q8, s=s), [i8, sc]),
        (lambda: K.rms_norm_quant(BF16, x, w, xn=e(4, 256)), [None, None]),
        (lambda: rope(), [row, kv]),
        (lambda: rope(k=None), [row, None]),
        (lambda: rope(out_q=q), [row, kv]),
        (lambda: rope(out_k=k), [row, kv]),
        (lambda: rope(out_q=q, out_k=k), [row, kv]),
        (lambda: store(), [row]),
        (lambda: store(out_q=q, out_k=k), [row]),
        (lambda: store(out_k=k, **fp8), [row]),
        (lambda: packed(), [row]),
        (lambda: packed(lse=lse), [row]),
        (lambda: packed(out=e(4, 256), lse=lse), [row]),
        (lambda: paged(), [row]),
        (lambda: paged(lse=lse, **fp8), [row]),
        (lambda: paged(out=e(4, 256)), [row]),
    ]


def check_shapes(call, want, device):
    got = call()
    got = got if isinstance(got, tuple) else (got,)
    assert [None if t is None else (tuple(t.shape), t.dtype) for t in got] == want
    assert all(t is None or t.device.type == device for t in got)


@pytest.mark.parametrize("i", range(21))
def test_fake_and_meta_tensors(i):
    """Tracing sees every form's results by shape, without data: fake CUDA tensors (as torch.compile makes them) and
    meta tensors."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    assert len(decoder_calls("meta")) == 21
    check_shapes(*decoder_calls("meta")[i], "meta")
    with FakeTensorMode():
        check_shapes(*decoder_calls("cuda")[i], "cuda")


def test_fake_tensors_of_wrong_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        e = lambda *shape, dtype=BF: torch.empty(*shape, dtype=dtype, device="cuda")
        f, a, i = e(64, dtype=torch.float64), e(64, dtype=torch.int32), e(4, dtype=torch.int32)
        for call in (lambda: K.rms_norm_quant(I8, e(256), e(256)), lambda: K.rope_axes(e(4, 200), None, i, f, a, 128),
                     lambda: K.attention_packed(e(4, 256), e(4, 256), e(4, 256), i, i, 3, 3),
                     lambda: K.attention_paged(e(4, 256), e(2, 4, 128), e(2, 4, 128), e(4, 2), i)):
            with pytest.raises(ValueError, match="must be"):
                call()


@pytest.mark.parametrize("name", OPS)
def test_schemas_say_what_is_written_and_returned(name):
    from qi_b200 import torch_ops

    torch_ops.load()
    packet = getattr(torch.ops.qi_b200, name)
    assert sorted(packet.overloads()) == ["default", "fresh", "out"]
    fresh, out = packet.fresh._schema, packet.out._schema
    assert fresh.returns and all(r.alias_info is None for r in fresh.returns)
    assert not out.returns
    written = {"rms_norm_quant": {"x_out", "q", "s", "xn"}, "rope_axes": {"out_q", "out_k"},
               "rope_axes_store": {"k_cache", "v_cache", "out_q", "out_k"}, "attention_packed": {"out", "lse"},
               "attention_paged": {"out", "lse"}}[name]
    mutable = lambda schema: {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write}
    assert mutable(out) == written and mutable(fresh) < written
    # the form that takes either: what it returns may be the argument that it names
    whole = packet.default._schema
    sets = {a.name: a.alias_info.before_set for a in whole.arguments if a.alias_info is not None}
    returned = [next(n for n, b in sets.items() if b == r.alias_info.before_set) for r in whole.returns]
    assert returned == {"rms_norm_quant": ["q", "s"], "rope_axes": ["out_q", "out_k"], "rope_axes_store": ["out_q"],
                        "attention_packed": ["out"], "attention_paged": ["out"]}[name]


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: for machines without a device")
def test_c_abi_flags_of_packed_attention():
    """Flags other than the two are refused; without sequences there is work only where rows are to become zeros."""
    call = lambda flags, n=1, out=0x1000: _lib.load().qi_b200_attention_packed(
        0x1000, 256, 0x1000, 128, 0x1000, 128, out, 256, None, 0x1000, 0x1000, n, 4, 4, 2, 1, 128, flags, 1.0, None, 0, None)
    assert call(4) == call(-1) == _lib.EINVAL
    assert call(0, n=0) == call(1, n=0, out=None) == _lib.OK
    assert call(3, n=0, out=None) == call(2, out=None) == _lib.EINVAL
    assert call(2, n=0) == call(3) == _lib.ECUDA  # the device is asked for


def test_scales_that_overflow_in_powers_of_two():
    """A finite scale whose product with log2(e) is not: it would make every score of zero a NaN."""
    edge = 3.4028234e38 / 1.4426950408889634
    for call in (packed, paged):
        for scale in (edge * 1.00001, 3.4e38):
            with pytest.raises(ValueError, match="scale must be"):
                call(scale=scale)
        with pytest.raises(ValueError, match="CUDA tensor"):
            call(scale=edge * 0.99999)


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: for machines without a device")
def test_c_abi_scales_that_overflow_in_powers_of_two():
    lib, p = _lib.load(), 0x1000
    c = _lib.PagedCache(k=p, v=p, pages=4, page_size=16)
    for field in (c.page_stride, c.slot_stride, c.head_stride):
        field[:] = (128, 128)
    for scale, status in ((2.4e38, _lib.EINVAL), (2.3e38, _lib.ECUDA)):  # log2(e) 2.36e38 is the largest number
        assert lib.qi_b200_attention_packed(p, 256, p, 128, p, 128, p, 256, None, p, p, 1, 4, 4, 2, 1, 128, 1, scale,
                                            None, 0, None) == status
        assert lib.qi_b200_attention_paged(p, 256, ctypes.byref(c), p, 4, 4, p, p, 256, None, 2, 2, 1, 128, scale, p,
                                           1 << 30, None) == status
