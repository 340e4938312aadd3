"""The 8-bit integer (W8A8) path against its definition in 64 bits: row quantisers, read-back, integer product, and the
feed-forward block they make together."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
FLOOR = 2.0 ** -120


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, seed, dtype=F32):
    return torch.randn(shape, generator=_gen(seed), device="cuda").to(dtype)


def _codes(rows, k, seed):
    from velogb10_b200.quant import codec
    return codec.rows16(torch.randint(-127, 128, (rows, k), generator=_gen(seed), device="cuda").to(torch.int8))


def _check_rows(act, y, n, rel, err):
    """``act`` holds the quantised rows ``y`` (fp64). ``rel`` bounds the relative error of a value the kernel quantised
    (and so of the scale, plus its own two roundings); a code is off by half a step, plus that error in steps."""
    from velogb10_b200.ops import lib
    torch.cuda.synchronize()
    lib.check_err_word()
    s = (y.abs().amax(-1) / 127).clamp_min(FLOOR)
    got = act.scale[:n].double()
    assert ((got - s).abs() <= (rel + 2 * 2.0 ** -24) * s).all(), err
    off = (act.q[:n].double() * got[:, None] - y).abs() / got[:, None]
    assert off.max().item() <= 0.5 + 127 * (2 * rel + 4 * 2.0 ** -24), (err, off.max().item())
    assert (act.q[:n].abs().amax(-1) <= 127).all()


# every width class: one element, odd, below a vector, one CTA with one / two groups a thread, clusters of 2, 4 and 8
WIDTHS = [1, 7, 8, 255, 512, 4111, 5120, 8192, 8200, 16384, 17408, 17411, 40000, 131071]


@pytest.mark.parametrize("k", WIDTHS)
@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_quantise_rows(k, dtype):
    from velogb10_b200.ops import int8 as I8
    for n in (1, 5):
        x = _randn((n, k), k + n, dtype)
        _check_rows(I8.quantize_act_int8(x), x.double(), n, 0.0, (k, n))


@pytest.mark.parametrize("k", WIDTHS)
def test_swiglu_rows(k):
    from velogb10_b200.ops import int8 as I8
    for n in (1, 3):
        gu = (_randn((n, 2 * k), 3 * k + n) * 3).to(BF)
        g, u = gu[:, :k].double(), gu[:, k:].double()
        # e^-g to 2 + 1.173 |g| ulp (|g| < 20 here: 26 * 2^-23), quotient 2 ulp, two products
        _check_rows(I8.swiglu_int8(gu), g * torch.sigmoid(g) * u, n, 30 * 2.0 ** -23, (k, n))


@pytest.mark.parametrize("h", WIDTHS)
@pytest.mark.parametrize("delta,plus_one,f16", [(True, True, True), (False, False, False), (True, False, False), (False, True, True)])
def test_add_rmsnorm_rows(h, delta, plus_one, f16):
    from velogb10_b200.ops import int8 as I8
    for n in (1, 4):
        res, d = _randn((n, h), h + n, BF), _randn((n, h), 7 * h + n, BF) if delta else None
        w = _randn((h,), 11 * h) * 0.2 + (0.0 if plus_one else 1.0)
        out16 = torch.empty((n, h), dtype=F16, device="cuda") if f16 else None
        want = (res.double() + d.double()).to(BF) if delta else res.clone()
        act = I8.add_rmsnorm_int8(res, d, w, 1e-6, out16=out16, plus_one=plus_one)
        x = want.double()
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (w.double() + (1.0 if plus_one else 0.0))
        # sum of squares: 16 terms a thread, 5 + 5 shuffles, 8 ranks, the square: 35 roundings, halved by the root;
        # reciprocal root 2 ulp; mean, eps, (w + 1) and two products: 5 roundings
        rel = (35 / 2 + 2 * 2 + 5) * 2.0 ** -24
        _check_rows(act, y, n, rel, (h, n))
        assert torch.equal(res, want)
        if f16:
            assert ((out16.double() - y).abs() <= y.abs() * (2.0 ** -11 + rel) + 2.0 ** -24).all()


def test_rows_with_strides_and_spare_rows():
    """Views with a pitch, an unaligned start, and buffers with more rows than are asked for."""
    from velogb10_b200.ops import int8 as I8
    for off, k in ((0, 512), (3, 512), (8, 509), (0, 17408)):
        base = _randn((9, 2 * k + 40), k + off, BF)
        x = base[:, off:off + k]
        out = I8.act_buffers(12, k, "cuda")
        out.q.fill_(99)
        out.scale.fill_(-1.0)
        I8.quantize_act_int8(x, n=7, out=out)
        _check_rows(out, x[:7].double(), 7, 0.0, (off, k))
        assert (out.q[7:] == 99).all() and (out.scale[7:] == -1).all()
        gu = base[:, off:off + 2 * k]
        act = I8.swiglu_int8(gu, n=2)
        g, u = gu[:2, :k].double(), gu[:2, k:].double()
        _check_rows(act, g * torch.sigmoid(g) * u, 2, 30 * 2.0 ** -23, (off, k))
        keep = base.clone()
        w = torch.zeros(k + 1, device="cuda")[1:]                    # 4-byte aligned weights
        act = I8.add_rmsnorm_int8(x, x.clone(), w, 1e-6, n=3, out=out)
        y = (x[:3].double())
        assert torch.equal(x[:3], (keep[:3, off:off + k].float() * 2).to(BF)) and torch.equal(base[3:], keep[3:])
        _check_rows(act, y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6), 3, 27 * 2.0 ** -24, (off, k))
        back = torch.full((9, k + 3), 5.0, dtype=F32, device="cuda")
        I8.dequantize_act_int8(out, n=3, out=back[:, 2:2 + k])
        assert torch.equal(back[:3, 2:2 + k], out.q[:3].float() * out.scale[:3, None])
        assert (back[3:] == 5).all() and (back[:, :2] == 5).all() and (back[:, 2 + k:] == 5).all()


@pytest.mark.parametrize("off", range(8))
@pytest.mark.parametrize("k", [1, 5, 9, 24, 250, 263, 4111, 16391])
def test_rows_at_every_offset(off, k):
    """Rows and codes that start anywhere: every distance from a 16-byte boundary, for the input, the residual that is written
    back, the codes and the f16 copy, with nothing touched next to them."""
    from velogb10_b200.ops import int8 as I8
    n, pitch = 5, k + off + 3
    for dtype in (BF, F16, F32):
        x = _randn((n, pitch), k + off, dtype)[:, off:off + k]
        q = torch.full((n, pitch), 77, dtype=torch.int8, device="cuda")
        act = I8.quantize_act_int8(x, out=I8.Int8Act(q[:, off // 2:off // 2 + k], torch.empty(n, device="cuda")))
        _check_rows(act, x.double(), n, 0.0, (off, k, dtype))
        assert (q[:, :off // 2] == 77).all() and (q[:, off // 2 + k:] == 77).all()
        assert torch.equal(I8.quantize_act_int8(x.contiguous()).q, act.q)
    res = _randn((n, pitch), off, BF)
    delta, w = _randn((n, k + 1), off + 9, BF)[:, 1:], _randn((k + off,), off)[off:] * 0.1
    keep, out16 = res.clone(), torch.full((n, pitch), 5.0, dtype=F16, device="cuda")
    act = I8.add_rmsnorm_int8(res[:, off:off + k], delta, w, 1e-6, out16=out16[:, 2:2 + k])
    x = (keep[:, off:off + k].double() + delta.double()).to(BF)
    assert torch.equal(res[:, off:off + k], x)
    assert torch.equal(res[:, :off], keep[:, :off]) and torch.equal(res[:, off + k:], keep[:, off + k:])
    y = x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-6) * (1 + w.double())
    _check_rows(act, y, n, 27 * 2.0 ** -24, (off, k))
    assert ((out16[:, 2:2 + k].double() - y).abs() <= y.abs() * (2.0 ** -11 + 27 * 2.0 ** -24) + 2.0 ** -24).all()
    assert (out16[:, :2] == 5).all() and (out16[:, 2 + k:] == 5).all()
    gu = _randn((n, 2 * k + off), off + 3, BF)[:, off:]
    g, u = gu[:, :k].double(), gu[:, k:].double()
    _check_rows(I8.swiglu_int8(gu), g * torch.sigmoid(g) * u, n, 30 * 2.0 ** -23, (off, k))
    for dtype in (BF, F16, F32):
        out = torch.full((n, pitch), 3.0, dtype=dtype, device="cuda")
        I8.dequantize_act_int8(act, out=out[:, off:off + k])
        assert torch.equal(out[:, off:off + k], I8.dequantize_act_int8(act, dtype=dtype))
        assert torch.equal(out[:, off:off + k], (act.q.float() * act.scale[:, None]).to(dtype))
        assert (out[:, :off] == 3).all() and (out[:, off + k:] == 3).all()


# rows enough for the ring of whole rows: several blocks an SM, two, one, and one of two halves; with and without a tail
@pytest.mark.parametrize("n,k", [(1184, 8), (1300, 512), (2777, 2048), (1200, 5120), (150, 8200), (333, 17408), (149, 20480), (301, 12800)])
def test_many_rows(n, k):
    from velogb10_b200.ops import int8 as I8
    spare = 3
    for dtype in (BF, F16, F32):
        x = _randn((n + spare, k), k, dtype)
        out = I8.act_buffers(n + spare, k, "cuda")
        out.q.fill_(99)
        I8.quantize_act_int8(x, n=n, out=out)
        _check_rows(out, x[:n].double(), n, 0.0, (n, k, dtype))
        assert (out.q[n:] == 99).all()
        for r in (0, n // 2, n - 1):                         # a row's bits do not depend on the form
            one = I8.quantize_act_int8(x[r:r + 1])
            assert torch.equal(one.q[0], out.q[r]) and torch.equal(one.scale[0], out.scale[r])
    gu = (_randn((n + spare, 2 * k), k + 1) * 3).to(BF)
    act = I8.swiglu_int8(gu, n=n)
    g, u = gu[:n, :k].double(), gu[:n, k:].double()
    _check_rows(act, g * torch.sigmoid(g) * u, n, 30 * 2.0 ** -23, (n, k))
    res, delta, w = _randn((n + spare, k), 3, BF), _randn((n + spare, k), 4, BF), _randn((k,), 5) * 0.2
    for d in (delta, None):
        x = res.clone()
        want = (res.double() + d.double()).to(BF) if d is not None else res
        out16 = torch.empty((n, k), dtype=F16, device="cuda") if d is not None else None
        act = I8.add_rmsnorm_int8(x, d, w, 1e-6, n=n, out16=out16)
        y = want[:n].double()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * (1 + w.double())
        # per thread at most 40 terms, then 10 shuffles: 51 roundings halved, and 9 more
        rel = (51 / 2 + 9) * 2.0 ** -24
        _check_rows(act, y, n, rel, (n, k))
        assert torch.equal(x[:n], want[:n]) and torch.equal(x[n:], res[n:])
        if out16 is not None:
            assert ((out16.double() - y).abs() <= y.abs() * (2.0 ** -11 + rel) + 2.0 ** -24).all()
    x = _randn((n, k), 6, BF)
    x[n // 3] = float("nan")
    x[n - 1] = 0
    act = I8.quantize_act_int8(x)
    assert act.scale[n // 3].isnan() and (act.q[n // 3] == 0).all() and float(act.scale[n - 1]) == FLOOR
    assert act.scale.isnan().sum() == 1


def test_wide_rows_under_load():
    """Two halves of a block share a ring of three rows whose copies may land in any order: the same bits every time, with
    other kernels (on another stream, and the read-back right behind) competing for memory."""
    from velogb10_b200.ops import int8 as I8, lib
    n, k = 4096, 17408
    gu = torch.randn((n, 2 * k), generator=_gen(0), device="cuda").to(BF)
    want = I8.swiglu_int8(gu)
    for r in (0, 1, 147, 148, 149, 1000, n - 1):
        one = I8.swiglu_int8(gu[r:r + 1])
        assert torch.equal(one.q[0], want.q[r]) and torch.equal(one.scale[0], want.scale[r])
    side, noise = torch.cuda.Stream(), torch.empty_like(gu)
    for i in range(20):
        if i % 2:
            with torch.cuda.stream(side):
                noise.copy_(gu)
        act = I8.swiglu_int8(gu)
        back = I8.dequantize_act_int8(act)
        assert torch.equal(act.q, want.q) and torch.equal(act.scale, want.scale)
        assert back.isfinite().all()
    torch.cuda.synchronize()
    lib.check_err_word()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("k", [1, 8, 33, 4096, 131071])
def test_read_back(dtype, k):
    from velogb10_b200.ops import int8 as I8
    act = I8.Int8Act(_codes(3, k, k), torch.tensor([0.5, 1e-3, 700.0], device="cuda"))
    got = I8.dequantize_act_int8(act, dtype=dtype)
    want = act.q.float() * act.scale[:, None]
    assert torch.equal(got, want.clamp(-65504, 65504).to(dtype) if dtype == F16 else want.to(dtype))


def test_rows_that_are_zero_tiny_or_not_finite():
    from velogb10_b200.models.weights import QLinear
    from velogb10_b200.ops import int8 as I8
    for k in (64, 67, 20000):
        x = _randn((6, k), k)
        x[0] = 0.0
        x[1] *= 1e-37                                               # below the scale's floor
        x[2, k // 2] = float("inf")
        x[3, k - 1] = float("nan")
        x[4] = 3e38
        act = I8.quantize_act_int8(x)
        assert (act.q[0] == 0).all() and float(act.scale[0]) == FLOOR
        assert float(act.scale[1]) == FLOOR and (act.q[1].double() * FLOOR - x[1].double()).abs().max() <= 0.5001 * FLOOR
        assert (act.q[2:4] == 0).all() and act.scale[2:4].isnan().all()
        assert (act.q[4] == 127).all() and act.scale[4].isfinite()
        assert I8.dequantize_act_int8(act)[2:4].isnan().all() and I8.dequantize_act_int8(act, dtype=F16)[2:4].isnan().all()
        q = QLinear.from_dense(_randn((40, k), k + 1), "int8")
        out = I8.linear_int8(q, act, out_f32=True)
        # row 4 is 3e38 * (the sum of a weight row): beyond fp32 (3.4e38) as soon as that sum exceeds 1.13
        ref = act.scale[4].double() * 127 * q.codes.double().sum(-1) * q.row_scale.double()
        assert torch.equal(out[4].isinf(), ref.abs() > 3.4028235e38) and not out[4].isnan().any()
        assert (out[0] == 0).all() and out[2:4].isnan().all() and out[5].isfinite().all() and out[:2].isfinite().all()
        gu = torch.zeros((3, 2 * k), dtype=BF, device="cuda")
        gu[0, :k], gu[0, k:] = -1e4, 1.0                             # silu underflows to zero
        gu[1, 0], gu[1, k:] = float("-inf"), 1.0
        gu[2, 0], gu[2, k] = 300.0, 2.0
        act = I8.swiglu_int8(gu)
        assert (act.q[0] == 0).all() and float(act.scale[0]) == FLOOR
        assert act.scale[1].isnan() and (act.q[1] == 0).all()
        assert int(act.q[2, 0]) == 127 and (act.q[2, 1:] == 0).all() and abs(float(act.scale[2]) - 600 / 127) < 1e-4
        res = torch.zeros((4, k), dtype=BF, device="cuda")
        res[1, 3] = float("nan")
        res[2] = 3e38                                                # the sum of squares leaves fp32
        res[3, 5] = float("inf")
        out16 = torch.empty((4, k), dtype=F16, device="cuda")
        act = I8.add_rmsnorm_int8(res, None, torch.zeros(k, device="cuda"), 1e-6, out16=out16)
        assert (act.q == 0).all() and float(act.scale[0]) == FLOOR and act.scale[1:].isnan().all()
        assert (out16[0] == 0).all() and out16[1:].isnan().all()


def _product(q, act, n, out_f32, m=None):
    from velogb10_b200.ops import int8 as I8, lib
    got = I8.linear_int8(q, act, n=n, out_f32=out_f32)
    torch.cuda.synchronize()
    lib.check_err_word()
    ref = (act.q[:n].double() @ q.codes.double().t()) * act.scale[:n].double()[:, None] * q.row_scale.double()
    # exact sum; its conversion and two products round to fp32, the store to bf16
    tol = 3.1 * 2.0 ** -24 + (0.0 if out_f32 else 2.0 ** -8)
    assert ((got.double() - ref).abs() <= tol * ref.abs()).all(), (q.m, q.k, n)
    return got


def _weights(m, k, seed):
    from velogb10_b200.models.weights import QLinear
    return QLinear("int8", m, k, codes=_codes(m, k, seed), row_scale=0.01 * (1 + torch.rand(m, generator=_gen(seed), device="cuda")))


def _tokens(n, k, seed):
    from velogb10_b200.ops import int8 as I8
    return I8.Int8Act(_codes(n, k, seed), 0.02 * (1 + torch.rand(n, generator=_gen(seed), device="cuda")))


@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (5, 17), (128, 127), (129, 129), (1001, 2063), (256, 8192), (640, 5120),
                                 (5120, 1024), (2000, 4160)])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 32, 33, 63, 65, 128, 129, 255, 256, 257, 511, 700, 1111])
def test_product(m, k, n):
    _product(_weights(m, k, m + k), _tokens(n, k, n), n, (m + n) % 2 == 0)


@pytest.mark.parametrize("m,k,n", [(34816, 5120, 1), (5120, 17408, 16), (34816, 5120, 300), (5120, 17408, 2048), (100000, 512, 7),
                                   (8192, 256, 4096), (131, 64, 70000)])
def test_product_at_model_widths(m, k, n):
    _product(_weights(m, k, 1), _tokens(n, k, 2), n, False)


def test_product_extremes_do_not_overflow():
    """Every code at its limit over the longest sum: 128 * 128 * 131071 fits 32 bits."""
    from velogb10_b200.models.weights import QLinear
    from velogb10_b200.ops import int8 as I8
    k = I8.MAX_K
    for n in (1, 40, 300):
        q, act = _weights(130, k, 3), _tokens(n, k, 4)
        q.codes.fill_(-128)
        act.q.fill_(-128)
        q.codes[1::2] = 127
        _product(q, act, n, True)
        assert float(I8.linear_int8(q, act, out_f32=True)[0, 0]) > 0 > float(I8.linear_int8(q, act, out_f32=True)[0, 1])


def test_product_does_not_depend_on_the_batch():
    from velogb10_b200.ops import int8 as I8
    for m, k in ((5120, 4160), (1001, 2063), (300, 300)):
        q, act = _weights(m, k, 5), _tokens(1030, k, 6)
        whole = I8.linear_int8(q, act)
        for n in (1, 3, 16, 17, 50, 128, 200, 257, 600):
            assert torch.equal(I8.linear_int8(q, act, n=n), whole[:n]), (m, k, n)
        one = I8.linear_int8(q, I8.Int8Act(act.q[1029:], act.scale[1029:]))
        assert torch.equal(one[0], whole[1029])
        assert torch.equal(I8.linear_int8(q, act), whole)


def test_product_into_views_leaves_the_rest_alone():
    from velogb10_b200.ops import int8 as I8
    for m, k, n in ((200, 64, 3), (129, 300, 20), (1000, 512, 290)):
        q, act = _weights(m, k, 7), _tokens(n + 5, k, 8)
        for dtype in (BF, F32):
            buf = torch.full((n + 4, m + 9), 3.0, dtype=dtype, device="cuda")
            view = buf[1:, 5:5 + m]
            I8.linear_int8(q, act, n=n, out=view)
            assert torch.equal(view[:n], I8.linear_int8(q, act, n=n, out_f32=dtype == F32))
            buf[1:n + 1, 5:5 + m] = 3.0
            assert (buf == 3).all()
        # wide pitches on the inputs
        wide = torch.zeros((m, 2 * ((k + 15) // 16 * 16)), dtype=torch.int8, device="cuda")
        wide[:, :k] = q.codes
        q2 = type(q)("int8", m, k, codes=wide[:, :k], row_scale=q.row_scale)
        assert torch.equal(I8.linear_int8(q2, act, n=n), I8.linear_int8(q, act, n=n))


def _spread(t, pitch):
    """The matrix with its rows `pitch` elements apart; what lies between is never touched."""
    buf = torch.empty((t.shape[0] - 1) * pitch + t.shape[1], dtype=t.dtype, device="cuda")
    view = buf.as_strided(t.shape, (pitch, 1))
    view.copy_(t)
    return view


@pytest.mark.parametrize("n,k,pitch", [(3, 264, (1 << 30) + 64), (3, 263, (1 << 30) + 48), (1200, 264, 1800016)])
def test_offsets_past_32_bits(n, k, pitch):
    """Rows that start more than 2^31 elements into their buffer, few of them and many: the bits of near rows. These start
    at the same places within 16 bytes, since the order of the norm's sum goes by that."""
    from velogb10_b200.ops import int8 as I8
    assert (n - 1) * pitch > 1 << 31 and pitch % 16 == 0
    far, near = (lambda t: _spread(t, pitch)), (lambda t: _spread(t, 1072))
    x, d, gu, w = _randn((n, k), 1, BF), _randn((n, k), 3, BF), _randn((n, 2 * k), 2, BF), _randn((k,), 4)
    got = []
    for place in (far, near):
        out = I8.Int8Act(place(torch.zeros((n, k), dtype=torch.int8, device="cuda")), torch.zeros(n, device="cuda"))
        f16, res, r = place(torch.zeros((n, k), dtype=F16, device="cuda")), place(x), []
        I8.quantize_act_int8(res, out=out)
        r += [out.q.clone(), out.scale.clone()]
        I8.dequantize_act_int8(out, out=f16)
        r += [f16.clone()]
        I8.swiglu_int8(place(gu), out=out)
        r += [out.q.clone(), out.scale.clone()]
        I8.add_rmsnorm_int8(res, place(d), w, 1e-6, out=out, out16=f16)
        got.append(r + [out.q.clone(), out.scale.clone(), f16.clone(), res.clone()])
    _check_rows(I8.Int8Act(got[0][0], got[0][1]), x.double(), n, 0.0, (n, k))
    assert [torch.equal(a, b) for a, b in zip(*got)] == [True] * 9


@pytest.mark.parametrize("m,k,n,pitch", [(136, 264, 3, (1 << 30) + 64), (264, 520, 70, (1 << 25) + 16), (200, 264, 1200, 1800016)])
def test_product_offsets_past_32_bits(m, k, n, pitch):
    """Tokens and results (and with three tokens weights too) that lie beyond 2^31 elements."""
    from velogb10_b200.ops import int8 as I8
    assert (n - 1) * pitch > 1 << 31
    q, act = _weights(m, k, 5), _tokens(n, k, 6)
    want = I8.linear_int8(q, act)
    far = I8.Int8Act(_spread(act.q, pitch), act.scale)
    out = _spread(torch.zeros_like(want), pitch)
    wide = type(q)("int8", m, k, codes=_spread(q.codes, 1 << 24), row_scale=q.row_scale)
    I8.linear_int8(wide, far, out=out)
    assert torch.equal(out, want)


def test_first_call_may_not_be_captured(monkeypatch):
    from velogb10_b200.ops import int8 as I8, lib
    x = torch.zeros((1, 16), device="cuda")
    monkeypatch.setattr(I8, "_err", {})
    monkeypatch.setattr(lib, "_err_words", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(lib.KernelError, match="before capturing"):
        I8.quantize_act_int8(x)
    monkeypatch.undo()
    I8.quantize_act_int8(x)


def test_calls_on_two_streams_at_once():
    """Every form of the product and the quantisers in flight on two streams: nothing is shared between calls."""
    from velogb10_b200.ops import int8 as I8, lib
    jobs = []
    for i, (m, k, n) in enumerate(((5120, 4160, 3), (640, 5120, 40), (1001, 2063, 203), (5120, 6144, 256), (5120, 1024, 1200))):
        q, x = _weights(m, k, i), _randn((n, k), i, BF)
        act = I8.quantize_act_int8(x)
        jobs.append((q, x, act.q.clone(), act.scale.clone(), I8.linear_int8(q, act)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for r in range(10):
        for i, (q, x, *_) in enumerate(jobs):
            with torch.cuda.stream(streams[(r + i) % 2]):
                act = I8.quantize_act_int8(x)
                got.append((i, act, I8.linear_int8(q, act)))
    torch.cuda.synchronize()
    lib.check_err_word()
    for i, act, out in got:
        _, _, codes, scale, want = jobs[i]
        assert torch.equal(act.q, codes) and torch.equal(act.scale, scale) and torch.equal(out, want), i


def test_no_rows():
    from velogb10_b200.ops import int8 as I8
    act = I8.quantize_act_int8(torch.zeros((0, 64), device="cuda"))
    assert act.q.shape == (0, 64) and I8.linear_int8(_weights(8, 64, 0), act).shape == (0, 8)
    assert I8.dequantize_act_int8(act).shape == (0, 64)
    assert I8.swiglu_int8(torch.zeros((4, 64), dtype=BF, device="cuda"), n=0).q.shape == (0, 32)


def _block(res, delta, w, gate_up, down):
    from velogb10_b200.ops import int8 as I8
    act = I8.add_rmsnorm_int8(res, delta, w, 1e-6)
    act = I8.swiglu_int8(I8.linear_int8(gate_up, act))
    return I8.linear_int8(down, act)


@pytest.mark.parametrize("n,h,inter", [(1, 256, 512), (16, 2048, 512), (33, 640, 1111), (300, 1000, 776)])
def test_feed_forward_block(n, h, inter):
    """The operators as a decoder layer runs them, on their own stream and as a replayed graph: the same bits."""
    from velogb10_b200.models.weights import QLinear
    from velogb10_b200.ops import lib
    gate_up = QLinear.from_dense(_randn((2 * inter, h), 1) / h ** 0.5, "int8")
    down = QLinear.from_dense(_randn((h, inter), 2) / inter ** 0.5, "int8")
    w, res, delta = _randn((h,), 3) * 0.1, _randn((n, h), 4, BF), _randn((n, h), 5, BF)
    res0 = res.clone()
    out = _block(res, delta, w, gate_up, down)
    torch.cuda.synchronize()
    lib.check_err_word()
    # the same definition in 64 bits, rounded where the operators store bf16
    x = (res0.double() + delta.double()).to(BF).double()
    assert torch.equal(res.double(), x)
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1 + w.double())

    def quantised(y, q):
        s = (y.abs().amax(-1, keepdim=True) / 127)
        return torch.round(y / s) * s @ (q.codes.double() * q.row_scale.double()[:, None]).t()

    gu = quantised(y, gate_up).to(BF).double()
    g, u = gu[:, :inter], gu[:, inter:]
    ref = quantised(g * torch.sigmoid(g) * u, down)
    # a code that falls on the other side of a tie moves a value by one step (1 / 127 of the row's largest) in a few
    # places out of k: far below the rounding of the bf16 output, which is 2^-8 of each value
    assert ((out.double() - ref).norm() / ref.norm()).item() <= 2.0 ** -8
    # another stream
    res2, side = res0.clone(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out2 = _block(res2, delta, w, gate_up, down)
    side.synchronize()
    assert torch.equal(out2, out) and torch.equal(res2, res)
    # two captured graphs that share nothing, replayed on changed inputs
    res3, res4 = res0.clone(), res0.clone()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out3 = _block(res3, delta, w, gate_up, down)
    with torch.cuda.graph(g2):
        out4 = _block(res4, delta, w, gate_up, down)
    res3.copy_(res0)
    res4.copy_(res0 * 2)
    g1.replay()
    g2.replay()
    torch.cuda.synchronize()
    assert torch.equal(out3, out) and torch.equal(res3, res)
    res5 = res0 * 2
    assert torch.equal(out4, _block(res5, delta, w, gate_up, down)) and torch.equal(res4, res5)
    lib.check_err_word()


def _exact_codes(y):
    """rint(127 y / max|y|), half to even: in 64 bits the product is exact, and a quotient of 24-bit numbers that is not a half
    lies 2^-33 or more of its size away from one."""
    amax = y.double().abs().amax(-1, keepdim=True).clamp_min(127 * FLOOR)
    return torch.round(y.double() * 127 / amax).to(torch.int8), (amax / torch.full_like(amax, 127.0)).float().squeeze(-1)


# row form (whole words, shifted, two groups a thread, clusters) and ring form (several blocks an SM, one)
@pytest.mark.parametrize("n,k", [(64, 6144), (64, 4111), (700, 4111), (9, 20000), (9, 17411), (1300, 512), (1200, 5120), (333, 17408)])
@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_exact_halves_round_to_even(n, k, dtype):
    from velogb10_b200.ops import int8 as I8
    from velogb10_b200.quant import codec
    x = _randn((n, k), 3 * n + k, BF).to(dtype)                     # bf16 values in every type: halves are frequent
    ratio = x.double() * 254 / x.double().abs().amax(-1, keepdim=True)
    assert ((ratio == ratio.round()) & (ratio % 2 == 1)).sum() > n * k // 50000
    act = I8.quantize_act_int8(x)
    codes, scale = _exact_codes(x)
    assert torch.equal(act.scale, scale)
    assert torch.equal(act.q, codes)
    q = codec.quantize_int8(x)                                      # weight rows: the same rule
    assert torch.equal(q.codes, codes) and torch.equal(q.row_scale, scale)


def test_codes_next_to_a_half_are_decided_exactly():
    """fp32 values at a half and one and two fp32 steps beside it, for every code and several largest values; tiny rows at the
    floor of the scale and rows near the end of fp32 among them."""
    from velogb10_b200.ops import int8 as I8
    h = torch.arange(-127, 127, dtype=F64, device="cuda") + 0.5
    rows = []
    for amax in (1.0, 127.0, 1.9999999, 3.3e38, 0.7, 1e-30, 2.0 ** -100, 127 * FLOOR, 3 * 127 * FLOOR / 4):
        a = torch.tensor(amax, dtype=F32, device="cuda")
        y = (h * a.double().clamp_min(127 * FLOOR) / 127).float()
        near = [y]
        for way in (float("inf"), -float("inf")):
            b = y
            for _ in range(2):
                b = torch.nextafter(b, torch.full_like(b, way))
                near.append(b)
        t = torch.cat(near).clamp(-a, a)
        rows.append(torch.cat([t, a[None]]))
    x = torch.stack(rows)
    codes, scale = _exact_codes(x)
    for w in (x, torch.cat([x, torch.zeros_like(x)], 1)[:, :x.shape[1] + 1].contiguous()):
        act = I8.quantize_act_int8(w)
        assert torch.equal(act.scale, scale)
        assert torch.equal(act.q[:, :x.shape[1]], codes)


@pytest.mark.parametrize("dtype,bits,exps", [(BF, 8, (-110, -3, 99, 110, 120)), (F16, 11, (-14, 4))])
def test_every_pair_of_16_bit_significands(dtype, bits, exps):
    """All values whose code is not 0, against all largest values: exact quotients, exact halves, rows near the end of the range."""
    from velogb10_b200.ops import int8 as I8
    sig = torch.arange(1 << (bits - 1), 1 << bits, dtype=F64, device="cuda")
    vals = torch.cat([sig * 2.0 ** -e for e in range(9)])
    vals = torch.cat([vals, -vals])
    for exp in exps:
        x = (vals[None, :] * 2.0 ** (exp - bits + 1) * (vals.abs()[None, :] <= sig[:, None])).to(dtype)     # f16: subnormals among them
        act = I8.quantize_act_int8(x)
        codes, scale = _exact_codes(x)
        assert torch.equal(act.scale, scale) and torch.equal(act.q, codes), exp


# ring form (one, two, four groups a thread) against the row form alone and in clusters; odd widths; every start within 16 bytes
@pytest.mark.parametrize("n,k", [(1300, 256), (1300, 2048), (1200, 5120), (150, 8200), (170, 17408), (149, 20480), (7, 40000),
                                 (1200, 2051), (300, 8209), (5, 131071)])
def test_norm_of_a_row_does_not_depend_on_the_call(n, k):
    """A row's codes, scale and f16 copy have the same bits alone, among a few and among many, with and without a residual
    update, aligned or not."""
    from velogb10_b200.ops import int8 as I8
    res, w = _randn((n, k), k, BF) * 3, _randn((k,), n) * 0.3
    many, f16 = res.clone(), torch.empty((n, k), dtype=F16, device="cuda")
    act = I8.add_rmsnorm_int8(many, None, w, 1e-6, out16=f16)
    rows = sorted({0, 1, 2, 3, n // 2, n - 2, n - 1})
    for lo, hi in [(r, r + 1) for r in rows] + [(0, min(n, 5)), (n // 3, min(n, n // 3 + 100))]:
        for off in (0, 1, 3, 4):
            x = torch.zeros((hi - lo, k + 8), dtype=BF, device="cuda")[:, off:off + k]
            x.copy_(res[lo:hi])
            d, o = (torch.zeros_like(x), torch.empty((hi - lo, k), dtype=F16, device="cuda"))
            got = I8.add_rmsnorm_int8(x, d if off else None, w, 1e-6, out16=o)
            assert torch.equal(got.q, act.q[lo:hi]) and torch.equal(got.scale, act.scale[lo:hi]) and torch.equal(o, f16[lo:hi]), (lo, hi, off)
    _check_rows(act, res.double() * torch.rsqrt(res.double().square().mean(-1, keepdim=True) + 1e-6) * (1 + w.double()), n,
                27 * 2.0 ** -24, (n, k))


@pytest.mark.parametrize("n,k", [(1300, 512), (1200, 5120), (150, 8200), (333, 17408), (149, 20480)])
def test_swiglu_of_a_row_does_not_depend_on_the_call(n, k):
    from velogb10_b200.ops import int8 as I8
    gu = _randn((n, 2 * k), k, BF) * 2
    act = I8.swiglu_int8(gu)
    for lo, hi in ((0, 1), (n - 1, n), (n // 2, n // 2 + 40)):
        for off in (0, 1):
            x = torch.zeros((hi - lo, 2 * k + 8), dtype=BF, device="cuda")[:, off:off + 2 * k]
            x.copy_(gu[lo:hi])
            got = I8.swiglu_int8(x)
            assert torch.equal(got.q, act.q[lo:hi]) and torch.equal(got.scale, act.scale[lo:hi]), (lo, hi, off)


def test_without_pytorchs_private_calls(monkeypatch):
    from velogb10_b200.ops import int8 as I8, lib
    x, q = _randn((5, 300), 1, BF), _weights(64, 300, 2)
    want = I8.linear_int8(q, I8.quantize_act_int8(x))
    monkeypatch.setattr(lib, "_raw_stream", None)
    monkeypatch.setattr(lib, "_empty_strided_cuda", None)
    monkeypatch.setattr(lib, "current_index", torch.cuda.current_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert lib.raw_stream(0) == side.cuda_stream
        got = I8.linear_int8(q, I8.quantize_act_int8(x))
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("eps", [2.0 ** -100, 1e-12, 1.0, 2.0 ** 127])
@pytest.mark.parametrize("k", [64, 67, 20000])
def test_norm_over_the_range_of_eps(eps, k):
    """Zero rows, rows whose squares leave fp32 at the lower end, ordinary ones; the largest eps leaves only rows of 0."""
    from velogb10_b200.ops import int8 as I8
    x = _randn((5, k), k, BF)
    for r, e in enumerate((-140, -60, -49, 0)):
        x[r] = (x[r].double() * 2.0 ** e).to(BF)
    x[4] = 0
    w = _randn((k,), 1) * 0.2
    act = I8.add_rmsnorm_int8(x, None, w, eps)
    # subnormal inputs count as zero (less than 2^-126 of eps^(1/2) or more)
    y = torch.where(x.double().abs() < 2.0 ** -126, 0.0, x.double())
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * (1 + w.double())
    _check_rows(act, y, 5, 27 * 2.0 ** -24, (eps, k))
    assert float(act.scale[4]) == FLOOR and act.scale.isfinite().all()


@pytest.mark.parametrize("n,k", [(1300, 512), (1200, 5120), (150, 8200), (333, 17408), (149, 20480)])
def test_rows_of_infinities_and_nan_among_many(n, k):
    """Forms for many rows: such a row gives scale NaN, codes 0 and an f16 row of NaN, its residual is updated like any other,
    and its neighbours have the bits they have without it."""
    from velogb10_b200.ops import int8 as I8, lib
    res, delta, w = _randn((n, k), 1, BF), _randn((n, k), 2, BF), _randn((k,), 3) * 0.2
    clean, clean16 = res.clone(), torch.empty((n, k), dtype=F16, device="cuda")
    want = I8.add_rmsnorm_int8(clean, delta, w, 1e-6, out16=clean16)
    bad = {0: float("nan"), 1: float("inf"), n // 2: float("-inf"), n - 1: float("nan")}
    dirty_d = delta.clone()
    for r, v in bad.items():
        dirty_d[r, (r * 37) % k] = v
    x, out16 = res.clone(), torch.zeros((n, k), dtype=F16, device="cuda")
    act = I8.add_rmsnorm_int8(x, dirty_d, w, 1e-6, out16=out16)
    good = torch.ones(n, dtype=torch.bool, device="cuda")
    good[list(bad)] = False
    assert act.scale[~good].isnan().all() and (act.q[~good] == 0).all() and out16[~good].isnan().all()
    sums = (res.double() + dirty_d.double()).to(BF)
    assert torch.equal(x.isnan(), sums.isnan()) and torch.equal(x.nan_to_num(7.0), sums.nan_to_num(7.0))
    assert torch.equal(act.q[good], want.q[good]) and torch.equal(act.scale[good], want.scale[good]) and torch.equal(out16[good], clean16[good])
    gu = _randn((n, 2 * k), 4, BF)
    want = I8.swiglu_int8(gu)
    for r, v in bad.items():
        gu[r, (r * 37) % (2 * k)] = v
    act = I8.swiglu_int8(gu)
    assert act.scale[~good].isnan().all() and (act.q[~good] == 0).all()
    assert torch.equal(act.q[good], want.q[good]) and torch.equal(act.scale[good], want.scale[good])
    torch.cuda.synchronize()
    lib.check_err_word()
