"""8-bit operators on the GPU: kernels against 64-bit arithmetic and against their plain forms, at the sizes, layouts and
values where they can go wrong; the training path that uses them."""
import pytest
import torch

from dcp_b200.ops import fp8_ops as F
from dcp_b200.ops import optim_ops as O

pytestmark = pytest.mark.gpu
E4M3, E5M2 = F.E4M3, F.E5M2
TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # half a step, relative


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def _status():
    yield
    if torch.cuda.is_available():
        F.check_status()


def _bits(t):
    return t.contiguous().view(torch.uint8)


def _same(q, p):
    """Codes and scales bit by bit; zeros of either sign and all NaN count as one."""
    a, b = q.codes.float(), p.codes.float()
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(1e9), b.nan_to_num(1e9))
    assert q.block == p.block and torch.equal(_bits(q.scales), _bits(p.scales))


def _values(rows, cols, dtype, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, cols, device=dev, generator=g) * torch.exp2(torch.randint(-6, 6, (rows, 1), device=dev, generator=g).float())
    if rows > 2:
        x[rows // 2] = 0
    return x.to(dtype)


# --------------------------------------------------------------------------- codes
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("code", [E4M3, E5M2])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (2, 127), (127, 128), (128, 129), (129, 136), (300, 1000), (257, 1001)])
def test_quantize(dev, dtype, code, rows, cols):
    x = _values(rows, cols, dtype, dev)
    for block in ((1, 128), (128, 1), (128, 128)):
        _same(F.quantize(x, block, code), F.quantize_reference(x, block, code))
    for q, block in zip(F.quantize_both(x, code), ((1, 128), (128, 1))):
        _same(q, F.quantize_reference(x, block, code))


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_of_any_values(dev, dtype):
    """Infinities, NaN, the type's largest and smallest values, every exponent."""
    info = torch.finfo(dtype)
    x = torch.randn(260, 392, device=dev)
    x *= torch.exp2(torch.linspace(-140, 127, 260, device=dev).round())[:, None]
    x = x.to(dtype)
    x[3, 130], x[7, 5], x[200, 391] = float("nan"), float("inf"), -float("inf")
    x[11], x[12], x[13, ::2] = info.max, info.tiny, info.min
    x[14] = info.smallest_normal * info.eps
    for block in ((1, 128), (128, 1), (128, 128)):
        _same(F.quantize(x, block), F.quantize_reference(x, block))


@pytest.mark.parametrize("how", ["pitch", "odd pitch", "shifted", "columns", "one column"])
def test_quantize_of_any_layout(dev, how):
    base = _values(200, 600, torch.bfloat16, dev)
    x = {"pitch": base[:, :264], "odd pitch": base.view(-1)[:200 * 599].view(200, 599)[:, :264], "shifted": base[:, 3:259],
         "columns": base[:, :256].t(), "one column": base[:, 5:6]}[how]
    for block in ((1, 128), (128, 1), (128, 128)):
        _same(F.quantize(x, block), F.quantize_reference(x.contiguous(), block))


# --------------------------------------------------------------------------- RMSNorm
def _check_norm(x, w, eps, residual, y, h, rstd, code):
    h64 = (x.double() + residual.double()).to(x.dtype) if residual is not None else x
    # fp32 and fp64 sums of two values of x's type round to the same
    assert torch.equal(h, (x.float() + residual.float()).to(x.dtype) if residual is not None else x)
    assert residual is None or (h.double() - h64.double()).abs().max() <= (h64.double().abs().max() * 2 * HALF[x.dtype])
    r64 = torch.rsqrt(h.double().pow(2).mean(-1) + eps)
    # a mean of squares through at most 8 * 4 + 10 additions, a root and its reciprocal
    assert ((rstd.double() - r64).abs() <= r64 * 32 * 2.0 ** -23).all()
    y64 = h.double() * r64[:, None] * w.double()
    ones = y._replace(codes=torch.ones_like(y.codes)).dequantize(torch.float64)
    step, least, largest = (2.0 ** -4, 2.0 ** -10, 448.0) if code == E4M3 else (2.0 ** -3, 2.0 ** -17, 57344.0)
    slack = 36 * 2.0 ** -23
    assert ((y.dequantize(torch.float64) - y64).abs() <= torch.maximum(y64.abs() * (step + slack), ones * (least + slack * largest))).all()
    amax = torch.zeros(y64.shape[0], y.scales.shape[1] * 128, dtype=torch.float64, device=y64.device)
    amax[:, :y64.shape[1]] = y64.abs()
    amax, s = amax.view(y64.shape[0], -1, 128).amax(-1), y.scales.double()
    assert (amax <= largest * s * (1 + slack)).all() and ((amax >= largest / 2 * s * (1 - slack)) | (s == 2.0 ** -127)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 8), (3, 77), (5, 128), (299, 1000), (600, 1001), (2, 4096), (400, 5120), (7, 16384), (300, 9001)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm(dev, dtype, rows, width, with_residual):
    x, residual = _values(rows, width, dtype, dev), _values(rows, width, dtype, dev, 1) if with_residual else None
    w = (torch.randn(width, device=dev) + 1).to(dtype)
    for code in (E4M3, E5M2):
        y, h, rstd = F.rmsnorm_quant(x, w, 1e-5, residual, code)
        _check_norm(x, w, 1e-5, residual, y, h, rstd, code)


@pytest.mark.parametrize("how", ["pitch", "shifted", "columns"])
def test_norm_of_any_layout(dev, how):
    base, other = _values(300, 512, torch.bfloat16, dev), _values(300, 512, torch.bfloat16, dev, 2)
    cut = {"pitch": lambda t: t[:, :256], "shifted": lambda t: t[:, 3:259], "columns": lambda t: t[:, :256].t()}[how]
    x, res, dy = cut(base), cut(other), cut(base.flip(0))
    w = torch.randn(512 + 3, device=dev).bfloat16()[3:3 + x.shape[1]]
    y, h, rstd = F.rmsnorm_quant(x, w, 1e-5, res)
    _check_norm(x, w, 1e-5, res, y, h, rstd, E4M3)
    got = F.rmsnorm_quant_bwd(cut(base), w, rstd, dy, res)
    want = F.rmsnorm_quant_bwd(x.contiguous(), w.contiguous(), rstd, dy.contiguous(), res.contiguous())
    for a, b in zip(got, want):
        assert (a.double() - b.double()).abs().max() <= b.double().abs().max() * 2 * HALF[torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 8), (3, 77), (149, 1000), (601, 1001), (5, 4096), (700, 1024), (1000, 2048), (461, 5120),
                                        (300, 8192), (150, 12288), (7, 16384), (160, 9001)])
@pytest.mark.parametrize("with_add", [False, True])
def test_norm_backward(dev, dtype, rows, width, with_add):
    h, dy, add = (_values(rows, width, dtype, dev, s) for s in range(3))
    add = add if with_add else None
    w = (torch.randn(width, device=dev) + 1).to(dtype)
    rstd = torch.rsqrt(h.double().pow(2).mean(-1) + 1e-5).float()
    dx, dw = F.rmsnorm_quant_bwd(h, w, rstd, dy, add)
    r, xh = rstd.double()[:, None], h.double() * rstd.double()[:, None]
    g = dy.double() * w.double()
    # what is added up in fp32, in magnitudes: 60 roundings bound its sums (chains of 32 additions, trees, a few products)
    size = r * (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)) + (0 if add is None else add.double().abs())
    want = r * (g - xh * (g * xh).mean(-1, keepdim=True)) + (0 if add is None else add.double())
    assert ((dx.double() - want).abs() <= want.abs() * HALF[dtype] + size * 60 * 2.0 ** -24 + 2.0 ** -25).all()   # and fp16's denormals
    want, size = (dy.double() * xh).sum(0), (dy.double() * xh).abs().sum(0)
    # a CTA's chain of rows, then an eighth of the CTAs at a time
    assert ((dw.double() - want).abs() <= size * (rows / 100 + 150) * 2.0 ** -24).all()
    again = F.rmsnorm_quant_bwd(h, w, rstd, dy, add)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_norm_without_rows(dev):
    x = torch.zeros(0, 256, device=dev)
    y, h, rstd = F.rmsnorm_quant(x, torch.ones(256, device=dev))
    dx, dw = F.rmsnorm_quant_bwd(x, torch.ones(256, device=dev), rstd, x)
    assert y.codes.shape == (0, 256) and dx.shape == (0, 256) and torch.equal(dw, torch.zeros(256, device=dev))


def test_a_row_that_is_not_finite_leaves_the_others(dev):
    x = _values(5, 1024, torch.bfloat16, dev)
    x[1, 7], x[3, 900] = float("nan"), float("inf")
    y, _, rstd = F.rmsnorm_quant(x, torch.ones(1024, device=dev, dtype=torch.bfloat16))
    d = y.dequantize()
    assert torch.isnan(d[1]).all() and torch.isnan(d[3, 896:]).all() and torch.isfinite(d[[0, 2, 4]]).all() and torch.isnan(rstd[1])


# --------------------------------------------------------------------------- products
def _operands(m, n, k, how, dev, a_code=E4M3, b_code=E4M3, seed=0):
    a = _values(*((k, m) if how == "wgrad" else (m, k)), torch.float32, dev, seed)
    b = _values(*((n, k) if how == "forward" else (k, n)), torch.float32, dev, seed + 1)
    return (F.quantize(a, (128, 1) if how == "wgrad" else (1, 128), a_code),
            F.quantize(b, (128, 1) if how == "wgrad" else (128, 128), b_code), dict(trans_a=how == "wgrad", trans_b=how == "forward"))


def _check_product(got, a, b, kw, add=None):
    x, y = a.dequantize(torch.float64), b.dequantize(torch.float64)
    x, y = (x.t() if kw["trans_a"] else x), (y.t() if kw["trans_b"] else y)
    want, size = x @ y, x.abs() @ y.abs()
    if add is not None:
        want, size = want + add.double(), size + add.double().abs()
    # the tensor cores add 32 products to the running sum at a time and cut each result to 24 bits; a split sum is added up
    # in eight parts at most
    steps = x.shape[1] / 32 + 12
    bound = want.abs() * HALF[got.dtype] + size * steps * 2.0 ** -23
    # beyond the type's range the nearest value is infinite: fp16 ends at 65504, and what reaches 65504 + 16 rounds to infinity
    past = (want.abs() + bound >= torch.finfo(got.dtype).max * (1 + HALF[got.dtype] / 2)) & (got.double() == torch.sign(want) * float("inf"))
    ok = ((got.double() - want).abs() <= bound) | past
    assert ok.all(), ((got.double() - want).abs() / bound.clamp(min=1e-300))[~ok].max()


SIZES = [(1, 1, 1), (1, 128, 128), (16, 128, 512), (17, 300, 1000), (33, 256, 513), (64, 130, 640), (100, 200, 700), (128, 128, 128),
         (129, 257, 129), (256, 256, 256), (257, 300, 1500), (600, 1000, 2048), (700, 64, 4096)]


@pytest.mark.parametrize("how", ["forward", "dgrad", "wgrad"])
@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("form", [0, 1, 2])
def test_matmul(dev, how, m, n, k, form):
    a, b, kw = _operands(m, n, k, how, dev)
    got = F.matmul(a, b, **kw, out_dtype=torch.float32, form=form)
    _check_product(got, a, b, kw)
    assert torch.equal(F.matmul(a, b, **kw, out_dtype=torch.float32, form=form), got)


@pytest.mark.parametrize("how", ["forward", "dgrad", "wgrad"])
@pytest.mark.parametrize("m,n,k", [(5000, 4100, 640), (3, 2000, 16384), (1024, 1536, 16500)])
def test_matmul_of_many_tiles_and_long_sums(dev, how, m, n, k):
    a, b, kw = _operands(m, n, k, how, dev)
    _check_product(F.matmul(a, b, **kw, out_dtype=torch.float32), a, b, kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", [1, 2])
@pytest.mark.parametrize("m,n,k", [(30, 77, 300), (300, 520, 1030)])
def test_matmul_results_and_additions(dev, dtype, form, m, n, k):
    a, b, kw = _operands(m, n, k, "forward", dev)
    add = _values(m, n, dtype, dev, 5)
    _check_product(F.matmul(a, b, **kw, out_dtype=dtype, form=form), a, b, kw)
    _check_product(F.matmul(a, b, **kw, out_dtype=dtype, add=add, form=form), a, b, kw, add)
    # into a part of a larger tensor, whose rest stays as it was, and on top of what is there
    whole = torch.full((m + 2, n + 5), 7.0, dtype=dtype, device=dev)
    out = whole[1:-1, 3:3 + n]
    assert F.matmul(a, b, **kw, out=out, form=form) is out
    _check_product(out, a, b, kw)
    before = out.clone()
    F.matmul(a, b, **kw, out=out, add=out, form=form)
    _check_product(out, a, b, kw, before)
    whole[1:-1, 3:3 + n] = 7.0
    assert (whole == 7.0).all()


@pytest.mark.parametrize("a_code,b_code", [(E5M2, E4M3), (E4M3, E5M2), (E5M2, E5M2)])
@pytest.mark.parametrize("form", [1, 2])
def test_matmul_of_mixed_codes(dev, a_code, b_code, form):
    a, b, kw = _operands(200, 300, 400, "dgrad", dev, a_code, b_code)
    _check_product(F.matmul(a, b, **kw, out_dtype=torch.float32, form=form), a, b, kw)


@pytest.mark.parametrize("form", [1, 2])
def test_matmul_operands_of_any_layout(dev, form):
    a, b, kw = _operands(100, 200, 300, "forward", dev)
    want = F.matmul(a, b, **kw, form=form)
    plain = lambda q: q._replace(codes=q.codes.contiguous(), scales=q.scales.contiguous())  # noqa: E731  rows of 300 bytes, 3 scales
    assert torch.equal(F.matmul(plain(a), plain(b), **kw, form=form), want)
    columns = a._replace(codes=a.codes.t().contiguous().t(), scales=a.scales.t().contiguous().t())
    assert torch.equal(F.matmul(columns, b, **kw, form=form), want)
    shifted = torch.empty(100 * 304 + 8, dtype=torch.uint8, device=dev)[8:].view(E4M3).view(100, 304)[:, :300].copy_(a.codes)
    assert torch.equal(F.matmul(a._replace(codes=shifted), b, **kw, form=form), want)
    # a weight with a scale per row and block, as an activation has it
    rows = F.quantize(b.dequantize(), (1, 128))
    _check_product(F.matmul(a, rows, **kw, form=form), a, rows, kw)
    by_blocks = F.quantize(a.dequantize(), (128, 128))
    _check_product(F.matmul(by_blocks, rows, **kw, form=form), by_blocks, rows, kw)


@pytest.mark.parametrize("form", [1, 2])
def test_matmul_keeps_rows_that_are_not_finite_apart(dev, form):
    x = _values(300, 512, torch.float32, dev)
    x[7, 200], x[290, 3] = float("nan"), float("inf")
    a, b = F.quantize(x), F.quantize(_values(260, 512, torch.float32, dev, 1), (128, 128))
    got = F.matmul(a, b, form=form)
    bad = torch.isnan(got).all(1)
    assert bad.nonzero().view(-1).tolist() == [7, 290] and torch.isfinite(got[~bad]).all()


def test_matmul_extreme_scales(dev):
    """Scales at both ends of their range, whose product is representable."""
    x = torch.randn(64, 256, device=dev)
    a, b = F.quantize(x * 2.0 ** 100), F.quantize(torch.randn(96, 256, device=dev) * 2.0 ** -118, (128, 128))
    kw = dict(trans_a=False, trans_b=True)
    _check_product(F.matmul(a, b, out_dtype=torch.float32), a, b, kw)
    z = F.quantize(torch.zeros(96, 256, device=dev), (128, 128))
    assert torch.equal(F.matmul(a, z), torch.zeros(64, 96, device=dev, dtype=torch.bfloat16))


def test_captured_and_on_another_stream(dev):
    """All calls of a layer in a graph on a side stream, replayed with new inputs; the same calls eagerly meanwhile."""
    w = F.quantize(_values(384, 256, torch.bfloat16, dev, 3), (128, 128))
    nw = torch.randn(256, device=dev).bfloat16()
    x, res, dy = (_values(300, 256, torch.bfloat16, dev, s) for s in range(3))

    def layer(x, res, dy):
        y, h, rstd = F.rmsnorm_quant(x, nw, 1e-5, res)
        out = F.matmul(y, w)
        rows, cols = F.quantize_both(out)
        g = F.matmul(rows, w, trans_b=False)
        dx, dw = F.rmsnorm_quant_bwd(h, nw, rstd, g, dy)
        return out, dx, dw, F.matmul(cols, F.quantize(dy, (128, 1)), trans_a=True, trans_b=False)

    want = layer(x, res, dy)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        layer(x, res, dy)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = layer(x, res, dy)
        graph.replay()
        eager = layer(x, res, dy)
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, eager):
        assert torch.equal(a, b) and torch.equal(a, c)
    x.copy_(_values(300, 256, torch.bfloat16, dev, 8))
    graph.replay()
    for a, b in zip(layer(x, res, dy), got):
        assert torch.equal(a, b)


def test_two_threads_at_once(dev):
    import threading
    a, b, kw = _operands(300, 520, 700, "forward", dev)
    want, got = F.matmul(a, b, **kw), {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream(dev)):
            got[i] = [F.matmul(a, b, **kw) for _ in range(20)]
            torch.cuda.current_stream(dev).synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in threads], [t.join() for t in threads]
    assert all(torch.equal(o, want) for outs in got.values() for o in outs)


# --------------------------------------------------------------------------- AdamW
HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)


def _adam_state(sizes, bits, ptype, gtype, dev, offset=0, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def place(t):   # `offset` values behind an aligned address
        return torch.empty(t.numel() + offset, dtype=t.dtype, device=dev)[offset:].copy_(t)

    rnd = lambda n: torch.randn(n, device=dev, generator=g)  # noqa: E731
    params = [place(rnd(n).to(ptype)) for n in sizes]
    st = {"params": params, "grads": [place((rnd(n) * 1e-2).to(gtype)) for n in sizes],
          "masters": None if ptype == torch.float32 else [place(p.float()) for p in params],
          "step": torch.full((1,), 4, dtype=torch.int64, device=dev)}
    m, v = [rnd(n) * 1e-2 for n in sizes], [(rnd(n) * 1e-2).square() for n in sizes]
    if bits == 32:
        return {**st, "m": [place(t) for t in m], "v": [place(t) for t in v]}
    em, ev = [O.encode_state(t) for t in m], [O.encode_state(t.sqrt(), root=True) for t in v]
    return {**st, "m": [place(c) for c, _ in em], "v": [place(c) for c, _ in ev], "m_scales": [s for _, s in em], "v_scales": [s for _, s in ev]}


def _copy(st):
    return {k: [t.clone() for t in x] if isinstance(x, list) else x.clone() if torch.is_tensor(x) else x for k, x in st.items()}


def _weights(st):
    return [t.double() for t in (st["masters"] or st["params"])]


def _check_adam(st, ref, before):
    """``before``: a copy of the state before the step."""
    w, w_ref, w_old = _weights(st), _weights(ref), _weights(before)
    for i in range(len(w)):
        # The step is a sum of two terms of a handful of roundings (2^-24 each) and approximations of an ulp or two: 2^-20 of
        # its size, which is at most its length and twice lr wd w.  Then it is added to the weight, which rounds once.
        step = (w_ref[i] - w_old[i]).abs()
        if "m_scales" not in st:
            # m is a sum of two terms that may cancel; its roundings (three of 2^-24, fused or not) go by the terms' sizes
            terms = before["m"][i].double().abs() + before["grads"][i].double().abs()
            assert ((st["m"][i].double() - ref["m"][i].double()).abs() <= terms * 3 * 2.0 ** -24).all(), i
            # v is a sum of positive terms: five roundings of either
            assert ((st["v"][i].double() - ref["v"][i].double()).abs() <= ref["v"][i].double() * 10 * 2.0 ** -24).all(), i
            step = step * (terms / ref["m"][i].double().abs().clamp(min=1e-300)).clamp(min=1.0)
        step = step + 2 * HYPER["lr"] * HYPER["weight_decay"] * w_old[i].abs()
        off = (w[i] - w_ref[i]).abs()
        assert torch.equal(torch.isnan(w[i]), torch.isnan(w_ref[i]))
        assert (off <= step * 2.0 ** -20 + w_ref[i].abs() * 2.0 ** -23).logical_or(torch.isnan(off)).all(), i
        torch.testing.assert_close(st["params"][i].float(), w[i].float().to(st["params"][i].dtype).float(), rtol=0, atol=0, equal_nan=True)
        if "m_scales" in st:
            for k in ("m", "v"):
                a, b = _bits(st[k][i]), _bits(ref[k][i])
                # the plain form rounds each operation as the kernel does; a root in a million differs in its last place, which
                # moves a code where 16 random bits decide that closely
                assert (a != b).sum() <= 1 + a.numel() // 10000, (i, k)
                assert torch.equal(_bits(st[k + "_scales"][i]), _bits(ref[k + "_scales"][i])), (i, k)
    assert torch.equal(st["step"], ref["step"])


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("ptype,gtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32),
                                         (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("clip", [None, 0.5])
def test_adamw(dev, bits, ptype, gtype, clip):
    st = _adam_state([1, 7, 256, 257, 2048, 5000, 3, 100_001], bits, ptype, gtype, dev)
    ref = _copy(st)
    for i in range(3):
        for g, h in zip(st["grads"], ref["grads"]):
            g.copy_(torch.randn(g.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(i)) * 1e-2), h.copy_(g)
        before = _copy(st)
        norm = O.adamw_multi(**st, **HYPER, grad_scale=0.5, clip=clip, seed=3)
        want = O.adamw_multi_reference(**ref, **HYPER, grad_scale=0.5, clip=clip, seed=3)
        assert (norm is None) == (clip is None) and (clip is None or abs(norm.item() / want.item() - 1) < 1e-6)
        _check_adam(st, ref, before)
        ref = _copy(st)    # a code that moved does not count twice


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("offset", [1, 8])
def test_adamw_of_any_alignment(dev, bits, offset):
    st = _adam_state([5, 300, 4096, 10_001], bits, torch.bfloat16, torch.bfloat16, dev, offset)
    ref, before = _copy(st), _copy(st)
    O.adamw_multi(**st, **HYPER, clip=1.0)
    O.adamw_multi_reference(**ref, **HYPER, clip=1.0)
    _check_adam(st, ref, before)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_of_many_tensors(dev, bits):
    """More tensors than a launch takes, empty ones among them."""
    st = _adam_state([(i * 37) % 600 for i in range(300)], bits, torch.bfloat16, torch.bfloat16, dev)
    ref, before = _copy(st), _copy(st)
    norm = O.adamw_multi(**st, **HYPER, clip=0.1)
    want = O.adamw_multi_reference(**ref, **HYPER, clip=0.1)
    assert abs(norm.item() / want.item() - 1) < 1e-6
    _check_adam(st, ref, before)


def test_adamw_without_values(dev):
    st = _adam_state([0, 0], 8, torch.bfloat16, torch.bfloat16, dev)
    assert O.adamw_multi(**st, **HYPER, clip=0.1).item() == 0 and int(st["step"]) == 5


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_adamw_keeps_a_bad_gradient_to_its_element(dev, bits, bad):
    st = _adam_state([700, 2048], bits, torch.bfloat16, torch.bfloat16, dev)
    st["grads"][1][300] = bad
    ref = _copy(st)
    for _ in range(2):
        O.adamw_multi(**st, **HYPER)
    w = st["masters"][1]
    assert torch.isnan(w).nonzero().view(-1).tolist() == [300] and torch.isfinite(st["masters"][0]).all()
    if bits == 8:
        assert torch.isnan(st["m"][1].float()).nonzero().view(-1).tolist() == [300] == torch.isnan(st["v"][1].float()).nonzero().view(-1).tolist()
        clean = _copy(ref)
        clean["grads"][1][300] = 0.0
        O.adamw_multi(**ref, **HYPER), O.adamw_multi(**clean, **HYPER)
        keep = torch.arange(2048, device=dev) != 300
        assert torch.equal(_bits(ref["m"][1])[keep], _bits(clean["m"][1])[keep]) or not torch.equal(_bits(ref["m_scales"][1]), _bits(clean["m_scales"][1]))


def test_adamw_of_huge_and_tiny_moments(dev):
    """Scales beyond the range in which one factor takes a value to its code, and moments that vanish."""
    st = _adam_state([1024, 1024, 1024], 8, torch.float32, torch.float32, dev)
    for g, f in zip(st["grads"], (1e16, 1e-30, 0.0)):
        g.mul_(f)
    for k in ("m", "v"):
        for i in range(3):
            c, s = O.encode_state(torch.zeros(1024, device=dev))
            st[k][i].copy_(c), _bits(st[k + "_scales"][i]).copy_(_bits(s))
            st[k + "_scales"][i].view(torch.uint8).copy_(_bits(s))
    ref = _copy(st)
    for _ in range(2):
        before = _copy(st)
        O.adamw_multi(**st, **HYPER)
        O.adamw_multi_reference(**ref, **HYPER)
        _check_adam(st, ref, before)
        ref = _copy(st)
    assert (st["m"][2].float() == 0).all() and (st["v"][2].float() == 0).all()


def test_adamw_is_replayed_and_repeats_to_the_bit(dev):
    st = _adam_state([300, 4096, 77], 8, torch.bfloat16, torch.bfloat16, dev)
    eager = _copy(st)
    O.adamw_multi(**_copy(st), **HYPER, clip=1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = O.adamw_multi(**st, **HYPER, clip=1.0)
    for _ in range(3):
        graph.replay()
        want = O.adamw_multi(**eager, **HYPER, clip=1.0)
    assert torch.equal(norm, want) and int(st["step"]) == 7
    for k in ("params", "masters", "m", "v", "m_scales", "v_scales"):
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(st[k], eager[k])), k


def test_adamw_refuses_a_tensor_given_twice(dev):
    st = _adam_state([300, 300], 8, torch.bfloat16, torch.bfloat16, dev)
    for k in ("params", "m", "v_scales"):
        bad = _copy(st)
        bad[k][1] = bad[k][0]
        with pytest.raises(ValueError, match="given twice"):
            O.adamw_multi(**bad, **HYPER)
    with pytest.raises(ValueError, match="either clip"):
        O.adamw_multi(**st, **HYPER, clip=1.0, factor=torch.ones(1, device=dev))
    with pytest.raises(ValueError, match="tensor 1"):
        O.adamw_multi(**{**st, "grads": [st["grads"][0], st["grads"][1][::2]]}, **HYPER)


def test_refusals_on_the_gpu(dev):
    x, w = torch.zeros(4, 256, device=dev), torch.zeros(8, 256, device=dev)
    q, wq = F.quantize(x), F.quantize(w, (128, 128))
    for call, words in [
            (lambda: F.quantize(x[0]), "matrix"), (lambda: F.quantize(x.double()), "bfloat16"),
            (lambda: F.rmsnorm_quant(x, w[0].cpu()), "device"), (lambda: F.rmsnorm_quant(x, w[0, :255]), "w has to be"),
            (lambda: F.rmsnorm_quant(x, w[0], 1e-5, x.bfloat16()), "residual"),
            (lambda: F.rmsnorm_quant_bwd(x, w[0], torch.zeros(4, device=dev), x[:2]), "dy"),
            (lambda: F.matmul(q, wq._replace(codes=wq.codes.cpu(), scales=wq.scales.cpu())), "two devices"),
            (lambda: F.matmul(q, wq, out=torch.zeros(8, 4, device=dev).t()), "contiguous"),
            (lambda: F.matmul(q, wq, out=torch.zeros(1, 8, device=dev).expand(4, 8)), "contiguous"),
            (lambda: F.matmul(q, wq, add=torch.zeros(4, 8, device=dev)), "add has to be"),
            (lambda: F.matmul(q._replace(scales=q.scales[:, :1]), wq), "scales"), (lambda: F.matmul(q, wq, form=7), "form")]:
        with pytest.raises(ValueError, match=words):
            call()
    # a broadcast addition is taken, row by row
    got = F.matmul(q, wq, add=torch.ones(1, 8, device=dev, dtype=torch.bfloat16).expand(4, 8))
    assert torch.equal(got, torch.ones(4, 8, device=dev, dtype=torch.bfloat16))
    assert torch.equal(F.matmul(F.quantize(x[:0]), wq), torch.zeros(0, 8, device=dev, dtype=torch.bfloat16))
    assert torch.equal(F.matmul(F.quantize(x[:, :0]), F.quantize(w[:, :0], (128, 128))), torch.zeros(4, 8, device=dev, dtype=torch.bfloat16))


def test_a_graph_needs_one_call_before(dev, monkeypatch):
    q, wq = F.quantize(torch.zeros(4, 256, device=dev)), F.quantize(torch.zeros(8, 256, device=dev), (128, 128))
    monkeypatch.setattr(F, "_STATUS", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before capturing"):
        F.matmul(q, wq)


def test_adamw_status_and_factor(dev):
    st = _adam_state([300, 4096], 8, torch.bfloat16, torch.bfloat16, dev)
    ref, before = _copy(st), _copy(st)
    word = torch.ones(1, dtype=torch.int32, device=dev)
    O.adamw_multi(**st, **HYPER, clip=1.0, status=[torch.zeros_like(word), word])
    for k in ("params", "masters", "m", "v"):
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(st[k], before[k]))
    assert int(st["step"]) == 4
    O.adamw_multi(**st, **HYPER, factor=torch.full((1,), 0.25, device=dev), status=[torch.zeros_like(word)])
    O.adamw_multi(**ref, **HYPER, grad_scale=0.25)
    for k in ("params", "masters", "m", "v"):
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(st[k], ref[k]))


def test_optimizer_class(dev):
    params = [torch.randn(40, 33, device=dev).bfloat16(), torch.randn(500, device=dev).bfloat16()]
    opts = [O.MultiTensorAdamW([p.clone() for p in params], lr=1e-2, state_bits=b, clip_grad=1.0) for b in (8, 32)]
    ref = O.MultiTensorAdamW([p.cpu() for p in params], lr=1e-2, state_bits=8, clip_grad=1.0)
    for i in range(3):
        grads = [torch.randn(p.shape, generator=torch.Generator().manual_seed(i)).bfloat16() for p in params]
        for o in (*opts, ref):
            for p, g in zip(o.params, grads):
                p.grad = g.to(p.device)
            o.step()
    assert (opts[0].master.cpu() - ref.master).abs().max() < 1e-6 + 3 * 1e-2 * 2.0 ** -3 * (opts[0].m.cpu().float() != ref.m.float()).any()
    assert (opts[0].master - opts[1].master).abs().max() < 3 * 1e-2 * 0.6


# --------------------------------------------------------------------------- sharded optimizer
def _sharded(dev, bits, seed=0):
    from dcp_b200.parallel.dist_optimizer import FlatBuffers, ShardedAdamW
    buckets = [(0, 4096), (4096, 8 * 1001), (4096 + 8 * 1001, 8), (4096 + 8 * 1002, 8 * 3333)]
    bufs = FlatBuffers(sum(b[1] for b in buckets), dev)
    g = torch.Generator(device=dev).manual_seed(7)
    bufs.params.copy_(torch.randn(bufs.n_flat, device=dev, generator=g).bfloat16())
    return bufs, ShardedAdamW(bufs, lr=1e-2, clip_grad=0.5, buckets=buckets, state_bits=bits, seed=seed)


def _grads(bufs, i):
    g = torch.Generator(device=bufs.grads.device).manual_seed(i)
    bufs.grads.copy_(torch.randn(bufs.n_flat, device=bufs.grads.device, generator=g).bfloat16())


def test_sharded_optimizer_with_8_bit_state(dev):
    (bufs, opt), (bufs32, opt32) = _sharded(dev, 8), _sharded(dev, 32)
    params = [bufs.params[s.flat_off:s.flat_off + s.length].clone() for s in opt.shards]
    ref = {"params": params, "masters": [p.float() for p in params], "step": torch.zeros(1, dtype=torch.int64, device=dev)}
    zero = [O.encode_state(torch.zeros(p.numel(), device=dev)) for p in params]
    ref |= {"m": [c.clone() for c, _ in zero], "v": [c.clone() for c, _ in zero], "m_scales": [s.clone() for _, s in zero],
            "v_scales": [s.clone() for _, s in zero]}
    for i in range(3):
        _grads(bufs, i), _grads(bufs32, i)
        opt.step(0.5), opt32.step(0.5)
        grads = [bufs.grads[s.flat_off:s.flat_off + s.length] for s in opt.shards]
        O.adamw_multi_reference(**ref, grads=grads, lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, grad_scale=0.5,
                                clip=0.5)
        assert abs(opt.grad_norm() / opt32.grad_norm() - 1) < 1e-6
    err = (opt.master - torch.cat(ref["masters"])).abs()
    # codes that moved (see above) change a step by 2^-3 of it at most
    assert err.max() < 3 * 1e-2 * 2.0 ** -2 and (err > 1e-6).sum() < 10
    assert torch.equal(bufs.params.float(), opt.master.bfloat16().float())
    assert (opt.master - opt32.master).abs().max() < 3 * 1e-2 * 0.6


def test_sharded_8_bit_state_in_a_checkpoint(dev):
    (bufs, opt), (bufs2, opt2), (bufs3, opt3) = _sharded(dev, 8), _sharded(dev, 8), _sharded(dev, 32)
    for i in range(2):
        _grads(bufs, i)
        opt.step()
    sd = opt.state_dict()
    assert sd["m"].dtype == torch.float32 and sd["m"].device.type == "cpu"
    for o in (opt2, opt3):
        o.load_state_dict(sd)
        o.rebuild_params()
    assert all(torch.equal(opt2.state_dict()[k], sd[k]) for k in ("m", "v"))
    assert torch.equal(opt3.m.cpu(), sd["m"]) and torch.equal(opt3.v.cpu(), sd["v"])
    _grads(bufs, 5), _grads(bufs2, 5)
    opt.step(), opt2.step()
    assert torch.equal(opt.master, opt2.master) and torch.equal(bufs.params, bufs2.params)
    assert torch.equal(_bits(opt.m), _bits(opt2.m)) and torch.equal(_bits(opt.v), _bits(opt2.v))
    bufs.arena.status.fill_(1)
    before = opt.master.clone()
    opt.step()
    assert torch.equal(opt.master, before)
    bufs.arena.status.zero_()


# --------------------------------------------------------------------------- training
def _engine(dev, **kw):
    from dcp_b200.data import synth
    from dcp_b200.models.llama import tiny_config
    from dcp_b200.train import EngineConfig, TrainEngine
    cfg = EngineConfig(tiny_config(n_layers=2, hidden=1024, n_heads=8, n_kv_heads=2, ffn=2048, vocab=512), tokens_per_step=1024,
                       block_size=512, length_dist=synth.LengthDist("lognormal", 300.0, 0.6, 64, 800), planner_workers=0, lookahead=1, **kw)
    return TrainEngine(cfg, dev)


def _gradients(eng):
    plan = eng.plans.get(0)
    toks, labels, pos = eng.stage_inputs(plan)
    eng.model.grads_flat.zero_()
    loss = eng.model.loss(toks, labels, pos, 1.0 / plan.n_global_tokens, write_grads=eng.model.layer_levels is not None)
    loss.backward()
    torch.cuda.synchronize()
    eng.check_status()
    return loss.item(), {k: t.grad.double().clone() for k, t in eng.model.p.items()}


@pytest.mark.parametrize("level", [None, 0, 1, 2])    # None: autograd and recomputation
def test_model_in_8_bits(dev, level):
    """Gradients of all parameters against the same model in bf16: a product of operands rounded to three bits is off by
    2^-4 of its size per operand at most where the errors add up, in the mean by 2^-4 / sqrt(3) * sqrt(2) = 0.05; a gradient passes
    at most eleven products one after the other: sqrt(11) * 0.05 = 0.17 in the mean, 0.35 allowed.  Levels give the same."""
    budget = -1.0 if level is None else 0.0
    eng, plain = _engine(dev, fp8=True, activation_budget_gb=budget), _engine(dev, activation_budget_gb=budget)
    try:
        if level is not None:
            eng.model.layer_levels = [level, level]
        (loss, grads), (loss0, grads0) = _gradients(eng), _gradients(plain)
        assert abs(loss - loss0) < 0.02 * loss0
        for k, g in grads.items():
            assert (g - grads0[k]).norm() <= 0.35 * grads0[k].norm(), (k, ((g - grads0[k]).norm() / grads0[k].norm()).item())
        if level:
            base = _engine(dev, fp8=True, activation_budget_gb=0.0)
            try:
                _, same = _gradients(base)
            finally:
                base.close()
            # embeddings and attention's dQ add in an order that may differ between runs
            for k, g in grads.items():
                assert (g - same[k]).norm() <= 2.0 ** -8 * same[k].norm(), k
    finally:
        eng.close()
        plain.close()


def test_training_steps_in_8_bits(dev, tmp_path):
    """Steps, a checkpoint and a resumed run with 8-bit products and 8-bit moments."""
    mk = lambda: _engine(dev, fp8=True, optimizer_state_bits=8, lr=1e-3)  # noqa: E731
    eng, other = mk(), mk()
    try:
        losses = [eng.train_step() for _ in range(3)]
        assert all(torch.isfinite(torch.tensor(losses)))
        eng.save_checkpoint(str(tmp_path))
        other.load_checkpoint(str(tmp_path))
        assert other.iteration == 3 and torch.equal(other.bufs.params, eng.bufs.params)
        a, b = eng.optimizer.state_dict(), other.optimizer.state_dict()
        assert torch.equal(a["m"], b["m"]) and torch.equal(a["v"], b["v"]) and torch.equal(a["master"], b["master"])
        assert abs(eng.train_step() - other.train_step()) < 1e-4
    finally:
        eng.close()
        other.close()


@pytest.mark.parametrize("form", [1, 2])
def test_what_a_product_is_added_to_on_the_gpu(dev, form):
    """Beside the output in one matrix, the output itself, or refused."""
    m, n, k = 130, 200, 300
    a, b = F.quantize(_values(m, k, torch.bfloat16, dev)), F.quantize(_values(n, k, torch.bfloat16, dev, 1), (128, 128))
    buf = torch.randn(m + 2, 2 * n + 3, device=dev)
    beside = buf[:m, n + 1:2 * n + 1]
    for out, add in ((buf[:m, :n], beside), (beside, buf[:m, :n]), (buf[:m, :n], buf[:m, :n])):
        want = F.matmul(a, b, out_dtype=torch.float32, add=add.clone(), form=form)
        kept = buf.clone()
        assert torch.equal(F.matmul(a, b, add=add, out=out, form=form), want)
        out.copy_(kept[:m, :n] if out.data_ptr() == buf.data_ptr() else kept[:m, n + 1:2 * n + 1])
        assert torch.equal(buf, kept)
    for out, add in ((buf[:m, :n], buf[1:m + 1, :n]), (buf[:m, :n], buf[:m, 1:n + 1]), (buf[:m, 3:n + 3], buf[2:m + 2, :n])):
        with pytest.raises(ValueError, match="lie apart"):
            F.matmul(a, b, add=add, out=out, form=form)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_refuses_overlapping_memory_and_betas_on_the_gpu(dev, bits):
    st = _adam_state([300, 300], bits, torch.bfloat16, torch.bfloat16, dev)
    kept = _copy(st)
    for key in ("params", "masters", "m", "v") + (("m_scales", "v_scales") if bits == 8 else ()):
        n, size = st[key][0].numel(), st[key][0].element_size()
        flat = torch.zeros(2 * n * size, dtype=torch.uint8, device=dev).view(st[key][0].dtype)
        for skip in (n - 1, 1):
            if skip < n:
                with pytest.raises(ValueError, match="given twice"):
                    O.adamw_multi(**{**st, **HYPER, key: [flat[skip:skip + n], flat[:n]]})
        O.adamw_multi(**{**_copy(st), **HYPER, key: [flat[n:], flat[:n]]})   # beside one another
    for bad in (dict(beta1=1.0), dict(beta2=1.0), dict(beta1=float("nan"))):
        with pytest.raises(ValueError, match="betas"):
            O.adamw_multi(**{**st, **HYPER, **bad})
    assert int(st["step"]) == int(kept["step"]) and all(torch.equal(_bits(a), _bits(b)) for a, b in zip(st["params"], kept["params"]))


def _laid(q, offset, pitch):
    """The operand with its codes `offset` bytes behind an aligned address, rows `pitch` bytes apart."""
    rows, cols = q.codes.shape
    pitch = max(pitch, cols)
    buf = torch.full((offset + rows * pitch + 64,), 0x7F, dtype=torch.uint8, device=q.codes.device)   # NaN all around
    codes = buf[offset:].as_strided((rows, cols), (pitch, 1), offset)
    codes.copy_(q.codes.contiguous().view(torch.uint8))
    return q._replace(codes=codes.view(q.codes.dtype))


@pytest.mark.parametrize("how", ["forward", "dgrad", "wgrad"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 65, 17), (33, 130, 129), (130, 257, 1001), (513, 64, 15), (300, 1030, 511)])
def test_products_of_codes_that_do_not_begin_on_16_bytes(dev, how, m, n, k):
    a, b = _values(*((k, m) if how == "wgrad" else (m, k)), torch.bfloat16, dev), _values(*((n, k) if how == "forward" else (k, n)), torch.bfloat16, dev, 1)
    qa = F.quantize(a, (128, 1) if how == "wgrad" else (1, 128))
    qb = F.quantize(b, (128, 1) if how == "wgrad" else (128, 128), E5M2)
    call = lambda a, b: F.matmul(a, b, trans_a=how == "wgrad", trans_b=how == "forward")  # noqa: E731
    want = call(qa, qb)
    assert not torch.isnan(want).any()
    for offset, extra in ((0, 0), (1, 0), (8, 3), (15, 16), (16, 1), (6, 2)):
        pa, pb = qa.codes.shape[1] + extra, qb.codes.shape[1] + extra
        for x, y in ((_laid(qa, offset, pa), _laid(qb, 16 - offset, pb)), (qa, _laid(qb, offset, pb)), (_laid(qa, offset, pa), qb)):
            assert torch.equal(call(x, y), want), (offset, extra)
    for x, y in ((qa._replace(codes=qa.codes.t().contiguous().t()), qb), (qa, qb._replace(codes=qb.codes.t().contiguous().t()))):   # by columns
        assert torch.equal(call(x, y), want)


def test_codes_laid_out_inside_a_graph_and_beside_another_stream(dev):
    m, n, k = 200, 300, 391
    qa, qb = (F.quantize(_values(r, k, torch.bfloat16, dev, r), b) for r, b in ((m, (1, 128)), (n, (128, 128))))
    x, y = _laid(qa, 3, k), _laid(qb, 5, k)
    graph, out = torch.cuda.CUDAGraph(), torch.zeros(m, n, dtype=torch.bfloat16, device=dev)
    want = F.matmul(qa, qb)
    with torch.cuda.graph(graph):
        F.matmul(x, y, out=out)
    other = F.quantize(_values(m, k, torch.bfloat16, dev, 9))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        graph.replay()
        with torch.cuda.stream(side):
            beside = F.matmul(_laid(other, 1, k), y)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(beside, F.matmul(other, qb))
    x.codes.view(torch.uint8).copy_(other.codes.contiguous().view(torch.uint8))   # a replay lays out what is there then
    x.scales.view(torch.uint8).copy_(other.scales.view(torch.uint8))
    graph.replay()
    assert torch.equal(out, F.matmul(other, qb))


def test_more_columns_than_the_kernels_count_are_refused_on_the_gpu(dev):
    from test_fp8_ops import _too_wide
    _too_wide(dev)


def _exact_adamw(st, coef, hyper=HYPER):
    """Weights and moments after a step in 64 bits, of a state before it."""
    t = int(st["step"]) + 1
    out = []
    for i, g in enumerate(st["grads"]):
        w, g = _weights(st)[i], g.double() * coef
        m, v = (st["m"][i].double(), st["v"][i].double()) if "m_scales" not in st else \
            (O.decode_state(st["m"][i], st["m_scales"][i]).double(), O.decode_state(st["v"][i], st["v_scales"][i]).double().square())
        m, v = hyper["beta1"] * m + (1 - hyper["beta1"]) * g, hyper["beta2"] * v + (1 - hyper["beta2"]) * g * g
        step = hyper["lr"] * (m / (1 - hyper["beta1"] ** t)) / ((v / (1 - hyper["beta2"] ** t)).sqrt() + hyper["eps"])
        out.append((w - step - hyper["lr"] * hyper["weight_decay"] * w, m, v, step))
    return out


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("gtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("at", [5, 9_000, 20_479, 30_001])
def test_adamw_clips_a_gradient_whose_square_fp32_does_not_hold(dev, bits, gtype, offset, at):
    st = _adam_state([300, 30_002], bits, torch.bfloat16, gtype, dev, offset)
    st["grads"][1][at] = -1e20
    before = _copy(st)
    length = sum(g.double().square().sum() for g in before["grads"]).sqrt().item()
    norm = O.adamw_multi(**st, **HYPER, clip=0.5)
    # Squares in fp32: one rounding each, four added in turn and eight of these by pairs (the first addition is to zero): seven
    # roundings at most of the sum, half of that of its root, which is rounded once.
    assert abs(norm.item() / length - 1) <= 4.5 * 2.0 ** -24
    for i, (w, m, v, step) in enumerate(_exact_adamw(before, 0.5 / (length + 1e-6))):
        # The coefficient carries the norm's error and three roundings (itself, the scaled one, the gradient's product): 8 * 2^-24
        # of m's part, 16 of v's; with the roundings of the sums below 2^-19.  m's terms may cancel.
        terms = 0.9 * (before["m"][i].double() if bits == 32 else O.decode_state(before["m"][i], before["m_scales"][i]).double()).abs() \
            + 0.1 * before["grads"][i].double().abs() * 0.5 / length
        near = step.abs() * (terms / m.abs().clamp(min=1e-300)).clamp(min=1.0) * 2.0 ** -18
        assert ((_weights(st)[i] - w).abs() <= near + w.abs() * 2.0 ** -23).all()
        if bits == 32:
            assert ((st["m"][i].double() - m).abs() <= terms * 2.0 ** -19).all() and ((st["v"][i].double() - v).abs() <= v * 2.0 ** -19).all()
    assert (_weights(st)[1][at] - _weights(before)[1][at]).item() > 0     # by about lr


@pytest.mark.parametrize("gtype,size", [(torch.float32, 1e-25), (torch.float32, 1e-41), (torch.bfloat16, 1e-25), (torch.bfloat16, 1e30), (torch.float16, 6e-8),
                                        (torch.float32, 0.0)])
def test_adamw_norm_of_tiny_and_huge_gradients(dev, gtype, size):
    st = _adam_state([77, 50_000], 32, torch.float32, gtype, dev)
    for g in st["grads"]:
        g.copy_(torch.randn(g.shape, device=dev) * size)
    want = sum(g.double().square().sum() for g in st["grads"]).sqrt().item()
    norm = O.adamw_multi(**st, **HYPER, clip=1.0).item()
    assert abs(norm - want) <= want * 4.5 * 2.0 ** -24 + 2.0 ** -150     # fp32's smallest values lie 2^-149 apart


def test_adamw_norm_of_many_values(dev):
    n = 100_000_003
    g = torch.empty(n, dtype=torch.bfloat16, device=dev).normal_(generator=torch.Generator(device=dev).manual_seed(1))
    w, m, v, step = torch.zeros(n, device=dev), torch.zeros(n, device=dev), torch.zeros(n, device=dev), torch.zeros(1, dtype=torch.int64, device=dev)
    norm = O.adamw_multi([w], [g], None, [m], [v], step, **HYPER, clip=1.0).item()
    want = sum(part.double().square().sum().item() for part in g.split(1 << 24)) ** 0.5
    assert abs(norm / want - 1) <= 4.5 * 2.0 ** -24


@pytest.mark.parametrize("gtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("size", [1e20, 2e19, 1e-16, 1e-18, 1e-19, 1e-20, 1e-21, 3e-23])
@pytest.mark.parametrize("eps", [1e-8, 1e-19, 0.0])
def test_adamw_of_second_moments_at_the_ends_of_fp32(dev, gtype, offset, size, eps):
    """A v that overflows has an infinite root and leaves its weight to the decay; one below 2^-126 keeps its root, in a block of
    its like and beside larger ones."""
    hyper = {**HYPER, "eps": eps}
    st = _adam_state([700, 2048, 5000], 8, torch.bfloat16, gtype, dev, offset)
    rnd = lambda g, seed: torch.randn(g.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed))  # noqa: E731
    for i, g in enumerate(st["grads"]):
        values = (rnd(g, i).abs() + 0.1) * rnd(g, i + 9).sign() * size
        if i == 2:
            values = values * torch.exp2((rnd(g, i + 20) * 20).clamp(max=0.0 if size > 1 else 60.0).round())
        g.copy_(values)
        for k in ("m", "v"):
            c, s = O.encode_state(rnd(g, i + 30).abs() * size if size < 1 else torch.zeros(g.shape, device=dev), root=k == "v")
            st[k][i].copy_(c), st[k + "_scales"][i].view(torch.uint8).copy_(_bits(s))
    ref = _copy(st)
    for _ in range(2):
        before = _copy(st)
        O.adamw_multi(**st, **hyper), O.adamw_multi_reference(**ref, **hyper)
        _check_adam(st, ref, before)
        if size > 1 and _ == 0:   # 0.05 g^2 passes fp32's 3.4e38 from 8.2e19 on: in hundreds of values of 1e20, hardly in one of 2e19
            assert all(torch.isfinite(w).all() for w in st["masters"])
            assert size < 1e20 or any(torch.isnan(v.float()).any() for v in st["v"])
        ref = _copy(st)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_product_that_gave_up_stops_the_optimizer(dev, bits):
    """The word is set from the host; whatever the gradients are then, the step changes nothing and the check raises."""
    eng = _engine(dev, fp8=True, optimizer_state_bits=bits)
    try:
        eng.train_step()
        opt = eng.optimizer
        state = [eng.bufs.params, opt.master, opt.m, opt.v] + ([opt.m_scale, opt.v_scale, opt.step_tensor] if bits == 8 else [])
        before = [t.clone() for t in state]
        F.status_word(dev).fill_(1)
        inputs = eng.stage_inputs(eng.plans.get(1))
        eng.run_step(*inputs, 1000)
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(state, before))
        with pytest.raises(RuntimeError, match="gave up waiting"):
            eng.check_status()
        eng.check_status()
        eng.run_step(*inputs, 1000)     # the word is cleared
        assert not torch.equal(eng.bufs.params, before[0])
    finally:
        eng.close()


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_every_status_word_stops_the_kernels_of_several_ranks(dev, which):
    """The kernels that several ranks take, as a world of one."""
    import ctypes
    from dcp_b200.ops import _lib
    from dcp_b200.ops.attention import _ptr_array
    lib, n = _lib.load(), 4096
    grads, params = torch.ones(n, device=dev).bfloat16(), torch.ones(n, device=dev).bfloat16()
    master, m, v, main, sq = (torch.ones(k, device=dev) for k in (n, n, n, n, 1))
    words = [torch.zeros(1, dtype=torch.int32, device=dev) for _ in range(4)]
    pointers = _ptr_array([w.data_ptr() for w in words])

    def run():
        f, p = ctypes.c_float, _lib.ptr
        _lib.check(lib.dcpk_grad_reduce_scatter(_ptr_array([grads.data_ptr()]), ctypes.c_int(1), ctypes.c_long(0), ctypes.c_long(n), f(2.0), p(main),
                                                p(sq), ctypes.c_int(0), pointers, ctypes.c_int(4), _lib.stream_handle()), "grad_reduce_scatter")
        _lib.check(lib.dcpk_adamw_all_gather(p(master), p(m), p(v), p(main), _ptr_array([params.data_ptr()]), ctypes.c_int(1), ctypes.c_long(0),
                                             ctypes.c_long(n), f(0.1), f(0.9), f(0.95), f(1e-8), f(0.1), ctypes.c_int(1), ctypes.c_void_p(0), pointers,
                                             ctypes.c_int(4), _lib.stream_handle()), "adamw_all_gather")
        _lib.check(lib.dcpk_fused_rs_adamw_ag(_ptr_array([grads.data_ptr()]), _ptr_array([params.data_ptr()]), ctypes.c_int(1), ctypes.c_long(0),
                                              ctypes.c_long(n), f(1.0), p(master), p(m), p(v), f(0.1), f(0.9), f(0.95), f(1e-8), f(0.1), ctypes.c_int(1),
                                              ctypes.c_void_p(0), pointers, ctypes.c_int(4), _lib.stream_handle()), "fused_rs_adamw_ag")

    words[which].fill_(1)
    run()
    assert all((t == 1).all() for t in (params, master, m, v, main, sq))
    words[which].zero_()
    run()
    assert not any((t == 1).any() for t in (params, master, main, sq))
    assert lib.dcpk_grad_reduce_scatter(_ptr_array([grads.data_ptr()]), ctypes.c_int(1), ctypes.c_long(0), ctypes.c_long(n), ctypes.c_float(1.0),
                                        _lib.ptr(main), _lib.ptr(sq), ctypes.c_int(0), pointers, ctypes.c_int(5), _lib.stream_handle()) == -3


def test_status_words_of_the_optimizers(dev):
    from dcp_b200.parallel.dist_optimizer import FlatBuffers, ShardedAdamW
    bufs = FlatBuffers(64, dev)
    word = torch.zeros(1, dtype=torch.int32, device=dev)
    for bad in ([word] * 4, torch.zeros(1, device=dev), word.cpu(), [word[:0]]):
        with pytest.raises(ValueError, match="status"):
            ShardedAdamW(bufs, extra_status=bad)
    ShardedAdamW(bufs, extra_status=word), ShardedAdamW(bufs, extra_status=(word, word, word)), ShardedAdamW(bufs)
    p = torch.ones(300, device=dev).bfloat16()
    p.grad = torch.ones_like(p)
    opt = O.MultiTensorAdamW([p], lr=0.1, state_bits=8, status=[F.status_word(dev), word])
    word.fill_(3)
    opt.step()
    assert (p == 1).all() and int(opt.step_count) == 0
    word.zero_()
    opt.step()
    assert (p != 1).all() and int(opt.step_count) == 1


def test_autograd_sees_what_is_written_on_the_gpu(dev):
    from test_fp8_ops import _check_versions
    _check_versions(dev)
    with torch.inference_mode():
        frozen = torch.zeros(5, 7, device=dev)
        a, b = F.quantize(torch.ones(5, 130, device=dev)), F.quantize(torch.ones(7, 130, device=dev), (128, 128))
        assert (F.matmul(a, b, out=frozen) == 130).all()
    with pytest.raises(RuntimeError, match="inference"):
        F.matmul(a, b, out=frozen)


@pytest.mark.parametrize("bits", [8, 32])
def test_resuming_takes_no_room_for_the_file_on_the_gpu(dev, bits, tmp_path, monkeypatch):
    """What a checkpoint holds comes from the host slice by slice."""
    eng, other = (_engine(dev, optimizer_state_bits=bits) for _ in range(2))
    try:
        eng.train_step()
        eng.save_checkpoint(str(tmp_path))
        load, found = torch.load, []

        def tensors(x):
            return [x] if torch.is_tensor(x) else [t for y in (x.values() if isinstance(x, dict) else x if isinstance(x, (list, tuple)) else ()) for t in tensors(y)]

        monkeypatch.setattr(torch, "load", lambda *a, **kw: found.append(load(*a, **kw)) or found[-1])
        torch.cuda.synchronize(), torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        if bits == 8:
            pieces = other.optimizer._state_pieces
            monkeypatch.setattr(other.optimizer, "_state_pieces", lambda: pieces(1 << 16))
        other.load_checkpoint(str(tmp_path))
        assert len(tensors(found)) > 4 and all(t.device.type == "cpu" for t in tensors(found))
        # pieces of 2^16 values with a few temporaries of up to 8 bytes each; in 32 bits none
        assert torch.cuda.max_memory_allocated() - held <= (1 << 16) * 8 * 16 + (1 << 20)
        assert torch.equal(other.bufs.params, eng.bufs.params) and torch.equal(other.optimizer.master, eng.optimizer.master)
        # value for value, not bit for bit: a block's largest code may be 224 after rounding down, 448 with half its scale
        monkeypatch.undo()
        a, b = eng.optimizer.state_dict(), other.optimizer.state_dict()
        assert torch.equal(a["m"].cpu(), b["m"].cpu()) and torch.equal(a["v"].cpu(), b["v"].cpu())
        assert abs(eng.train_step() - other.train_step()) < 1e-4
    finally:
        eng.close()
        other.close()


@pytest.mark.parametrize("most", [256, 1024, 1 << 24])
def test_8_bit_state_in_pieces_is_the_whole(dev, most):
    (_, opt), (_, other) = _sharded(dev, 8), _sharded(dev, 8)
    for i in range(2):
        _grads(opt.bufs, i)
        opt.step()
    whole = opt.state_dict()
    pieces = opt._state_pieces
    opt._state_pieces = lambda: pieces(most)
    assert all(torch.equal(opt.state_dict()[k], whole[k]) for k in ("m", "v"))
    pieces2 = other._state_pieces
    other._state_pieces = lambda: pieces2(most)
    other.load_state_dict(whole)
    assert all(torch.equal(other.state_dict()[k], whole[k]) for k in ("m", "v"))


def test_adamw_refuses_to_read_what_it_writes_on_the_gpu(dev):
    from test_fp8_ops import _check_read_memory
    _check_read_memory(dev)


def test_adamw_of_leaves_and_its_norm_on_the_gpu(dev):
    from test_fp8_ops import _check_leaves_and_norm
    _check_leaves_and_norm(dev)


def test_pieces_pass_no_gradient_on_the_gpu(dev):
    from test_fp8_ops import _check_pieces_pass_no_gradient
    _check_pieces_pass_no_gradient(dev)


def test_linear_of_nothing_on_the_gpu(dev):
    from test_fp8_ops import _check_linear_of_nothing
    _check_linear_of_nothing(dev)


def test_status_across_streams(dev, monkeypatch):
    """A new word is zero for every stream, and the check waits for what runs on another one."""
    monkeypatch.setattr(F, "_STATUS", {})
    side, busy = torch.cuda.Stream(), torch.randn(8192, 8192, device=dev)
    # memory that was not zero, whose next owner is the word
    used = [torch.full((1,), 7, dtype=torch.int32, device=dev) for _ in range(64)]
    torch.cuda.synchronize()
    del used
    for _ in range(20):
        busy @ busy
    word = F.status_word(dev)
    with torch.cuda.stream(side):
        seen = word.clone()
    side.synchronize()
    assert seen.item() == 0
    with torch.cuda.stream(side):
        for _ in range(20):
            busy @ busy
        word.fill_(1)
    with pytest.raises(RuntimeError, match="gave up"):
        F.check_status()
    with torch.cuda.stream(side):
        assert word.clone().item() == 0
    F.check_status()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("at", [0, 300, 2047, 2500])
@pytest.mark.parametrize("offset", [0, 1])
def test_a_bad_gradient_leaves_its_block_alone(dev, bad, at, offset):
    """Codes and scales of all other elements, with the bad one's old moments at zero, so that it cannot be its block's largest."""
    st = _adam_state([700, 2600], 8, torch.bfloat16, torch.bfloat16, dev, offset)
    for k in ("m", "v"):
        st[k][1].view(torch.uint8)[at] = 0
    clean = _copy(st)
    st["grads"][1][at], clean["grads"][1][at] = bad, 0.0
    O.adamw_multi(**st, **HYPER), O.adamw_multi(**clean, **HYPER)
    keep = torch.arange(2600, device=dev) != at
    for k in ("m", "v", "masters", "params"):
        assert torch.isnan(st[k][1][at].float()), k
        assert torch.equal(_bits(st[k][0]), _bits(clean[k][0])) and torch.equal(st[k][1].float()[keep], clean[k][1].float()[keep]), k
    for k in ("m_scales", "v_scales"):
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(st[k], clean[k])), k


def test_overlapped_step_with_8_bit_state(dev):
    """The step of several ranks (slices reduced on a side stream, the update, the new parameters to every rank) as a world of one:
    gradients times 0.5 are exact, so without a norm, whose sum has no fixed order there, it gives the bits of the other."""
    (bufs, opt), (bufs2, opt2) = _sharded(dev, 8), _sharded(dev, 8)
    for o in (opt, opt2):
        o.clip = None
    opt2.overlap, opt2.side = True, torch.cuda.Stream()
    opt2.main_grad = torch.zeros(opt2.master.numel(), device=dev)
    for i in range(3):
        _grads(bufs, i), _grads(bufs2, i)
        for b in (3, 2):
            opt2.grad_scale = 0.5
            opt2.reduce_bucket(b)
        opt.step(0.5), opt2.step(0.5)
        for k in ("m", "v", "m_scale", "v_scale", "master", "step_tensor"):
            assert torch.equal(_bits(getattr(opt, k)), _bits(getattr(opt2, k))), k
        assert torch.equal(bufs.params, bufs2.params)
    opt2.clip = 0.5
    _grads(bufs2, 7)
    before = opt2.master.clone()
    want = {"params": [bufs2.params[s.flat_off:s.flat_off + s.length].clone() for s in opt2.shards], "step": opt2.step_tensor.clone()}
    parts = [slice(s.state_off, s.state_off + s.length) for s in opt2.shards]
    want |= {"masters": [before[p].clone() for p in parts], "m": [opt2.m[p].clone() for p in parts], "v": [opt2.v[p].clone() for p in parts],
             "m_scales": [opt2._scales(opt2.m_scale, i).clone() for i in range(4)], "v_scales": [opt2._scales(opt2.v_scale, i).clone() for i in range(4)]}
    opt2.step(0.5)
    O.adamw_multi(**want, grads=[bufs2.grads[s.flat_off:s.flat_off + s.length] for s in opt2.shards], lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8,
                  weight_decay=0.1, grad_scale=0.5, clip=0.5)
    step = (torch.cat(want["masters"]) - before).abs()
    # the norm in fp32, its 40000 squares added in any order: 2^-24 times at most some 300 additions of one chain
    assert ((opt2.master - torch.cat(want["masters"])).abs() <= step * 2.0 ** -14 + before.abs() * 2.0 ** -23).all()
    assert torch.equal(bufs2.params.float(), opt2.master.bfloat16().float())


# --------------------------------------------------------------------------- the layers, compared closely
# Two runs in 8 bits that differ by d somewhere differ by sqrt(2^-3 d) after the next quantizer, so whole gradients of two forms
# cannot be compared closely.  Instead every call is compared on the very operands it had, and how the layer is put together is
# compared with quantizers that round nothing.
@pytest.mark.parametrize("level", [None, 0, 1, 2])
def test_every_call_of_the_layers_in_8_bits(dev, level, monkeypatch):
    calls = {k: getattr(F, k) for k in ("quantize", "quantize_both", "matmul", "rmsnorm_quant", "rmsnorm_quant_bwd")}
    count = dict.fromkeys(calls, 0)

    def quantize(x, block=(1, 128), dtype=E4M3):
        count["quantize"] += 1
        got = calls["quantize"](x, block, dtype)
        _same(got, F.quantize_reference(x, block, dtype))
        return got

    def quantize_both(x, dtype=E4M3):
        count["quantize_both"] += 1
        got = calls["quantize_both"](x, dtype)
        for q, block in zip(got, ((1, 128), (128, 1))):
            _same(q, F.quantize_reference(x, block, dtype))
        return got

    def matmul(a, b, *, trans_a=False, trans_b=True, out_dtype=torch.bfloat16, add=None, out=None):
        count["matmul"] += 1
        was = None if add is None else add.clone()
        got = calls["matmul"](a, b, trans_a=trans_a, trans_b=trans_b, out_dtype=out_dtype, add=add, out=out)
        _check_product(got, a, b, dict(trans_a=trans_a, trans_b=trans_b), was)
        return got

    def rmsnorm_quant(x, w, eps=1e-5, residual=None, dtype=E4M3):
        count["rmsnorm_quant"] += 1
        y, h, rstd = calls["rmsnorm_quant"](x, w, eps, residual, dtype)
        _check_norm(x, w, eps, residual, y, h, rstd, dtype)
        return y, h, rstd

    def rmsnorm_quant_bwd(h, w, rstd, dy, add=None):
        count["rmsnorm_quant_bwd"] += 1
        dx, dw = calls["rmsnorm_quant_bwd"](h, w, rstd, dy, add)
        r, xh, g = rstd.double()[:, None], h.double() * rstd.double()[:, None], dy.double() * w.double()
        more = 0 if add is None else add.double()
        want, size = r * (g - xh * (g * xh).mean(-1, keepdim=True)) + more, r * (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)) + abs(more)
        assert ((dx.double() - want).abs() <= want.abs() * HALF[h.dtype] + size * 60 * 2.0 ** -24).all()
        assert ((dw.double() - (dy.double() * xh).sum(0)).abs() <= (dy.double() * xh).abs().sum(0) * (h.shape[0] / 100 + 150) * 2.0 ** -24).all()
        return dx, dw

    for k, f in dict(quantize=quantize, quantize_both=quantize_both, matmul=matmul, rmsnorm_quant=rmsnorm_quant, rmsnorm_quant_bwd=rmsnorm_quant_bwd).items():
        monkeypatch.setattr(F, k, f)
    eng = _engine(dev, fp8=True, activation_budget_gb=-1.0 if level is None else 0.0)
    try:
        if level is not None:
            eng.model.layer_levels = [level, level]
        _gradients(eng)
        # of each layer four products forward and eight back; again QKV, output and gate | up, or what of them is not kept
        assert count["quantize_both"] == count["rmsnorm_quant_bwd"] * 2 == 8 and count["matmul"] >= 2 * (12 + (3, 1, 0)[level or 0]), count
    finally:
        eng.close()


@pytest.mark.parametrize("level,ranks", [(None, "one"), (0, "one"), (1, "one"), (2, "one"), (0, "as of several"), (1, "as of several"),
                                         (2, "as of several")])
def test_how_the_layers_in_8_bits_are_put_together(dev, level, ranks, monkeypatch):
    """With quantizers that round nothing the layers are those of the model in 16 bits, up to roundings to 16 bits: of a gradient's
    eleven products two operands and a result each, in two forms, 66 roundings of 2^-8 / sqrt(3) in the mean: 2^-5.8; 2^-5
    allowed.  ``as of several``: the form that tensor parallelism takes, with sums over one rank."""
    budget = -1.0 if level is None else 0.0
    eng, other = _engine(dev, fp8=True, activation_budget_gb=budget), _engine(dev, activation_budget_gb=budget)
    kept = lambda x, block=(1, 128): F.BlockScaled(x.float(), torch.ones(1, device=dev), block)  # noqa: E731

    def norm(x, w, eps=1e-5, residual=None):
        h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
        rstd = torch.rsqrt(h.float().square().mean(-1) + eps)
        return kept(h.float() * rstd[:, None] * w.float()), h, rstd

    def product(a, b, *, trans_a=False, trans_b=True, out_dtype=torch.bfloat16, add=None, out=None):
        got = (a.codes.t() if trans_a else a.codes) @ (b.codes.t() if trans_b else b.codes) + (0 if add is None else add.float())
        return got.to(out_dtype) if out is None else out.copy_(got)

    try:
        if level is not None:
            for e in (eng, other):
                e.model.layer_levels = [level, level]
        loss0, want = _gradients(other)
        for k, f in dict(quantize=kept, quantize_both=lambda x: (kept(x), kept(x)), matmul=product, rmsnorm_quant=norm).items():
            monkeypatch.setattr(F, k, f)
        if ranks != "one":
            eng.model.tp_group, eng.model.tp_sum = object(), lambda t: t
        loss, grads = _gradients(eng)
        assert abs(loss - loss0) <= 2.0 ** -9 * loss0
        off = {k: ((g - want[k]).norm() / want[k].norm()).item() for k, g in grads.items()}
        assert max(off.values()) <= 2.0 ** -5, sorted(off.items(), key=lambda t: -t[1])[:4]
    finally:
        eng.close()
        other.close()


@pytest.mark.parametrize("level", [0, 2])
def test_layers_in_8_bits_add_to_gradients(dev, level):
    """With ``accumulate_grads`` a layer adds to what is there, rounded once: a gradient of its own is rounded when it is written,
    the sum when it is."""
    eng = _engine(dev, fp8=True, activation_budget_gb=0.0)
    try:
        eng.model.layer_levels = [level, level]
        plan = eng.plans.get(0)
        inputs = eng.stage_inputs(plan)

        def run(base):
            eng.model.grads_flat.copy_(base)
            eng.model.loss(*inputs, 1.0 / plan.n_global_tokens).backward()
            torch.cuda.synchronize()
            return {k: t.grad.double().clone() for k, t in eng.model.p.items()}

        base = torch.zeros_like(eng.model.grads_flat)
        own = run(base)
        base.copy_(torch.randn(base.shape, device=dev) * eng.model.grads_flat.float().std())
        eng.model.accumulate_grads = True
        got = run(base)
        eng.model.grads_flat.copy_(base)
        there = {k: t.grad.double().clone() for k, t in eng.model.p.items()}
        for k in own:
            if not k.startswith("l"):
                continue
            near = 2.0 ** -8 * (own[k].abs() + (own[k] + there[k]).abs() * (1 + 2.0 ** -7))
            off = (got[k] - own[k] - there[k]).abs()
            if k in ("l1.wd", "l1.wgu", "l1.norm2"):
                assert (off <= near).all(), k    # nothing before them adds in an order that may differ
            # attention's dQ does
            assert off.norm() <= near.norm() + 2.0 ** -8 * own[k].norm(), k
        # and a second time over the same codes
        again = run(base)
        for k in ("l1.wd", "l1.wgu", "l1.norm2"):
            assert torch.equal(again[k], got[k]), k
    finally:
        eng.close()


@pytest.mark.parametrize("how", ["forward", "dgrad", "wgrad"])
@pytest.mark.parametrize("m,n,k", [(512, 5120, 300), (256, 9729, 130), (300, 5120, 513), (768, 3328, 1000), (1535, 1537, 257)])
def test_matmul_around_a_round_of_small_tiles(dev, how, m, n, k):
    """Outputs of about as many tiles of 128 x 128 as there are processors, where the rule goes from one kernel to the other."""
    a, b, kw = _operands(m, n, k, how, dev)
    _check_product(F.matmul(a, b, **kw), a, b, kw)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("at", [0, 4103, 12_110, 30_003])
def test_sharded_optimizer_clips_a_gradient_whose_square_fp32_does_not_hold(dev, bits, at):
    bufs, opt = _sharded(dev, bits)
    _grads(bufs, 0)
    bufs.grads[at] = 1e20
    length = bufs.grads.double().norm().item()
    w = opt.master.double()
    opt.step()
    assert abs(opt.grad_norm() / length - 1) <= 2.0 ** -20
    # the first step is g / (|g| + eps) of the clipped gradient, whatever its length: the one moves by lr, the others, 1e-20 of it, not
    g = bufs.grads.double() * (0.5 / length)
    want = w - 1e-2 * (g / (g.abs() + 1e-8) + 0.1 * w)
    # m / (sqrt(v) + eps) of a dozen roundings, and moments that are not rounded yet
    assert ((opt.master.double() - want).abs() <= 1e-2 * 2.0 ** -18 + w.abs() * 2.0 ** -23).all()
