"""8-bit operators on the CPU: their plain forms against 64-bit arithmetic, their gradients against the formulas and against
differences, and what they refuse.  The kernels themselves are in test_gpu_fp8.py."""
import pytest
import torch

from dcp_b200.ops import fp8_ops as F
from dcp_b200.ops import optim_ops as O

E4M3, E5M2, E8M0 = F.E4M3, F.E5M2, F.E8M0


def _scale_bounds(x, q):
    """The scale is the smallest power of two with amax <= largest code * scale."""
    largest = torch.finfo(q.codes.dtype).max
    rows, cols = x.shape
    for i in range(q.scales.shape[0]):
        for j in range(q.scales.shape[1]):
            part = x[i * q.block[0]:(i + 1) * q.block[0], j * q.block[1]:(j + 1) * q.block[1]].double().abs().max().item()
            s = q.scales[i, j].double().item()
            assert part <= largest * s and (part > largest * s / 2 or s == 2.0 ** -127), (i, j, part, s)


@pytest.mark.parametrize("block", [(1, 128), (128, 1), (128, 128)])
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("shape", [(1, 1), (3, 127), (130, 257)])
def test_quantize_reference(block, dtype, shape):
    torch.manual_seed(0)
    x = torch.randn(shape) * torch.exp2(torch.randint(-20, 20, (shape[0], 1)).float())
    x[0] = 0
    q = F.quantize(x, block, dtype)
    _scale_bounds(x, q)
    s = q._replace(codes=torch.ones_like(q.codes)).dequantize(torch.float64)
    step, least = (2.0 ** -4, 2.0 ** -10) if dtype == E4M3 else (2.0 ** -3, 2.0 ** -17)   # half a step; of the denormals
    err = (q.dequantize(torch.float64) - x.double()).abs()
    assert (err <= torch.maximum(x.double().abs() * step, s * least)).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_block_with_a_value_that_is_not_finite_reads_back_as_nan(bad):
    x = torch.ones(2, 300)
    x[1, 130] = bad
    d = F.quantize(x).dequantize()
    assert torch.isnan(d[1, 128:256]).all() and torch.equal(d[0], x[0]) and torch.equal(d[1, :128], x[1, :128]) and \
        torch.equal(d[1, 256:], x[1, 256:])


def test_extreme_magnitudes_are_representable():
    x = torch.zeros(4, 128)
    x[0, 0], x[1, 0], x[2, 0] = 3.4028234e38, 1e-38, 2.0 ** -149
    q = F.quantize(x)
    d = q.dequantize(torch.float64)
    assert abs(d[0, 0].item() / 3.4028234663852886e38 - 1) <= 2.0 ** -4 and abs(d[1, 0].item() / 1e-38 - 1) <= 2.0 ** -4
    assert d[2, 0] == 0 and q.scales.view(torch.uint8).tolist() == [[247], [0], [0], [0]]   # 2^-149 is below half a step of 2^-136


def _numeric(f, x, i, eps):
    a, b = x.clone(), x.clone()
    a.view(-1)[i] += eps
    b.view(-1)[i] -= eps
    return (f(a) - f(b)) / (2 * eps)


@pytest.mark.parametrize("with_add", [False, True])
def test_norm_backward_against_formula_and_differences(with_add):
    torch.manual_seed(1)
    rows, width, eps = 3, 40, 1e-5
    h, w, dy, add = (torch.randn(s, dtype=torch.float64) for s in ((rows, width), (width,), (rows, width), (rows, width)))
    norm = lambda t, u: t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + eps) * u  # noqa: E731
    f = lambda t, u: ((norm(t, u) * dy).sum() + ((t * add).sum() if with_add else 0.0))  # noqa: E731
    rstd = torch.rsqrt(h.pow(2).mean(-1) + eps)
    dx, dw = F.rmsnorm_quant_bwd(h.float(), w.float(), rstd.float(), dy.float(), add.float() if with_add else None)
    leaf, leaf_w = h.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(f(leaf, leaf_w), (leaf, leaf_w))
    # a few dozen fp32 roundings of values of order one
    assert (dx.double() - gx).abs().max() < 2e-5 and (dw.double() - gw).abs().max() < 2e-5
    for i in (0, 17, 63, rows * width - 1):
        assert abs(_numeric(lambda t: f(t, w), h, i, 1e-5) - gx.view(-1)[i]) < 1e-7
    assert abs(_numeric(lambda u: f(h, u), w, 5, 1e-5) - gw[5]) < 1e-7


def test_linear_and_norm_linear_are_their_products():
    torch.manual_seed(2)
    x, w, nw = torch.randn(5, 7, 200), torch.randn(48, 200), torch.randn(200)
    res, d_out, d_h = torch.randn(5, 7, 200), torch.randn(5, 7, 48), torch.randn(5, 7, 200)
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    out = F.linear(*leaves)
    out.backward(d_out)
    deq = lambda t, b: F.quantize(t.reshape(-1, t.shape[-1]), b).dequantize(torch.float64)  # noqa: E731
    near = lambda a, b: torch.testing.assert_close(a.double().reshape(b.shape), b, rtol=1e-5, atol=1e-4)  # fp32 sums of up to 200 products
    near(out, deq(x, (1, 128)) @ deq(w, (128, 128)).t())
    near(leaves[0].grad, deq(d_out, (1, 128)) @ deq(w, (128, 128)))
    near(leaves[1].grad, deq(d_out, (128, 1)).t() @ deq(x, (128, 1)))
    # the norm's, with the gradient of the sum from elsewhere
    lx, lr, lw, ln = (t.clone().requires_grad_() for t in (x, res, w, nw))
    out, h = F.norm_linear(lx, ln, lw, 1e-5, lr)
    torch.autograd.backward([out, h], [d_out, d_h])
    h2 = (x + res).reshape(-1, 200)
    y, _, rstd = F.rmsnorm_quant(h2, nw, 1e-5)
    near(out, y.dequantize(torch.float64) @ deq(w, (128, 128)).t())
    assert torch.equal(h.reshape(-1, 200), h2)
    dy = (deq(d_out, (1, 128)) @ deq(w, (128, 128))).float()
    dx, dn = F.rmsnorm_quant_bwd(h2, nw, rstd, dy, d_h.reshape(-1, 200))
    near(lx.grad, dx.double()), near(ln.grad, dn.double())
    assert torch.equal(lx.grad, lr.grad)
    near(lw.grad, deq(d_out, (128, 1)).t() @ deq(h2 * rstd[:, None] * nw, (128, 1)))
    # only the sum is used
    lx, lr = x.clone().requires_grad_(), res.clone().requires_grad_()
    F.norm_linear(lx, nw, w, 1e-5, lr)[1].backward(d_h)
    assert torch.equal(lx.grad, d_h) and torch.equal(lr.grad, d_h)


def test_refusals_of_the_8_bit_operators():
    x, w = torch.zeros(4, 256), torch.zeros(8, 256)
    q, wq = F.quantize(x), F.quantize(w, (128, 128))
    for call, words in [
            (lambda: F.quantize(x, (1, 64)), "blocks are"),
            (lambda: F.quantize(x[0]), "matrix"),
            (lambda: F.quantize(x.double()), "bfloat16, float16 or float32"),
            (lambda: F.quantize(x, dtype=torch.float16), "codes are"),
            (lambda: F.quantize_both(x.int()), "bfloat16, float16 or float32"),
            (lambda: F.rmsnorm_quant(x, torch.zeros(255)), "w has to be"),
            (lambda: F.rmsnorm_quant(x, torch.zeros(256, dtype=torch.bfloat16)), "w has to be"),
            (lambda: F.rmsnorm_quant(x, torch.zeros(256), residual=torch.zeros(4, 255)), "residual"),
            (lambda: F.rmsnorm_quant(torch.zeros(1, 16385), torch.zeros(16385)), "16384"),
            (lambda: F.rmsnorm_quant(torch.zeros(3, 0), torch.zeros(0)), "16384"),
            (lambda: F.rmsnorm_quant_bwd(x, torch.zeros(256), torch.zeros(4), torch.zeros(4, 255)), "dy"),
            (lambda: F.rmsnorm_quant_bwd(x, torch.zeros(256), torch.zeros(5), x), "rstd"),
            (lambda: F.rmsnorm_quant_bwd(x, torch.zeros(256), torch.zeros(4), x, x.bfloat16()), "add"),
            (lambda: F.matmul(q, F.quantize(torch.zeros(8, 128))), "contraction"),
            (lambda: F.matmul(F.quantize(x, (128, 1)), wq), "scale per 128"),
            (lambda: F.matmul(q, wq, trans_a=True, trans_b=False), "contraction"),
            (lambda: F.matmul(q._replace(codes=x), wq), "codes"),
            (lambda: F.matmul(q._replace(scales=q.scales[:2]), wq), "scales"),
            (lambda: F.matmul(q._replace(scales=q.scales.float()), wq), "scales"),
            (lambda: F.matmul(q._replace(block=(2, 128)), wq), "blocks are"),
            (lambda: F.matmul(q, wq, out_dtype=torch.float64), "results are"),
            (lambda: F.matmul(q, wq, out=torch.zeros(4, 9)), "out has to be"),
            (lambda: F.matmul(q, wq, out=torch.zeros(8, 4).t()), "contiguous"),
            (lambda: F.matmul(q, wq, add=torch.zeros(4, 8)), "add has to be"),
            (lambda: F.matmul(q, wq, form=3), "form"),
            (lambda: F.linear(x, w.bfloat16()), "of one type"),
            (lambda: F.norm_linear(x, torch.zeros(256), w, 1e-5, x[:2]), "residual")]:
        with pytest.raises(ValueError, match=words):
            call()


def test_empty_operands():
    q, wq = F.quantize(torch.zeros(0, 256)), F.quantize(torch.zeros(8, 256), (128, 128))
    assert F.matmul(q, wq).shape == (0, 8) and q.scales.shape == (0, 2)
    none = F.quantize(torch.zeros(3, 0)), F.quantize(torch.zeros(5, 0), (128, 128))
    assert torch.equal(F.matmul(*none, out_dtype=torch.float32), torch.zeros(3, 5))


# --------------------------------------------------------------------------- AdamW
def _state(sizes, bits, ptype, gtype, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda n: torch.randn(n, generator=g)  # noqa: E731
    params = [rnd(n).to(ptype).to(device) for n in sizes]
    st = {"params": params, "grads": [(rnd(n) * 1e-2).to(gtype).to(device) for n in sizes],
          "masters": None if ptype == torch.float32 else [p.float() for p in params], "step": torch.full((1,), 4, device=device)}
    m, v = [rnd(n).to(device) * 1e-2 for n in sizes], [(rnd(n).to(device) * 1e-2).square() for n in sizes]
    if bits == 32:
        return {**st, "m": m, "v": v}
    em, ev = [O.encode_state(t) for t in m], [O.encode_state(t.sqrt(), root=True) for t in v]
    return {**st, "m": [c for c, _ in em], "v": [c for c, _ in ev], "m_scales": [s for _, s in em], "v_scales": [s for _, s in ev]}


HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)


def test_plain_adamw_is_torchs():
    p0 = [torch.randn(7, 3), torch.randn(11)]
    mine = [p.clone() for p in p0]
    leaves = [p.clone().requires_grad_() for p in p0]
    opt = torch.optim.AdamW(leaves, lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    m, v, step = [torch.zeros_like(p) for p in mine], [torch.zeros_like(p) for p in mine], torch.zeros(1, dtype=torch.int64)
    for i in range(4):
        grads = [torch.randn(p.shape, generator=torch.Generator().manual_seed(i)) for p in p0]
        for leaf, g in zip(leaves, grads):
            leaf.grad = g.clone() * 0.5
        norm = torch.nn.utils.clip_grad_norm_(leaves, 1.0)
        opt.step()
        got = O.adamw_multi(mine, grads, None, m, v, step, **HYPER, grad_scale=0.5, clip=1.0)
        assert abs(got.item() - norm.item()) < 1e-5
    for a, b in zip(mine, leaves):
        assert (a - b).abs().max() < 1e-6       # ten roundings of values of order one, four times


def test_stochastic_rounding_is_right_on_average():
    torch.manual_seed(3)
    x = torch.randn(256)
    bits = torch.arange(0, 65536, 37)[:, None].expand(-1, 256)
    n = bits.shape[0]
    codes, scales = O.encode_state(x.repeat(n), bits.reshape(-1))
    mean = O.decode_state(codes, scales).view(n, 256).double().mean(0)
    # random bits at distances of 37 of 65536 and cut at 16 bits: a step (2^-3 of the value at most) is hit within 38 / 65536
    s = O.decode_state(torch.ones(256).to(E4M3), scales[:1]).double()
    assert ((mean - x.double()).abs() <= torch.maximum(x.abs().double() * 2.0 ** -3, s * 2.0 ** -9) * 40 / 65536).all()


def test_state_codes_come_back_to_the_bit():
    torch.manual_seed(4)
    for root in (False, True):
        x = torch.randn(5000) * torch.exp2(torch.randint(-30, 5, (5000,)).float())
        x = x.abs() if root else x
        x[::7] = 0
        c, s = O.encode_state(x, torch.randint(0, 65536, (5000,)), root)
        value = O.decode_state(c, s)
        c2, s2 = O.encode_state(value, root=root)
        assert torch.equal(O.decode_state(c2, s2), value)
        assert not root or ((value > 0) == (x > 0)).all()


def test_optimizer_class_on_the_cpu():
    torch.manual_seed(5)
    params = [torch.randn(300, dtype=torch.bfloat16), torch.randn(4, 5, dtype=torch.bfloat16)]
    opts = [O.MultiTensorAdamW([p.clone() for p in params], lr=1e-2, state_bits=b, clip_grad=1.0) for b in (8, 32)]
    for i in range(3):
        for o in opts:
            for p in o.params:
                p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(i)).bfloat16()
            o.step()
    eight, full = opts
    assert int(eight.step_count) == 3 and eight.m.dtype == E4M3 and eight.master.dtype == torch.float32
    # steps of lr each, whose direction differs by the roundings of m and of sqrt(v): each within a step of 2^-3
    assert (eight.master - full.master).abs().max() < 3 * 1e-2 * 0.6
    other = O.MultiTensorAdamW([p.clone() for p in params], lr=1e-2, state_bits=8, clip_grad=1.0)
    other.load_state_dict(eight.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(other.params, eight.params)) and torch.equal(other.m.view(torch.uint8), eight.m.view(torch.uint8))
    with pytest.raises(ValueError, match="another width"):
        full.load_state_dict(eight.state_dict())


def test_refusals_of_adamw():
    ok = lambda **kw: {**_state([5, 300], 8, torch.bfloat16, torch.bfloat16), **HYPER, **kw}  # noqa: E731
    st = ok()
    for bad, words in [(dict(params=[], grads=[]), "no parameters"), (dict(grads=st["grads"][:1]), "2 parameters"),
                       (dict(masters=None), "need fp32 masters"), (dict(v_scales=None), "scales of m and of v"),
                       (dict(step=torch.zeros(1)), "int64"), (dict(m=[t.float() for t in st["m"]]), "tensor 0"),
                       (dict(m_scales=[s[:1] for s in st["m_scales"]]), "tensor 1"),
                       (dict(grads=[torch.zeros(10)[::2], torch.zeros(300)]), "tensor 0"),
                       (dict(grads=[st["grads"][0], st["grads"][1].float()]), "tensor 1"),
                       (dict(params=[p.double() for p in st["params"]]), "parameters and gradients"),
                       (dict(clip=0.0), "positive"), (dict(factor=torch.zeros(2)), "factor"),
                       (dict(clip=1.0, factor=torch.ones(1)), "either clip"), (dict(params=[st["params"][1], st["params"][1]][:1] * 2,
                        grads=[st["grads"][1]] * 2, masters=[st["masters"][1]] * 2, m=[st["m"][1]] * 2, v=[st["v"][1]] * 2,
                        m_scales=[st["m_scales"][1]] * 2, v_scales=[st["v_scales"][1]] * 2), "given twice"),
                       (dict(status=[torch.zeros(1)]), "status")]:
        with pytest.raises(ValueError, match=words):
            O.adamw_multi(**ok(**bad))
    with pytest.raises(ValueError, match="8 or 32"):
        O.MultiTensorAdamW([torch.zeros(3)], state_bits=16)
    with pytest.raises(ValueError, match="no gradient"):
        O.MultiTensorAdamW([torch.zeros(3)]).step()


def test_a_status_word_stops_the_step():
    st = _state([5, 300], 8, torch.bfloat16, torch.bfloat16)
    before = [p.clone() for p in st["params"]]
    O.adamw_multi(**st, **HYPER, status=[torch.zeros(1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)])
    assert all(torch.equal(a, b) for a, b in zip(before, st["params"])) and int(st["step"]) == 4


def test_what_a_product_is_added_to_is_the_output_or_lies_apart():
    torch.manual_seed(0)
    a, b = F.quantize(torch.randn(5, 130)), F.quantize(torch.randn(7, 130), (128, 128))
    buf = torch.randn(40 * 20)
    at = lambda start, pitch: buf[start:].as_strided((5, 7), (pitch, 1), buf.storage_offset() + start)  # noqa: E731
    for out, add, ok in ((at(0, 20), at(0, 20), True), (at(0, 20), at(7, 20), True), (at(7, 20), at(0, 20), True), (at(0, 20), at(13, 20), True),
                         (at(0, 20), at(6, 20), False), (at(0, 20), at(14, 20), False), (at(0, 20), at(20, 20), False), (at(0, 20), at(0, 7), False),
                         (at(0, 7), at(34, 7), False), (at(0, 7), at(35, 7), True), (at(35, 7), at(0, 7), True), (at(1, 7), at(0, 7), False),
                         (at(0, 20), at(27, 20), True), (at(0, 8), at(40, 9), True), (at(0, 9), at(3, 8), False)):
        used = [{t.storage_offset() + i * t.stride(0) + j for i in range(5) for j in range(7)} for t in (out, add)]
        same = (out.storage_offset(), out.stride()) == (add.storage_offset(), add.stride())
        if out.stride() == add.stride():   # of one pitch the rule is exact
            assert ok == (same or not used[0] & used[1])
        if ok:
            want = F.matmul(a, b, out_dtype=torch.float32, add=add.clone())
            assert torch.equal(F.matmul(a, b, add=add, out=out), want)
        else:
            with pytest.raises(ValueError, match="lie apart"):
                F.matmul(a, b, add=add, out=out)


@pytest.mark.parametrize("key", ["params", "masters", "m", "v", "m_scales", "v_scales"])
def test_adamw_refuses_memory_that_overlaps(key):
    """Also where it does not begin at one address; parts of one buffer beside one another are taken."""
    st = _state([300, 300], 8, torch.bfloat16, torch.bfloat16)
    for skip, ok in ((st[key][0].numel(), True), (st[key][0].numel() - 1, False), (1, False)):
        n = st[key][0].numel()
        flat = torch.zeros(2 * n, dtype=torch.uint8).view(st[key][0].dtype) if st[key][0].element_size() == 1 else torch.zeros(2 * n, dtype=st[key][0].dtype)
        call = lambda: O.adamw_multi(**{**st, **HYPER, key: [flat[skip:skip + n], flat[:n]]})  # noqa: B023, E731
        if ok:
            call()
        else:
            with pytest.raises(ValueError, match="given twice"):
                call()


@pytest.mark.parametrize("bad", [dict(beta1=1.0), dict(beta2=1.0), dict(beta1=-0.1), dict(beta2=float("nan"))])
def test_adamw_refuses_betas_that_it_would_divide_by_zero_with(bad):
    with pytest.raises(ValueError, match="betas"):
        O.adamw_multi(**{**_state([5], 8, torch.bfloat16, torch.bfloat16), **HYPER, **bad})


def test_a_second_derivative_is_refused():
    torch.manual_seed(0)
    x, w, nw = (torch.randn(s, requires_grad=True) for s in ((4, 130), (6, 130), (130,)))
    for y in (F.linear(x, w), F.norm_linear(x, nw, w)[0]):
        dx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            dx.sum().backward()


def _too_wide(device="cpu"):
    """Calls with more columns than the kernels count, of tensors that take no memory."""
    wide, one = 2 ** 31, lambda dtype: torch.zeros(1, dtype=torch.uint8 if dtype.itemsize == 1 else dtype, device=device).view(dtype)  # noqa: E731
    x = one(torch.bfloat16).expand(1, wide)
    scaled = lambda rows, k: F.BlockScaled(one(E4M3).expand(rows, k), one(F.E8M0).expand(rows, -(-k // 128)), (1, 128))  # noqa: E731
    for call in (lambda: F.quantize(x), lambda: F.quantize(x, (128, 1)), lambda: F.quantize(x, (128, 128)), lambda: F.quantize_both(x),
                 lambda: F.quantize(one(torch.bfloat16).expand(1, 2 ** 33)), lambda: F.quantize(x[:, :wide - 127]),
                 lambda: F.quantize(x.t()), lambda: F.matmul(scaled(2, wide - 127), scaled(3, wide - 127)),
                 lambda: F.matmul(scaled(2, 2 ** 33), scaled(3, 2 ** 33))):
        with pytest.raises(ValueError, match="up to 2147483"):
            call()


def test_more_columns_than_the_kernels_count_are_refused():
    _too_wide()


def test_status_words_are_those_of_devices():
    with pytest.raises(ValueError, match="CUDA devices"):
        F.status_word(torch.device("cpu"))
    word = torch.ones(1, dtype=torch.int32)
    p = torch.ones(300)
    p.grad = torch.ones(300)
    opt = O.MultiTensorAdamW([p], lr=0.1, status=[torch.zeros(1, dtype=torch.int32), word])
    opt.step()
    assert (p == 1).all() and int(opt.step_count) == 0
    word.zero_()
    opt.step()
    assert (p != 1).all()
    with pytest.raises(ValueError, match="up to four"):
        O.MultiTensorAdamW([p], status=[word] * 5).step()


def _check_versions(device):
    """Autograd sees what the operators write: a graph that saved it raises instead of giving other gradients."""
    for bits, ptype in ((8, torch.bfloat16), (32, torch.float32)):
        p = [torch.randn(300, device=device).to(ptype).requires_grad_(), torch.randn(7, 3, device=device).to(ptype).requires_grad_()]
        opt = O.MultiTensorAdamW(p, state_bits=bits)
        graphs = [t.square().sum() for t in p]
        for t in p:
            t.grad = torch.randn_like(t).detach()
        opt.step()
        for g in graphs:
            with pytest.raises(RuntimeError, match="inplace operation"):
                g.backward()
        p[0].square().sum().backward()
        kept = [opt.m, opt.v, opt.step_count] + [t for t in (opt.master, opt.m_scale, opt.v_scale) if t is not None]
        before, grads = [t._version for t in kept], [t.grad._version for t in p]
        opt.step()
        assert all(t._version > v for t, v in zip(kept, before)) and [t.grad._version for t in p] == grads
    a, b = F.quantize(torch.randn(5, 130, device=device)), F.quantize(torch.randn(7, 130, device=device), (128, 128))
    out, scale = torch.zeros(6, 7, device=device), torch.ones(6, 7, device=device, requires_grad=True)
    graph = (out * scale).sum()
    F.matmul(a, b, out=out[:5])
    with pytest.raises(RuntimeError, match="inplace operation"):
        graph.backward()
    add = torch.zeros(5, 7, device=device)
    versions = [t._version for t in (add, a.codes, b.codes)]
    F.matmul(a, b, add=add, out=out[:5])
    assert [t._version for t in (add, a.codes, b.codes)] == versions


def test_autograd_sees_what_is_written():
    _check_versions("cpu")


def _check_read_memory(device):
    """Gradients, factor and status words that lie in what the step writes, wherever in it."""
    for bits in (8, 32):
        st = _state([300, 300], bits, torch.bfloat16, torch.bfloat16, device=device)
        buf = torch.zeros(4000, dtype=torch.uint8, device=device)
        f32 = buf.view(torch.float32)
        word = lambda i: buf[4 * i:4 * i + 4].view(torch.int32)  # noqa: E731
        masters = [f32[100:400], f32[500:800]]
        bf16 = buf.view(torch.bfloat16)
        # in 16-bit values the masters are [200, 800) and [1000, 1600)
        for lo, ok in ((0, False), (250, False), (799, False), (800, False), (1599, False), (1600, True), (1700, True)):
            given = {**st, **HYPER, "masters": masters, "grads": [st["grads"][0], bf16[lo:lo + 300]]}
            if ok:
                O.adamw_multi(**given)
            else:
                with pytest.raises(ValueError, match="share memory"):
                    O.adamw_multi(**given)
        for i, ok in ((99, True), (100, False), (399, False), (400, True), (799, False), (800, True)):
            for extra in (dict(factor=f32[i:i + 1]), dict(status=[word(i)])):
                given = {**st, **HYPER, "masters": masters, **extra}
                if ok:
                    O.adamw_multi(**given)
                else:
                    with pytest.raises(ValueError, match="share memory"):
                        O.adamw_multi(**given)
        moments = buf[:1200].view(torch.float32) if bits == 32 else buf[:300].view(E4M3)
        with pytest.raises(ValueError, match="given twice"):
            O.adamw_multi(**{**st, **HYPER, "m": [st["m"][0], moments], "step": buf[:8].view(torch.int64)})


def test_adamw_refuses_to_read_what_it_writes():
    _check_read_memory("cpu")


def _check_leaves_and_norm(device):
    """Parameters that are leaves of a graph are stepped whatever the grad mode; a step that a status word stops has its norm."""
    for bits, ptype in ((8, torch.bfloat16), (32, torch.float32)):
        st = _state([300, 7], bits, ptype, ptype, device=device)
        plain = {k: [t.clone() for t in x] if isinstance(x, list) else x.clone() if torch.is_tensor(x) else x for k, x in st.items()}
        for k in ("params", "grads"):
            for t in st[k]:
                t.requires_grad_()
        want = sum(g.double().square().sum() for g in plain["grads"]).sqrt().item() * 0.5
        stopped = O.adamw_multi(**st, **HYPER, grad_scale=0.5, clip=1.0, status=[torch.ones(1, dtype=torch.int32, device=device)])
        assert torch.equal(st["params"][0], plain["params"][0]) and abs(stopped.item() / want - 1) < 1e-6
        norm = O.adamw_multi(**st, **HYPER, grad_scale=0.5, clip=1.0)
        O.adamw_multi(**plain, **HYPER, grad_scale=0.5, clip=1.0)
        assert torch.equal(norm, stopped) and not norm.requires_grad
        assert all(torch.equal(a, b) and a.requires_grad for a, b in zip(st["params"], plain["params"]))
        assert st["masters"] is None or not any(w.requires_grad for w in st["masters"])


def test_adamw_of_leaves_and_its_norm():
    _check_leaves_and_norm("cpu")


def _check_pieces_pass_no_gradient(device):
    """No result carries a graph, and a product that would drop a gradient is refused where one would be recorded."""
    x, w = torch.randn(3, 130, device=device, requires_grad=True), torch.ones(130, device=device, requires_grad=True)
    y, h, rstd = F.rmsnorm_quant(x, w, residual=x.detach())
    dx, dw = F.rmsnorm_quant_bwd(h, w, rstd, x)
    b = F.quantize(torch.randn(5, 130, device=device, requires_grad=True), (128, 128))
    out = F.matmul(y, b, out_dtype=torch.float32)
    assert not any(t.requires_grad for t in (y.codes, y.scales, h, rstd, dx, dw, b.codes, b.scales, out, *F.quantize(x)[:2]))
    leaf = torch.zeros(3, 5, device=device, requires_grad=True)
    for call in (lambda: F.matmul(y, b, out_dtype=torch.float32, add=leaf), lambda: F.matmul(y, b, out=leaf), lambda: F.matmul(y, b, out=leaf * 1),
                 lambda: F.matmul(y, b, add=leaf, out=torch.zeros(3, 5, device=device))):
        with pytest.raises(ValueError, match="no gradient"):
            call()
    with torch.no_grad():
        assert torch.equal(F.matmul(y, b, out_dtype=torch.float32, add=leaf), out) and torch.equal(F.matmul(y, b, out=leaf), out)


def test_pieces_pass_no_gradient():
    _check_pieces_pass_no_gradient("cpu")


def _check_linear_of_nothing(device):
    """No tokens, no outputs, nothing to add up: empty results or zeros, and gradients of zero."""
    for shape, n in (((0, 256), 8), ((3, 0, 256), 8), ((4, 256), 0), ((2, 3, 256), 0), ((4, 0), 8), ((0, 0), 8), ((256,), 8)):
        x = torch.zeros(shape, device=device, requires_grad=True)
        w = torch.zeros(n, shape[-1], device=device, requires_grad=True)
        out = F.linear(x, w)
        assert out.shape == (*shape[:-1], n) and not out.any()
        out.sum().backward()
        assert x.grad.shape == x.shape and w.grad.shape == w.shape and not x.grad.any() and not w.grad.any()
        if shape[-1] == 0:
            continue
        leaves = [t.detach().clone().requires_grad_() for t in (x, torch.ones(shape[-1], device=device), w, x)]
        out, h = F.norm_linear(leaves[0], leaves[1], leaves[2], 1e-5, leaves[3])
        assert out.shape == (*shape[:-1], n) and h.shape == x.shape
        (out.sum() + 2 * h.sum()).backward()
        assert not leaves[1].grad.any() and not leaves[2].grad.any() and (leaves[0].grad == 2).all() and torch.equal(leaves[0].grad, leaves[3].grad)


def test_linear_of_nothing():
    _check_linear_of_nothing("cpu")
