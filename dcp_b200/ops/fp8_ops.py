"""Training in 8 bits: block-scaled codes, their makers and their products (csrc/kernels/fp8_quant.cu, fp8_gemm.cu), each
with a plain fp32 PyTorch form.

A matrix is kept as ``BlockScaled``: codes in ``torch.float8_e4m3fn`` or ``torch.float8_e5m2`` and a power-of-two scale
(``torch.float8_e8m0fnu``) per block of 1 x 128, 128 x 1 or 128 x 128 values; ``value = code * scale``.  The scale is the
smallest power of two with which the block's largest magnitude is representable; a block with a value that is not finite
has the scale NaN and reads back as NaN.

A product's scales have to run along the contraction in blocks of 128, so

* ``y  = x  w^T``   takes x by rows (1 x 128) and w by blocks (128 x 128):  ``matmul(x, w)``
* ``dx = dy w``     takes dy by rows and the same codes of w:               ``matmul(dy, w, trans_b=False)``
* ``dw = dy^T x``   takes both by tokens (128 x 1):                         ``matmul(dy, x, trans_a=True, trans_b=False)``

``linear`` and ``norm_linear`` are these three as autograd functions (of a first derivative; a second is refused); the pieces
that they are made of pass no gradient on.  On a CUDA tensor the kernels always run (a missing library raises); CPU tensors
take the plain forms.  All calls run on the current stream of their tensors' device, allocate their results there and may be
captured into a CUDA graph once a call has been made on the device.  (As with torch's own functions, a backward pass is
captured together with its forward pass, not while an eager graph of the same leaves lives.)
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib

BLOCK = 128
E4M3, E5M2, E8M0 = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu
MAX_NORM_WIDTH = 16384
MAX_ROWS = 2 ** 31 - 1
MAX_BLOCKED = MAX_ROWS - (BLOCK - 1)    # columns of a quantizer, and what a product adds up: whole blocks are counted in 32 bits
_CODES = {E4M3: 0, E5M2: 1}
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_KINDS = {(1, BLOCK): 1, (BLOCK, 1): 2, (BLOCK, BLOCK): 4}
_WAYS = {1: [(1, BLOCK)], 2: [(BLOCK, 1)], 3: [(1, BLOCK), (BLOCK, 1)], 4: [(BLOCK, BLOCK)]}


class BlockScaled(NamedTuple):
    """``codes`` [R, C] and ``scales`` [ceil(R / block[0]), ceil(C / block[1])]."""
    codes: torch.Tensor
    scales: torch.Tensor
    block: Tuple[int, int]

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        wide = torch.float64 if dtype == torch.float64 else torch.float32
        s = self.scales.to(wide)
        for dim in (0, 1):
            if self.block[dim] > 1:
                s = s.repeat_interleave(self.block[dim], dim).narrow(dim, 0, self.codes.shape[dim])
        return (self.codes.to(wide) * s).to(dtype)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _up(n: int, to: int) -> int:
    return -(-n // to) * to


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A 2-D tensor whose rows are contiguous and apart, of any pitch (and any strides without values)."""
    return t if t.numel() == 0 or (t.stride(1) == 1 or t.shape[1] <= 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


_NATIVE = None


def _native():
    """The native host side (``csrc/host/ops8.cpp``), looked up once."""
    global _NATIVE
    if _NATIVE is None:
        _NATIVE = _lib.calls()
    return _NATIVE


def _taken(got):
    """What the native call gave for tensors that are known to be right and have been brought into shape."""
    if got is None:
        raise RuntimeError("the native call does not take these tensors")
    _lib.count(1)
    return got


_STATUS = {}


def _status(device: torch.device) -> torch.Tensor:
    """The device's status word, which bounded waits report to; shared by all calls and graphs, written on failure only."""
    if device.index not in _STATUS:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call one of the 8-bit operators on this device before capturing a graph with them")
        word = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()    # other streams read it
        _STATUS.setdefault(device.index, word)
    return _STATUS[device.index]


def status_word(device: torch.device) -> torch.Tensor:
    """The int32 word of a device that the products and the norm's backward pass report a wait that ran out to (0: none).  What
    they gave is not complete then: an optimizer that reads the word (``status`` of ``optim_ops.adamw_multi``,
    ``extra_status`` of ``ShardedAdamW``) leaves the weights alone until ``check_status`` has raised and cleared it."""
    device = torch.device(device)
    _need(device.type == "cuda", f"status words are those of CUDA devices, not of {device}")
    return _status(device if device.index is not None else torch.device("cuda", torch.cuda.current_device()))


def check_status() -> None:
    """Raise if a bounded wait inside a product ran out since the last call (waits for all streams of the devices)."""
    for index, word in list(_STATUS.items()):
        torch.cuda.synchronize(index)
        code = int(word.item())
        if code:
            word.zero_()
            torch.cuda.synchronize(index)
            raise RuntimeError(f"8-bit product on cuda:{index} gave up waiting (status {code}): its results are not complete")


# --------------------------------------------------------------------------- plain forms (fp32; like the kernels without autograd)
def _scale_bytes(amax: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    mantissa, exponent = torch.frexp(amax)
    k = exponent - (9 if dtype == E4M3 else 16) + (mantissa > 0.875).to(exponent.dtype)   # largest code: 0.875 * 2^9 or 2^16
    k = torch.where(amax > 0, k, torch.full_like(k, -127)).clamp(-127, 127) + 127
    return torch.where(torch.isfinite(amax), k, torch.full_like(k, 255)).to(torch.uint8)


@torch.no_grad()
def quantize_reference(x: torch.Tensor, block: Tuple[int, int] = (1, BLOCK), dtype: torch.dtype = E4M3) -> BlockScaled:
    rows, cols = x.shape
    br, bc = block
    full = torch.zeros(_up(rows, br), _up(cols, bc), dtype=torch.float32, device=x.device)
    full[:rows, :cols] = x
    tiles = full.view(full.shape[0] // br, br, full.shape[1] // bc, bc)
    scales = _scale_bytes(tiles.abs().amax((1, 3)), dtype).view(E8M0)
    largest = torch.finfo(dtype).max
    codes = (tiles / scales.float()[:, None, :, None]).clamp(-largest, largest).view(full.shape)[:rows, :cols]
    return BlockScaled(codes.to(dtype), scales, (br, bc))


@torch.no_grad()
def rmsnorm_quant_reference(x, w, eps, residual=None, dtype=E4M3):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hf = h.float()
    rstd = torch.rsqrt(hf.pow(2).mean(-1) + eps)
    return quantize_reference(hf * rstd[:, None] * w.float(), (1, BLOCK), dtype), h, rstd


@torch.no_grad()
def rmsnorm_quant_bwd_reference(h, w, rstd, dy, add=None):
    xh, g = h.float() * rstd[:, None], dy.float() * w.float()
    dx = rstd[:, None] * (g - xh * (g * xh).mean(-1, keepdim=True))
    if add is not None:
        dx = dx + add.float()
    return dx.to(h.dtype), (dy.float() * xh).sum(0)


@torch.no_grad()
def matmul_reference(a, b, trans_a=False, trans_b=True, out_dtype=torch.bfloat16, add=None):
    x, y = a.dequantize(), b.dequantize()
    out = (x.t() if trans_a else x) @ (y.t() if trans_b else y)
    return (out if add is None else out + add.float()).to(out_dtype)


# --------------------------------------------------------------------------- codes
def _check_matrix(x: torch.Tensor, what: str) -> None:
    _need(x.dim() == 2, f"{what} has to be a matrix, not {tuple(x.shape)}")
    _need(x.dtype in _TYPES, f"{what} has to be bfloat16, float16 or float32, not {x.dtype}")


def _quantize(x: torch.Tensor, ways: int, dtype: torch.dtype):
    kinds = _WAYS[ways]
    got = _native().quantize8(x, ways, dtype == E5M2) if x.is_cuda and dtype in _CODES else None
    if got is None:
        _check_matrix(x, "x")
        _need(dtype in _CODES, f"codes are float8_e4m3fn or float8_e5m2, not {dtype}")
        _need(x.shape[0] <= MAX_ROWS and x.shape[1] <= MAX_BLOCKED, f"up to {MAX_ROWS} rows of {MAX_BLOCKED} columns, not {tuple(x.shape)}")
        if not x.is_cuda:
            return [quantize_reference(x, k, dtype) for k in kinds]
        got = _native().quantize8(_rows(x), ways, dtype == E5M2)
    _taken(got)
    return [BlockScaled(got[2 * i], got[2 * i + 1], k) for i, k in enumerate(kinds)]


def quantize(x: torch.Tensor, block: Tuple[int, int] = (1, BLOCK), dtype: torch.dtype = E4M3) -> BlockScaled:
    """Codes of a matrix (bf16, fp16 or fp32, any pitch) with a scale per block: (1, 128), (128, 1) or (128, 128).  Up to 2^31 - 128
    columns: a longer flat buffer is viewed as several rows."""
    _need(tuple(block) in _KINDS, f"blocks are (1, 128), (128, 1) or (128, 128), not {block}")
    return _quantize(x, _KINDS[tuple(block)], dtype)[0]


def quantize_both(x: torch.Tensor, dtype: torch.dtype = E4M3) -> Tuple[BlockScaled, BlockScaled]:
    """``quantize`` by rows (1, 128) and by columns (128, 1) from one pass over ``x``: what a gradient needs for the input
    gradient and for the weight gradient."""
    return tuple(_quantize(x, 3, dtype))


# --------------------------------------------------------------------------- RMSNorm
def rmsnorm_quant(x: torch.Tensor, w: torch.Tensor, eps: float = 1e-5, residual: Optional[torch.Tensor] = None,
                  dtype: torch.dtype = E4M3):
    """(y, h, rstd): h = x + residual in x's type (x itself without a residual), y = rmsnorm(h) * w as ``BlockScaled`` by rows,
    rounded once; rstd fp32 [rows].  x, residual [rows, width] of any pitch, w [width], all of one type; no autograd."""
    got = _native().norm8(x, w, eps, residual, dtype == E5M2) if x.is_cuda and dtype in _CODES else None
    if got is None:
        _check_matrix(x, "x")
        _need(dtype in _CODES, f"codes are float8_e4m3fn or float8_e5m2, not {dtype}")
        width = x.shape[1]
        _need(w.shape == (width,) and w.dtype == x.dtype, f"w has to be {x.dtype} of {width} channels")
        _need(1 <= width <= MAX_NORM_WIDTH, f"rows of 1 to {MAX_NORM_WIDTH} channels, not {width}")
        _need(residual is None or (residual.shape == x.shape and residual.dtype == x.dtype), "the residual has to be like x")
        _need(all(t.device == x.device for t in (w, residual) if t is not None), "all tensors have to be on x's device")
        if not x.is_cuda:
            return rmsnorm_quant_reference(x, w, eps, residual, dtype)
        got = _native().norm8(_rows(x), w.contiguous(), eps, None if residual is None else _rows(residual), dtype == E5M2)
    codes, scales, h, rstd = _taken(got)
    return BlockScaled(codes, scales, (1, BLOCK)), (x if residual is None else h), rstd


def rmsnorm_quant_bwd(h: torch.Tensor, w: torch.Tensor, rstd: torch.Tensor, dy: torch.Tensor, add: Optional[torch.Tensor] = None):
    """(dx, dw fp32) for what ``rmsnorm_quant`` returned and the gradient ``dy`` of y (of the values the codes stand for);
    ``add``, the gradient of h from elsewhere, is added to dx, which is the gradient of x and of the residual.  Sums in fp32
    and in a fixed order: the same bits in every run."""
    got = _native().norm8_bwd(h, w, rstd, dy, add, _status(h.device)) if h.is_cuda else None
    if got is None:
        _check_matrix(h, "h")
        rows, width = h.shape
        _need(w.shape == (width,) and w.dtype == h.dtype, f"w has to be {h.dtype} of {width} channels")
        _need(1 <= width <= MAX_NORM_WIDTH, f"rows of 1 to {MAX_NORM_WIDTH} channels, not {width}")
        _need(dy.shape == h.shape and dy.dtype == h.dtype, "dy has to be like h")
        _need(add is None or (add.shape == h.shape and add.dtype == h.dtype), "add has to be like h")
        _need(rstd.shape == (rows,) and rstd.dtype == torch.float32, f"rstd has to be float32 of {rows} rows")
        _need(all(t.device == h.device for t in (w, rstd, dy, add) if t is not None), "all tensors have to be on h's device")
        if not h.is_cuda:
            return rmsnorm_quant_bwd_reference(h, w, rstd, dy, add)
        got = _native().norm8_bwd(_rows(h), w.contiguous(), rstd.contiguous(), _rows(dy), None if add is None else _rows(add),
                                     _status(h.device))
    dx, dw = _taken(got)
    return dx, dw


# --------------------------------------------------------------------------- products
def _check_scaled(q: BlockScaled, what: str) -> None:
    codes, scales, block = q
    _need(codes.dim() == 2 and codes.dtype in _CODES, f"{what}: codes have to be a float8_e4m3fn or float8_e5m2 matrix")
    _need(tuple(block) in _KINDS, f"{what}: blocks are (1, 128), (128, 1) or (128, 128), not {block}")
    want = tuple(-(-n // s) for n, s in zip(codes.shape, block))
    _need(scales.dtype == E8M0 and tuple(scales.shape) == want, f"{what}: scales have to be float8_e8m0fnu of shape {want}")
    _need(scales.device == codes.device, f"{what}: codes and scales on two devices")


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Two matrices of one shape and type whose rows are contiguous share no element; interleaved columns of one are apart."""
    (m, n), size = a.shape, a.element_size()
    if m == 0 or n == 0:
        return True
    (pa, pb), d = (t.stride(0) if m > 1 else n for t in (a, b)), b.data_ptr() - a.data_ptr()
    if d >= ((m - 1) * pa + n) * size or -d >= ((m - 1) * pb + n) * size:
        return True
    return pa == pb and n * size <= d % (pa * size) <= (pa - n) * size


def _same_place(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and (a.shape[0] <= 1 or a.stride(0) == b.stride(0))


def matmul(a: BlockScaled, b: BlockScaled, *, trans_a: bool = False, trans_b: bool = True, out_dtype: torch.dtype = torch.bfloat16,
           add: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, form: int = 0) -> torch.Tensor:
    """op(a) op(b) of the values the codes stand for, summed in fp32 and rounded once; ``add`` (of the output's type and shape,
    rows contiguous) is added before the rounding; it may be ``out`` itself, and shares nothing with it otherwise.  No autograd: an
    ``add`` or ``out`` that requires a gradient is refused where one would be recorded.

    a: [M, K], or [K, M] with ``trans_a``; b: [N, K], or [K, N] without ``trans_b`` -> [M, N] in bf16, fp16 or fp32.  Along K
    both need a scale per 128 values; along the other dimension one per value or per 128.  Codes whose rows begin on 16 bytes
    (as the makers here lay them out) are read where they are, others are laid out in each call first.  ``form``: 0 chooses the kernel, 1 and
    2 name it (measurements)."""
    if out is not None:
        out_dtype = out.dtype

    def call(a, b, add):
        return _native().matmul8(*a, *b, trans_a, trans_b, _TYPES.get(out_dtype, -1), add, out, form, _status(a.codes.device))

    got = call(a, b, add) if a.codes.is_cuda and form in (0, 1, 2) else None
    if got is None:
        _check_scaled(a, "a")
        _check_scaled(b, "b")
        ka, kb = (0 if trans_a else 1), (1 if trans_b else 0)
        m, n, k = a.codes.shape[1 - ka], b.codes.shape[1 - kb], a.codes.shape[ka]
        _need(k == b.codes.shape[kb], f"contraction over {k} values of a and {b.codes.shape[kb]} of b")
        _need(k <= MAX_BLOCKED and m <= MAX_ROWS and n <= MAX_ROWS, f"sums of up to {MAX_BLOCKED} values and up to {MAX_ROWS} rows and columns, not {(m, n, k)}")
        _need(a.block[ka] == BLOCK and b.block[kb] == BLOCK, "both operands need a scale per 128 values along the contraction")
        _need(a.codes.device == b.codes.device, "a and b are on two devices")
        _need(form in (0, 1, 2), "form is 0, 1 or 2")
        _need(out_dtype in _TYPES, f"results are bfloat16, float16 or float32, not {out_dtype}")
        if out is not None:
            _need(tuple(out.shape) == (m, n) and out.device == a.codes.device, f"out has to be {(m, n)} on a's device")
            _need(out is _rows(out), "rows of out have to be contiguous")
        if add is not None:
            _need(tuple(add.shape) == (m, n) and add.dtype == out_dtype and add.device == a.codes.device,
                  f"add has to be {out_dtype} {(m, n)} on a's device")
            if out is not None:
                rows = _rows(add)   # a copy where its rows are not contiguous
                _need(_same_place(rows, out) or _apart(rows, out), "add has to be out itself or lie apart from it")
        _need(not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (add, out))),
              "products pass no gradient on: add and out may not require one (see linear and norm_linear)")
        if not a.codes.is_cuda:
            got = matmul_reference(a, b, trans_a, trans_b, out_dtype, add)
            return got if out is None else out.copy_(got)
        if m == 0 or n == 0 or k == 0:
            out = torch.empty(m, n, dtype=out_dtype, device=a.codes.device) if out is None else out
            return out.zero_() if add is None else out.copy_(add)
        got = call(a._replace(codes=_rows(a.codes)), b._replace(codes=_rows(b.codes)), None if add is None else _rows(add))
    return _taken(got) if out is None else (_taken(got), out)[1]


# --------------------------------------------------------------------------- autograd
def _matrix(t: torch.Tensor) -> torch.Tensor:
    """[..., N] as a matrix, without values too."""
    return t.reshape(math.prod(t.shape[:-1]), t.shape[-1])


def _grad_products(dy: torch.Tensor, x: torch.Tensor, wq: BlockScaled, need_x: bool, need_w: bool):
    """(dx, dw) of y = x w^T in 8 bits, in the types of dy."""
    if need_x and need_w:
        by_rows, by_cols = quantize_both(dy)
    else:
        by_rows, by_cols = (quantize(dy) if need_x else None), (quantize(dy, (BLOCK, 1)) if need_w else None)
    dx = matmul(by_rows, wq, trans_b=False, out_dtype=dy.dtype) if need_x else None
    dw = matmul(by_cols, quantize(x, (BLOCK, 1)), trans_a=True, trans_b=False, out_dtype=dy.dtype) if need_w else None
    return dx, dw


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight):
        x2 = _matrix(x)
        wq = quantize(weight, (BLOCK, BLOCK))
        ctx.save_for_backward(x2, wq.codes, wq.scales)
        return matmul(quantize(x2), wq, out_dtype=x.dtype).view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, codes, scales = ctx.saved_tensors
        dx, dw = _grad_products(_matrix(dy), x2, BlockScaled(codes, scales, (BLOCK, BLOCK)), *ctx.needs_input_grad)
        return None if dx is None else dx.view(*dy.shape[:-1], x2.shape[1]), dw


def linear(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """x weight^T with all three products (result, input gradient, weight gradient) in 8 bits; x [..., K], weight [N, K] of one
    type."""
    _need(x.dtype == weight.dtype and weight.dim() == 2 and x.shape[-1] == weight.shape[1], "x [..., K] and weight [N, K] of one type")
    return _Linear.apply(x, weight)


class _NormLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, norm_weight, weight, eps, residual):
        x2 = _matrix(x)
        y, h, rstd = rmsnorm_quant(x2, norm_weight, eps, None if residual is None else residual.reshape(x2.shape))
        wq = quantize(weight, (BLOCK, BLOCK))
        ctx.save_for_backward(h, norm_weight, rstd, wq.codes, wq.scales)
        ctx.with_residual = residual is not None
        ctx.set_materialize_grads(False)
        out = matmul(y, wq, out_dtype=x.dtype).view(*x.shape[:-1], weight.shape[0])
        return out, (h.view(x.shape) if residual is not None else x.view(x.shape))

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dh):
        if dout is None:   # only h was used
            return dh, None, None, None, dh if ctx.with_residual else None
        h, norm_weight, rstd, codes, scales = ctx.saved_tensors
        d2 = _matrix(dout)
        need_w = ctx.needs_input_grad[2]
        # the weight gradient needs the norm's result by tokens: made again, in h's type
        y = (h.float() * rstd[:, None] * norm_weight.float()).to(h.dtype) if need_w else None
        dy, dw = _grad_products(d2, y, BlockScaled(codes, scales, (BLOCK, BLOCK)), True, need_w)
        dx, dnorm = rmsnorm_quant_bwd(h, norm_weight, rstd, dy, None if dh is None else dh.reshape(h.shape).contiguous())
        dx = dx.view(dout.shape[:-1] + h.shape[1:])
        return dx, dnorm.to(norm_weight.dtype), dw, None, dx if ctx.with_residual else None


def norm_linear(x: torch.Tensor, norm_weight: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                residual: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(rmsnorm(h) norm_weight weight^T, h) with h = x + residual, all products in 8 bits; the gradient of h from elsewhere is
    added in the norm's backward pass.  All tensors of one type."""
    _need(x.dtype == weight.dtype == norm_weight.dtype and weight.dim() == 2 and x.shape[-1] == weight.shape[1],
          "x [..., K], norm_weight [K] and weight [N, K] of one type")
    _need(residual is None or (residual.shape == x.shape and residual.dtype == x.dtype), "the residual has to be like x")
    return _NormLinear.apply(x, norm_weight, weight, eps, residual)
