"""AdamW over many tensors at once, moments in 32 or 8 bits (csrc/kernels/adamw_multi.cu), with a plain PyTorch form.

``adamw_multi`` is the operator; ``MultiTensorAdamW`` keeps the state of a list of parameters for it.
``parallel.dist_optimizer.ShardedAdamW`` is the optimizer for flat buffers that are shared between ranks.
"""
from __future__ import annotations

import bisect
from typing import List, Optional, Sequence

import torch

from . import _lib
from .fp8_ops import E4M3, E8M0, _native, _need, _scale_bytes

STATE_BLOCK = 256       # values that share a scale in an 8-bit moment
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _mix32(x):
    x = ((x ^ (x >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    x = ((x ^ (x >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def state_scales(n: int) -> int:
    """Scales of an 8-bit moment of ``n`` values."""
    return -(-n // STATE_BLOCK)


def encode_state(x: torch.Tensor, random: Optional[torch.Tensor] = None, root: bool = False):
    """(codes, scales) of an fp32 moment: to nearest, or with ``random`` (16 bits per value) as a step rounds.  Values that
    are not finite become NaN codes and do not count for their block's scale."""
    n = x.numel()
    flat = x.detach().reshape(-1).float()
    blocks = torch.zeros(state_scales(n) * STATE_BLOCK, device=x.device)
    blocks[:n] = torch.where(torch.isfinite(flat), flat.abs(), torch.zeros_like(flat))
    blocks = blocks.view(-1, STATE_BLOCK)
    scales = _scale_bytes(blocks.amax(1), E4M3).view(E8M0)
    y = (blocks / scales.float()[:, None]).view(-1)[:n]
    if random is None:
        code = y.to(E4M3).view(torch.uint8).long()
    else:
        # 2^-120 takes e4m3's smallest exponent to fp32's: the cut goes through its denormals too
        code = ((y * 2.0 ** -120).contiguous().view(torch.int32).long() + (random << 4) >> 20).clamp(max=0x7E)
    if root:
        code = torch.where(flat > 0, code.clamp(min=1), code)
    code = torch.where(torch.isfinite(flat), code, torch.full_like(code, 0x7F))
    code = code | (torch.signbit(flat).long() << 7)
    return code.to(torch.uint8).view(E4M3).view(x.shape), scales


def decode_state(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp32 values of an 8-bit moment."""
    flat = codes.reshape(-1)
    return (flat.float() * scales.float().repeat_interleave(STATE_BLOCK)[:flat.numel()]).view(codes.shape)


def _norm64(grads, grad_scale, device) -> torch.Tensor:
    total = torch.zeros(1, dtype=torch.float64, device=device)
    for g in grads:
        total += (g.double() * grad_scale).square().sum()
    return total.sqrt()


@torch.no_grad()
def adamw_multi_reference(params, grads, masters, m, v, step, *, lr, beta1, beta2, eps, weight_decay, grad_scale=1.0, clip=None,
                          m_scales=None, v_scales=None, seed=0):
    step += 1
    t = step.double()
    bc1, root_bc2 = (1 / (1 - beta1 ** t)).float(), (1 / (1 - beta2 ** t)).sqrt().float()
    coef, norm = grad_scale, None
    if clip is not None:
        norm = _norm64(grads, grad_scale, step.device)
        coef = grad_scale * (clip / (norm + 1e-6)).float().clamp(max=1.0)
        norm = norm.float()
    key = _mix32((seed + int(step) * 0x9E3779B1) & 0xFFFFFFFF)
    flat = lambda ts: None if ts is None else [t.view(-1) for t in ts]  # noqa: E731
    params, grads, masters, m, v = flat(params), flat(grads), flat(masters), flat(m), flat(v)
    for i, g in enumerate(grads):
        w = params[i] if masters is None else masters[i]
        g = g.float() * coef
        m32, v32 = (m[i], v[i]) if m_scales is None else (decode_state(m[i], m_scales[i]), decode_state(v[i], v_scales[i]).square())
        m32 = beta1 * m32 + (1 - beta1) * g
        v32 = beta2 * v32 + (1 - beta2) * g * g
        root = v32.sqrt()
        w -= lr * (m32 * bc1 / (root * root_bc2 + eps) + weight_decay * w)
        if masters is not None:
            params[i].copy_(w)
        if m_scales is None:
            m[i].copy_(m32), v[i].copy_(v32)
            continue
        at = torch.arange(g.numel(), device=g.device) & 0xFFFFFFFF
        r = _mix32((at * 0x9E3779B1 + _mix32((key + i * 0x85EBCA77) & 0xFFFFFFFF)) & 0xFFFFFFFF)
        for codes, scales, new, bits, root_ in ((m[i], m_scales[i], m32, r & 0xFFFF, False), (v[i], v_scales[i], root, r >> 16, True)):
            c, s = encode_state(new, bits, root_)
            codes.copy_(c), scales.view(torch.uint8).copy_(s.view(torch.uint8))
    return norm


def _check_written(written, read) -> None:
    """What is written shares memory with nothing else that is written or read."""
    span = lambda t: (t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())  # noqa: E731
    spans = sorted(span(t) for ts in written for t in ts or () if t.numel() > 0)
    _need(all(end <= start for (_, end), (start, _) in zip(spans, spans[1:])), "memory that the step writes is given twice")
    starts = [start for start, _ in spans]
    for lo, hi in (span(t) for t in read if t.numel() > 0):
        i = bisect.bisect_left(starts, lo)
        _need((i == len(spans) or starts[i] >= hi) and (i == 0 or spans[i - 1][1] <= lo), "gradients, factor or status share memory with what the step writes")


def _check_lists(params, grads, masters, m, v, step, m_scales, v_scales):
    n = len(params)
    _need(n > 0, "no parameters")
    for name, ts in (("grads", grads), ("masters", masters), ("m", m), ("v", v), ("m_scales", m_scales), ("v_scales", v_scales)):
        _need(ts is None or len(ts) == n, f"{n} parameters, but {0 if ts is None else len(ts)} {name}")
    _need((m_scales is None) == (v_scales is None), "8-bit moments have scales of m and of v")
    dev, ptype, gtype = params[0].device, params[0].dtype, grads[0].dtype
    _need(ptype in _TYPES and gtype in _TYPES, f"parameters and gradients are bfloat16, float16 or float32, not {ptype} and {gtype}")
    _need(masters is not None or ptype == torch.float32, f"{ptype} parameters need fp32 masters")
    _need(step.dtype == torch.int64 and step.numel() == 1 and step.device == dev, "step has to be one int64 on the parameters' device")
    state = torch.float32 if m_scales is None else E4M3
    for i in range(n):
        size = params[i].numel()
        group = [(params[i], ptype, size), (grads[i], gtype, size), (m[i], state, size), (v[i], state, size)]
        if masters is not None:
            group.append((masters[i], torch.float32, size))
        if m_scales is not None:
            group += [(m_scales[i], E8M0, state_scales(size)), (v_scales[i], E8M0, state_scales(size))]
        for t, dtype, count in group:
            if not (t.dtype == dtype and t.numel() == count and t.device == dev and t.is_contiguous()):
                raise ValueError(f"tensor {i}: {tuple(t.shape)} {t.dtype} on {t.device} where a contiguous one of {count} {dtype} on {dev} belongs")


def adamw_multi(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], masters: Optional[Sequence[torch.Tensor]],
                m: Sequence[torch.Tensor], v: Sequence[torch.Tensor], step: torch.Tensor, *, lr: float, beta1: float, beta2: float,
                eps: float, weight_decay: float, grad_scale: float = 1.0, clip: Optional[float] = None,
                m_scales: Optional[Sequence[torch.Tensor]] = None, v_scales: Optional[Sequence[torch.Tensor]] = None,
                seed: int = 0, factor: Optional[torch.Tensor] = None, status: Sequence[torch.Tensor] = ()) -> Optional[torch.Tensor]:
    """One AdamW step over lists of contiguous tensors, in place; returns the norm of the scaled gradients (fp32, one element)
    where ``clip`` limits it, else None.  What it writes shares memory with nothing else that it is given.

    params: bf16, fp16 or fp32, all of one type; grads: of one type; masters: fp32 (None: fp32 parameters are their own).
    m, v: fp32 moments; with ``m_scales`` and ``v_scales`` (float8_e8m0fnu, one per 256 values) codes in float8_e4m3fn of m and
    of sqrt(v), rounded stochastically by a hash of ``seed``, step, tensor and element: right on average, and the same bits
    for the same inputs.  ``step``: one int64 on the device, counted up by the call, so a captured step can be replayed; all
    other numbers are the call's.  ``status``: up to four int32 words, such as ``fp8_ops.status_word``: when one is not zero as
    the step runs, all stays as it is.  A gradient that is not finite makes its own element NaN, and with ``clip`` all."""
    def call():
        return _native().adamw8(params, grads, masters, m, v, step, lr, beta1, beta2, eps, weight_decay, grad_scale, clip or 0.0, m_scales,
                                   v_scales, seed & 0xFFFFFFFF, factor, status)

    taken, norm = call() if step.is_cuda and (clip is None or clip > 0) else (False, None)
    if not taken:
        _check_lists(params, grads, masters, m, v, step, m_scales, v_scales)
        _need(0 <= beta1 < 1 and 0 <= beta2 < 1, f"betas from 0 to below 1, not {beta1} and {beta2}")
        _need(clip is None or clip > 0, "clip has to be positive")
        _need(clip is None or factor is None, "either clip, or a factor from elsewhere")
        _need(factor is None or (factor.dtype == torch.float32 and factor.numel() == 1 and factor.device == step.device),
              "factor has to be one float32 on the parameters' device")
        _need(len(status) <= 4 and all(s.dtype == torch.int32 and s.numel() > 0 and s.device == step.device for s in status),
              "status: up to four int32 words on the parameters' device")
        _check_written((params, masters, m, v, m_scales, v_scales, [step]),
                       [*grads, *([] if factor is None else [factor]), *(s.reshape(-1)[:1] for s in status)])
        _need(not step.is_cuda, "the native call does not take these tensors")
        if any(int(s.reshape(-1)[0]) for s in status):
            return None if clip is None else _norm64(grads, grad_scale, step.device).float().detach()
        return adamw_multi_reference(params, grads, masters, m, v, step, lr=lr, beta1=beta1, beta2=beta2, eps=eps,
                                     weight_decay=weight_decay, grad_scale=grad_scale if factor is None else grad_scale * float(factor),
                                     clip=clip, m_scales=m_scales, v_scales=v_scales, seed=seed)
    _lib.count(1)
    return norm


class MultiTensorAdamW:
    """AdamW over a list of parameters with ``adamw_multi``: fp32 masters (for 16-bit parameters), moments in 32 or 8 bits.

    ``step()`` takes the parameters' ``.grad`` (all of them set, contiguous, of one type).  State of the whole list lies in
    flat tensors: ``master``, ``m``, ``v`` (in 8 bits: codes of m and of sqrt(v), with ``m_scale`` and ``v_scale``); each
    parameter's part begins at a multiple of 256 values.  ``status``: words that keep a step from changing anything while one
    is not zero; gradients that come of 8-bit products need ``fp8_ops.status_word`` among them."""

    def __init__(self, params: Sequence[torch.Tensor], lr: float = 3e-4, betas=(0.9, 0.95), eps: float = 1e-8, weight_decay: float = 0.1,
                 clip_grad: Optional[float] = None, state_bits: int = 32, seed: int = 0, status: Sequence[torch.Tensor] = ()):
        self.params: List[torch.Tensor] = list(params)
        _need(len(self.params) > 0, "no parameters")
        _need(state_bits in (8, 32), "moments are kept in 8 or 32 bits")
        self.lr, self.betas, self.eps, self.wd, self.clip, self.bits, self.seed = lr, betas, eps, weight_decay, clip_grad, state_bits, seed
        self.status = list(status)
        p0 = self.params[0]
        starts, at = [], 0
        for p in self.params:
            starts.append(at)
            at += state_scales(p.numel()) * STATE_BLOCK
        flat = lambda dtype, per=1: torch.zeros(at // per, dtype=dtype, device=p0.device)  # noqa: E731
        cut = lambda t, per=1: [t[s // per:-(-(s + p.numel()) // per)] for s, p in zip(starts, self.params)]  # noqa: E731
        self.master = flat(torch.float32) if p0.dtype != torch.float32 else None
        self._masters = None if self.master is None else cut(self.master)
        if self._masters is not None:
            for w, p in zip(self._masters, self.params):
                w.copy_(p.detach().reshape(-1))
        state = torch.float32 if state_bits == 32 else torch.uint8
        self.m, self.v = (flat(state) if state_bits == 32 else flat(state).view(E4M3) for _ in range(2))
        self.m_scale, self.v_scale = (None, None) if state_bits == 32 else (flat(torch.uint8, STATE_BLOCK).view(E8M0) for _ in range(2))
        self._m, self._v = cut(self.m), cut(self.v)
        self._m_scales, self._v_scales = (None, None) if state_bits == 32 else (cut(self.m_scale, STATE_BLOCK), cut(self.v_scale, STATE_BLOCK))
        self.step_count = torch.zeros(1, dtype=torch.int64, device=p0.device)

    @torch.no_grad()
    def step(self, grad_scale: float = 1.0) -> Optional[torch.Tensor]:
        """One update; returns the norm of the scaled gradients where it is clipped."""
        grads = [p.grad for p in self.params]
        _need(all(g is not None for g in grads), "a parameter has no gradient")
        return adamw_multi([p.detach() for p in self.params], grads, self._masters, self._m, self._v, self.step_count, lr=self.lr,
                           beta1=self.betas[0], beta2=self.betas[1], eps=self.eps, weight_decay=self.wd, grad_scale=grad_scale,
                           clip=self.clip, m_scales=self._m_scales, v_scales=self._v_scales, seed=self.seed, status=self.status)

    def state_dict(self) -> dict:
        keep = ("master", "m", "v", "m_scale", "v_scale", "step_count")
        return {"bits": self.bits, "sizes": [p.numel() for p in self.params], **{k: getattr(self, k) for k in keep}}

    def load_state_dict(self, sd: dict) -> None:
        _need(sd["bits"] == self.bits and list(sd["sizes"]) == [p.numel() for p in self.params], "state of other parameters or another width")
        for k in ("master", "m", "v", "m_scale", "v_scale", "step_count"):
            mine = getattr(self, k)
            if mine is not None:
                mine.copy_(sd[k]) if mine.dtype != E8M0 else mine.view(torch.uint8).copy_(sd[k].view(torch.uint8))
        if self._masters is not None:
            for w, p in zip(self._masters, self.params):
                p.detach().copy_(w.view(p.shape))
