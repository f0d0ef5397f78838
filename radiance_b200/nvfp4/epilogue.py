"""What follows a linear's product in a feed-forward sublayer: activation, dropout and residual.

radiance's ``FeedForward`` ends in ``nn.Dropout`` and its block adds the residual
(src/radiance/model/ffn.py:10-39, block.py:45-71), each a full pass over the output.  Here they run
where the product is (``epilogue_mm``), their backward is one pass that also yields what the
linear's backward needs of the gradient (``epilogue_backward``), and ``dropout`` stands alone for
outputs of other producers.

The dropout mask is a function of a 64-bit seed and the element's row-major index (Philox4x32-10),
drawn where it is needed and never stored; the three operators draw the same mask for the same seed.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from .. import _lib
from . import _trace
from .quantize import NVFP4Tensor, _require_cuda

# The current stream's handle without the Stream object around it (2 us a call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)

_DTYPES = {torch.bfloat16: _lib.RB_DTYPE_BF16, torch.float32: _lib.RB_DTYPE_F32}


def _dtype_of(x: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise ValueError(f"{what}: unsupported dtype {x.dtype} (bf16 or fp32)")
    return code


def _call(what: str, device: torch.device, fn, *args) -> None:
    """One C call (its stream argument appended) with ``device`` current, and its error raised."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, what)


def _tracked(*tensors: torch.Tensor | None) -> bool:
    """Whether autograd follows one of these: in reverse (it requires a gradient) or forward mode (it has a tangent,
    which can be only inside a ``dual_level``: asking each tensor outside one would cost a third of a microsecond)."""
    reverse, forward = torch.is_grad_enabled(), getattr(forward_ad, "_current_level", 0) >= 0
    if reverse or forward:
        for t in tensors:
            if t is not None and ((reverse and t.requires_grad)
                                  or (forward and forward_ad.unpack_dual(t).tangent is not None)):
                return True
    return False


class _Refuse(torch.autograd.Function):
    """Gradients as they are, which cannot be differentiated again."""

    @staticmethod
    def forward(ctx, *grads):
        return grads

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("radiance_b200.nvfp4: these gradients are of first order (once_differentiable) and cannot be "
                           "differentiated again")


class _NoGradient(torch.autograd.Function):
    """A call without a gradient formula on tensors that autograd follows: its results raise in backward, as those
    of ``mm`` do, instead of being taken for constants."""

    @staticmethod
    def forward(ctx, what, call, kwargs, *tensors):
        ctx.set_materialize_grads(False)
        ctx.what = what
        return call(*tensors, **kwargs)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.what} has no gradient formula: FP4Linear differentiates it")


def _no_gradient(what: str, call, out: torch.Tensor | None, kwargs, *tensors):
    """``call(*tensors, out=None, **kwargs)`` for tensors that autograd follows; refused with an ``out``."""
    if out is not None:
        raise ValueError(f"{what}: out= cannot be differentiated, and one of its tensors requires a gradient")
    return _NoGradient.apply(what, call, dict(kwargs, out=None), *tensors)


def _first_order(backward):
    """A Function's backward under ``create_graph``: its gradients raise when they are differentiated again.
    They depend on the upstream gradients, and on the inputs where the forward set ``ctx.curved``; what depends on
    neither is a constant and stays one.  (torch's ``once_differentiable`` asks for the upstream gradients only.)"""

    def wrapper(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not (getattr(ctx, "curved", False) or any(g is not None and g.requires_grad for g in grads)):
            return out
        refused = iter(_Refuse.apply(*(g.detach().requires_grad_() for g in out if g is not None)))
        return tuple(None if g is None else next(refused) for g in out)

    return wrapper


def _size(device: torch.device, fn, *args) -> int:
    """A workspace size, asked with ``device`` current (it goes by the device's SMs)."""
    if device.index == torch.cuda.current_device():
        return int(fn(*args))
    with torch.cuda.device(device):
        return int(fn(*args))


def _rows(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """A 2-D tensor whose rows are contiguous and do not overlap, and its row stride in elements."""
    r, c = x.shape
    if x.is_contiguous():
        return x, c
    if (c > 1 and x.stride(1) != 1) or (r > 1 and x.stride(0) < c):
        x = x.contiguous()
    return x, (x.stride(0) if r > 1 else c)


def _like(name: str, t: torch.Tensor, shape, dtype: torch.dtype, device: torch.device, what: str) -> None:
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != device:
        raise ValueError(f"{what}: {name} must be {dtype} of shape {tuple(shape)} on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")


def _probability(p: float, what: str) -> float:
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: the dropout probability must be in [0, 1], got {p}")
    return p


def dropout_seed(device: torch.device | str = "cuda") -> torch.Tensor:
    """A fresh dropout seed (0-d int64) from torch's CUDA generator: it follows ``torch.manual_seed``, the
    generator state that activation checkpointing restores, and replays of a captured graph."""
    return torch.empty((), dtype=torch.int64, device=device).random_()


def _seed_tensor(seed: torch.Tensor | int | None, device: torch.device, what: str) -> torch.Tensor:
    if seed is None:
        return dropout_seed(device)
    if not isinstance(seed, torch.Tensor):
        return torch.full((), int(seed), dtype=torch.int64, device=device)
    if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
        raise ValueError(f"{what}: seed must be an int or one int64 on {device}, got {seed.dtype} "
                         f"{tuple(seed.shape)} on {seed.device}")
    return seed


# ------------------------------------------------------------------------------------------------
# Dropout
# ------------------------------------------------------------------------------------------------


def _dropout(x: torch.Tensor, residual: torch.Tensor | None, p: float, seed: torch.Tensor | None) -> torch.Tensor:
    what = "nvfp4.dropout"
    code = _dtype_of(x, what)
    x = x.contiguous()
    if residual is not None:
        residual = residual.contiguous()
    y = torch.empty_like(x)
    n = x.numel()
    tok = _trace.begin("dropout", n * x.element_size() * (2 + (residual is not None)))
    _call(what, x.device, _lib.load().rb_nvfp4_dropout, x.data_ptr(),
          None if residual is None else residual.data_ptr(), code, n, p, None if seed is None else seed.data_ptr(),
          y.data_ptr())
    _trace.end(tok)
    return y


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed):
        ctx.p = p
        ctx.save_for_backward(seed)
        return _dropout(x, residual, p, seed)

    @staticmethod
    @_first_order
    def backward(ctx, grad):
        (seed,) = ctx.saved_tensors
        gx = None
        if ctx.needs_input_grad[0]:
            gx = grad if seed is None else _dropout(grad, None, ctx.p, seed)
        return gx, (grad if ctx.needs_input_grad[1] else None), None, None


def dropout(x: torch.Tensor, p: float = 0.5, *, seed: torch.Tensor | int | None = None,
            residual: torch.Tensor | None = None, training: bool = True) -> torch.Tensor:
    """``residual + drop(x)`` in one pass (``residual`` optional), differentiable in both.

    An element is dropped with probability ``t / 65536``, ``t = round(65536 p)``; a kept one is
    multiplied by ``65536 / (65536 - t)``, a dropped one contributes 0 whatever it holds.  bf16 or
    fp32, any shape; product and sum in fp32, rounded once.  ``seed``: an int, a 0-d int64 CUDA
    tensor (read on the device, so a captured graph can change it; it must keep its value until the
    backward pass, which draws the mask again), or None for a fresh ``dropout_seed``.  Equal seeds
    give equal masks for equal element counts.
    """
    what = "nvfp4.dropout"
    _require_cuda(x, what)
    _dtype_of(x, what)
    p = _probability(p, what) if training else 0.0
    if residual is not None:
        _like("residual", residual, x.shape, x.dtype, x.device, what)
    if p == 0.0 and residual is None:
        return x
    seed = _seed_tensor(seed, x.device, what) if p > 0.0 else None
    if _tracked(x, residual):
        return _DropoutFn.apply(x, residual, p, seed)
    return _dropout(x, residual, p, seed)


# ------------------------------------------------------------------------------------------------
# The GEMM with its sublayer's end, and the backward of that end
# ------------------------------------------------------------------------------------------------


def _activation_code(activation: str | None, what: str) -> int:
    code = _lib.RB_ACTIVATIONS.get(activation)
    if code is None:
        names = ", ".join(repr(a) for a in _lib.RB_ACTIVATIONS)
        raise ValueError(f"{what}: activation must be one of {names}, got {activation!r}")
    return code


def _tma_rows(x: torch.Tensor) -> torch.Tensor:
    """A 2-D tensor that a TMA tensor map can describe: 16-byte aligned, with 16-byte row strides."""
    x, ld = _rows(x)
    return x if x.data_ptr() % 16 == 0 and ld * x.element_size() % 16 == 0 else x.contiguous().clone()


def _share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two 2-D tensors of one shape and dtype, with contiguous rows, share an element; rows of
    one stride may interleave (column slices of one buffer)."""
    size, (rows, cols) = a.element_size(), a.shape
    lda, ldb = _rows(a)[1] * size, _rows(b)[1] * size
    width, pa, pb = cols * size, a.data_ptr(), b.data_ptr()
    if pa + (rows - 1) * lda + width <= pb or pb + (rows - 1) * ldb + width <= pa:
        return False
    at = (pb - pa) % lda
    return lda != ldb or at < width or at + width > lda


def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.stride() == b.stride()


def _operand(q: NVFP4Tensor, device: torch.device, what: str) -> None:
    """Refuses an operand whose tensors the kernel would read past or cannot read."""
    rows, k2 = q.packed.shape
    if q.packed.device != device or q.scale.device != device or q.global_scale.device != device:
        raise ValueError(f"{what}: all parts of both operands must be on {device}")
    if not q.packed.is_contiguous() or not q.scale.is_contiguous() or q.packed.element_size() != 1 \
            or q.scale.element_size() != 1 or q.scale.numel() < (rows // 128) * (k2 // 32) * 512 \
            or q.global_scale.dtype != torch.float32 or q.global_scale.numel() != 1:
        raise ValueError(f"{what}: an operand of {rows} x {2 * k2} needs contiguous packed codes, its block scales and "
                         "one fp32 global scale")


def epilogue_mm(a: NVFP4Tensor, b: NVFP4Tensor, *, bias: torch.Tensor | None = None, activation: str | None = None,
                dropout_p: float = 0.0, seed: torch.Tensor | int | None = None, residual: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None, save_preact: bool = False
                ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``residual + drop(act(z))`` with ``z = (a @ b.T) * (ga * gb) + bias``, in one GEMM.

    ``mm`` with the end of a sublayer in its epilogue: everything after the accumulator is fp32 and is
    rounded once, to ``out_dtype`` (bf16 or fp32).  ``activation``: None, "relu", "relu2", "silu", "gelu"
    (erf) or "gelu_tanh".  ``dropout_p`` and ``seed`` as in ``dropout`` (None: a fresh seed; a backward
    pass needs the seed, so keep it).  ``residual``: ``(M, N)`` of ``out_dtype``.  ``out`` may be the
    residual itself.  With ``save_preact`` also returns ``z`` in ``out_dtype``, which
    ``epilogue_backward`` takes.  No gradient formula (``FP4Linear`` has one): where ``bias`` or ``residual``
    requires a gradient, the result raises in backward, and ``out`` is refused.
    """
    if _tracked(bias, residual, out):
        return _no_gradient("nvfp4.epilogue_mm", _epilogue_mm, out,
                            dict(a=a, b=b, activation=activation, dropout_p=dropout_p, seed=seed, out_dtype=out_dtype,
                                 save_preact=save_preact), bias, residual)
    return _epilogue_mm(bias, residual, a, b, activation, dropout_p, seed, out_dtype, out, save_preact)


def _epilogue_mm(bias, residual, a, b, activation, dropout_p, seed, out_dtype, out, save_preact):
    what = "nvfp4.epilogue_mm"
    ap, bp = a.packed, b.packed
    _require_cuda(ap, what)
    dev = ap.device
    (m, k2), (n, k2b) = ap.shape, bp.shape
    if k2 != k2b:
        raise ValueError(f"{what}: contraction mismatch {2 * k2} vs {2 * k2b}")
    _operand(a, dev, what)
    _operand(b, dev, what)
    out_code = _DTYPES.get(out_dtype)
    if out_code is None:
        raise ValueError(f"{what}: unsupported output dtype {out_dtype} (bf16 or fp32)")
    act, p = _activation_code(activation, what), _probability(dropout_p, what)
    seed = _seed_tensor(seed, dev, what) if p > 0.0 else None
    bias_code = 0
    if bias is not None:
        if bias.shape != (n,) or bias.device != dev:
            raise ValueError(f"{what}: bias must have shape ({n},) on {dev}, got {tuple(bias.shape)} on {bias.device}")
        if bias.dtype not in _DTYPES:
            bias = bias.to(torch.float32)
        bias = bias.contiguous()
        if bias.data_ptr() % 16:  # the epilogue reads the bias in vectors
            bias = bias.clone()
        bias_code = _DTYPES[bias.dtype]
    if residual is not None:
        _like("residual", residual, (m, n), out_dtype, dev, what)
    ldo = ldr = n
    given = out is not None
    if not given:
        out = torch.empty(m, n, dtype=out_dtype, device=dev)
    else:
        _like("out", out, (m, n), out_dtype, dev, what)
        if _tma_rows(out) is not out:
            raise ValueError(f"{what}: out must be 16-byte aligned with contiguous rows and 16-byte row strides")
        if residual is not None and _share_memory(out, _rows(residual)[0]) and not _same(out, residual):
            raise ValueError(f"{what}: out overlaps the residual without being the residual")
        ldo = _rows(out)[1]
    if residual is not None:
        residual = _tma_rows(residual)
        ldr = _rows(residual)[1]
    z = torch.empty(m, n, dtype=out_dtype, device=dev) if save_preact else None
    tok = _trace.begin("gemm", 4.0 * m * n * k2)
    _call(what, dev, _lib.load().rb_nvfp4_gemm_epilogue, ap.data_ptr(), a.scale.data_ptr(), bp.data_ptr(),
          b.scale.data_ptr(), m, n, 2 * k2, a.global_scale.data_ptr(), b.global_scale.data_ptr(),
          None if bias is None else bias.data_ptr(), bias_code, act, p, None if seed is None else seed.data_ptr(),
          None if residual is None else residual.data_ptr(), ldr, None if z is None else z.data_ptr(), n,
          out.data_ptr(), out_code, ldo)
    _trace.end(tok)
    if given:
        torch.autograd.graph.increment_version(out)  # written behind autograd's back: who saved it must learn of it
    return (out, z) if save_preact else out


def epilogue_backward(grad_y: torch.Tensor, preact: torch.Tensor | None = None, *, activation: str | None = None,
                      dropout_p: float = 0.0, seed: torch.Tensor | int | None = None, bias_grad: bool = False,
                      out: torch.Tensor | None = None
                      ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """The gradient of ``epilogue_mm``'s pre-activations: ``grad_z = drop(grad_y) * act'(preact)``.

    One pass over ``grad_y`` and ``preact`` (2-D, the same dtype) that also takes the global scale of
    ``grad_z``, which the quantizer of the backward GEMMs needs, and with ``bias_grad`` its fp32 column
    sums.  ``seed`` is the forward call's.  Returns ``(grad_z, global_scale_of(grad_z), sums or None)``.
    The gradient of the residual is ``grad_y`` itself.  No gradient formula, as ``epilogue_mm``.
    """
    if _tracked(grad_y, preact, out):
        return _no_gradient("nvfp4.epilogue_backward", _epilogue_backward, out,
                            dict(activation=activation, dropout_p=dropout_p, seed=seed, bias_grad=bias_grad), grad_y,
                            preact)
    return _epilogue_backward(grad_y, preact, activation, dropout_p, seed, bias_grad, out)


def _epilogue_backward(grad_y, preact, activation, dropout_p, seed, bias_grad, out):
    what = "nvfp4.epilogue_backward"
    _require_cuda(grad_y, what)
    code, act = _dtype_of(grad_y, what), _activation_code(activation, what)
    p = _probability(dropout_p, what)
    if grad_y.dim() != 2 or grad_y.numel() == 0:
        raise ValueError(f"{what}: a non-empty 2-D gradient expected, got shape {tuple(grad_y.shape)}")
    dev, (rows, cols) = grad_y.device, grad_y.shape
    grad_y, ldg = _rows(grad_y)
    z, ldz = None, cols
    if act:
        if preact is None:
            raise ValueError(f"{what}: activation {activation!r} needs the pre-activations")
        _like("preact", preact, (rows, cols), grad_y.dtype, dev, what)
        z, ldz = _rows(preact)
    if p > 0.0:
        if seed is None:
            raise ValueError(f"{what}: dropout needs the forward call's seed")
        seed = _seed_tensor(seed, dev, what)
    ldo = cols
    given = out is not None
    if not given:
        out = torch.empty(rows, cols, dtype=grad_y.dtype, device=dev)
    else:
        _like("out", out, (rows, cols), grad_y.dtype, dev, what)
        if _rows(out)[0] is not out:
            raise ValueError(f"{what}: out must have contiguous rows")
        ldo = _rows(out)[1]
        for name, t in (("gradient", grad_y), ("pre-activations", z)):
            if t is not None and _share_memory(out, t) and not _same(out, t):
                raise ValueError(f"{what}: out overlaps the {name} without being the same tensor")
    gs = torch.empty((), dtype=torch.float32, device=dev)
    sums = torch.empty(cols, dtype=torch.float32, device=dev) if bias_grad else None
    lib = _lib.load()
    need = _size(dev, lib.rb_nvfp4_epilogue_backward_workspace, rows, cols)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    tok = _trace.begin("epilogue", rows * cols * grad_y.element_size() * (2 + (z is not None)))
    _call(what, dev, lib.rb_nvfp4_epilogue_backward, grad_y.data_ptr(), ldg, None if z is None else z.data_ptr(), ldz,
          code, rows, cols, act, p, seed.data_ptr() if p > 0.0 else None, out.data_ptr(), ldo, gs.data_ptr(),
          None if sums is None else sums.data_ptr(), ws.data_ptr(), need)
    _trace.end(tok)
    if given:
        torch.autograd.graph.increment_version(out)
    return out, gs, sums
