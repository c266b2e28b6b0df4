"""Functional op surface used by the models.

Each op has two implementations:

* the **HIP path** (``ops/hip_ops.py`` → ``_ddl_kernels.so``): hand-written gfx950 kernels on
  NHWC bf16 tensors, wrapped in ``torch.autograd.Function``s.  This is the path that runs on
  MI355X; it fails loudly if the kernel library is missing.
* the **reference path** (this file, plain PyTorch): used on CPU (tests, the gloo plumbing
  configuration of BASELINE.json) and as the fp32 numerical oracle for every kernel test.
  ``DDL_OPS=aten`` forces it on the GPU too, which is how the stock-PyTorch/MIOpen baseline
  in BASELINE.md is measured.

Semantics follow the reference's model code: conv without bias and explicit padding
(``HorovodTF/src/resnet_model.py:84-109``), training-mode BatchNorm with momentum 0.1
(= decay 0.9) and eps 1e-5 (``:10-11,40-49``) followed by ReLU, with the residual form
``relu(bn(x) + shortcut)`` (``:201-204``), 3×3/2 max-pool (``:264-266``), 7×7 global average
pool (``:287-289``), dense head (``:293-296``), mean softmax cross-entropy
(``imagenet_pytorch_horovod.py:340``).
"""
from __future__ import annotations

import ctypes
import functools
import math
import os

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

__all__ = ["use_hip", "conv2d", "conv_bn_act", "residual_block", "batchnorm_act", "maxpool3x3s2", "global_avgpool", "linear",
           "orthogonalize", "quantize_int8", "linear_int8", "softmax_cross_entropy", "topk_correct", "topk_hits", "NoHipKernel", "set_backend", "backend"]

_FORCED = os.environ.get("DDL_OPS", "auto").lower()  # auto | hip | aten


def set_backend(name: str) -> None:
    global _FORCED
    if name not in ("auto", "hip", "aten"):
        raise ValueError(name)
    _FORCED = name


def backend() -> str:
    return _FORCED


class NoHipKernel(RuntimeError):
    """A GPU tensor reached an op the HIP kernels do not serve.  There is ONE code path on the GPU:
    nothing falls back to ATen/MIOpen unless ``DDL_OPS=aten`` asks for the oracle explicitly."""


def use_hip(t: torch.Tensor) -> bool:
    """HIP kernels serve every GPU tensor (bf16 activations) unless ``DDL_OPS=aten`` selects the
    PyTorch oracle; CPU tensors always take the PyTorch path."""
    if _FORCED == "aten" or not t.is_cuda:
        return False
    if t.dtype != torch.bfloat16:
        raise NoHipKernel("the HIP kernels compute in bf16, got a %s tensor on %s: move the model with "
                          ".to_compute(device, torch.bfloat16) and feed bf16 batches, or set DDL_OPS=aten "
                          "for the PyTorch oracle" % (t.dtype, t.device))
    from . import kernels

    return kernels.require()


def _no_kernel(op, what):
    raise NoHipKernel("ops.%s: no HIP kernel for %s (set DDL_OPS=aten to run the PyTorch oracle instead)"
                      % (op, what))


# ------------------------------------------------------------------------------------------
def conv2d(x, weight, stride=1, padding=0):
    if use_hip(x):
        from . import hip_ops

        if hip_ops.conv_supported(weight, stride, padding):
            return hip_ops.conv2d(x, weight, stride, padding)
        _no_kernel("conv2d", "Cin=%d Cout=%d %dx%d stride %s" % (weight.shape[1], weight.shape[0],
                                                                  weight.shape[2], weight.shape[3], stride))
    return F.conv2d(x, weight.to(x.dtype), None, stride, padding)


def conv_bn_act(x, weight, stride, padding, gamma, beta, running_mean, running_var, training,
                momentum=0.1, eps=1e-5, relu=True, residual=None):
    """``act(bn(conv(x)) [+ residual])`` — on the HIP path the convolution's epilogue emits the
    per-channel batch-statistic partial sums, so BatchNorm never re-reads the conv output to
    compute them (SURVEY §2.6 K1 note / K6)."""
    if use_hip(x):
        from . import hip_ops

        if hip_ops.conv_supported(weight, stride, padding) and hip_ops.bn_supported(weight.shape[0]):
            y, stats = hip_ops.conv2d_stats(x, weight, stride, padding, bool(training))
            return hip_ops.batchnorm_act(y, gamma, beta, running_mean, running_var, training,
                                         momentum, eps, relu, residual, stats)
        _no_kernel("conv_bn_act", "weight %s stride %s" % (tuple(weight.shape), stride))
    y = conv2d(x, weight, stride, padding)
    return batchnorm_act(y, gamma, beta, running_mean, running_var, training, momentum, eps, relu,
                         residual)


def residual_block(x, units, downsample, training, momentum=0.1, eps=1e-5):
    """A whole residual block: ``units`` is the main path as a list of
    ``(weight, stride, padding, gamma, beta, running_mean, running_var)`` conv-BN-ReLU pairs (the
    last one adds the shortcut before its ReLU), ``downsample`` is None (identity shortcut) or
    ``(weight, stride, gamma, beta, running_mean, running_var)`` for the 1x1 projection
    (``HorovodTF/src/resnet_model.py:112-204``).  On the HIP path the block is one autograd
    node with a hand-scheduled backward (``hip_ops.ResidualBlockFn``)."""
    if use_hip(x):
        from . import hip_ops

        convs = [u[0] for u in units] + ([downsample[0]] if downsample is not None else [])
        if hip_ops.residual_block_supported(convs):
            return hip_ops.residual_block(x, units, downsample, training, momentum, eps)
        _no_kernel("residual_block", "convolutions %s" % [tuple(w.shape) for w in convs])
    shortcut = x
    if downsample is not None:
        w, s, g, b, rm, rv = downsample
        shortcut = conv_bn_act(x, w, s, 0, g, b, rm, rv, training, momentum, eps, False)
    cur = x
    for i, (w, s, p, g, b, rm, rv) in enumerate(units):
        last = i == len(units) - 1
        cur = conv_bn_act(cur, w, s, p, g, b, rm, rv, training, momentum, eps, True,
                          shortcut if last else None)
    return cur


def stem(x, weight, stride, padding, gamma, beta, running_mean, running_var, training, momentum=0.1,
         eps=1e-5):
    """ResNet stem: conv -> BatchNorm -> ReLU -> 3x3/2 max pool (``HorovodTF/src/resnet_model.py:
    256-266``).  In training mode on the HIP path this is one fused node (``hip_ops.StemFn``);
    otherwise the composition of the three ops."""
    if training and use_hip(x):
        from . import hip_ops

        if hip_ops.stem_supported(weight, stride, padding) and not x.requires_grad:
            return hip_ops.stem(x, weight, gamma, beta, running_mean, running_var, momentum, eps)
    y = conv_bn_act(x, weight, stride, padding, gamma, beta, running_mean, running_var, training,
                    momentum, eps, True)
    return maxpool3x3s2(y)


def residual_chain(x, blocks, training, momentum=0.1, eps=1e-5):
    """Consecutive residual blocks, ``blocks`` = list of ``(units, downsample)`` as taken by
    :func:`residual_block`.  The intermediate activations are not exposed, which lets the HIP
    path pass ReLU-masked gradients between the fused block nodes
    (``hip_ops.residual_chain``); elsewhere it is just the loop over the blocks."""
    if use_hip(x):
        from . import hip_ops

        if all(hip_ops.residual_block_supported(
                [u[0] for u in units] + ([ds[0]] if ds is not None else []))
               for units, ds in blocks):
            return hip_ops.residual_chain(x, blocks, training, momentum, eps)
        _no_kernel("residual_chain", "one of the blocks' convolutions")
    for units, ds in blocks:
        x = residual_block(x, units, ds, training, momentum, eps)
    return x


def batchnorm_act(x, gamma, beta, running_mean, running_var, training, momentum=0.1, eps=1e-5,
                  relu=True, residual=None):
    """``act(bn(x) [+ residual])`` with act = ReLU or identity; running stats updated in place
    when training (unbiased variance, like torch)."""
    if use_hip(x):
        from . import hip_ops

        if hip_ops.bn_supported(x.shape[1]):
            return hip_ops.batchnorm_act(x, gamma, beta, running_mean, running_var, training,
                                         momentum, eps, relu, residual)
        _no_kernel("batchnorm_act", "C=%d" % x.shape[1])
    y = F.batch_norm(x.float() if x.dtype != torch.float32 and not x.is_cuda else x,
                     running_mean, running_var, gamma, beta, training, momentum, eps)
    y = y.to(x.dtype)
    if residual is not None:
        y = y + residual
    return F.relu(y) if relu else y


def maxpool3x3s2(x):
    if use_hip(x):
        from . import hip_ops

        return hip_ops.maxpool3x3s2(x)
    return F.max_pool2d(x, kernel_size=3, stride=2, padding=1)


def global_avgpool(x):
    """[B,C,H,W] → [B,C]."""
    if use_hip(x):
        from . import hip_ops

        return hip_ops.global_avgpool(x)
    return x.mean(dim=(2, 3))


def linear(x, weight, bias=None):
    if use_hip(x):
        from . import hip_ops

        if x.dim() == 2 and hip_ops.linear_supported(weight):
            return hip_ops.linear(x, weight, bias)
        _no_kernel("linear", "in=%d out=%d on a %d-d input" % (weight.shape[1], weight.shape[0], x.dim()))
    return F.linear(x, weight.to(x.dtype), None if bias is None else bias.to(x.dtype))


def _has_tangent(t):
    """True for a dual tensor of forward-mode differentiation."""
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


ORTHO_COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # five steps take singular values from about 0.002 on into [0.7, 1.2]


@functools.lru_cache(maxsize=256)
def _steps_in_range(a, b, c, steps):
    """True when these steps keep every operand of the kernels in the range of scaled fp16 values: the largest |s (a + b s^2 + c s^4)| and
    |b s^2 + c s^4| over [0, top], top = what the step before leaves (1 at first), at the ends or where a derivative vanishes.
    The library has the same rule (``ddl_ortho_coefficients_ok``); here it holds on every device."""
    a, b, c = (ctypes.c_float(v).value for v in (a, b, c))
    if not all(map(math.isfinite, (a, b, c))):
        return False
    top = 1.0
    for _ in range(steps):
        end = top * top
        at, root = [0.0, end], 9.0 * b * b - 20.0 * a * c
        if c != 0.0:
            if root >= 0.0:
                at += [(-3.0 * b + math.sqrt(root)) / (10.0 * c), (-3.0 * b - math.sqrt(root)) / (10.0 * c)]
        elif b != 0.0:
            at.append(-a / (3.0 * b))
        f = max(math.sqrt(s) * abs(a + b * s + c * s * s) for s in at if 0.0 <= s <= end)
        mid = -b / (2.0 * c) if c != 0.0 and 0.0 < -b / (2.0 * c) < end else 0.0
        p = max(abs(b * s + c * s * s) for s in (end, mid))
        q = max(abs(a + b * s + c * s * s) for s in (0.0, end, mid))
        if not (f * 1.02 <= 8.0 and p * 1.02 <= 15.0 and end <= 15.0 and q <= 1024.0):
            return False
        top = max(f * 1.02, 1.0)
    return True


def _check_steps(steps, coefficients, eps):
    if not isinstance(steps, int) or not 1 <= steps <= 64:
        raise ValueError("orthogonalize: steps must be an integer from 1 to 64, got %r" % (steps,))
    if len(coefficients) != 3:
        raise ValueError("orthogonalize: three coefficients expected, got %r" % (coefficients,))
    if not _steps_in_range(*map(float, coefficients), steps):
        raise ValueError("orthogonalize: %d steps with the coefficients %r leave the range of the kernels' 16-bit operands"
                         % (steps, tuple(coefficients)))
    if not 1e-30 <= eps <= 3e38:
        raise ValueError("orthogonalize: eps must be from 1e-30 to 3e38, got %r" % (eps,))


def orthogonalize_plain(x, steps=5, coefficients=ORTHO_COEFFICIENTS, eps=1e-7):
    """The steps of :func:`orthogonalize` in plain PyTorch, computed and returned in fp32 (fp64 for an fp64 input)."""
    a, b, c = coefficients
    x = x if x.dtype == torch.float64 else x.float()
    turn = x.shape[-2] > x.shape[-1]
    if turn:
        x = x.transpose(-2, -1)
    x = x / x.double().square().sum(dim=(-2, -1), keepdim=True).sqrt().clamp_min(eps).to(x.dtype)
    for _ in range(steps):
        gram = x @ x.transpose(-2, -1).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-2, -1) if turn else x


def orthogonalize(x, steps=5, coefficients=ORTHO_COEFFICIENTS, eps=1e-7):
    """Newton-Schulz orthogonalisation: ``X = G / max(|G|_F, eps)``, then ``steps`` times ``X <- a X + (b A + c A^2) X``
    with ``A = X X^T`` over the shorter side - every singular value of ``G`` is driven towards 1, its vectors stay.

    On the GPU the result is, before its rounding to bf16, about 1e-3 off where both sides are above 32 (products of 16-bit operands), 1e-5 else.

    ``x``: a matrix [r, c], a stack [k, r, c], or a list / tuple of matrices of any shapes (they share the launches), fp32 or
    bf16 of any strides; returns bf16 of the same shape(s).  No gradient flows through it: an input that requires one is
    refused outside ``torch.no_grad()``, a dual tensor always.  Matrices do not influence each other; one that holds an infinity or a NaN
    gives NaN, a zero matrix zeros.  ``coefficients`` whose steps leave the range of 16-bit operands are refused on any device, and on the
    GPU matrices whose sides, rounded up to 64, have a product of 2^30 or more."""
    many = isinstance(x, (list, tuple))
    mats = list(x) if many else [x]
    _check_steps(steps, coefficients, eps)
    for m in mats:
        if m.dim() != 2 and (many or m.dim() != 3):
            raise ValueError("orthogonalize: a matrix, a stack of matrices or a list of matrices expected, got shape %s" % (tuple(m.shape),))
        if m.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("orthogonalize: fp32 or bf16 expected, got %s" % m.dtype)
        if m.device != mats[0].device or m.dtype != mats[0].dtype:
            raise ValueError("orthogonalize: the matrices of a list must share device and dtype")
        if m.requires_grad and torch.is_grad_enabled():
            raise ValueError("orthogonalize: no gradient flows through it; detach the input or call it under torch.no_grad()")
        if _has_tangent(m):
            raise ValueError("orthogonalize: no tangent flows through it; take the primal of the input")
    if not mats:
        return []
    out = None
    if mats[0].is_cuda and _FORCED != "aten":
        from . import kernels

        if kernels.require():
            from . import hip_ops

            out = hip_ops.orthogonalize(mats, steps, tuple(map(float, coefficients)), float(eps))
    if out is None:
        with torch.no_grad():
            out = [orthogonalize_plain(m, steps, coefficients, eps).to(torch.bfloat16).contiguous() for m in mats]
    return out if many else out[0]


_INT8_TINY = 1e-30


def quantize_int8(w):
    """8-bit codes of the rows of ``w`` [n, k] (fp32 or bf16): ``(q, scale)`` with ``q`` int8 [n, k], ``scale`` fp32 [n] and
    ``w ~ q * scale[:, None]``; ``scale = max|row| / 127``, ``q = round(row * (127 * (1 / max|row|)))`` to even, in fp32.  Rows of ``q`` start
    at multiples of 64 bytes, as :func:`linear_int8` reads them.  A row below 1e-30 counts as zero; one that holds an
    infinity or a NaN has the scale NaN.  No gradient and no tangent flows through it."""
    if w.dim() != 2 or w.dtype not in (torch.float32, torch.bfloat16) or w.shape[1] == 0:
        raise ValueError("quantize_int8: an fp32 or bf16 matrix with columns expected, got %s %s" % (w.dtype, tuple(w.shape)))
    w = w.detach()
    if _has_tangent(w):                       # (detach keeps it)
        w = forward_ad.unpack_dual(w).primal
    n, k = w.shape
    if w.is_cuda and _FORCED != "aten":
        from . import kernels

        if kernels.require():
            from . import hip_ops

            return hip_ops.quantize_int8(w)
    store = torch.zeros((n, (k + 63) // 64 * 64), dtype=torch.int8, device=w.device)
    q, scale = _int8_rows_plain(w)
    store[:, :k] = q
    return store[:, :k], scale


def _int8_rows_plain(x):
    x = x.float()
    top = x.abs().amax(dim=1)
    zero = top < _INT8_TINY
    bad = ~torch.isfinite(top)
    inv = torch.where(zero | bad, torch.zeros_like(top), 127.0 * top.reciprocal())
    q = torch.where((zero | bad)[:, None], torch.zeros_like(x), torch.round(x * inv[:, None]))
    scale = torch.where(zero, torch.zeros_like(top), torch.where(bad, torch.full_like(top, float("nan")), top / 127.0))
    return q.to(torch.int8), scale


def linear_int8(x, q, scale, bias=None):
    """Dense layer on 8-bit integers, for answering: the rows of ``x`` [..., k] (fp32 or bf16) are quantised like
    :func:`quantize_int8` does, each with a scale of its own, multiplied with the codes ``q`` [n, k] and ``scale`` [n] of the weights
    and summed exactly: ``y = (xq q^T) * sx * scale + bias`` in fp32, returned in ``x``'s dtype [..., n].  ``bias``: fp32 [n].
    ``q`` as :func:`quantize_int8` returns it (rows start at multiples of 16 bytes).  No gradient flows through it: an input
    that requires one is refused outside ``torch.no_grad()``, a dual tensor always.  ``k`` is at most 133 144."""
    if (x.dtype is not torch.float32 and x.dtype is not torch.bfloat16) or x.dim() < 1:
        raise ValueError("linear_int8: fp32 or bf16 rows expected, got %s" % x.dtype)
    shape, qshape, device = x.shape, q.shape, x.device
    k = shape[-1]
    if q.dtype is not torch.int8 or len(qshape) != 2 or qshape[1] != k or not 0 < k <= 133144:
        raise ValueError("linear_int8: int8 codes [n, %d] of 1 to 133144 columns expected, got %s %s" % (k, q.dtype, tuple(qshape)))
    for name, t in (("scale", scale), ("bias", bias)):
        if t is not None and (t.dtype is not torch.float32 or t.shape != qshape[:1]):
            raise ValueError("linear_int8: %s must be fp32 [%d], got %s %s" % (name, qshape[0], t.dtype, tuple(t.shape)))
    if q.device != device or scale.device != device or (bias is not None and bias.device != device):
        raise ValueError("linear_int8: input, codes, scales and bias must be on one device")
    if torch.is_grad_enabled() and (x.requires_grad or scale.requires_grad or (bias is not None and bias.requires_grad)):
        raise ValueError("linear_int8: no gradient flows through it; call it under torch.no_grad()")
    if _has_tangent(x) or _has_tangent(scale) or (bias is not None and _has_tangent(bias)):
        raise ValueError("linear_int8: no tangent flows through it; take the primal of the input")
    x2 = x if len(shape) == 2 else x.reshape(shape[:-1].numel(), k)
    if device.type == "cuda" and _FORCED != "aten":
        from . import kernels

        if kernels.require():
            from . import hip_ops

            y = hip_ops.linear_int8(x2, q, scale, bias)
            return y if len(shape) == 2 else y.view(shape[:-1] + qshape[:1])
    xq, sx = _int8_rows_plain(x2)
    # (fp64 sums: whole numbers up to 2^31 are exact)
    y = (xq.double() @ q.double().t()).float() * (sx[:, None] * scale[None, :])
    y = y if bias is None else y + bias
    return y.to(x.dtype).view(x.shape[:-1] + q.shape[:1])


def softmax_cross_entropy(logits, target):
    """Mean softmax cross-entropy, computed in fp32; returns an fp32 scalar."""
    if logits.is_cuda and _FORCED != "aten":
        from . import kernels

        if kernels.require():
            from . import hip_ops

            return hip_ops.softmax_cross_entropy(logits, target)
    return F.cross_entropy(logits.float(), target)


def topk_hits(logits, target, ks=(1, 5)):
    """Per-k count of samples whose label is within the top-k logits, as a float64 tensor on the
    logits' device - no host synchronisation, so evaluation loops accumulate it and read once
    (eval metric: ``imagenet_keras_horovod.py:307`` accuracy + top_k_categorical_accuracy,
    ``imagenet_estimator_tf_horovod.py:209-213``).  On the GPU this is K21: one wave per row finds
    the rank of the label's logit, no sort and no [B, k] index tensor."""
    if logits.is_cuda and _FORCED != "aten":
        from . import kernels as K

        K.require()
        if logits.dim() != 2:
            _no_kernel("topk_hits", "a %d-d logits tensor" % logits.dim())
        lg = logits.detach()
        if lg.dtype != torch.bfloat16 or lg.stride(1) != 1:
            lg = lg.to(torch.bfloat16).contiguous()   # the classifier head emits bf16; fp32 callers are rounded once
        rank = K.label_rank(lg, target.contiguous())
        return torch.stack([(rank < k).sum() for k in ks]).double()
    maxk = max(ks)
    _, pred = logits.detach().float().topk(maxk, dim=1)
    hit = pred.eq(target.view(-1, 1))
    return torch.stack([hit[:, :k].any(dim=1).sum() for k in ks]).double()


def topk_correct(logits, target, ks=(1, 5)):
    """:func:`topk_hits` as Python ints (one device synchronisation)."""
    return [int(v) for v in topk_hits(logits, target, ks).tolist()]
