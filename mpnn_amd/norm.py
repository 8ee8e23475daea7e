"""The join between two layers of a deep stack: residual, gate and the norms around them in one pass over the rows.

``block_norm`` computes, per row and in float32 whatever the storage,

    n      = norm(block) * post_weight + post_bias   (post_norm=True; otherwise n = block)
    stream = residual_scale * residual + branch_scale * gate * n
    normed = norm(stream) * weight + bias

The reference has no such operator: its stacks are one or two layers that end in a relu (models/mpnn.py:46-49).  The
forward reads the block's output and the residual stream once and writes both results; the backward reads the same
inputs once more with the two upstream gradients and forms the rows again, so that nothing besides the inputs is kept
between the passes.
"""
from __future__ import annotations

import ctypes
import struct

import torch
from torch.autograd.function import once_differentiable

from . import _lib

NORMS = {"rms": 0, "layer": 1}
OUTPUTS = ("both", "stream", "normed")
MAX_WIDTH = 2048

# struct mpnn_block_norm, field for field (the layout _lib.BlockNormDesc declares): one packing call fills it
_DESC = struct.Struct("@PqPqPq" "PPPP" "qiiiii" "fff" "PqPq" "PqPq" "PqPqPq" "PPPP" "P")
assert _DESC.size == ctypes.sizeof(_lib.BlockNormDesc)


def _p(t) -> int:
    return 0 if t is None else t.data_ptr()


class _Plan:
    """What a call's arguments come to: everything but the tensors."""
    __slots__ = ("norm", "post", "gate_kind", "eps", "rs", "bs", "outputs")


def _forward(plan, block, residual, gate, post_w, post_b, w, b):
    n, h = block.shape
    stream = normed = None
    if plan.outputs != "normed":
        stream = torch.empty((n, h), dtype=block.dtype, device=block.device)
    if plan.outputs != "stream":
        normed = torch.empty((n, h), dtype=block.dtype, device=block.device)
    d = _lib.BlockNormDesc()
    _DESC.pack_into(d, 0, *_inputs(plan, n, h, block, residual, gate, post_w, post_b, w, b),
                    _p(stream), h, _p(normed), h, *_NO_GRADIENTS)
    _lib.check(_lib.load().mpnn_block_norm_fwd(d, _lib.stream_handle(block.device)), "mpnn_block_norm_fwd")
    return stream, normed


_NO_GRADIENTS = (0,) * 15


def _inputs(plan, n, h, block, residual, gate, post_w, post_b, w, b):
    """The fields both directions share (through branch_scale)."""
    ld = _lib.leading
    return (block.data_ptr(), ld(block), _p(residual), ld(residual), _p(gate), ld(gate) if plan.gate_kind > 1 else 0,
            _p(post_w), _p(post_b), _p(w), _p(b), n, h, _lib.dtype_code(block.dtype), plan.norm, plan.gate_kind, plan.post,
            plan.eps, plan.rs, plan.bs)


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, block, residual, gate, post_w, post_b, w, b):
        ctx.set_materialize_grads(False)
        ctx.plan = plan
        ctx.save_for_backward(block, residual, gate, post_w, post_b, w, b)
        stream, normed = _forward(plan, block, residual, gate, post_w, post_b, w, b)
        if plan.outputs == "both":
            return stream, normed
        return stream if normed is None else normed

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        plan = ctx.plan
        tensors = ctx.saved_tensors
        block, residual, gate, post_w, post_b, w, b = tensors
        g_stream = grads[0] if plan.outputs != "normed" else None
        g_normed = grads[-1] if plan.outputs != "stream" else None
        if g_stream is None and g_normed is None:
            return (None,) * 8
        g_stream = None if g_stream is None else _lib.rows_in_place(g_stream)
        g_normed = None if g_normed is None else _lib.rows_in_place(g_normed)
        lib = _lib.load()
        n, h = block.shape
        outs = [torch.empty_like(t, memory_format=torch.contiguous_format)
                if t is not None and need else None for t, need in zip(tensors, ctx.needs_input_grad[1:])]
        g_block, g_residual, g_gate, g_post_w, g_post_b, g_w, g_b = outs
        partial = None
        if (plan.gate_kind == 1 and g_gate is not None) or not (g_post_w is g_post_b is g_w is g_b is None):
            partial = torch.empty(lib.mpnn_block_norm_partial_floats(n, h, _lib.dtype_code(block.dtype)),
                                  dtype=torch.float32, device=block.device)
        ld = _lib.leading
        d = _lib.BlockNormDesc()
        _DESC.pack_into(d, 0, *_inputs(plan, n, h, *tensors), 0, 0, 0, 0, _p(g_stream), ld(g_stream), _p(g_normed), ld(g_normed),
                        _p(g_block), h, _p(g_residual), h, _p(g_gate), 1 if plan.gate_kind == 2 else h,
                        _p(g_post_w), _p(g_post_b), _p(g_w), _p(g_b), _p(partial))
        _lib.check(lib.mpnn_block_norm_bwd(d, _lib.stream_handle(block.device)), "mpnn_block_norm_bwd")
        return (None, *outs)


def _refuse(name, t, like, shape):
    """Why ``t`` cannot stand next to ``like``."""
    _lib.require_device(t, name)
    if t.dtype != like.dtype or t.device != like.device:
        raise TypeError(f"{name} must be {like.dtype} on {like.device} like block, got {t.dtype} on {t.device}")
    raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _gate_kind(gate, n: int, h: int):
    """(kind, the gate in the layout of its kind)"""
    if gate.shape == (h,):
        return 1, gate.contiguous()
    if gate.shape == (n, h):
        return 3, _lib.rows_in_place(gate)
    if gate.shape == (n, 1):
        return 2, gate.contiguous()
    if gate.shape == (1, h):
        return 1, gate.contiguous().view(h)
    raise ValueError(f"gate must have shape [{h}], [1, {h}], [{n}, 1] or [{n}, {h}], got {tuple(gate.shape)}")


def block_norm(block: torch.Tensor, residual: torch.Tensor | None = None, *, norm: str = "rms", eps: float = 1e-5,
               post_norm: bool = False, post_weight: torch.Tensor | None = None, post_bias: torch.Tensor | None = None,
               gate: torch.Tensor | None = None, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               residual_scale: float = 1.0, branch_scale: float = 1.0, outputs: str = "both"):
    """Joins ``block`` [N, H] to the ``residual`` stream and normalises the sum: returns (stream, normed), or one of the
    two with ``outputs="stream"`` / ``"normed"`` (the other is then not computed).

    ``norm``: "rms" or "layer"; weights and biases [H] are optional.  ``gate`` multiplies the branch: [H] (one value per
    channel), [N, 1] (per node) or [N, H].  ``residual=None`` counts as zeros.  float32 or bfloat16 (all operands
    alike), 1 <= H <= 2048, any number of rows, rows at any stride; differentiable once with respect to every tensor."""
    call = _marked if torch.compiler.is_compiling() else _block_norm
    return call(block, residual, norm, eps, post_norm, post_weight, post_bias, gate, weight, bias, residual_scale,
                branch_scale, outputs)


def _block_norm(block, residual, norm, eps, post_norm, post_weight, post_bias, gate, weight, bias, residual_scale, branch_scale,
                outputs):
    _lib.require_device(block, "block")
    _lib.dtype_code(block.dtype)
    if block.dim() != 2 or not 1 <= block.size(1) <= MAX_WIDTH:
        raise ValueError(f"block must have shape [N, H] with 1 <= H <= {MAX_WIDTH}, got {tuple(block.shape)}")
    if norm not in NORMS or outputs not in OUTPUTS:
        raise ValueError(f"norm must be one of {tuple(NORMS)} and outputs one of {OUTPUTS}, got {norm!r}, {outputs!r}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if not post_norm and (post_weight is not None or post_bias is not None):
        raise ValueError("post_weight and post_bias belong to post_norm=True")
    if outputs == "stream" and (weight is not None or bias is not None):
        raise ValueError('weight and bias belong to the normed output, which outputs="stream" leaves out')
    n, h = block.shape
    dtype, device = block.dtype, block.device
    for name, t, shape in (("residual", residual, (n, h)), ("post_weight", post_weight, (h,)), ("post_bias", post_bias, (h,)),
                           ("weight", weight, (h,)), ("bias", bias, (h,)), ("gate", gate, None)):
        if t is not None and (t.dtype != dtype or t.device != device or (shape is not None and t.shape != shape)):
            _refuse(name, t, block, shape)
    plan = _Plan()
    plan.norm, plan.post, plan.eps, plan.outputs = NORMS[norm], int(bool(post_norm)), float(eps), outputs
    plan.rs, plan.bs, plan.gate_kind = float(residual_scale), float(branch_scale), 0
    if gate is not None:
        plan.gate_kind, gate = _gate_kind(gate, n, h)
    c = lambda t: None if t is None else t.contiguous()
    r = _lib.rows_in_place
    tensors = (r(block), None if residual is None else r(residual), gate, c(post_weight), c(post_bias), c(weight), c(bias))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return _BlockNorm.apply(plan, *tensors)
    stream, normed = _forward(plan, *tensors)
    return (stream, normed) if outputs == "both" else (stream if normed is None else normed)


_marked = torch.compiler.disable(_block_norm)      # for a tracing compiler: one graph break, no tracing into the operator
