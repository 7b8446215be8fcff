"""Host side of the linear layers of a feed-forward block: gated projections, dropout, 8-bit products.

They stand beside `mm` / `addmm` / `add` of `ops.py`, behind the same C-ABI, and are reached as
`torch.ops.b200.<name>` (`custom_ops.py`):

* `gated_linear`: act(x Wg^T) * (x Wu^T) in one kernel, with its backward pass. The weight is one tensor of
  2 F rows, the gate's first, so that both gradients are one product each.
* `dropout`: x / (1 - p) where a counter-based generator says so, plus the residual; the mask is drawn again in the
  backward pass, never stored.
* `quantize_rows`, `mm_int8`: rows to 8 bits with a scale each, and the product of 8-bit operands with a scale
  to each row and column.

Nothing here computes with torch: outputs are allocated, shapes and strides read, and the library called.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ops
from ._abi import check, lib

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "sigmoid": 4}  # B200_ACT_*
ELAUNCH = -3  # B200_ELAUNCH
INT8_MAX_K = 131071  # B200_INT8_MAX_K: |sum| <= K * 128 * 128 < 2^31


def _on_device_of(fn):
    """Run with the first tensor's device as the current one: streams and launches go by that."""

    def call(first, *args, **kwargs):
        if first.is_cuda and first.get_device() != torch.cuda.current_device():
            with torch.cuda.device(first.get_device()):
                return fn(first, *args, **kwargs)
        return fn(first, *args, **kwargs)

    call.__name__, call.__doc__ = fn.__name__, fn.__doc__
    return call


def _activation(name: str) -> int:
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"gated_linear: activation {name!r} is not one of {', '.join(ACTIVATIONS)}") from None


def _as_rows(t: torch.Tensor) -> torch.Tensor:
    """[..., K] as [rows, K], a view where the strides allow one, else a copy by the strided-copy kernel."""
    if t.dim() == 2:
        return t
    shape = (ops._prod(t.shape[:-1]), t.shape[-1])
    if t.numel() == 0:
        return ops._new(shape, t.dtype, t.device)
    try:
        return t.view(shape)
    except RuntimeError:
        return ops._contig(t).view(shape)


def _pair_args(input: torch.Tensor, weight: torch.Tensor, what: str) -> Tuple[int, int]:
    """(F, K), or the reason why there is none."""
    if input.dim() < 1 or weight.dim() != 2:
        raise RuntimeError(f"{what}: expected an input of one dimension or more and a weight of two, got {list(input.shape)} and {list(weight.shape)}")
    if weight.shape[0] % 2:
        raise RuntimeError(f"{what}: the weight holds the gate's rows and as many for the up projection, got {weight.shape[0]} rows")
    if weight.shape[1] != input.shape[-1]:
        raise RuntimeError(f"{what}: input {list(input.shape)} and weight {list(weight.shape)} cannot be multiplied")
    if input.dtype != weight.dtype:
        raise RuntimeError(f"{what}: expected input and weight to have the same dtype, but got: {input.dtype} != {weight.dtype}")
    if input.dtype not in ops._FLOATS:
        raise ops.UnsupportedByB200(f"{what}: dtype {input.dtype}")
    return weight.shape[0] // 2, weight.shape[1]


def _product(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """a @ b. Large fp32 products take two f16 planes an operand, whose sums are rounded to nearest slab by slab: their
    contractions are as long as a layer is wide, where sums that truncate drift."""
    (M, K), N = a.shape, b.shape[1]
    need = int(lib().b200_linear_f32_scratch_bytes(M, N, K)) if a.dtype == torch.float32 else 0
    if not need:
        return ops.mm_default(a, b)
    out, scratch = ops._new((M, N), a.dtype, a.device), ops._scratch(a.device, need)
    check(
        lib().b200_linear_f32(
            a.data_ptr(), b.data_ptr(), out.data_ptr(), M, N, K, a.stride(0), a.stride(1), b.stride(0), b.stride(1), scratch.data_ptr(), need, ops._status(a.device).data_ptr(), ops._stream_handle()
        ),
        "b200_linear_f32",
    )
    return out


def _scaled_product(a: torch.Tensor, most: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """a @ b in f16, of an `a` whose rows were scaled by powers of two that bring `most` to [2^14, 2^15): the fp32 sums take the factors back."""
    (M, K), N = a.shape, b.shape[1]
    out = ops._new((M, N), a.dtype, a.device)
    if out.numel():
        strides = (a.stride(0), a.stride(1), b.stride(0), b.stride(1))
        need = int(lib().b200_linear_scaled_scratch_bytes(a.data_ptr(), b.data_ptr(), M, N, K, *strides))
        scratch = ops._scratch(a.device, need) if need else None
        check(
            lib().b200_linear_scaled(
                a.data_ptr(), most.data_ptr(), b.data_ptr(), out.data_ptr(), M, N, K, *strides, scratch.data_ptr() if need else None, need, ops._status(a.device).data_ptr(), ops._stream_handle()
            ),
            "b200_linear_scaled",
        )
    return out


def _gated(input: torch.Tensor, weight: torch.Tensor, activation: str, keep: bool, what: str):
    ops._require_cuda(input, weight)
    act = _activation(activation)
    F, K = _pair_args(input, weight, what)
    lead = list(input.shape[:-1])
    out = ops._new(lead + [F], input.dtype, input.device)
    M, fp32 = ops._prod(lead), input.dtype == torch.float32
    planes = int(lib().b200_linear_f32_scratch_bytes(M, 2 * F, K)) if fp32 else 0
    if fp32 and not planes:
        # small fp32 products leave their sums to a gate of its own
        projections = ops.mm_default(_as_rows(input), weight.t())
        if out.numel():
            check(lib().b200_gate(projections.data_ptr(), out.data_ptr(), M, F, act, ops._stream_handle()), "b200_gate")
        return out, projections.view(lead + [2 * F])
    projections = ops._new(lead + [2 * F], torch.float32, input.device) if keep else None
    if fp32:
        x, scratch = _as_rows(input), ops._scratch(out.device, planes)
        check(
            lib().b200_gated_linear_f32(
                x.data_ptr(), weight.data_ptr(), out.data_ptr(), projections.data_ptr() if projections is not None else None, M, F, K, x.stride(0), x.stride(1), weight.stride(0), weight.stride(1), act,
                scratch.data_ptr(), planes, ops._status(out.device).data_ptr(), ops._stream_handle(),
            ),
            "b200_gated_linear_f32",
        )
        return out, projections
    if out.numel():
        x = _as_rows(input)
        args = (M, F, K, x.stride(0), x.stride(1), weight.stride(0), weight.stride(1))
        need = int(lib().b200_gated_linear_scratch_bytes(x.data_ptr(), weight.data_ptr(), *args))
        scratch = ops._scratch(out.device, need) if need else None
        check(
            lib().b200_gated_linear(
                x.data_ptr(), weight.data_ptr(), out.data_ptr(), projections.data_ptr() if projections is not None else None, *args, act, ops._dt(x.dtype),
                scratch.data_ptr() if need else None, need, ops._status(out.device).data_ptr(), ops._stream_handle(),
            ),
            "b200_gated_linear",
        )
    return out, projections


@_on_device_of
def gated_linear(input: torch.Tensor, weight: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """act(input @ weight[:F].T) * (input @ weight[F:].T), [..., K] x [2 F, K] -> [..., F]. One kernel on fp32 sums, with one
    rounding; large fp32 operands are split into two f16 planes before it (2^-22 of an element, 2^-39 of its row's largest
    magnitude), small ones take the package's fp32 product and a gate behind it. `activation`: silu, gelu (erf), gelu_tanh, relu or sigmoid."""
    return _gated(input, weight, activation, False, "gated_linear")[0]


@_on_device_of
def gated_linear_train(input: torch.Tensor, weight: torch.Tensor, activation: str = "silu") -> Tuple[torch.Tensor, torch.Tensor]:
    """(gated_linear's result, the projections [..., 2 F] that its backward pass wants: the fp32 sums, whatever the input's
    type)."""
    return _gated(input, weight, activation, True, "gated_linear_train")


@_on_device_of
def gated_linear_backward(grad_output: torch.Tensor, input: torch.Tensor, weight: torch.Tensor, projections: torch.Tensor, activation: str = "silu", output_mask=(True, True)):
    """(grad_input, grad_weight) of gated_linear, None where `output_mask` is False. With P = [g | u] the
    projections: dP = [grad u act'(g) | grad act(g)] (rounded to the type of the operands: it is one of the two
    products that follow; f16, whose range it need not keep to, holds it twice, scaled by a power of two to each row and to each column), grad_input = dP @ weight,
    grad_weight = dP^T @ input, in one launch where one product after the other would leave SMs idle."""
    ops._require_cuda(grad_output, input, weight, projections)
    act = _activation(activation)
    F, K = _pair_args(input, weight, "gated_linear_backward")
    lead = list(input.shape[:-1])
    if list(grad_output.shape) != lead + [F] or list(projections.shape) != lead + [2 * F]:
        raise RuntimeError(f"gated_linear_backward: input {list(input.shape)} and weight {list(weight.shape)} do not go with grad_output {list(grad_output.shape)} and projections {list(projections.shape)}")
    if grad_output.dtype != input.dtype or projections.dtype != torch.float32:
        raise RuntimeError(f"gated_linear_backward: expected grad_output like the input and fp32 projections, got {grad_output.dtype}, {input.dtype} and {projections.dtype}")
    want_dx, want_dw = (bool(m) for m in output_mask)
    if not (want_dx or want_dw):
        return None, None
    M = ops._prod(lead)
    J = 2 * F
    # rows on lines of 128 bytes for the copy engine (fp32 ones are split into planes from anywhere)
    pitch = J if input.dtype == torch.float32 or J % 64 == 0 else (J + 63) // 64 * 64 if J > 64 else (J + 7) // 8 * 8
    scaled = input.dtype == torch.float16 and M * J > 0
    dp = ops._new((M, pitch), input.dtype, input.device)[:, :J] if want_dx or not scaled else None
    dp_columns = most = None
    if scaled:
        # (the gradient that nobody wants has no dP)
        g, p = ops._contig(grad_output), ops._contig(projections)
        dp_columns = ops._new((M, pitch), input.dtype, input.device)[:, :J] if want_dw else dp
        dp = dp if want_dx else dp_columns
        most = ops._new((M + J,), torch.int32, input.device)
        check(
            lib().b200_gate_backward_scaled(
                g.data_ptr(), p.data_ptr(), dp.data_ptr() if want_dx else None, dp_columns.data_ptr() if want_dw else None, most.data_ptr(), pitch, M, F, act, ops._stream_handle()
            ),
            "b200_gate_backward_scaled",
        )
    elif dp.numel():
        g, p = ops._contig(grad_output), ops._contig(projections)
        check(lib().b200_gate_backward_rows(g.data_ptr(), p.data_ptr(), dp.data_ptr(), pitch, M, F, act, ops._dt(g.dtype), ops._stream_handle()), "b200_gate_backward_rows")
    x = _as_rows(input)
    if dp.numel():
        fp32 = dp.dtype == torch.float32
        xs, ws = (x.stride(0), x.stride(1)), (weight.stride(0), weight.stride(1))
        operands = (dp.data_ptr(), x.data_ptr(), weight.data_ptr())
        scratch_bytes = lib().b200_linear_grads_scaled_scratch_bytes if scaled else lib().b200_linear_grads_scratch_bytes
        need = int(lib().b200_linear_f32_grads_scratch_bytes(M, J, K) if fp32 else scratch_bytes(*operands, M, J, K, pitch, *xs, *ws))
        if need >= 0:
            dx = ops._new(input.shape, input.dtype, input.device) if want_dx else None
            dw = ops._new((J, K), input.dtype, input.device) if want_dw else None
            scratch = ops._scratch(dp.device, need) if need else None
            results = (dx.data_ptr() if want_dx else None, dw.data_ptr() if want_dw else None)
            behind = (scratch.data_ptr() if need else None, need, ops._status(dp.device).data_ptr(), ops._stream_handle())
            if fp32:
                rc = lib().b200_linear_f32_grads(*operands, *results, M, J, K, pitch, 1, *xs, *ws, *behind)
            elif scaled:
                rc = lib().b200_linear_grads_scaled(operands[0], dp_columns.data_ptr(), most.data_ptr(), *operands[1:], *results, M, J, K, pitch, xs[0], ws[0], *behind)
            else:
                rc = lib().b200_linear_grads(*operands, *results, M, J, K, pitch, xs[0], ws[0], ops._dt(dp.dtype), *behind)
            if rc != ELAUNCH:  # (a refused cluster launch: one product after the other)
                check(rc, "b200_linear_grads")
                return dx, dw
    if scaled:
        dx = _scaled_product(dp, most, weight).view(input.shape) if want_dx else None
        return dx, _scaled_product(dp_columns.t(), most[M:], x) if want_dw else None
    dx = _product(dp, weight).view(input.shape) if want_dx else None
    dw = _product(dp.t(), x) if want_dw else None
    return dx, dw


def _dropout(input: torch.Tensor, p: float, state: torch.Tensor, residual: Optional[torch.Tensor], subsequence: int, what: str) -> torch.Tensor:
    ops._require_cuda(input, state, residual)
    if input.dtype not in ops._FLOATS:
        raise ops.UnsupportedByB200(f"{what}: dtype {input.dtype}")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: p must be between 0 and 1, got {p}")
    if state.dtype != torch.int64 or list(state.shape) != [2]:
        raise RuntimeError(f"{what}: state must be two int64 (seed, offset), got {state.dtype} {list(state.shape)}")
    if residual is not None and (residual.shape != input.shape or residual.dtype != input.dtype):
        raise RuntimeError(f"{what}: residual must be like the input, got {residual.dtype} {list(residual.shape)} and {input.dtype} {list(input.shape)}")
    out = ops._new_like(input)
    if out.numel():
        x, r, s = ops._contig(input), ops._contig(residual) if residual is not None else None, ops._contig(state)
        check(
            lib().b200_dropout(x.data_ptr(), r.data_ptr() if r is not None else None, out.data_ptr(), x.numel(), float(p), s.data_ptr(), int(subsequence), ops._dt(x.dtype), ops._stream_handle()),
            "b200_dropout",
        )
    return out


@_on_device_of
def dropout(input: torch.Tensor, p: float, state: torch.Tensor, residual: Optional[torch.Tensor] = None, *, subsequence: int = 0) -> torch.Tensor:
    """residual + (keep ? input / (1 - p) : 0). Element i in row-major order of the shape, whatever the strides, is kept where word
    i % 4 of Philox-4x32-10 for the counter (state[1] + i / 4, subsequence) under the key state[0] is at
    least round(p 2^32). `state` is (seed, offset) in device memory, so that a captured graph draws
    anew when the program advances it between replays: by (numel + 3) // 4, or once a
    step with a `subsequence` to each layer. Dropped elements give 0 whatever they hold."""
    return _dropout(input, p, state, residual, subsequence, "dropout")


@_on_device_of
def dropout_backward(grad_output: torch.Tensor, p: float, state: torch.Tensor, *, subsequence: int = 0) -> torch.Tensor:
    """The gradient of `dropout` for its input: the same mask, drawn again (the residual's is grad_output itself)."""
    return _dropout(grad_output, p, state, None, subsequence, "dropout_backward")


@_on_device_of
def quantize_rows(input: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """[..., K] -> (int8 [..., K], fp32 scales [...]): scale = max|row| / 127, q = row * (127 / max|row|) rounded to even. A row
    whose largest magnitude is below 2^-118 counts as zeros (scale 0); a row that holds an infinity or a NaN has
    that as its scale, and zeros, so that what is made of it is not finite either."""
    ops._require_cuda(input)
    if input.dtype not in ops._FLOATS:
        raise ops.UnsupportedByB200(f"quantize_rows: dtype {input.dtype}")
    if input.dim() < 1:
        raise RuntimeError("quantize_rows: expected an input of one dimension or more")
    lead, cols = list(input.shape[:-1]), input.shape[-1]
    q, scale = ops._new(input.shape, torch.int8, input.device), ops._new(lead, torch.float32, input.device)
    if scale.numel():
        x = _as_rows(input)
        if x.stride(1) != 1 and cols > 1:
            x = ops._contig(x)
        check(lib().b200_quantize_rows(x.data_ptr(), q.data_ptr(), scale.data_ptr(), scale.numel(), cols, x.stride(0), ops._dt(x.dtype), ops._stream_handle()), "b200_quantize_rows")
    return q, scale


def _scales(t: torch.Tensor, n: int, column: bool, what: str) -> torch.Tensor:
    if t.dtype != torch.float32 or list(t.shape) not in ([n], [n, 1] if column else [1, n]):
        raise RuntimeError(f"mm_int8: {what} must be {n} fp32 values, one to each {'row' if column else 'column'}, got {t.dtype} {list(t.shape)}")
    return ops._contig(t)


@_on_device_of
def mm_int8(self: torch.Tensor, mat2: torch.Tensor, self_scale: torch.Tensor, mat2_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, *, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """(self @ mat2) * self_scale[:, None] * mat2_scale + bias: int8 [M, K] and [K, N] of any strides, exact 32-bit sums, fp32 scales to
    each row and column, one rounding to `out_dtype` (fp32, f16 or bf16; the bias's, or bf16). K up to 131071."""
    ops._require_cuda(self, mat2, self_scale, mat2_scale, bias)
    if self.dim() != 2 or mat2.dim() != 2:
        raise RuntimeError("mm_int8: self and mat2 must be matrices")
    (M, K), (K2, N) = self.shape, mat2.shape
    if K != K2:
        raise RuntimeError(f"mm_int8: mat1 and mat2 shapes cannot be multiplied ({M}x{K} and {K2}x{N})")
    if self.dtype != torch.int8 or mat2.dtype != torch.int8:
        raise ops.UnsupportedByB200(f"mm_int8: dtypes {self.dtype} and {mat2.dtype}, expected int8")
    if K > INT8_MAX_K:
        raise ops.UnsupportedByB200(f"mm_int8: a contraction of {K} could overflow 32-bit sums (at most {INT8_MAX_K})")
    if out_dtype is None:
        out_dtype = bias.dtype if bias is not None else torch.bfloat16
    if out_dtype not in ops._FLOATS:
        raise ops.UnsupportedByB200(f"mm_int8: out_dtype {out_dtype}")
    sa, sb = _scales(self_scale, M, True, "self_scale"), _scales(mat2_scale, N, False, "mat2_scale")
    if bias is not None and (bias.dtype != out_dtype or list(bias.shape) != [N]):
        raise RuntimeError(f"mm_int8: bias must be [{N}] of {out_dtype}, got {bias.dtype} {list(bias.shape)}")
    out = ops._new((M, N), out_dtype, self.device)
    if out.numel():
        c = ops._contig(bias) if bias is not None else None
        args = (M, N, K, self.stride(0), self.stride(1), mat2.stride(0), mat2.stride(1))
        need = int(lib().b200_mm_int8_scratch_bytes(self.data_ptr(), mat2.data_ptr(), *args))
        scratch = ops._scratch(out.device, need) if need else None
        check(
            lib().b200_mm_int8(
                self.data_ptr(), mat2.data_ptr(), sa.data_ptr(), sb.data_ptr(), c.data_ptr() if c is not None else None, out.data_ptr(), *args, ops._dt(out_dtype),
                scratch.data_ptr() if need else None, need, ops._status(out.device).data_ptr(), ops._stream_handle(),
            ),
            "b200_mm_int8",
        )
    return out


# --------------------------------------------------------------------- gradients
class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, activation):
        out, projections = torch.ops.b200.gated_linear_train(input, weight, activation)
        ctx.save_for_backward(input, weight, projections)
        ctx.activation = activation
        ctx.mark_non_differentiable(projections)
        return out, projections

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        dx, dw = torch.ops.b200.gated_linear_backward(grad, *ctx.saved_tensors, ctx.activation, list(ctx.needs_input_grad[:2]))
        return dx, dw, None


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, p, state, residual, subsequence):
        ctx.save_for_backward(state)
        ctx.p, ctx.subsequence = p, subsequence
        return torch.ops.b200.dropout(input, p, state, residual, subsequence=subsequence)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (state,) = ctx.saved_tensors
        dx = torch.ops.b200.dropout_backward(grad, ctx.p, state, subsequence=ctx.subsequence) if ctx.needs_input_grad[0] else None
        return dx, None, None, grad if ctx.needs_input_grad[3] else None, None


def _wants_gradient(*tensors) -> bool:
    if torch.autograd.forward_ad._current_level >= 0:  # the autograd functions refuse a forward-mode gradient
        return any(t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors)
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def gated_linear_autograd(input, weight, activation="silu"):
    if _wants_gradient(input, weight):
        return _GatedLinear.apply(input, weight, activation)[0]
    with torch._C._AutoDispatchBelowAutograd():
        return torch.ops.b200.gated_linear(input, weight, activation)


def gated_linear_train_autograd(input, weight, activation="silu"):
    if _wants_gradient(input, weight):
        return _GatedLinear.apply(input, weight, activation)
    with torch._C._AutoDispatchBelowAutograd():
        return torch.ops.b200.gated_linear_train(input, weight, activation)


def dropout_autograd(input, p, state, residual=None, *, subsequence=0):
    if _wants_gradient(input, residual):
        return _Dropout.apply(input, p, state, residual, subsequence)
    with torch._C._AutoDispatchBelowAutograd():
        return torch.ops.b200.dropout(input, p, state, residual, subsequence=subsequence)


# --------------------------------------------------------------------- shapes alone
def _fake_gated(input, weight, activation="silu"):
    F, _ = _pair_args(input, weight, "gated_linear")
    return input.new_empty(list(input.shape[:-1]) + [F])


def _fake_gated_train(input, weight, activation="silu"):
    F, _ = _pair_args(input, weight, "gated_linear_train")
    lead = list(input.shape[:-1])
    return input.new_empty(lead + [F]), input.new_empty(lead + [2 * F], dtype=torch.float32)


def _fake_gated_backward(grad_output, input, weight, projections, activation="silu", output_mask=(True, True)):
    return input.new_empty(input.shape) if output_mask[0] else None, weight.new_empty(weight.shape) if output_mask[1] else None


def _fake_dropout(input, p, state, residual=None, *, subsequence=0):
    return input.new_empty(input.shape)


def _fake_dropout_backward(grad_output, p, state, *, subsequence=0):
    return grad_output.new_empty(grad_output.shape)


def _fake_quantize(input):
    return input.new_empty(input.shape, dtype=torch.int8), input.new_empty(input.shape[:-1], dtype=torch.float32)


def _fake_mm_int8(self, mat2, self_scale, mat2_scale, bias=None, *, out_dtype=None):
    if out_dtype is None:
        out_dtype = bias.dtype if bias is not None else torch.bfloat16
    return self.new_empty((self.shape[0], mat2.shape[1]), dtype=out_dtype)


# name in the b200 namespace -> (schema after the name, fake kernel, autograd kernel or None); the CUDA kernel is the
# function of the same name above
OPERATORS = {
    "gated_linear": ('(Tensor input, Tensor weight, str activation="silu") -> Tensor', _fake_gated, gated_linear_autograd),
    "gated_linear_train": ('(Tensor input, Tensor weight, str activation="silu") -> (Tensor, Tensor)', _fake_gated_train, gated_linear_train_autograd),
    "gated_linear_backward": (
        '(Tensor grad_output, Tensor input, Tensor weight, Tensor projections, str activation="silu", bool[2] output_mask=[True, True]) -> (Tensor?, Tensor?)',
        _fake_gated_backward,
        None,
    ),
    "dropout": ("(Tensor input, float p, Tensor state, Tensor? residual=None, *, int subsequence=0) -> Tensor", _fake_dropout, dropout_autograd),
    "dropout_backward": ("(Tensor grad_output, float p, Tensor state, *, int subsequence=0) -> Tensor", _fake_dropout_backward, None),
    "quantize_rows": ("(Tensor input) -> (Tensor, Tensor)", _fake_quantize, None),
    "mm_int8": ("(Tensor self, Tensor mat2, Tensor self_scale, Tensor mat2_scale, Tensor? bias=None, *, ScalarType? out_dtype=None) -> Tensor", _fake_mm_int8, None),
}
