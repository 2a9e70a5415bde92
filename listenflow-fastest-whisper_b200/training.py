"""Scoring and training operators of the decoder's tail and of the norms, with gradients.

    layer_norm       y = LN(x + residual) with the statistics kept     (fp16 or bf16 rows)
    cross_entropy    -log p(label) under the logits x weight^T          per token
    distillation     T^2 KL(teacher's top logits || student)             per token

Each has a ``*_forward`` and a ``*_backward`` call, which allocate nothing but their results
and a workspace, and an autograd form of its plain name.  The two losses take the final
states [n, width] and the token table [vocab, width] (tied embedding and logits weight).
The logits are never held; their gradient is, in 16 bits, a piece of the vocabulary at a time
(512 MB at most for up to 2^20 rows, which up to some 5000 rows of a 51866-token table is
all of it).

Rows are fp16 or bf16, LayerNorm parameters, losses and log-sum-exps fp32.  Tensors are
contiguous CUDA tensors of one device; the work is queued on ``stream`` (a torch stream or a
cudaStream_t), by default that device's current stream, and results and workspaces are
allocated on it.  Inputs made on other streams are the caller's to wait for; they may be let
go of once a call returns if ``stream`` is a torch stream (their memory is recorded on it),
and with a cudaStream_t, or without ``stream`` where the current stream is not theirs, once
the work has run, as for any torch operator.  Every byte of arithmetic runs in
liblffw_b200.so.
"""

from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _native as native

MAX_TEACHER_ENTRIES = 256
IGNORE_INDEX = -100

_DTYPES = {torch.float16: native.DT_HALF, torch.bfloat16: native.DT_BF16}
_TEACHER_DTYPES = {**_DTYPES, torch.float32: native.DT_FLOAT}


# The current device's index and its current stream's handle, without the objects that
# torch.cuda wraps them in (a tenth of a small call's host time).
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _elsewhere(device: torch.device, stream) -> bool:
    """Whether a call has to make another device or stream current first (see _scope)."""
    return stream is not None or device.index != _current_device()


def _scope(device: torch.device, stream, *inputs: torch.Tensor | None):
    """Makes `device` and `stream` current: allocations follow the current stream.  The memory of
    `inputs` is kept from other uses until a torch stream has read it, should the caller let go
    of them; a cudaStream_t's life is its owner's, so nothing is recorded on one."""
    if stream is None:
        return torch.cuda.device(device)
    if not isinstance(stream, torch.cuda.Stream):
        handle = int(stream)
        stream = torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)
    if stream.device != device:
        raise ValueError(f"stream is on {stream.device}, the tensors on {device}")
    # A stream object around a handle has the handle as its id (the default stream's are 0 both).
    if stream.stream_id != stream.cuda_stream or stream.cuda_stream == 0:
        for t in inputs:
            if t is not None:
                t.record_stream(stream)
    return torch.cuda.stream(stream)


def _rows(t: torch.Tensor, name: str) -> int:
    """Checks 16-bit rows [n, width]; returns their type's code."""
    code = _DTYPES.get(t.dtype)
    if code is None or not t.is_cuda or t.dim() != 2 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous CUDA float16 or bfloat16 tensor [rows, width]")
    return code


def _like(t: torch.Tensor, other: torch.Tensor, name: str, what: str) -> None:
    if t.dtype != other.dtype or t.shape != other.shape or t.device != other.device or not t.is_contiguous():
        raise ValueError(f"{name} must match {what} in type, shape and device, and be contiguous")


def _vector(t: torch.Tensor, dtypes, count: int, device: torch.device, name: str) -> None:
    if t.dtype not in dtypes or t.dim() != 1 or t.shape[0] != count or t.device != device or not t.is_contiguous():
        kinds = " or ".join(str(d).removeprefix("torch.") for d in dtypes)
        raise ValueError(f"{name} must be a contiguous {kinds} tensor [{count}] on {device}")


def _run(call, args, name: str, device: torch.device) -> None:
    status = call(ctypes.byref(args), _raw_stream(device.index))
    if status:
        native.check(status, name)


_FLOAT = (torch.float32,)
_LABELS = (torch.int32, torch.int64)


# ---- LayerNorm ------------------------------------------------------------------


def layer_norm_forward(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-5, *,
                       residual: torch.Tensor | None = None, stream=None):
    """Returns (sum, y, stats): sum = x + residual in the rows' type (x itself without a
    residual), y its LayerNorm, stats fp32 [2, rows] (mean, reciprocal standard deviation)."""
    dtype = _rows(x, "x")
    rows, cols = x.shape
    device = x.device
    _vector(gamma, _FLOAT, cols, device, "gamma")
    _vector(beta, _FLOAT, cols, device, "beta")
    if residual is not None:
        _like(residual, x, "residual", "x")
    if _elsewhere(device, stream):
        with _scope(device, stream, x, gamma, beta, residual):
            return layer_norm_forward(x, gamma, beta, eps, residual=residual)
    total = x if residual is None else torch.empty_like(x)
    y = torch.empty_like(x)
    stats = gamma.new_empty((2, rows))
    if rows:
        a = native.LayerNormTrainArgs(
            ctypes.sizeof(native.LayerNormTrainArgs), rows, cols, dtype, x.data_ptr(),
            None if residual is None else residual.data_ptr(), None if residual is None else total.data_ptr(),
            gamma.data_ptr(), beta.data_ptr(), eps, y.data_ptr(), stats.data_ptr())
        _run(native.library().lffw_layer_norm_train, a, "lffw_layer_norm_train", device)
    return total, y, stats


def layer_norm_backward(dy: torch.Tensor, total: torch.Tensor, gamma: torch.Tensor, stats: torch.Tensor, *,
                        dsum: torch.Tensor | None = None, want_dx: bool = True, want_params: bool = True,
                        stream=None):
    """Gradients of layer_norm_forward: (dx, dgamma, dbeta) from dy, the summed rows and their
    stats.  `dsum` is the gradient that arrives at the sum by the residual stream; dx (the
    gradient of x and of the residual alike) includes it."""
    dtype = _rows(total, "total")
    rows, cols = total.shape
    device = total.device
    _like(dy, total, "dy", "total")
    if dsum is not None:
        _like(dsum, total, "dsum", "total")
    _vector(gamma, _FLOAT, cols, device, "gamma")
    if (stats.dtype != torch.float32 or stats.shape != (2, rows) or stats.device != device
            or not stats.is_contiguous()):
        raise ValueError("stats must be layer_norm_forward's float32 [2, rows]")
    if not want_dx and not want_params:
        raise ValueError("nothing to compute: want_dx and want_params are both false")
    if _elsewhere(device, stream):
        with _scope(device, stream, dy, total, gamma, stats, dsum):
            return layer_norm_backward(dy, total, gamma, stats, dsum=dsum, want_dx=want_dx, want_params=want_params)
    dx = torch.empty_like(total) if want_dx else None
    dgamma = dbeta = workspace = None
    size = 0
    if not rows:
        return (dx, torch.zeros_like(gamma), torch.zeros_like(gamma)) if want_params else (dx, None, None)
    lib = native.library()
    if want_params:
        dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(gamma)
        size = lib.lffw_layer_norm_grad_workspace(rows, cols)
        if size > 0:
            workspace = gamma.new_empty(size // 4)
    a = native.LayerNormGradArgs(
        ctypes.sizeof(native.LayerNormGradArgs), rows, cols, dtype, dy.data_ptr(), total.data_ptr(),
        gamma.data_ptr(), stats.data_ptr(), None if dsum is None else dsum.data_ptr(),
        dx.data_ptr() if want_dx else None, dgamma.data_ptr() if want_params else None,
        dbeta.data_ptr() if want_params else None, None if workspace is None else workspace.data_ptr(), size)
    _run(lib.lffw_layer_norm_grad, a, "lffw_layer_norm_grad", device)
    return dx, dgamma, dbeta


# ---- losses over the vocabulary -----------------------------------------------------


def _operands(x: torch.Tensor, weight: torch.Tensor) -> native.VocabLossArgs:
    dtype = _rows(x, "x")
    _rows(weight, "weight")
    (rows, width), (vocab, weight_width) = x.shape, weight.shape
    if weight.dtype != x.dtype or weight.device != x.device or weight_width != width or not vocab:
        raise ValueError("weight must be [vocab, width] of x's type and device")
    return native.VocabLossArgs(ctypes.sizeof(native.VocabLossArgs), rows, width, vocab, dtype, x.data_ptr(),
                                weight.data_ptr())


def _with_labels(a: native.VocabLossArgs, x: torch.Tensor, labels: torch.Tensor, ignore_index: int) -> None:
    _vector(labels, _LABELS, a.rows, x.device, "labels")
    a.labels, a.label_bytes, a.ignore_index = labels.data_ptr(), labels.element_size(), ignore_index
    a.temperature = 1.0


def _check_teacher(rows: int, device: torch.device, tokens: torch.Tensor, logits: torch.Tensor,
                   temperature: float) -> None:
    if (tokens.dtype != torch.int32 or tokens.dim() != 2 or tokens.shape[0] != rows
            or not 1 <= tokens.shape[1] <= MAX_TEACHER_ENTRIES or tokens.device != device
            or not tokens.is_contiguous()):
        raise ValueError(f"teacher_tokens must be a contiguous int32 tensor [rows, 1 to {MAX_TEACHER_ENTRIES}] "
                         "on x's device")
    if (logits.dtype not in _TEACHER_DTYPES or logits.shape != tokens.shape or logits.device != device
            or not logits.is_contiguous()):
        raise ValueError("teacher_logits must be a contiguous float16, bfloat16 or float32 tensor like teacher_tokens")
    if not 2.0 ** -6 <= temperature <= 2.0 ** 6:
        raise ValueError("temperature must lie in [2^-6, 2^6]")


def _with_teacher(a: native.VocabLossArgs, x: torch.Tensor, tokens: torch.Tensor, logits: torch.Tensor,
                  temperature: float) -> None:
    _check_teacher(a.rows, x.device, tokens, logits, temperature)
    a.teacher_entries, a.teacher_dtype = tokens.shape[1], _TEACHER_DTYPES[logits.dtype]
    a.teacher_tokens, a.teacher_logits, a.temperature = tokens.data_ptr(), logits.data_ptr(), temperature


def _workspace(a: native.VocabLossArgs, x: torch.Tensor, grad: int) -> torch.Tensor:
    size = native.library().lffw_vocab_loss_workspace(ctypes.byref(a), grad)
    if size < 0:
        native.check(native.INVALID_ARGUMENT, "lffw_vocab_loss_workspace")
    workspace = x.new_empty((size + 1) // 2)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), size
    return workspace


def _loss_forward(a: native.VocabLossArgs, x: torch.Tensor, stream, *others: torch.Tensor):
    device, rows = x.device, a.rows
    if _elsewhere(device, stream):
        with _scope(device, stream, x, *others):
            return _loss_forward(a, x, None)
    losses = torch.empty(rows, dtype=torch.float32, device=device)
    lse = torch.empty_like(losses)
    if rows:
        a.losses, a.lse = losses.data_ptr(), lse.data_ptr()
        workspace = _workspace(a, x, 0)  # noqa: F841 (freed after the call is queued)
        _run(native.library().lffw_vocab_loss, a, "lffw_vocab_loss", device)
    return losses, lse


def _loss_backward(a: native.VocabLossArgs, x: torch.Tensor, weight: torch.Tensor, lse: torch.Tensor,
                   dloss: torch.Tensor, want_dx: bool, want_dweight: bool, stream, *targets: torch.Tensor):
    device, rows = x.device, a.rows
    _vector(lse, _FLOAT, rows, device, "lse")
    _vector(dloss, _FLOAT, rows, device, "dloss")
    if not want_dx and not want_dweight:
        raise ValueError("nothing to compute: want_dx and want_dweight are both false")
    if _elsewhere(device, stream):
        with _scope(device, stream, x, weight, lse, dloss, *targets):
            return _loss_backward(a, x, weight, lse, dloss, want_dx, want_dweight, None)
    dx = torch.empty_like(x) if want_dx else None
    if not rows:
        return dx, torch.zeros_like(weight) if want_dweight else None
    dweight = torch.empty_like(weight) if want_dweight else None
    a.lse, a.dloss = lse.data_ptr(), dloss.data_ptr()
    a.dx = dx.data_ptr() if want_dx else None
    a.dweight = dweight.data_ptr() if want_dweight else None
    workspace = _workspace(a, x, 1)  # noqa: F841 (freed after the call is queued)
    _run(native.library().lffw_vocab_loss_grad, a, "lffw_vocab_loss_grad", device)
    return dx, dweight


def cross_entropy_forward(x: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *,
                          ignore_index: int = IGNORE_INDEX, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-token cross entropy of the logits x weight^T: (losses, lse), fp32 [rows].
    labels: int32 or int64 [rows]; a row labelled `ignore_index` has loss 0."""
    a = _operands(x, weight)
    _with_labels(a, x, labels, ignore_index)
    return _loss_forward(a, x, stream, weight, labels)


def cross_entropy_backward(x: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, lse: torch.Tensor,
                           dloss: torch.Tensor, *, ignore_index: int = IGNORE_INDEX, want_dx: bool = True,
                           want_dweight: bool = True, stream=None):
    """(dx, dweight) in x's type from the forward's lse and the losses' gradients dloss."""
    a = _operands(x, weight)
    _with_labels(a, x, labels, ignore_index)
    return _loss_backward(a, x, weight, lse, dloss, want_dx, want_dweight, stream, labels)


def distillation_forward(x: torch.Tensor, weight: torch.Tensor, teacher_tokens: torch.Tensor,
                         teacher_logits: torch.Tensor, *, temperature: float = 1.0,
                         stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-token T^2 KL(t || softmax(x weight^T / T)) with t the softmax of the teacher's
    entries over T: (losses, lse), fp32 [rows].  teacher_tokens int32 [rows, k] (negative:
    entry left out), teacher_logits fp16, bf16 or fp32 [rows, k]."""
    a = _operands(x, weight)
    _with_teacher(a, x, teacher_tokens, teacher_logits, temperature)
    return _loss_forward(a, x, stream, weight, teacher_tokens, teacher_logits)


def distillation_backward(x: torch.Tensor, weight: torch.Tensor, teacher_tokens: torch.Tensor,
                          teacher_logits: torch.Tensor, lse: torch.Tensor, dloss: torch.Tensor, *,
                          temperature: float = 1.0, want_dx: bool = True, want_dweight: bool = True, stream=None):
    """(dx, dweight) in x's type from the forward's lse and the losses' gradients dloss."""
    a = _operands(x, weight)
    _with_teacher(a, x, teacher_tokens, teacher_logits, temperature)
    return _loss_backward(a, x, weight, lse, dloss, want_dx, want_dweight, stream, teacher_tokens, teacher_logits)


def token_error(device: torch.device | int | str | None = None) -> int:
    """Waits for the work queued on `device` (by default the current one), on any stream, then
    reads and clears its token error: 1 when a label or teacher token outside the vocabulary was
    met since the last call (it was treated as ignored), else 0.  A loss sets it on its tensors'
    device."""
    code = ctypes.c_int32(0)
    with contextlib.nullcontext() if device is None else torch.cuda.device(device):
        native.check(native.library().lffw_vocab_loss_error(ctypes.byref(code)), "lffw_vocab_loss_error")
    return int(code.value)


# ---- autograd --------------------------------------------------------------------


def _grad(g: torch.Tensor | None) -> torch.Tensor | None:
    """A gradient the kernels can read: dense and on a 16-byte boundary."""
    if g is None:
        return None
    g = g.contiguous()
    return g if g.data_ptr() % 16 == 0 else g.clone()


# Casts and views between an input and its leaf that _guard_capture looks through.
_GUARDED_STEPS = 8


def _accumulator(t: torch.Tensor):
    """The gradient accumulator of a leaf, also where t is made from it alone by a few casts or
    views (a 16-bit copy of 32-bit weights); None for other tensors."""
    if t.is_leaf:
        return torch.autograd.graph.get_gradient_edge(t).node
    node = t.grad_fn
    for _ in range(_GUARDED_STEPS):
        before = [n for n, _ in node.next_functions if n is not None]
        if len(before) != 1:
            return None
        node = before[0]
        if node.name() == "torch::autograd::AccumulateGrad":
            return node
    return None


def _guard_capture(*inputs: torch.Tensor | None) -> list:
    """Refuses to record, in a CUDA graph capture, an autograd graph over a leaf that an eager
    graph of these operators still holds: the engine would join the eager graph's stream to
    the capture in the backward pass, which invalidates it.  A leaf's gradient accumulator
    lives as long as a graph holds it, and so does the mark left on it here.  Returns the
    accumulators, for the caller to hold until the new graph does."""
    accumulators = []
    if not torch.is_grad_enabled():
        return accumulators
    capturing = None
    for t in inputs:
        if t is None or not t.requires_grad or not t.is_cuda:
            continue
        accumulator = _accumulator(t)
        if accumulator is None:
            continue
        accumulators.append(accumulator)
        if capturing is None:
            capturing = torch.cuda.is_current_stream_capturing()
        mark = accumulator.metadata
        stream = torch.cuda.current_stream(t.device).cuda_stream
        if capturing and mark.get("lffw_stream", stream) != stream:
            raise RuntimeError(
                "an eager autograd graph of this leaf is alive: release its losses before capturing a backward "
                "pass over it, or capture the *_forward and *_backward calls")
        mark["lffw_stream"] = stream
    return accumulators


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, eps, residual):
        total, y, stats = layer_norm_forward(x, gamma, beta, eps, residual=residual)
        ctx.save_for_backward(total, gamma, stats)
        ctx.set_materialize_grads(False)
        return (y,) if residual is None else (y, total)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dsum=None):
        total, gamma, stats = ctx.saved_tensors
        need_x, need_gamma, need_beta, _, need_residual = ctx.needs_input_grad
        if dy is None:
            zero = torch.zeros_like(gamma)
            return (dsum if need_x else None, zero if need_gamma else None, zero.clone() if need_beta else None, None,
                    dsum if need_residual else None)
        dx, dgamma, dbeta = layer_norm_backward(_grad(dy), total, gamma, stats, dsum=_grad(dsum),
                                                want_dx=need_x or need_residual, want_params=need_gamma or need_beta)
        return (dx if need_x else None, dgamma if need_gamma else None, dbeta if need_beta else None, None,
                dx if need_residual else None)


def layer_norm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-5, *,
               residual: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Differentiable (sum, y): sum = x + residual (x itself without one), y its LayerNorm."""
    held = _guard_capture(x, gamma, beta, residual)  # noqa: F841 (kept until the graph holds them)
    out = _LayerNorm.apply(x, gamma, beta, eps, residual)
    return (x, out[0]) if residual is None else (out[1], out[0])


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, labels, ignore_index):
        losses, lse = cross_entropy_forward(x, weight, labels, ignore_index=ignore_index)
        ctx.save_for_backward(x, weight, labels, lse)
        ctx.ignore_index = ignore_index
        return losses

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        x, weight, labels, lse = ctx.saved_tensors
        dx, dweight = cross_entropy_backward(x, weight, labels, lse, _grad(dloss), ignore_index=ctx.ignore_index,
                                             want_dx=ctx.needs_input_grad[0], want_dweight=ctx.needs_input_grad[1])
        return dx, dweight, None, None


def cross_entropy(x: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *,
                  ignore_index: int = IGNORE_INDEX) -> torch.Tensor:
    """Differentiable per-token cross entropy [rows] (see cross_entropy_forward)."""
    held = _guard_capture(x, weight)  # noqa: F841 (kept until the graph holds them)
    return _CrossEntropy.apply(x, weight, labels, ignore_index)


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, teacher_tokens, teacher_logits, temperature):
        losses, lse = distillation_forward(x, weight, teacher_tokens, teacher_logits, temperature=temperature)
        ctx.save_for_backward(x, weight, teacher_tokens, teacher_logits, lse)
        ctx.temperature = temperature
        return losses

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        x, weight, tokens, logits, lse = ctx.saved_tensors
        dx, dweight = distillation_backward(x, weight, tokens, logits, lse, _grad(dloss), temperature=ctx.temperature,
                                            want_dx=ctx.needs_input_grad[0], want_dweight=ctx.needs_input_grad[1])
        return dx, dweight, None, None, None


def distillation(x: torch.Tensor, weight: torch.Tensor, teacher_tokens: torch.Tensor, teacher_logits: torch.Tensor, *,
                 temperature: float = 1.0) -> torch.Tensor:
    """Differentiable per-token distillation loss [rows] (see distillation_forward); the
    teacher's logits are constants."""
    held = _guard_capture(x, weight)  # noqa: F841 (kept until the graph holds them)
    return _Distillation.apply(x, weight, teacher_tokens, teacher_logits, temperature)
