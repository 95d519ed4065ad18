"""Products of a language model next to matrix_mul, exported by tilec_b200.ext.

* ``linear_cross_entropy``: the output projection fused with its loss and gradients; the
  [tokens, vocabulary] logits are never kept.

The kernels are behind the C ABI (tilec_linear_ce_* in include/tilec_mm.h).  Like the rest
of the package there is no CPU path: CPU tensors raise, and a missing kernel library raises.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _native

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}             # TILEC_REDUCE_*
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # TILEC_DTYPE_*


def _rows(x):
    """(tensor, row stride) of a 2-D tensor with unit column stride and rows that do not
    overlap, copying only when it must."""
    r, c = x.shape
    s0, s1 = x.stride()
    if (c <= 1 or s1 == 1) and (r <= 1 or s0 >= c):
        return x, (s0 if r > 1 else c)
    return x.contiguous(), c


def _workspace(nbytes, device):
    """Scratch for one call, from torch's allocator: calls on different streams, and graphs
    captured one after the other, never share it."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    from . import ext
    return ext._current_stream(device.index)


def _check_device(stream):
    from . import ext
    if ext._check_enabled():
        ext.check_device(stream)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction):
        lib = _native.load()
        xr, ldx = _rows(x)
        wr, ldw = _rows(weight)
        t, d = x.shape
        v = weight.shape[0]
        dt, red = _DTYPES[x.dtype], _REDUCTIONS[reduction]
        with torch.cuda.device(x.device):
            loss = torch.empty(t if reduction == "none" else (), dtype=torch.float32, device=x.device)
            stats = torch.empty(2 * t + 1, dtype=torch.float32, device=x.device)
            nbytes = lib.tilec_linear_ce_workspace_bytes(_ptr(xr), _ptr(wr), dt, t, v, d, ldx, ldw, red, 0)
            ws = _workspace(nbytes, x.device)
            stream = _stream(x.device)
            rc = lib.tilec_linear_ce_forward(_ptr(xr), _ptr(wr), _ptr(target), dt, t, v, d, ldx, ldw, ignore_index,
                                             red, _ptr(loss), _ptr(stats), _ptr(ws), nbytes, stream)
            _native.check(rc, "tilec_linear_ce_forward")
            _check_device(stream)
        ctx.save_for_backward(x, weight, target, stats)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, target, stats = ctx.saved_tensors
        lib = _native.load()
        xr, ldx = _rows(x)
        wr, ldw = _rows(weight)
        t, d = x.shape
        v = weight.shape[0]
        dt, red = _DTYPES[x.dtype], _REDUCTIONS[ctx.reduction]
        with torch.cuda.device(x.device):
            grad = grad.to(torch.float32).contiguous()
            dx = torch.empty(t, d, dtype=x.dtype, device=x.device) if ctx.needs_input_grad[0] else None
            dw = torch.empty(v, d, dtype=x.dtype, device=x.device) if ctx.needs_input_grad[1] else None
            grads = (1 if dx is not None else 0) | (2 if dw is not None else 0)
            nbytes = lib.tilec_linear_ce_workspace_bytes(_ptr(xr), _ptr(wr), dt, t, v, d, ldx, ldw, red, grads)
            ws = _workspace(nbytes, x.device)
            stream = _stream(x.device)
            rc = lib.tilec_linear_ce_backward(_ptr(xr), _ptr(wr), _ptr(target), dt, t, v, d, ldx, ldw,
                                              ctx.ignore_index, red, _ptr(stats), _ptr(grad), _ptr(dx), _ptr(dw),
                                              _ptr(ws), nbytes, stream)
            _native.check(rc, "tilec_linear_ce_backward")
            _check_device(stream)
        return dx, dw, None, None, None


def linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean"):
    """Cross entropy of softmax(x @ weight.T) against `target`, differentiable in x and weight.

    x [..., D] and weight [V, D]: CUDA tensors of one dtype, float32, float16 or bfloat16;
    target [...]: int64 class indices with x's leading shape.  reduction: "mean" (over the
    tokens whose target is not ignore_index; NaN when there are none), "sum", or "none".
    Returns the float32 loss: a scalar, or one value per token for "none".

    Logits and their softmax are computed in fp32 and never kept: the forward pass keeps two
    floats per token, the backward pass computes the logits again a piece of the vocabulary
    at a time.  Its workspace is at most 512 MiB for a piece (or 4096 vocabulary entries, for
    very many tokens), a copy of x, fp32 sums of x's shape, and a copy of `weight` when its
    rows are not 16-byte aligned.  The gradients are sums in fp32 rounded once to x's dtype;
    the logits' gradient is rounded to the operands' dtype on the way (float32: not at all).

    A token whose target is ignore_index has loss 0 and gradient 0 whatever its row holds; a
    16-bit call does no products for it.  Any other target outside [0, V) makes the token's
    loss and the gradients NaN and sets a device status bit (ext.check_device raises it).
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: unknown reduction {reduction!r}; expected 'mean', 'sum' or 'none'")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_cross_entropy: shapes {tuple(x.shape)} and {tuple(weight.shape)} don't match "
                         "(x [..., D], weight [V, D])")
    if x.dtype not in _DTYPES or weight.dtype != x.dtype:
        raise TypeError(f"linear_cross_entropy: x and weight must share float32, float16 or bfloat16, "
                        f"got {x.dtype} and {weight.dtype}")
    if target.dtype != torch.int64:
        raise TypeError(f"linear_cross_entropy: target must be int64, got {target.dtype}")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: target has shape {tuple(target.shape)}, expected "
                         f"{tuple(x.shape[:-1])}")
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"linear_cross_entropy: weight {tuple(weight.shape)} is empty")
    if not (x.is_cuda and weight.device == x.device and target.device == x.device):
        raise ValueError(f"linear_cross_entropy: inputs must be CUDA tensors on one device (got {x.device}, "
                         f"{weight.device} and {target.device}); tilec_b200 has no CPU path")
    loss = _LinearCrossEntropy.apply(x.reshape(-1, x.shape[-1]), weight, target.reshape(-1).contiguous(),
                                     int(ignore_index), reduction)
    return loss.view(target.shape) if reduction == "none" else loss
