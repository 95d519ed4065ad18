"""Products of a language model next to matrix_mul, exported by tilec_b200.ext.

* ``linear_cross_entropy``: the output projection fused with its loss and gradients; the
  [tokens, vocabulary] logits are never kept.
* ``matrix_mul_w4``: x @ W.T with W in 4-bit codes and a scale per group; ``pack_w4`` lays
  out given codes, ``quantize_w4`` makes them from a weight matrix.

The kernels are behind the C ABI (tilec_linear_ce_*, tilec_mm_w4 in include/tilec_mm.h).
Like the rest of the package there is no CPU path for the products: CPU tensors raise, and a
missing kernel library raises.  (Packing and quantising are plain torch and run anywhere.)
"""
from types import SimpleNamespace

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native, select

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


def _library():
    """The kernel library, with the selection table that the fp32 forms' products go by."""
    if not select._installed:
        select.ensure_installed()
    return _native.load()


# torch's count of forward-mode levels: below 0 outside all of them, where no tensor has a tangent.
_levels = forward_ad if hasattr(forward_ad, "_current_level") else SimpleNamespace(_current_level=0)


def _refuse_tangents(where, *tensors):
    """Raises for a tensor with a forward-mode tangent, which the kernels would drop."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{where}: no forward-mode derivative; detach the inputs")


_ext = None   # tilec_b200.ext, which imports this module


def _stream(device):
    global _ext
    if _ext is None:
        from . import ext
        _ext = ext
    return _ext._current_stream(device.index)


def _check_device(stream):
    if _ext._check_enabled():
        _ext.check_device(stream)


class _OnDevice:
    """torch.cuda.device without its cost where the device is already the current one."""

    __slots__ = ("index", "prev")

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        self.prev = torch.cuda.current_device()
        if self.prev != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.prev != self.index:
            torch.cuda.set_device(self.prev)


_CE_BYTES = {}   # arguments that decide it -> workspace bytes of tilec_linear_ce_*


def _ce_workspace(lib, px, pw, dt, t, v, d, ldx, ldw, red, grads, device):
    """(workspace, bytes); operands count as far as their alignment goes."""
    key = (dt, t, v, d, ldx, ldw, red, grads, (px or 0) & 15, pw & 15, device.index)
    nbytes = _CE_BYTES.get(key)
    if nbytes is None:
        nbytes = lib.tilec_linear_ce_workspace_bytes(px, pw, dt, t, v, d, ldx, ldw, red, grads)
        if len(_CE_BYTES) >= 4096:   # a process that sees many shapes: start over
            _CE_BYTES.clear()
        _CE_BYTES[key] = nbytes
    return _workspace(nbytes, device), nbytes


def _ce_forward(x, weight, target, ignore_index, reduction):
    """(loss, statistics for the backward pass)"""
    lib, fast, dev = _library(), _native.fast(), x.device
    xr, ldx = _rows(x)
    wr, ldw = _rows(weight)
    t, d = x.shape
    v = weight.shape[0]
    dt, red = _DTYPES[x.dtype], _REDUCTIONS[reduction]
    with _OnDevice(dev.index):
        stats = torch.empty(2 * t + 1, dtype=torch.float32, device=dev)
        loss = stats.new_empty(t if reduction == "none" else ())
        px, pw = xr.data_ptr(), wr.data_ptr()
        ws, nbytes = _ce_workspace(lib, px, pw, dt, t, v, d, ldx, ldw, red, 0, dev)
        stream = _stream(dev)
        rc = (fast.ce_forward if fast is not None else lib.tilec_linear_ce_forward)(
            px, pw, target.data_ptr(), dt, t, v, d, ldx, ldw, ignore_index, red, loss.data_ptr(), stats.data_ptr(),
            _ptr(ws), nbytes, stream)
        _native.check(rc, "tilec_linear_ce_forward")
        _check_device(stream)
    return loss, stats


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction):
        loss, stats = _ce_forward(x, weight, target, ignore_index, reduction)
        ctx.save_for_backward(x, weight, target, stats)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, target, stats = ctx.saved_tensors
        lib, fast, dev = _library(), _native.fast(), x.device
        xr, ldx = _rows(x)
        wr, ldw = _rows(weight)
        t, d = x.shape
        v = weight.shape[0]
        dt, red = _DTYPES[x.dtype], _REDUCTIONS[ctx.reduction]
        with _OnDevice(dev.index):
            grad = grad.to(torch.float32).contiguous()
            dx = x.new_empty(t, d) if ctx.needs_input_grad[0] else None
            dw = weight.new_empty(v, d) if ctx.needs_input_grad[1] else None
            grads = (1 if dx is not None else 0) | (2 if dw is not None else 0)
            px, pw = xr.data_ptr(), wr.data_ptr()
            ws, nbytes = _ce_workspace(lib, px, pw, dt, t, v, d, ldx, ldw, red, grads, dev)
            stream = _stream(dev)
            rc = (fast.ce_backward if fast is not None else lib.tilec_linear_ce_backward)(
                px, pw, target.data_ptr(), dt, t, v, d, ldx, ldw, ctx.ignore_index, red, stats.data_ptr(),
                grad.data_ptr(), _ptr(dx), _ptr(dw), _ptr(ws), nbytes, stream)
            _native.check(rc, "tilec_linear_ce_backward")
            _check_device(stream)
        return dx, dw, None, None, None


def linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean"):
    """Cross entropy of softmax(x @ weight.T) against `target`, differentiable in x and weight.

    x [..., D] and weight [V, D]: CUDA tensors of one dtype, float32, float16 or bfloat16;
    target [...]: int64 class indices with x's leading shape.  reduction: "mean" (over the
    tokens whose target is not ignore_index; NaN when there are none), "sum", or "none".
    Returns the float32 loss: a scalar, or one value per token for "none".  Gradients are
    reverse-mode and of first order: forward-mode tangents are refused.

    Logits and their softmax are computed in fp32 and never kept whole: the forward pass keeps
    two floats per token, the backward pass computes the logits again a piece of the vocabulary
    at a time.  The gradients are sums in fp32 rounded once to x's dtype; the logits' gradient is
    rounded to the operands' dtype on the way (float32: not at all).

    Workspace of a forward pass: 16 bytes per token and 256 vocabulary entries (512 MiB for 65536
    tokens and 131072 entries); of 16-bit operands a copy of x above 256 tokens; of float32 ones a
    piece of the logits.  Of a backward pass: a piece of the logits' gradient and a copy of x,
    fp32 sums of x's shape where there are several pieces, at most 20 MB of partial sums, and,
    where D is no multiple of 8, a 16-bit copy of a piece's gradient (of the whole weight's, where
    one piece is all of the vocabulary).  Of either: a copy of `weight` when its 16-bit rows are
    not 16-byte aligned, and what the float32 products take (operands that are not aligned,
    partial sums).  A piece is at most 512 MiB, or 4096 vocabulary entries for very many tokens.

    A token whose target is ignore_index has loss 0 and gradient 0 whatever its row holds; with
    16-bit operands a backward pass, and a forward pass of more than 256 tokens, do no products
    for it.  Any other target outside [0, V) makes the token's loss and the gradients NaN and
    sets a device status bit (ext.check_device raises it).

    Forward and backward can be captured into a CUDA graph.  As with any torch operator, drop
    the losses of eager calls on the same leaves before capturing a backward() (or capture
    torch.autograd.grad): torch adds to a leaf's .grad on the stream of the oldest live graph
    that uses it, which is not the captured one.
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
    if _levels._current_level >= 0:
        _refuse_tangents("linear_cross_entropy", x, weight)
    if not (x.is_cuda and weight.device == x.device and target.device == x.device):
        raise ValueError(f"linear_cross_entropy: inputs must be CUDA tensors on one device (got {x.device}, "
                         f"{weight.device} and {target.device}); tilec_b200 has no CPU path")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    y = target if target.dim() == 1 else target.reshape(-1)
    if not y.is_contiguous():
        y = y.contiguous()
    if torch.is_grad_enabled() and (x2.requires_grad or weight.requires_grad):
        loss = _LinearCrossEntropy.apply(x2, weight, y, int(ignore_index), reduction)
    else:
        loss = _ce_forward(x2, weight, y, int(ignore_index), reduction)[0]
    return loss.view(target.shape) if reduction == "none" and target.dim() != 1 else loss


# ---------------------------------------------------------------- 4-bit weights
_BLOCK = 128   # k per 64-byte block of codes (tilec_mm_w4 in include/tilec_mm.h)


def _check_group(group_size, where):
    if not isinstance(group_size, int) or not (group_size in (32, 64) or (group_size > 0 and group_size % _BLOCK == 0)):
        raise ValueError(f"{where}: group_size must be 32, 64 or a multiple of 128, got {group_size!r}")


class W4Weight:
    """A weight [N, K] in 4-bit codes, laid out for matrix_mul_w4 (see pack_w4).

    shape (N, K); group_size; scale_dtype; data uint8 [row tiles of 16, blocks of 128 k, bytes]:
    each piece's group words, then its codes (tilec_mm_w4 in include/tilec_mm.h).
    matrix_mul_w4 reads it in place, so the four are checked against each other here and are
    read-only."""

    def __init__(self, shape, group_size, scale_dtype, data):
        n, k = (int(i) for i in shape)
        _check_group(group_size, "W4Weight")
        if n < 0 or k < 1:
            raise ValueError(f"W4Weight: shape must be (N, K) with K >= 1, got {(n, k)}")
        if scale_dtype not in _DTYPES:
            raise TypeError(f"W4Weight: scales must be float32, float16 or bfloat16, got {scale_dtype}")
        if data.dtype != torch.uint8:
            raise TypeError(f"W4Weight: data must be uint8, got {data.dtype}")
        words = 16 * max(1, _BLOCK // group_size) * (8 if scale_dtype == torch.float32 else 4)
        want = (-(-n // 16), -(-k // _BLOCK), words + 1024)
        if tuple(data.shape) != want or not data.is_contiguous() or data.data_ptr() % 16:
            raise ValueError(f"W4Weight: data must be contiguous, 16-byte aligned and of shape {want}, "
                             f"got shape {tuple(data.shape)}")
        self._shape, self._group_size, self._scale_dtype, self._data = (n, k), group_size, scale_dtype, data

    shape = property(lambda self: self._shape)
    group_size = property(lambda self: self._group_size)
    scale_dtype = property(lambda self: self._scale_dtype)
    data = property(lambda self: self._data)
    device = property(lambda self: self._data.device)

    def to(self, device):
        return W4Weight(self.shape, self.group_size, self.scale_dtype, self.data.to(device))

    def unpack(self):
        """The codes as uint8 [N, K], one per byte, in k order."""
        n, k = self.shape
        codes = self.data[:, :, -1024:].reshape(*self.data.shape[:2], 16, 64)
        w = codes.transpose(1, 2).reshape(-1, self.data.shape[1], 4, 4, 4)   # row, block, t, j, byte of the word
        nib = torch.stack((w & 15, w >> 4), -1).flatten(-2)        # nibbles 0..7 of the word
        nib = nib.view(*nib.shape[:-1], 2, 4).transpose(-1, -2)    # (i, parity): k = 2i + parity
        return nib.flatten(-2).transpose(2, 3).reshape(-1, self.data.shape[1] * _BLOCK)[:n, :k]

    def _words(self):
        """The group words as int32 [N, groups, 1 or 2]."""
        n, k = self.shape
        tiles, blocks = self.data.shape[:2]
        wide = 2 if self.scale_dtype == torch.float32 else 1
        words = self.data[:, :, :-1024].contiguous().view(torch.int32).view(tiles, blocks, 16, -1, wide)
        words = words.transpose(1, 2).reshape(tiles * 16, -1, wide)[:n, ::max(1, self.group_size // _BLOCK)]
        return words[:, :-(-k // self.group_size)]

    def scales(self):
        """[N, ceil(K / group_size)], as given."""
        words = self._words()
        if self.scale_dtype == torch.float32:
            return words[..., 1].contiguous().view(torch.float32)
        return (words[..., 0] >> 16).to(torch.int16).view(self.scale_dtype)

    def zeros(self):
        """[N, ceil(K / group_size)] uint8."""
        return (self._words()[..., 0] & 15).to(torch.uint8)

    def dequantize(self):
        """(code - zero) * scale as float32 [N, K]."""
        k = self.shape[1]
        scales = self.scales().float().repeat_interleave(self.group_size, 1)[:, :k]
        zeros = self.zeros().float().repeat_interleave(self.group_size, 1)[:, :k]
        return (self.unpack().float() - zeros) * scales

    def __repr__(self):
        return (f"W4Weight(shape={self.shape}, group_size={self.group_size}, scales={self.scale_dtype}, "
                f"device={self.device})")


def pack_w4(codes, scales, zeros=None, group_size=128):
    """Lays 4-bit codes out for matrix_mul_w4, once per weight.

    codes uint8 [N, K], one code 0..15 per byte; scales [N, ceil(K / group_size)] float32,
    float16 or bfloat16; zeros: None (zero point 8 everywhere) or uint8 of scales' shape,
    0..15.  The weight is (code - zero) * scale.  group_size: consecutive k that share a
    scale: 32, 64 or a multiple of 128 (the last group may be short)."""
    _check_group(group_size, "pack_w4")
    if codes.dim() != 2 or codes.shape[1] == 0:
        raise ValueError(f"pack_w4: codes must be [N, K] with K >= 1, got shape {tuple(codes.shape)}")
    if codes.dtype != torch.uint8:
        raise TypeError(f"pack_w4: codes must be uint8, got {codes.dtype}")
    n, k = codes.shape
    groups = -(-k // group_size)
    if tuple(scales.shape) != (n, groups):
        raise ValueError(f"pack_w4: scales have shape {tuple(scales.shape)}, expected {(n, groups)}")
    if scales.dtype not in _DTYPES:
        raise TypeError(f"pack_w4: scales must be float32, float16 or bfloat16, got {scales.dtype}")
    if zeros is not None:
        if tuple(zeros.shape) != (n, groups):
            raise ValueError(f"pack_w4: zeros have shape {tuple(zeros.shape)}, expected {(n, groups)}")
        if zeros.dtype != torch.uint8:
            raise TypeError(f"pack_w4: zeros must be uint8, got {zeros.dtype}")
    if scales.device != codes.device or (zeros is not None and zeros.device != codes.device):
        raise ValueError("pack_w4: codes, scales and zeros must be on one device")
    if n and (int(codes.max()) > 15 or (zeros is not None and int(zeros.max()) > 15)):
        raise ValueError("pack_w4: codes and zeros must be 0..15")
    blocks, tiles = -(-k // _BLOCK), -(-n // 16)
    pad = torch.nn.functional.pad
    codes = pad(codes, (0, blocks * _BLOCK - k, 0, tiles * 16 - n))
    c = codes.reshape(-1, blocks, 4, 4, 4, 2)          # j, t, i, parity: k = 32j + 8t + 2i + parity
    c = c.permute(0, 1, 3, 2, 5, 4).reshape(tiles, 16, blocks, 16, 4, 2)   # word, then nibbles 4 * parity + i
    packed = (c[..., 0] | c[..., 1] << 4).reshape(tiles, 16, blocks, 64).transpose(1, 2).reshape(tiles, blocks, 1024)
    wide = scales.dtype == torch.float32
    bits = scales.contiguous()
    bits = bits.view(torch.int32) if wide else bits.view(torch.int16).to(torch.int32) << 16
    zero = torch.full_like(bits, 8) if zeros is None else zeros.to(torch.int32)
    words = torch.stack((zero, bits), 2) if wide else (zero | bits)[:, :, None]
    if group_size > _BLOCK:
        words = words.repeat_interleave(group_size // _BLOCK, 1)[:, :blocks]
    per_block = max(1, _BLOCK // group_size)
    words = pad(words, (0, 0, 0, blocks * per_block - words.shape[1], 0, tiles * 16 - n))
    words = words.reshape(tiles, 16, blocks, per_block * words.shape[2]).transpose(1, 2)
    words = words.reshape(tiles, blocks, 16 * per_block * (2 if wide else 1)).contiguous().view(torch.uint8)
    return W4Weight((n, k), group_size, scales.dtype, torch.cat((words, packed), 2))


def quantize_w4(weight, group_size=128, symmetric=False):
    """A W4Weight whose values are the nearest of 16 steps to weight [N, K], group by group.

    symmetric: steps of max|w| / 7 around zero (zero point 8).  Otherwise 15 steps over the
    group's range, widened to hold zero, which stays exact.  Scales have weight's dtype
    (float32, float16 or bfloat16); codes are chosen for the rounded scale, so an error is at
    most half a step, plus what the scale's rounding cuts off the ends of the range and, where
    zero lies between two steps of it, up to half a step more at one end (so a magnitude above 15/16
    of the type's largest may become infinite).  A weight with infinities or NaN is refused."""
    _check_group(group_size, "quantize_w4")
    if weight.dim() != 2 or weight.shape[1] == 0:
        raise ValueError(f"quantize_w4: weight must be [N, K] with K >= 1, got shape {tuple(weight.shape)}")
    if weight.dtype not in _DTYPES:
        raise TypeError(f"quantize_w4: weight must be float32, float16 or bfloat16, got {weight.dtype}")
    weight = weight.detach()
    if not bool(torch.isfinite(weight).all()):
        raise ValueError("quantize_w4: weight holds infinities or NaN")
    n, k = weight.shape
    groups = -(-k // group_size)
    w = torch.nn.functional.pad(weight.float(), (0, groups * group_size - k)).view(n, groups, group_size)
    if symmetric:
        scales = w.abs().amax(2) / 7
    else:
        low, high = w.amin(2).clamp(max=0), w.amax(2).clamp(min=0)
        scales = (high / 2 - low / 2) / 7.5   # high - low itself can overflow
    scales = scales.to(weight.dtype)
    step = torch.where(scales > 0, scales.float(), 1.0)
    if symmetric:
        zeros, zf = None, torch.full_like(step, 8)
    else:
        zf = torch.round(-low / step).clamp(0, 15)
        zeros = zf.to(torch.uint8)
    codes = (torch.round(w / step[:, :, None]) + zf[:, :, None]).clamp(0, 15).to(torch.uint8)
    return pack_w4(codes.view(n, -1)[:, :k], scales, zeros, group_size)


def matrix_mul_w4(x, weight, bias=None, out=None):
    """x @ W.T (+ bias) with W a W4Weight of shape (N, K); x [..., K] float32, float16 or
    bfloat16 on the weight's device; bias None or [N] of x's dtype.  Returns (or writes into
    `out`, [..., N] with unit column stride, sharing no memory with x or bias) x's dtype.

    Up to 8 rows of x, the decoding case (many 16-bit calls of up to 16), the codes are read once
    and enter exactly, as x does: sums are fp32, with one rounding at the end.  With more rows the
    weight is rounded once to x's dtype (float16: what is past 65504 becomes infinite) and
    multiplied on the tensor cores: up to 256 rows of 16-bit x with scales of its dtype it is
    expanded on the way, once per 128 rows; otherwise into the workspace, at most 256 MiB (or
    256 rows of it) at a time (float32: exact, and the 3xTF32 product of matrix_mul).  So a token's
    bits depend on how many rows it comes with.

    Infinities and NaN in x stay in their rows, as in the formula (float32 from 9 rows on: NaN).
    Up to 16 rows, outputs whose sums leave float32's range before the scales bring them back (x of
    2^117 or more), and those of a single 16-bit row with infinities, are computed one at a time,
    which takes 0.5 to 5 ms.  Not differentiable: inputs that require a gradient or carry a
    forward-mode tangent are refused."""
    if not isinstance(weight, W4Weight):
        raise TypeError(f"matrix_mul_w4: weight must be a W4Weight (pack_w4, quantize_w4), got {type(weight).__name__}")
    n, k = weight.shape
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"matrix_mul_w4: shapes {tuple(x.shape)} and {weight.shape} don't match (x [..., K], "
                         "weight [N, K])")
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise TypeError(f"matrix_mul_w4: x must be float32, float16 or bfloat16, got {x.dtype}")
    if _levels._current_level >= 0:
        _refuse_tangents("matrix_mul_w4", x, bias, out)
    dev = x.device
    if not (x.is_cuda and weight.device == dev):
        raise ValueError(f"matrix_mul_w4: x and weight must be on one CUDA device (got {dev} and {weight.device}); "
                         "tilec_b200 has no CPU path")
    if bias is not None and (bias.dtype != x.dtype or bias.dim() != 1 or bias.shape[0] != n or bias.device != dev):
        raise ValueError(f"matrix_mul_w4: bias must be a {x.dtype} [{n}] tensor on {dev}")
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        raise ValueError("matrix_mul_w4: not differentiable; call it under torch.no_grad() or detach the inputs")
    if x.is_contiguous():
        xr, ldx, m = x, k, x.numel() // k
    else:
        xr, ldx = _rows(x if x.dim() == 2 else x.reshape(-1, k))
        m = xr.shape[0]
    if out is None:
        out = out2 = x.new_empty(x.shape[:-1] + (n,))
        ldo = n
    else:
        out2, ldo = _w4_out(out, x, dev, m, n)
    if m == 0 or n == 0:
        return out
    if bias is not None:
        bias = bias.contiguous()
    if not select._installed:
        select.ensure_installed()
    fast = _native.fast()
    index = dev.index
    prev = torch.cuda.current_device()
    switch = prev != index
    if switch:
        torch.cuda.set_device(index)
    try:
        stream = _stream(dev)
        px, po, sdt, group = xr.data_ptr(), out2.data_ptr(), _DTYPES[weight.scale_dtype], weight.group_size
        # The size depends on the operands' alignment only as far as their low bits tell.
        key = (dt, m, ldx, sdt, n, k, group, ldo, px & 15, po & 15, index)
        nbytes = _W4_BYTES.get(key)
        if nbytes is None:
            nbytes = _native.load().tilec_mm_w4_workspace_bytes(px, dt, m, ldx, sdt, n, k, group, po, ldo)
            if len(_W4_BYTES) >= 4096:  # a process that sees many shapes: start over
                _W4_BYTES.clear()
            _W4_BYTES[key] = nbytes
        ws = _workspace(nbytes, dev)
        rc = (fast.w4 if fast is not None else _native.load().tilec_mm_w4)(
            px, dt, m, ldx, weight.data.data_ptr(), sdt, n, k, group, _ptr(bias), po, ldo, _ptr(ws), nbytes, stream)
        _native.check(rc, "tilec_mm_w4")
        _check_device(stream)
    finally:
        if switch:
            torch.cuda.set_device(prev)
    return out


_W4_BYTES = {}   # arguments that decide it -> workspace bytes of tilec_mm_w4


def _w4_out(out, x, dev, m, n):
    """(the [m, n] view of a caller's out, its row stride)"""
    shape = x.shape[:-1] + (n,)
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("matrix_mul_w4: not differentiable, but out requires a gradient")
    if out.dtype != x.dtype or out.shape != shape or out.device != dev:
        raise ValueError(f"matrix_mul_w4: out must be a {x.dtype} {tuple(shape)} tensor on {dev}")
    try:
        out2 = out.view(m, n)
    except RuntimeError:
        raise ValueError("matrix_mul_w4: the rows of out must lie at one stride") from None
    s0, s1 = out2.stride()
    if not ((n <= 1 or s1 == 1) and (m <= 1 or s0 >= n)):
        raise ValueError("matrix_mul_w4: out must have unit column stride and non-overlapping rows")
    return out2, (s0 if m > 1 else n)
