"""ctypes bindings of the encoder operators (``include/tsnecuda/tsne_operators.h``):
block-scaled 8-bit matrices and their products, a teacher's top list, and
distillation from such a list with its gradient.

Arguments and results are torch CUDA tensors.  Every call only enqueues work on
the current stream of its arguments' device; workspaces come from torch's
allocator, on that stream.  Arguments that the library cannot take raise
``ValueError`` (``TypeError`` for what is no tensor of a supported type); a call
that fails raises ``RuntimeError`` with the library's message.  What a call
writes into a tensor that it is given, autograd is told of, as of torch's own
operations in place.
"""
import collections
import ctypes

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import stages

_vp, _ci, _cf, _c64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_int64
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_LISTED = 1024
MAX_DISTILLED = 1 << 20
_LEAST, _INFINITE = 2.0 ** -126, 2.0 ** 128 * (1 - 2.0 ** -25)  # (of temperatures, as floats hold them)

_bound = None


def _lib():
    global _bound
    if _bound is None:
        L = stages.lib()
        L.tsne_hip_quantize_blocks.argtypes = [_vp, _ci, _c64, _c64, _c64, _ci, _vp, _vp, _vp, _vp, _vp]
        L.tsne_hip_matmul_blocks.argtypes = [_vp, _vp, _vp, _vp, _c64, _c64, _c64, _vp, _ci, _c64, _ci, _vp, _c64, _vp]
        L.tsne_hip_linear_blocks.argtypes = [_vp, _ci, _c64, _c64, _c64, _vp, _vp, _c64, _vp, _c64, _vp, _c64, _vp]
        L.tsne_hip_top_logits.argtypes = [_vp, _ci, _c64, _c64, _c64, _ci, _cf, _vp, _vp, _vp, _vp, _c64, _vp]
        L.tsne_hip_distill.argtypes = [_vp, _ci, _c64, _c64, _c64, _vp, _vp, _ci, _vp, _vp, _cf, _ci, _vp, _vp, _c64,
                                       _vp, _c64, _vp]
        L.tsne_hip_matmul_blocks_workspace.argtypes = [_c64, _c64, _c64, _ci, _ci]
        L.tsne_hip_linear_blocks_workspace.argtypes = [_c64, _c64, _c64, _ci]
        L.tsne_hip_top_logits_workspace.argtypes = [_c64, _c64, _ci, _ci]
        L.tsne_hip_distill_workspace.argtypes = [_c64, _c64, _ci, _ci]
        for name in ("quantize_blocks", "matmul_blocks", "linear_blocks", "top_logits", "distill"):
            getattr(L, "tsne_hip_" + name).restype = _ci
        for name in ("matmul_blocks", "linear_blocks", "top_logits", "distill"):
            getattr(L, "tsne_hip_%s_workspace" % name).restype = _c64
        _bound = L
    return _bound


def _ptr(t):
    return None if t is None else t.data_ptr()


def _matrix(t, who, name):
    if not isinstance(t, torch.Tensor) or t.dtype not in _TYPES:
        raise TypeError("%s: %s must be a tensor of float32, float16 or bfloat16" % (who, name))
    if t.dim() != 2:
        raise ValueError("%s: %s must have two dimensions (got %s)" % (who, name, tuple(t.shape)))
    if not t.is_cuda:
        raise ValueError("%s: %s must be on the GPU" % (who, name))
    return t


def _rows(t, who, name):
    """(the matrix with values of a row side by side, copied where they are not; its rows, columns and row stride)."""
    t = _matrix(t, who, name)
    rows, cols = t.shape
    across, along = t.stride()
    if rows and cols and (along == 1 or cols == 1) and (rows == 1 or across >= cols):
        return t, rows, cols, cols if rows == 1 else across
    return t.contiguous(), rows, cols, cols


def _vector(t, n, dtype, device, who, name):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise TypeError("%s: %s must be a tensor of %s" % (who, name, dtype))
    if t.shape != n or t.device != device:
        raise ValueError("%s: %s must be of shape %s on %s (got %s on %s)" % (who, name, n, device, tuple(t.shape), t.device))
    return t if t.is_contiguous() else t.contiguous()


# (torch's handle of the current stream, which torch.cuda.current_stream() takes 2 us to wrap)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _call(fn, index, *args):
    """fn(*args, stream) on the current stream of GPU `index`."""
    if index == _device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        raise RuntimeError(_lib().tsne_hip_last_error().decode())


def _workspace(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


_NOWHERE = None, None


def _padded(n, to):
    return -(-n // to) * to


class BlockScaled(object):
    """A matrix in 8-bit floating point with a power-of-two scale for each block
    of 128 values of a row.

    data    (rows, columns rounded up to a multiple of 128) float8_e4m3fn, zeros behind a row's end
    scales  (rows, columns / 128 rounded up to a multiple of 4) float8_e8m0fnu
    shape   (rows, columns)
    """

    __slots__ = ("shape", "_data", "_scales", "_buffer", "_pointers", "_device")

    def __init__(self, data, scales, cols):
        if data.dtype != torch.float8_e4m3fn or scales.dtype != torch.float8_e8m0fnu:
            raise TypeError("BlockScaled: data must be float8_e4m3fn and scales float8_e8m0fnu")
        rows = data.shape[0] if data.dim() == 2 else -1
        if cols < 0 or data.shape != (rows, _padded(cols, 128)) or scales.shape != (rows, _padded(cols, 512) // 128):
            raise ValueError("BlockScaled: %d columns do not go with data of shape %s and scales of shape %s"
                             % (cols, tuple(data.shape), tuple(scales.shape)))
        if data.device != scales.device or not data.is_cuda:
            raise ValueError("BlockScaled: data and scales must be on one GPU")
        self._pointers = data.data_ptr(), scales.data_ptr()
        if not (data.is_contiguous() and scales.is_contiguous() and (self._pointers[0] | self._pointers[1]) % 16 == 0):
            raise ValueError("BlockScaled: data and scales must be contiguous and aligned to 16 bytes")
        self._data, self._scales, self._buffer, self._device = data, scales, None, data.device
        self.shape = rows, cols

    @classmethod
    def empty(cls, rows, cols, device):
        # (Both in one allocation, and no tensor made of either before somebody asks for it: each would cost a call as much
        # as a small kernel takes.)
        size = rows * (_padded(cols, 128) + _padded(cols, 512) // 128)
        return cls._of(torch.empty(size, dtype=torch.float8_e4m3fn, device=device), rows, cols)

    @classmethod
    def _of(cls, buffer, rows, cols):
        """The matrix whose data and scales are one allocation."""
        made = cls.__new__(cls)
        at = buffer.data_ptr()
        made._buffer, made._pointers = buffer, (at, at + rows * _padded(cols, 128))
        made._data = made._scales = None
        made._device = buffer.device
        made.shape = rows, cols
        return made

    @property
    def data(self):
        if self._data is None:
            rows, width = self.shape[0], _padded(self.shape[1], 128)
            self._data = self._buffer.as_strided((rows, width), (width, 1))
        return self._data

    @property
    def scales(self):
        if self._scales is None:
            rows, width = self.shape[0], _padded(self.shape[1], 512) // 128
            self._scales = self._buffer.view(torch.float8_e8m0fnu).as_strided(
                (rows, width), (width, 1), rows * _padded(self.shape[1], 128))
        return self._scales

    @property
    def device(self):
        return self._device

    def dequantize(self):
        """The values as float32."""
        rows, cols = self.shape
        blocks = _padded(cols, 128) // 128
        v = self.data.to(torch.float32).view(rows, blocks, 128) * self.scales[:, :blocks].to(torch.float32)[:, :, None]
        return v.view(rows, blocks * 128)[:, :cols]


def _quantize(x, square, plain, transposed, who):
    x = _matrix(x, who, "x")
    across, along = x.stride()
    if across == 1 and along != 1 and x.shape[0] > 1 and x.shape[1] > 1 and along >= x.shape[0]:
        b, a = _quantize(x.t(), square, transposed, plain, who)  # (a transposed view is read as what it is a view of)
        return a, b
    x, rows, cols, stride = _rows(x, who, "x")
    device = x.device
    a = BlockScaled.empty(rows, cols, device) if plain else None
    b = BlockScaled.empty(cols, rows, device) if transposed else None
    _call(_lib().tsne_hip_quantize_blocks, device.index, x.data_ptr(), _TYPES[x.dtype], rows, cols, stride,
          1 if square else 0, *(a._pointers if a else _NOWHERE), *(b._pointers if b else _NOWHERE))
    return a, b


def quantize_blocks(x, square=False):
    """x as a BlockScaled matrix, a block being 128 values of a row or, with
    square, 128 x 128 values."""
    return _quantize(x, square, True, False, "quantize_blocks")[0]


def quantize_blocks_transposed(x, square=False):
    """The transpose of x as a BlockScaled matrix (blocks run down x's columns)."""
    return _quantize(x, square, False, True, "quantize_blocks_transposed")[1]


def quantize_blocks_both(x, square=False):
    """(quantize_blocks(x), quantize_blocks_transposed(x)) from one reading of x:
    what a training step needs of a layer's input, weights and output gradient."""
    return _quantize(x, square, True, True, "quantize_blocks_both")


def matmul_blocks(a, b, out_dtype=torch.bfloat16, out=None, exact=False):
    """a (m x k) times the transpose of b (n x k), both BlockScaled.  A half or
    float32 result, and with exact any, is summed in 32 bits from exact products.
    A bfloat16 one is otherwise summed by the 8-bit matrix instructions, at twice
    the rate: of every eight products they drop what lies 2^-13 below the largest,
    which for normally distributed factors is 1.5e-5 of a result, a hundredth of its
    rounding, and more than its rounding where large products cancel."""
    if not isinstance(a, BlockScaled) or not isinstance(b, BlockScaled):
        raise TypeError("matmul_blocks: both factors must be BlockScaled")
    (m, k), (n, kb) = a.shape, b.shape
    device = a._device
    if k != kb or device != b._device:
        raise ValueError("matmul_blocks: factors of %s and %s on %s and %s" % (a.shape, b.shape, a.device, b.device))
    given = out
    out, stride = _result(out, m, n, out_dtype, device, "matmul_blocks")
    kind = _TYPES[out.dtype]
    lib = _lib()
    size = lib.tsne_hip_matmul_blocks_workspace(m, n, k, kind, 1 if exact else 0)
    space = _workspace(size, device)
    _call(lib.tsne_hip_matmul_blocks, device.index, *a._pointers, *b._pointers, m, n, k, out.data_ptr(), kind, stride,
          1 if exact else 0, _ptr(space), size)
    if given is not None:
        increment_version(given)
    return out


def _result(out, m, n, dtype, device, who):
    """(where an m x n result goes, and its row stride)."""
    if out is None:
        if dtype not in _TYPES:
            raise TypeError("%s: a result of float32, float16 or bfloat16, not %s" % (who, dtype))
        return torch.empty((m, n), dtype=dtype, device=device), n
    _matrix(out, who, "out")
    if tuple(out.shape) != (m, n) or out.device != device or (n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n):
        raise ValueError("%s: out must be %d x %d on %s with rows' values side by side" % (who, m, n, device))
    return out, out.stride(0) if m > 1 else n


def linear_blocks(x, weight, exact=False):
    """x (m x k) through a layer with BlockScaled weight (n x k): x is quantised
    and multiplied, in one call, into a result of x's type.  What a trained
    encoder places points with; the bits are those of
    matmul_blocks(quantize_blocks(x), weight, x.dtype, exact=exact).  It has no
    gradient, and where autograd would ask x for one it is refused."""
    if not isinstance(weight, BlockScaled):
        raise TypeError("linear_blocks: weight must be BlockScaled")
    x, m, k, stride = _rows(x, "linear_blocks", "x")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("linear_blocks has no gradient, and x requires one: block_linear has, and torch.no_grad() or x.detach() "
                         "say that none is wanted")
    n, device = weight.shape[0], x.device
    if k != weight.shape[1] or device != weight._device:
        raise ValueError("linear_blocks: x of %s on %s and a weight of %s on %s" % (tuple(x.shape), device, weight.shape, weight.device))
    if exact and x.dtype == torch.bfloat16:  # (the one type whose products are not exact anyway)
        return matmul_blocks(_quantize(x, False, True, False, "linear_blocks")[0], weight, x.dtype, exact=True)
    kind = _TYPES[x.dtype]
    out = x.new_empty((m, n))
    lib = _lib()
    size = lib.tsne_hip_linear_blocks_workspace(m, n, k, kind)
    space = _workspace(size, device)
    _call(lib.tsne_hip_linear_blocks, device.index, x.data_ptr(), kind, m, k, stride, *weight._pointers, n, out.data_ptr(), n,
          _ptr(space), size)
    return out


class _BlockLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, exact):
        need_x, need_w, _ = ctx.needs_input_grad
        xq, xt = _quantize(x, False, True, need_w, "block_linear")
        wq, wt = _quantize(weight, True, True, need_x, "block_linear")
        ctx.save_for_backward(xt and xt._buffer, wt and wt._buffer)
        ctx.how = x.shape, weight.shape, x.dtype, weight.dtype, exact
        return matmul_blocks(xq, wq, out_dtype=x.dtype, exact=exact)

    @staticmethod
    def _kept(buffer, rows, cols):
        # (A saved tensor is what the hooks on it give back: whatever they do, the kernels read aligned rows, and all of them.)
        size = rows * (_padded(cols, 128) + _padded(cols, 512) // 128)
        if buffer.dtype != torch.float8_e4m3fn or buffer.shape != (size,):
            raise RuntimeError("block_linear: a hook has put %s of shape %s in the place of %d saved values"
                               % (buffer.dtype, tuple(buffer.shape), size))
        buffer = buffer.contiguous()
        return BlockScaled._of(buffer.clone() if buffer.data_ptr() % 16 else buffer, rows, cols)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_w, _ = ctx.needs_input_grad
        xt, wt = ctx.saved_tensors
        (t, k), (n, _), x_type, w_type, exact = ctx.how
        dyq, dyt = _quantize(dy, False, need_x, need_w, "block_linear")
        dx = matmul_blocks(dyq, _BlockLinear._kept(wt, k, n), out_dtype=x_type, exact=exact) if need_x else None
        dw = matmul_blocks(dyt, _BlockLinear._kept(xt, k, t), out_dtype=w_type, exact=exact) if need_w else None
        return dx, dw, None


def block_linear(x, weight, exact=False):
    """x times the transpose of weight, differentiable: all three products of a
    training step are of 8-bit operands (x and the output's gradient scaled by 128
    values along what is summed over, the weights by squares).  The result and its
    gradient are of x's type, the weight's gradient of the weight's, and each is
    summed as matmul_blocks sums that type, with exact from exact products."""
    x, weight = _matrix(x, "block_linear", "x"), _matrix(weight, "block_linear", "weight")
    if x.shape[1] != weight.shape[1] or x.device != weight.device:
        raise ValueError("block_linear: x of %s on %s and a weight of %s on %s" % (tuple(x.shape), x.device, tuple(weight.shape), weight.device))
    if not (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)):  # (nothing to keep)
        return matmul_blocks(_quantize(x, False, True, False, "block_linear")[0],
                             _quantize(weight, True, True, False, "block_linear")[0], out_dtype=x.dtype, exact=exact)
    return _BlockLinear.apply(x, weight, exact)


TopLogits = collections.namedtuple("TopLogits", "values indices lse")


def top_logits(logits, k, temperature=1.0):
    """A teacher's list: of every row the k largest logits (float32, descending,
    equal ones by ascending column), their columns (int32; -1 where a row has
    fewer than k that are not -infinity) and ln sum exp(logits / temperature).  A
    teacher's list is a constant: no gradient goes through it."""
    logits, rows, cols, stride = _rows(logits, "top_logits", "logits")
    if not 1 <= k <= min(cols, MAX_LISTED):
        raise ValueError("top_logits: k must be in [1, %d] (got %s)" % (min(cols, MAX_LISTED), k))
    if not _LEAST <= temperature < _INFINITE:
        raise ValueError("top_logits: the temperature must be positive, as a float (got %s)" % temperature)
    device = logits.device
    values = torch.empty((rows, k), dtype=torch.float32, device=device)
    indices = torch.empty((rows, k), dtype=torch.int32, device=device)
    lse = torch.empty(rows, dtype=torch.float32, device=device)
    kind = _TYPES[logits.dtype]
    lib = _lib()
    size = lib.tsne_hip_top_logits_workspace(rows, cols, kind, k)
    space = _workspace(size, device)
    _call(lib.tsne_hip_top_logits, device.index, logits.data_ptr(), kind, rows, cols, stride, k, temperature,
          values.data_ptr(), indices.data_ptr(), lse.data_ptr(), _ptr(space), size)
    return TopLogits(values, indices, lse)


def _distill(logits, indices, values, lse, weights, temperature, rest, want_grad, out, who):
    logits, rows, cols, stride = _rows(logits, who, "logits")
    device = logits.device
    if not 1 <= cols <= MAX_DISTILLED:
        raise ValueError("%s: logits of 1 to %d columns (got %d)" % (who, MAX_DISTILLED, cols))
    if not isinstance(indices, torch.Tensor) or indices.dim() != 2 or not 1 <= indices.shape[1] <= MAX_LISTED:
        raise ValueError("%s: indices must be a matrix of 1 to %d columns" % (who, MAX_LISTED))
    k = indices.shape[1]
    indices = _vector(indices, (rows, k), torch.int32, device, who, "indices")
    values = _vector(values, (rows, k), torch.float32, device, who, "values")
    lse = None if lse is None else _vector(lse, (rows,), torch.float32, device, who, "lse")
    weights = None if weights is None else _vector(weights, (rows,), torch.float32, device, who, "weights")
    if not _LEAST <= temperature < _INFINITE:
        raise ValueError("%s: the temperature must be positive, as a float (got %s)" % (who, temperature))
    if rest and lse is None:
        raise ValueError("%s: rest needs the teacher's lse" % who)
    grad, grad_stride = _result(out, rows, cols, logits.dtype, device, who) if want_grad else (None, 0)
    if grad is not None and grad.dtype != logits.dtype:
        raise TypeError("%s: out must be of the logits' type" % who)
    loss = torch.empty(rows, dtype=torch.float32, device=device)
    kind = _TYPES[logits.dtype]
    lib = _lib()
    size = lib.tsne_hip_distill_workspace(rows, cols, kind, k)
    space = _workspace(size, device)
    _call(lib.tsne_hip_distill, device.index, logits.data_ptr(), kind, rows, cols, stride, indices.data_ptr(),
          values.data_ptr(), k, _ptr(lse), _ptr(weights), temperature, 1 if rest else 0, loss.data_ptr(), _ptr(grad),
          grad_stride, _ptr(space), size)
    if out is not None:
        increment_version(out)
    return loss, grad


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, indices, values, lse, weights, temperature, rest):
        ctx.save_for_backward(logits, indices, values, lse, weights)
        ctx.how = temperature, rest
        return _distill(logits, indices, values, lse, weights, temperature, rest, False, None, "distill_loss")[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, up):
        logits, indices, values, lse, weights = ctx.saved_tensors
        up = up.to(torch.float32) if weights is None else up.to(torch.float32) * weights
        grad = _distill(logits, indices, values, lse, up.contiguous(), *ctx.how, True, None, "distill_loss")[1]
        return grad, None, None, None, None, None, None


def distill_loss(logits, indices, values, lse=None, weights=None, temperature=1.0, rest=False):
    """Divergence of every row's softmax(logits / temperature) from a teacher's
    list (columns, logits, and ln sum exp of the teacher's row at the same
    temperature; without lse the list's probabilities are made to sum to 1),
    times the row's weight.  With rest what the list leaves out counts as one
    event.  Differentiable by the logits, and by nothing else: a teacher or a
    weight that wants a gradient is refused."""
    if torch.is_grad_enabled():
        for name, t in (("values", values), ("lse", lse), ("weights", weights)):
            if isinstance(t, torch.Tensor) and t.requires_grad:
                raise ValueError("distill_loss: %s require a gradient, and there is none but the logits': detach them" % name)
    if isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled():
        return _Distill.apply(logits, indices, values, lse, weights, temperature, rest)
    return _distill(logits, indices, values, lse, weights, temperature, rest, False, None, "distill_loss")[0]


def distill(logits, indices, values, lse=None, weights=None, temperature=1.0, rest=False, out=None):
    """(distill_loss, its gradient by the logits) in one pass, for training loops
    whose loss is the rows' sum: what each row's gradient is multiplied by goes into
    weights.  Neither is part of autograd's graph.  out: where the gradient goes; the
    logits themselves are allowed, where no backward pass still needs them."""
    return _distill(logits, indices, values, lse, weights, temperature, rest, True, out, "distill")
