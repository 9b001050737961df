"""Matrix operators beside the convolutions: the dense layer with its epilogue in one product (`linear`, differentiable),
the orthogonalisation of matrices by Newton-Schulz products (`orthogonalize`) and the optimizer step built on it
(`muon_step`, what `train_class.FusedMuon` runs).

Tensors are float32 or bfloat16 on one GPU; every call enqueues its work on the current stream of the tensors' device
and takes its workspace from torch's allocator, so it can be captured into a graph.
"""
import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib, engine
from ._lib import lib, check

ACTIVATIONS = {None: 0, 'silu': 1, 'gelu': 2, 'relu': 3}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_Z_DTYPES = {torch.float32: torch.float32, torch.bfloat16: torch.float16}         # the pre-activation kept for the backward pass
MATRIX_DTYPE = np.dtype([('offset', '<i8'), ('rows', '<i4'), ('cols', '<i4')])      # odamd_matrix
_MOST = 2 ** 31 - 2 ** 16                                       # rows, columns and matrices of a call, elements of a matrix
RANGE_DTYPE = np.dtype([('offset', '<i8'), ('len', '<i8')])                         # odamd_range


# the stream's handle and the device's number alone, without a Stream object or a check for lazy initialisation (a CUDA tensor
# is at hand wherever they are asked): 0.1 us each instead of 2.8 and 0.25
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)
_current_device = getattr(torch._C, '_cuda_getDevice', torch.cuda.current_device)


def _stream(device):
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


_dispatch_modes = torch._C._len_torch_dispatch_stack


def _call(device, fn, *args):
    """fn(*args, current stream of `device`) with that device as the current one; its return code."""
    if _dispatch_modes() and torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None:
        raise RuntimeError('make_fx does not see a launch: the graph would hold an empty result')
    if _current_device() == device.index:
        return fn(*args, _stream(device))
    with torch.cuda.device(device):
        return fn(*args, _stream(device))


_tracing_state = torch._C._get_tracing_state


def _watched():
    """Whether something other than the backward pass follows operations on tensors: forward-mode differentiation or torch.jit.trace.
    What is launched through raw pointers escapes both; an autograd function does not: it refuses a tangent, and a trace
    records it."""
    return forward_ad._current_level >= 0 or _tracing_state() is not None


def _refuse_trace(name):
    if _tracing_state() is not None:
        raise RuntimeError(f'{name} writes to its arguments, which a trace does not record')


def _written(*tensors):
    """Tensors of the caller's were written through raw pointers: a backward pass that saved one of them has to raise, plans that
    hold folded weights have to fold them again."""
    torch.autograd.graph.increment_version([t for t in tensors if t is not None])
    engine.touch_weights()


def _overlap(a, b):
    """Whether two contiguous tensors share memory."""
    first, second = a.data_ptr(), b.data_ptr()
    return first < second + b.numel() * b.element_size() and second < first + a.numel() * a.element_size()


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _workspace(size, device):
    return torch.empty((size,), dtype=torch.uint8, device=device) if size else None


def _check_tensor(name, t, dtype=None, device=None):
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in _DTYPES and (dtype is None or t.dtype is dtype) and (
            device is None or t.device == device):
        return
    if not torch.is_tensor(t) or not t.is_cuda:
        raise ValueError(f'{name} must be a CUDA tensor')
    if t.dtype not in _DTYPES:
        raise ValueError(f'{name} must be float32 or bfloat16, not {t.dtype}')
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f'{name} is {t.dtype}, the input {dtype}: one type for all')
    if device is not None and t.device != device:
        raise ValueError(f'{name} is on {t.device}, the input on {device}')


def _rows(t):
    """(..., c) -> (rows, c) with contiguous rows that do not overlap: a view where the strides allow one."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    elif t.is_contiguous():
        return t
    c = t.shape[1]
    if (c > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < c):
        t = t.contiguous()
    return t


# ---------------------------------------------------------------------------------------------
# dense layer
# ---------------------------------------------------------------------------------------------
def _linear_forward(x, weight, bias, residual, act, keep_z):
    """2-D operands as `_rows` leaves them -> (y, z or None)."""
    m, k = x.shape
    n = weight.shape[0]
    dtype, device = x.dtype, x.device
    y = x.new_empty((m, n))
    z = x.new_empty((m, n), dtype=_Z_DTYPES[dtype]) if keep_z else None
    # a single row may have any stride: at least its length
    d = _lib.LinearDesc(x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(residual), y.data_ptr(), _ptr(z), max(x.stride(0), k),
                        max(weight.stride(0), k), 0 if residual is None else max(residual.stride(0), n), n, n, m, k, n, act,
                        _DTYPES[dtype])
    size = lib.odamd_linear_workspace_bytes(d)
    ws = _workspace(size, device)
    check(_call(device, lib.odamd_linear_forward, d, _ptr(ws), size), 'linear_forward')
    return y, z


def _linear_backward(dy, z, x, weight, act, want_dx, want_dw, want_db):
    """Gradients of `_linear_forward` from 2-D operands; x and weight may be None where they are not needed."""
    m, n = dy.shape
    k = weight.shape[1] if want_dx else x.shape[1] if want_dw else 1
    device = dy.device
    dx = dy.new_empty((m, k)) if want_dx else None
    dw = dy.new_empty((n, k)) if want_dw else None
    db = dy.new_empty((n,)) if want_db else None
    d = _lib.LinearGradDesc(dy.data_ptr(), _ptr(z), x.data_ptr() if want_dw else None, weight.data_ptr() if want_dx else None,
                            _ptr(dx), _ptr(dw), _ptr(db), max(dy.stride(0), n), n if z is None else max(z.stride(0), n),
                            max(x.stride(0), k) if want_dw else 0, max(weight.stride(0), k) if want_dx else 0, k, k, m, k, n,
                            act, _DTYPES[dy.dtype])
    size = lib.odamd_linear_backward_workspace_bytes(d)
    ws = _workspace(size, device)
    check(_call(device, lib.odamd_linear_backward, d, _ptr(ws), size), 'linear_backward')
    return dx, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        x2, w2 = _rows(x), _rows(weight)
        need = ctx.needs_input_grad
        keep_z = act != 0 and (need[0] or need[1] or need[2])
        y, z = _linear_forward(x2, w2, bias if bias is None else bias.contiguous(),
                               None if residual is None else _rows(residual), act, keep_z)
        ctx.act, ctx.x_shape = act, x.shape
        ctx.save_for_backward(x2 if need[1] else None, w2 if need[0] else None, z)
        return y if x.dim() == 2 else y.view(x.shape[:-1] + (weight.shape[0],))

    @staticmethod
    def backward(ctx, dy):
        # under create_graph the gradients have to refuse a second derivative; the wrapper that sees to it costs 5 us a call
        return _Linear.gradients_once(ctx, dy) if torch.is_grad_enabled() else _Linear.gradients(ctx, dy)

    @staticmethod
    def gradients(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[1] or need[2]:
            dx, dw, db = _linear_backward(_rows(dy), z, x, weight, ctx.act, *need[:3])
            if dx is not None and len(ctx.x_shape) != 2:
                dx = dx.view(ctx.x_shape)
        return dx, dw, db, dy if need[3] else None, None


_Linear.gradients_once = staticmethod(torch.autograd.function.once_differentiable(_Linear.gradients))


def linear(x, weight, bias=None, activation=None, residual=None):
    """act(x W^T + bias) + residual in one product.  x: (..., k); weight: (n, k); bias: (n,); residual: (..., n); all of one
    type, float32 or bfloat16.  activation: None, 'silu', 'gelu' (the erf form) or 'relu'.  Rows may be strided (a slice of a
    wider, concatenated buffer is read in place).  Differentiable once in all four tensors, backward only; in bfloat16 the pre-activation
    that the backward pass keeps is float16 and the gradient at it bfloat16.  As with every differentiable torch operation,
    a backward pass is captured into a graph on leaves that no eager graph holds any more (detached copies of them will do).
    float32 products carry 22 bits per value, counted from the largest magnitude of its row; a float32 row with an infinity
    gives NaN or infinity."""
    if activation not in ACTIVATIONS:
        raise ValueError(f'activation {activation!r}: one of {list(ACTIVATIONS)}')
    _check_tensor('x', x)
    dtype, device = x.dtype, x.device
    _check_tensor('weight', weight, dtype, device)
    k = x.shape[-1] if x.dim() else 0
    if weight.dim() != 2 or weight.shape[1] != k or min(weight.shape) < 1:
        raise ValueError(f'x (..., k) and weight (n, k) do not fit: {tuple(x.shape)} and {tuple(weight.shape)}')
    n, flat = weight.shape[0], x.dim() == 2
    if bias is not None:
        _check_tensor('bias', bias, dtype, device)
        if bias.shape != (n,):
            raise ValueError(f'bias must have shape ({n},), not {tuple(bias.shape)}')
    if residual is not None:
        _check_tensor('residual', residual, dtype, device)
        if residual.shape != ((x.shape[0], n) if flat else x.shape[:-1] + (n,)):
            raise ValueError(f'residual must have shape {tuple(x.shape[:-1]) + (n,)}, not {tuple(residual.shape)}')
    act = ACTIVATIONS[activation]
    if x.numel() // k > _MOST or k > _MOST or n > _MOST:
        raise ValueError(f'at most {_MOST} rows, inputs and outputs')
    if x.numel() == 0:
        # no rows: nothing to launch; the empty result stays connected to its inputs
        y = x.new_empty(x.shape[:-1] + (n,))
        if torch.is_grad_enabled():
            y = y + 0 * x.sum() + 0 * weight.sum()
            y = y if bias is None else y + 0 * bias.sum()
            y = y if residual is None else y + residual
        return y
    if (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                     or (residual is not None and residual.requires_grad))) or _watched():
        return _Linear.apply(x, weight, bias, residual, act)
    y, _ = _linear_forward(_rows(x), _rows(weight), bias if bias is None else bias.contiguous(),
                           None if residual is None else _rows(residual), act, False)
    return y if flat else y.view(x.shape[:-1] + (n,))


# ---------------------------------------------------------------------------------------------
# orthogonalisation and the optimizer step
# ---------------------------------------------------------------------------------------------
class _Orthogonalize(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, steps, eps):
        return _orthogonalize(x, steps, eps, x.new_empty(x.shape))

    @staticmethod
    def backward(ctx, dy):
        raise RuntimeError('orthogonalize has no backward pass: detach its argument or its result')


def _orthogonalize(x, steps, eps, out):
    rows, cols = x.size(-2), x.size(-1)
    batch = x.numel() // max(rows * cols, 1)
    if batch == 0 or rows * cols == 0:
        return out
    src = x if x.is_contiguous() else x.detach().contiguous()
    size = lib.odamd_orthogonalize_workspace_bytes(batch, rows, cols)
    ws = _workspace(size, x.device)
    check(_call(x.device, lib.odamd_orthogonalize, src.data_ptr(), out.data_ptr(), batch, rows, cols, steps, eps,
                _DTYPES[x.dtype], ws.data_ptr(), size), 'orthogonalize')
    return out


def orthogonalize(x, steps=5, eps=1e-7, out=None):
    """Brings the singular values of every matrix of x (..., rows, cols) near one and keeps its singular vectors: `steps`
    Newton-Schulz products with the coefficients (3.4445, -4.7750, 2.0315) from x / (|x|_F + eps) on.  Five steps take
    singular values from 0.003 of the norm up to between 0.68 and 1.21.  float32 or bfloat16, rounded once.  Matrices with a
    side of at most 64 are computed in 64 bits (over ten steps rounded to float32 after every ten), others with products of 22
    bits; bfloat16 results of those are off by up to 1e-3 of their norm in directions of small singular values (half a bfloat16
    step).  A matrix with a NaN or an infinity gives NaN.  `out` may be x itself.  Not differentiable: a backward pass that
    reaches the result raises, and `out` belongs to no graph."""
    _check_tensor('x', x)
    if x.dim() < 2:
        raise ValueError(f'x must have rows and columns, not shape {tuple(x.shape)}')
    if not 1 <= int(steps) <= 32 or not eps >= 0:
        raise ValueError('steps must be 1 to 32, eps must not be negative')
    rows, cols = x.size(-2), x.size(-1)
    if rows * cols > _MOST or x.numel() // max(rows * cols, 1) > _MOST:
        raise ValueError(f'at most {_MOST} elements of a matrix and matrices')
    steps, eps = int(steps), float(eps)
    if out is None:
        if (x.requires_grad and torch.is_grad_enabled()) or _watched():
            return _Orthogonalize.apply(x, steps, eps)
        return _orthogonalize(x, steps, eps, x.new_empty(x.shape))
    _check_tensor('out', out, x.dtype, x.device)
    if out.shape != x.shape or not out.is_contiguous():
        raise ValueError('out must be contiguous and have the shape of x')
    if x.is_contiguous() and x.data_ptr() != out.data_ptr() and _overlap(x, out):
        raise ValueError('out shares a part of the memory of x: it may be x itself or lie beside it')
    _refuse_trace('orthogonalize into `out`')
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise RuntimeError('orthogonalize into `out` has no tangent')
    _orthogonalize(x, steps, eps, out)
    _written(out)
    return out


class MatrixTable:
    """The matrices of a flat buffer, [(offset, rows, cols)], checked once: in the buffer, not overlapping."""

    def __init__(self, matrices):
        given = np.asarray(list(matrices)).reshape(-1, 3)
        with np.errstate(invalid='ignore'):
            a = given.astype(np.int64) if given.dtype.kind in 'iuf' else np.zeros((0, 3), np.int64)
        size = a[:, 1] * a[:, 2]
        if (len(a) == 0 or (a != given).any() or (a[:, 0] < 0).any() or (a[:, 0] > 2 ** 62).any() or (a[:, 1:] < 1).any()
                or (a[:, 1:] >= 2 ** 31).any() or (size > _MOST).any()):
            raise ValueError(f'matrices: at least one (offset, rows, cols) of whole numbers, offsets from 0 to 2^62, sizes from 1, at '
                             f'most {_MOST} elements each')
        order = np.argsort(a[:, 0], kind='stable')
        ends = (a[:, 0] + size)[order]
        if (a[order, 0][1:] < ends[:-1]).any():
            raise ValueError('matrices overlap')
        self.end = int(ends[-1])
        self.table = np.zeros(len(a), MATRIX_DTYPE)
        for i, name in enumerate(('offset', 'rows', 'cols')):
            self.table[name] = a[:, i]
        self.workspace_bytes = int(lib.odamd_muon_workspace_bytes(self.table.ctypes.data, len(a)))

    def __len__(self):
        return len(self.table)

    def gaps(self, numel):
        """What lies between the matrices of a buffer of `numel` elements, as (offset, length)."""
        found, at = [], 0
        for e in np.sort(self.table, order='offset'):
            if e['offset'] > at:
                found.append((at, int(e['offset']) - at))
            at = int(e['offset']) + int(e['rows']) * int(e['cols'])
        if numel > at:
            found.append((at, numel - at))
        return found


def muon_step(param, grad, momentum, matrices, lr, momentum_decay=0.95, nesterov=True, weight_decay=0.0, ema=None,
              ema_decay=0.0, grad_scale=1.0, steps=5, eps=1e-7):
    """One optimizer step with orthogonalised momentum over the matrices of flat float32 buffers, in place:

        m = momentum_decay m + grad_scale g;  u = grad_scale g + momentum_decay m  (nesterov; else m)
        p = p (1 - lr weight_decay) - lr 0.2 sqrt(max(rows, cols)) orthogonalize(u)
        ema = ema_decay ema + (1 - ema_decay) p

    `matrices`: [(offset, rows, cols)] or a MatrixTable of them.  What lies between the matrices is not touched.  The
    orthogonalised direction is accurate to 1e-3 of its norm, where every matrix has a side of at most 64 to float32's rounding."""
    table = matrices if isinstance(matrices, MatrixTable) else MatrixTable(matrices)
    _check_tensor('param', param)
    for name, t in (('param', param), ('grad', grad), ('momentum', momentum), ('ema', ema)):
        if t is None and name == 'ema':
            continue
        _check_tensor(name, t, device=param.device)
        if t.dtype != torch.float32 or t.dim() != 1 or not t.is_contiguous() or t.numel() != param.numel():
            raise ValueError(f'{name} must be a flat contiguous float32 buffer of the length of param')
    buffers = [('param', param), ('grad', grad), ('momentum', momentum)] + ([] if ema is None else [('ema', ema)])
    for i, (name, t) in enumerate(buffers):
        for other, u in buffers[:i]:
            if _overlap(t, u):
                raise ValueError(f'{name} shares memory with {other}')
    if table.end > param.numel():
        raise ValueError(f'matrices end at {table.end}, the buffers at {param.numel()}')
    if not 1 <= int(steps) <= 32 or not eps >= 0:
        raise ValueError('steps must be 1 to 32, eps must not be negative')
    _refuse_trace('muon_step')
    ws = _workspace(table.workspace_bytes, param.device)
    check(_call(param.device, lib.odamd_muon_ema_step, param.data_ptr(), grad.data_ptr(), momentum.data_ptr(), _ptr(ema),
                table.table.ctypes.data, len(table), lr, momentum_decay, int(nesterov), weight_decay, int(steps), eps,
                ema_decay, grad_scale, ws.data_ptr(), table.workspace_bytes), 'muon_ema_step')
    _written(param, momentum, ema)
