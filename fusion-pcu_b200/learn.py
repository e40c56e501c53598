"""Learning operators beside the strict path (include/pcu_b200_learn.h): group norm with an
activation, distillation from a teacher's top logits, and the product of 8-bit operands with a
scale for each block of 128.

The calls follow the node calls of the package: they return their outputs without waiting, faults
stay in `status` (a device word) until the caller reads it -- element_fault(word, extent) decodes
it -- and `chain=GuardedChain.stage(s)` runs a call as a stage of a guarded chain.  Outputs and
workspaces that are not passed are allocated.  Tensors of another device than the current one are
worked on on their own device.  The reference has no counterpart of these operators.
"""
import functools
import inspect
import struct

from . import _check, _rate_bits, _torch, library, new_status

__all__ = ["ACTIVATIONS", "group_norm", "group_norm_backward", "distill_loss", "distill_loss_backward",
           "distill_loss_step", "block_quantize", "block_matmul"]

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
DISTILL_TOP_MAX = 1024

# The kernels of small calls take a few microseconds, so the host's part is kept short: pointers go as
# plain integers, devices are compared by index, workspace sizes are remembered by their arguments.
_FLOAT, _WORD = struct.Struct("f"), struct.Struct("I")


def _bits(value):
    """The binary32 pattern of `value` as it is now.  Nothing is remembered: a 0-dimensional tensor is a number
    whose value changes, 0.0 equals -0.0, and an annealed temperature is another number in each step.  A Python
    float takes a short way (0.2 us against 1.8)."""
    return _WORD.unpack(_FLOAT.pack(value))[0] if type(value) is float else _rate_bits(value)


@functools.lru_cache(maxsize=None)
def _types():
    torch = _torch()
    codes = {torch.float32: 0, torch.float64: 1, torch.float16: 2, torch.bfloat16: 3}
    wide = {t: torch.float64 if t == torch.float64 else torch.float32 for t in codes}
    return codes, wide


@functools.lru_cache(maxsize=None)
def _entry(name, guarded):
    return getattr(library(), ("pcu_b200_guarded_" if guarded else "pcu_b200_") + name)


@functools.lru_cache(maxsize=1024)
def _need(name, device, *sizes):
    """Workspace bytes of a call on `device` (which is current)."""
    return getattr(library(), f"pcu_b200_{name}_workspace_size")(*sizes)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(name, args, status, chain, like):
    """pcu_b200_<name>(*args, status, stream) on the current stream; with chain=(records, stage), its
    guarded form."""
    stream = _torch()._C._cuda_getCurrentRawStream(like.get_device())
    if chain is None:
        rc = _entry(name, False)(*args, status.data_ptr(), stream)
    else:
        rc = _entry(name, True)(*args, chain[0].data_ptr(), int(chain[1]), stream)
    if rc:
        _check(rc)


def _code(t):
    try:
        return _types()[0][t.dtype]
    except KeyError:
        raise TypeError(f"learning operators handle float32/float64/float16/bfloat16, got {t.dtype}") from None


def _on_device(call):
    """Runs `call` with its first tensor's device current, and on `stream` when one is given, so that
    what the call allocates belongs to the stream that uses it."""
    name = next(iter(inspect.signature(call).parameters))

    @functools.wraps(call)
    def wrapped(*args, **kwargs):
        torch = _torch()
        first = args[0] if args else kwargs[name]
        if first.get_device() == torch._C._cuda_getDevice() and kwargs.get("stream") is None:  # -1: not on a GPU
            return call(*args, **kwargs)
        if not first.is_cuda:
            raise ValueError(f"{name}: a CUDA tensor is wanted, got one on {first.device}")
        stream = kwargs.get("stream")
        if stream is not None:
            if stream.device != first.device:
                raise ValueError(f"stream is on {stream.device}, {name} on {first.device}")
            with torch.cuda.stream(stream):
                return call(*args, **kwargs)
        with torch.cuda.device(first.device):
            return call(*args, **kwargs)
    return wrapped


def _want(name, t, like, shape=None, dtype=None):
    """`t` is a dense tensor of the given shape and type on the device of `like`."""
    if t is None or (t.get_device() == like.get_device() and (dtype is None or t.dtype == dtype) and
                     (shape is None or t.shape == shape) and t.is_contiguous()):
        return
    if not t.is_cuda or t.get_device() != like.get_device():
        raise ValueError(f"{name} is on {t.device}, not on {like.device}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, {dtype} is wanted")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, {tuple(shape)} is wanted")
    if not t.is_contiguous():
        raise ValueError(f"{name} is not contiguous")


def _alike(name, t, like):
    if t.shape != like.shape or t.dtype != like.dtype or not t.is_cuda or t.get_device() != like.get_device():
        raise ValueError(f"{name} is {tuple(t.shape)} {t.dtype} on {t.device}, "
                         f"{tuple(like.shape)} {like.dtype} on {like.device} is wanted")


def _status(status, chain, like):
    if chain is not None:
        if not chain[0].is_cuda or chain[0].get_device() != like.get_device():
            raise ValueError(f"the chain's records are on {chain[0].device}, not on {like.device}")
        return status
    if status is None:
        return new_status(device=like.device)
    if not status.is_cuda or status.get_device() != like.get_device() or status.element_size() != 8 or status.numel() < 1:
        raise ValueError(f"status is one 64-bit word on {like.device}")
    return status


# ------------------------------------------------------------------ group norm

def _maps(name, t, like=None):
    """(batch, positions, channels, batch stride, row stride) of a channels-last tensor: [batch,
    positions, channels], or [batch, channels] with one position."""
    if t.dim() not in (2, 3):
        raise ValueError(f"{name} is [batch, positions, channels] or [batch, channels], got {tuple(t.shape)}")
    if like is not None:
        _alike(name, t, like)
    shape, strides = t.shape, t.stride()
    n, c, batch_stride = shape[0], shape[-1], strides[0]
    if len(shape) == 2:
        s, stride = 1, max(c, batch_stride)
    else:
        s, stride = shape[1], strides[1]
    if strides[-1] != 1 and c > 1 and n and s:
        raise ValueError(f"{name}: channels must be adjacent (channels last)")
    return n, s, c, batch_stride, stride


def _norm_shape(x, groups, weight, bias, activation):
    n, s, c, batch_stride, stride = _maps("input", x)
    groups = int(groups)
    if groups < 1 or c % groups:
        raise ValueError(f"{c} channels are not {groups} equal groups")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation is one of {sorted(ACTIVATIONS)}, got {activation!r}")
    wide = _types()[1][x.dtype]
    _want("weight", weight, x, (c,), wide)
    _want("bias", bias, x, (c,), wide)
    return n, s, c, groups, batch_stride, stride, wide


def _workspace(workspace, need, like):
    if workspace is None:
        return _torch().empty(need, dtype=_torch().uint8, device=like.device) if need else None
    if not workspace.is_cuda or workspace.get_device() != like.get_device() or workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace holds {need} bytes on {like.device}")
    return workspace


@_on_device
def group_norm(x, groups, weight=None, bias=None, activation="none", eps=1e-5, out=None, stats=None, workspace=None,
               status=None, *, stream=None, chain=None):
    """activation(group_norm(x) * weight + bias), channels last: x is [batch, positions, channels] or
    [batch, channels], its rows may be strided.  weight and bias are float32 (float64 for float64).
    Returns (out, stats); stats is [batch, groups, 2] with mean and 1 / sqrt(variance + eps), for
    group_norm_backward.  out may be x."""
    torch = _torch()
    code = _code(x)
    n, s, c, groups, batch_stride, stride, wide = _norm_shape(x, groups, weight, bias, activation)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if stats is None:
        stats = torch.empty((n, groups, 2), dtype=wide, device=x.device)
    _want("stats", stats, x, (n, groups, 2), wide)
    _, _, _, out_batch, out_stride = _maps("out", out, x)
    status = _status(status, chain, x)
    need = _need("group_norm", x.get_device(), code, n, s, c, groups)
    workspace = _workspace(workspace, need, x)
    _call("group_norm", (code, ACTIVATIONS[activation], _ptr(x), _ptr(weight), _ptr(bias), _ptr(out), _ptr(stats),
          n, s, c, groups, batch_stride, stride, out_batch, out_stride, _bits(eps), _ptr(workspace), need), status,
          chain, x)
    return out, stats


@_on_device
def group_norm_backward(x, upstream, groups, stats, weight=None, bias=None, activation="none", dx=None, dweight=None,
                        dbias=None, workspace=None, status=None, *, stream=None, chain=None):
    """Gradients of group_norm for `upstream`, the gradient of its output: (dx, dweight, dbias), the
    last two None without weight (bias).  dx may be x or upstream."""
    torch = _torch()
    code = _code(x)
    n, s, c, groups, batch_stride, stride, wide = _norm_shape(x, groups, weight, bias, activation)
    _, _, _, up_batch, up_stride = _maps("upstream", upstream, x)
    _want("stats", stats, x, (n, groups, 2), wide)
    if dx is None:
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _, _, _, dx_batch, dx_stride = _maps("dx", dx, x)
    if dweight is None and weight is not None:
        dweight = torch.empty_like(weight)
    if dbias is None and bias is not None:
        dbias = torch.empty_like(bias)
    _want("dweight", dweight, x, (c,), wide)
    _want("dbias", dbias, x, (c,), wide)
    status = _status(status, chain, x)
    need = _need("group_norm_backward", x.get_device(), code, n, s, c, groups)
    workspace = _workspace(workspace, need, x)
    _call("group_norm_backward", (code, ACTIVATIONS[activation], _ptr(x), _ptr(upstream), _ptr(weight),
          _ptr(bias), _ptr(stats), _ptr(dx), _ptr(dweight), _ptr(dbias), n, s, c, groups, batch_stride, stride,
          up_batch, up_stride, dx_batch, dx_stride, _ptr(workspace), need), status, chain, x)
    return dx, dweight, dbias


# ------------------------------------------------------------------ distillation

def _rows(name, t, like=None):
    """Row stride of a matrix with adjacent columns."""
    if t.dim() != 2:
        raise ValueError(f"{name} is a matrix, got {tuple(t.shape)}")
    if like is not None:
        _alike(name, t, like)
    (rows, columns), (stride, step) = t.shape, t.stride()
    if step != 1 and columns > 1 and rows:
        raise ValueError(f"{name}: columns must be adjacent")
    return stride if rows > 1 else columns


def _distill(logits, top_indices, top_logits, temperature, row_weights):
    """(wide type, the arguments that every call begins with)."""
    torch = _torch()
    code = _code(logits)
    wide = _types()[1][logits.dtype]
    stride = _rows("logits", logits)
    rows, vocab = logits.shape
    if top_indices.dim() != 2 or top_indices.shape[0] != rows:
        raise ValueError(f"top_indices is [{rows}, entries], got {tuple(top_indices.shape)}")
    k = top_indices.shape[1]
    if k > DISTILL_TOP_MAX:
        raise ValueError(f"at most {DISTILL_TOP_MAX} teacher entries a row, got {k}")
    _want("top_indices", top_indices, logits, dtype=torch.int64)
    _want("top_logits", top_logits, logits, (rows, k), wide)
    _want("row_weights", row_weights, logits, (rows,), wide)
    return wide, (code, _ptr(logits), rows, vocab, stride, _ptr(top_indices), _ptr(top_logits), k, _ptr(row_weights),
                  _bits(temperature))


def _upstream(upstream, logits, wide):
    if upstream is None:
        return (None, 0)
    _want("upstream", upstream, logits, dtype=wide)
    if upstream.numel() == 1:
        return (_ptr(upstream), 1)
    if upstream.shape != (logits.shape[0],):
        raise ValueError(f"upstream is one value or one for each of {logits.shape[0]} rows, got {tuple(upstream.shape)}")
    return (_ptr(upstream), 0)


@_on_device
def distill_loss(logits, top_indices, top_logits, temperature=1.0, row_weights=None, loss=None, stats=None, status=None,
                 *, stream=None, chain=None):
    """Each row's loss against a teacher's top logits: T^2 KL(softmax(top / T) || softmax(logits / T)),
    times row_weights.  logits is [rows, vocab] (rows may be strided), top_indices int64 [rows, k]
    (negative: absent), top_logits float32 (float64 for float64) [rows, k].  Returns (loss, stats):
    loss [rows], stats [rows, 2] for distill_loss_backward."""
    torch = _torch()
    wide, inputs = _distill(logits, top_indices, top_logits, temperature, row_weights)
    rows = logits.shape[0]
    if loss is None:
        loss = torch.empty(rows, dtype=wide, device=logits.device)
    if stats is None:
        stats = torch.empty((rows, 2), dtype=wide, device=logits.device)
    _want("loss", loss, logits, (rows,), wide)
    _want("stats", stats, logits, (rows, 2), wide)
    status = _status(status, chain, logits)
    _call("distill_loss", inputs + (_ptr(loss), _ptr(stats)), status, chain, logits)
    return loss, stats


@_on_device
def distill_loss_backward(logits, top_indices, top_logits, stats, upstream=None, temperature=1.0, row_weights=None,
                          gradient=None, status=None, *, stream=None, chain=None):
    """The gradient of sum(upstream * loss) with respect to the logits; upstream is one value, one for
    each row, or None (1).  gradient may be logits."""
    torch = _torch()
    wide, inputs = _distill(logits, top_indices, top_logits, temperature, row_weights)
    _want("stats", stats, logits, (logits.shape[0], 2), wide)
    if gradient is None:
        gradient = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    stride = _rows("gradient", gradient, logits)
    up, uniform = _upstream(upstream, logits, wide)
    status = _status(status, chain, logits)
    _call("distill_loss_backward", inputs + (_ptr(stats), up, uniform, _ptr(gradient), stride), status, chain,
          logits)
    return gradient


@_on_device
def distill_loss_step(logits, top_indices, top_logits, upstream=None, temperature=1.0, row_weights=None, loss=None,
                      stats=None, gradient=None, status=None, *, stream=None, chain=None):
    """distill_loss and distill_loss_backward in one call, for an upstream that does not depend on the
    loss.  Returns (loss, stats, gradient).  gradient may be logits."""
    torch = _torch()
    wide, inputs = _distill(logits, top_indices, top_logits, temperature, row_weights)
    rows = logits.shape[0]
    if loss is None:
        loss = torch.empty(rows, dtype=wide, device=logits.device)
    if stats is None:
        stats = torch.empty((rows, 2), dtype=wide, device=logits.device)
    if gradient is None:
        gradient = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    _want("loss", loss, logits, (rows,), wide)
    _want("stats", stats, logits, (rows, 2), wide)
    stride = _rows("gradient", gradient, logits)
    up, uniform = _upstream(upstream, logits, wide)
    status = _status(status, chain, logits)
    _call("distill_loss_step", inputs + (_ptr(loss), _ptr(stats), up, uniform, _ptr(gradient), stride), status,
          chain, logits)
    return loss, stats, gradient


# ------------------------------------------------------------------ 8-bit block product

def _codes(name, t, like=None):
    if t.dtype not in _code_types():
        raise TypeError(f"{name} is {t.dtype}, float8_e4m3fn (or its bytes, uint8) is wanted")
    if like is not None and t.get_device() != like.get_device():
        raise ValueError(f"{name} is on {t.device}, not on {like.device}")
    return _rows(name, t)


@functools.lru_cache(maxsize=None)
def _code_types():
    return frozenset((_torch().float8_e4m3fn, _torch().uint8))


@_on_device
def block_quantize(x, block_rows=1, codes=None, scales=None, status=None, *, stream=None, chain=None):
    """(codes, scales) of the matrix x: float8_e4m3fn codes and a float32 power of two for each block of
    block_rows (1: activations, 128: weights) rows x 128 columns, x ~ codes * scale.  Allocated codes
    have rows of a multiple of 16 bytes, as block_matmul's tensor core path wants them."""
    torch = _torch()
    if x.dtype == torch.float64:
        raise TypeError("block_quantize handles float32/float16/bfloat16, got torch.float64")
    code = _code(x)
    stride = _rows("input", x)
    rows, columns = x.shape
    if block_rows not in (1, 128):
        raise ValueError(f"block_rows is 1 or 128, got {block_rows}")
    if codes is None:
        room = (columns + 15) // 16 * 16
        codes = torch.empty((rows, room), dtype=torch.float8_e4m3fn, device=x.device)[:, :columns]
    shape = (-(-rows // block_rows), -(-columns // 128))
    if scales is None:
        scales = torch.empty(shape, dtype=torch.float32, device=x.device)
    if codes.shape != x.shape:
        raise ValueError(f"codes has shape {tuple(codes.shape)}, {tuple(x.shape)} is wanted")
    codes_stride = _codes("codes", codes, x)
    _want("scales", scales, x, shape, torch.float32)
    status = _status(status, chain, x)
    _call("block_quantize", (code, _ptr(x), rows, columns, stride, block_rows, _ptr(codes), codes_stride,
          _ptr(scales)), status, chain, x)
    return codes, scales


@_on_device
def block_matmul(left, left_scales, right, right_scales, out=None, dtype=None, status=None, *, stream=None, chain=None):
    """left [rows, inner] times the transpose of right [columns, inner], both codes of block_quantize:
    left with block_rows 1, right (the weights, output features as rows) with 128.  Returns out
    [rows, columns], of type `dtype` (bfloat16 by default, float16 or float32) when it is not given."""
    torch = _torch()
    left_stride, right_stride = _codes("left", left), _codes("right", right, left)
    (rows, inner), (columns, right_inner) = left.shape, right.shape
    if right_inner != inner:
        raise ValueError(f"MatMulShape {tuple(left.shape)} {tuple(right.shape)}")
    blocks = -(-inner // 128)
    _want("left_scales", left_scales, left, (rows, blocks), torch.float32)
    _want("right_scales", right_scales, left, (-(-columns // 128), blocks), torch.float32)
    if out is None:
        out = torch.empty((rows, columns), dtype=dtype or torch.bfloat16, device=left.device)
    elif dtype is not None and out.dtype != dtype:
        raise TypeError(f"out is {out.dtype}, {dtype} is wanted")
    if out.dtype == torch.float64 or out.shape != (rows, columns) or out.get_device() != left.get_device():
        raise ValueError(f"out is a {rows} x {columns} float32/float16/bfloat16 matrix on {left.device}")
    code = _code(out)
    out_stride = _rows("out", out)
    status = _status(status, chain, left)
    _call("block_matmul", (code, _ptr(left), _ptr(left_scales), _ptr(right), _ptr(right_scales), _ptr(out), rows,
          inner, columns, left_stride, right_stride, out_stride), status, chain, left)
    return out
