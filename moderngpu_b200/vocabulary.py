"""The vocabulary operators of libmgpu_b200.so: embedding lookup and gradient,
distillation from a teacher's top logits, token sampling. Formulas and rules for
empty rows: include/moderngpu_b200.h.

As in binding.py, tensor arguments are torch CUDA tensors, all of one call on
one device; work is enqueued on torch's current stream of that device. Matrices
may have more than `width` elements from row to row (a padded vocabulary's
view); everything else is contiguous.
"""
import ctypes

import torch

from .binding import (_DTYPES, _check, _on, _require_cuda, _scratch, _stream,
                      _workspace, load_library)

F16, BF16 = 4, 5
_REALS = {torch.float32: _DTYPES[torch.float32], torch.float16: F16,
          torch.bfloat16: BF16}
_MOST = 0x7fffffff
_TOKENS = {torch.int32: _DTYPES[torch.int32],
           torch.int64: _DTYPES[torch.int64]}


def declare(lib):
    """Argument types of the entry points (called by load_library)."""
    c_void_p, c_int, c_size_t = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
    c_int64, c_float = ctypes.c_int64, ctypes.c_float
    lib.mgpu_b200_embedding_lookup.restype = c_int
    lib.mgpu_b200_embedding_lookup.argtypes = [
        c_int, c_void_p, c_int, c_int, c_int64, c_int, c_void_p, c_int,
        c_float, c_void_p, c_void_p]
    lib.mgpu_b200_embedding_gradient_workspace_bytes.restype = c_size_t
    lib.mgpu_b200_embedding_gradient_workspace_bytes.argtypes = [
        c_int, c_int, c_int, c_int]
    lib.mgpu_b200_embedding_gradient.restype = c_int
    lib.mgpu_b200_embedding_gradient.argtypes = [
        c_int, c_void_p, c_int64, c_int, c_int, c_void_p, c_int, c_int,
        c_float, c_int, c_int, c_void_p, c_void_p, c_size_t, c_void_p]
    lib.mgpu_b200_distill_loss.restype = c_int
    lib.mgpu_b200_distill_loss.argtypes = [
        c_int, c_void_p, c_int64, c_int, c_int, c_int, c_void_p, c_int,
        c_void_p, c_int, c_float, c_void_p, c_void_p]
    lib.mgpu_b200_distill_loss_gradient.restype = c_int
    lib.mgpu_b200_distill_loss_gradient.argtypes = [
        c_int, c_void_p, c_int64, c_int, c_int, c_int, c_void_p, c_int,
        c_void_p, c_int, c_float, c_void_p, c_void_p, c_void_p, c_int64,
        c_void_p]
    lib.mgpu_b200_sample_tokens.restype = c_int
    lib.mgpu_b200_sample_tokens.argtypes = [
        c_int, c_void_p, c_int64, c_int, c_int, c_void_p, c_float, c_void_p,
        c_int, c_void_p, c_float, c_void_p, c_float, c_void_p, c_void_p,
        c_void_p]


# The address of the current stream and the number of the current device without
# the objects around them, which cost as much as the launch of a small kernel; the
# public ways where a torch does not have these.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_raw_device = getattr(torch._C, "_cuda_getDevice", None)


def _stream_of(device):
    if _raw_stream is None or device.index is None:
        return _stream(device)
    return _raw_stream(device.index)


def _call(device, entry, *arguments):
    """entry(*arguments, current stream) with `device` the current one; raises
    MgpuError."""
    if _raw_device is not None and device.index == _raw_device():
        code = entry(*arguments, _stream_of(device))
    else:
        with _on(device):
            code = entry(*arguments, _stream_of(device))
    if code:
        _check(code)


def _require(t, name, dtypes, device=None):
    """A dense CUDA tensor of one of the dtypes, on the call's device."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or \
            not t.is_contiguous():
        _require_cuda(t, name)
    if t.dtype not in dtypes:
        raise TypeError("%s must have one of the dtypes %s" %
                        (name, ", ".join(str(d) for d in dtypes)))
    if device is not None and t.device != device:
        raise ValueError("%s must be on %s" % (name, device))


def _matrix(t, name, dtypes, device=None):
    """Checks a matrix whose rows are dense; returns (rows, width, stride)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA tensor" % name)
    if t.dtype not in dtypes:
        raise TypeError("%s must have one of the dtypes %s" %
                        (name, ", ".join(str(d) for d in dtypes)))
    if device is not None and t.device != device:
        raise ValueError("%s must be on %s" % (name, device))
    if t.dim() != 2:
        raise ValueError("%s must have two dimensions" % name)
    (rows, width), (stride, step) = t.shape, t.stride()
    if width > 1 and step != 1:
        raise ValueError("the rows of %s must be contiguous" % name)
    if rows < 2:
        stride = width
    if stride < width:
        raise ValueError("the rows of %s must not overlap" % name)
    if rows > _MOST or width > _MOST:
        raise ValueError("%s is too large: %d x %d" % (name, rows, width))
    return rows, width, stride


def _fits(n, name):
    """The library's sizes are 32 bits wide; ctypes would cut off the rest."""
    if n > _MOST:
        raise ValueError("%s is too large: %d" % (name, n))
    return n


def _shaped(out, name, shape, dtypes, device):
    """Checks a caller's output, or makes one (of the first dtype)."""
    if out is None:
        return torch.empty(shape, dtype=dtypes[0], device=device)
    _require(out, name, dtypes, device)
    if tuple(out.shape) != tuple(shape):
        raise ValueError("%s must have the shape %s" % (name, tuple(shape)))
    return out


def _call_workspace(device, nbytes):
    """The stream's scratch buffer; while a graph is captured, memory of the
    graph's own, so that graphs which are replayed at the same time share
    none."""
    if _raw_device is not None and device.index == _raw_device():
        capturing = torch.cuda.is_current_stream_capturing()
    else:
        with _on(device):
            capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    if _raw_stream is not None and device.index is not None:
        # _workspace's buffer, by the same key.
        buf = _scratch.get((device.index, _raw_stream(device.index)))
        if buf is not None and buf.numel() >= nbytes:
            return buf
    return _workspace(device, nbytes)


def embedding_lookup(table, tokens, scale=1.0, out=None):
    """out[..., :] = scale * table[tokens[...], :]; a token outside of the
    table (-1 for padding) gives zeros.

    table: (rows, width) float32, float16 or bfloat16; tokens: int32 or int64
    of any shape; out: tokens.shape + (width,), of the table's dtype.
    """
    lib = load_library()
    rows, width, stride = _matrix(table, "table", _REALS)
    dtype, device = table.dtype, table.device
    _require(tokens, "tokens", _TOKENS, device)
    count = _fits(tokens.numel(), "tokens")
    out = _shaped(out, "out", tokens.shape + (width,), (dtype,), device)
    _call(device, lib.mgpu_b200_embedding_lookup,
          _REALS[dtype], table.data_ptr(), rows, width, stride,
          _TOKENS[tokens.dtype], tokens.data_ptr(), count, scale,
          out.data_ptr())
    return out


def embedding_gradient(grad, tokens, rows, scale=1.0, out=None,
                       accumulate=False, workspace=None):
    """The gradient of embedding_lookup for its table: out[r] = scale * the sum
    of grad[i] over the positions i whose token is r, zero for rows without one.

    grad: tokens.shape + (width,), float32, float16 or bfloat16 (as a matrix it
    may have a row stride); out: (rows, width) of grad's dtype or float32. With
    accumulate the sums are added to `out` and other rows stay as they are.
    Sums are held in 32 bits in the order of the positions.
    """
    lib = load_library()
    if not isinstance(grad, torch.Tensor) or not grad.is_cuda:
        raise TypeError("grad must be a CUDA tensor")
    _require(tokens, "tokens", _TOKENS, grad.device)
    if grad.dim() < 1 or tuple(grad.shape[:-1]) != tuple(tokens.shape):
        raise ValueError("grad must have one row for each token")
    device = grad.device
    width, count = grad.shape[-1], _fits(tokens.numel(), "tokens")
    _fits(rows, "rows")
    if grad.dim() != 2:
        if not grad.is_contiguous():
            raise ValueError("grad must be contiguous, or a matrix")
        grad = grad.view(count, width)
    _, _, stride = _matrix(grad, "grad", _REALS)
    if accumulate and out is None:
        raise ValueError("accumulate needs out")
    out = _shaped(out, "out", (rows, width), (grad.dtype, torch.float32),
                  device)
    if workspace is None:
        # A size out of range asks for 0 bytes here and is refused below.
        workspace = _call_workspace(
            device, lib.mgpu_b200_embedding_gradient_workspace_bytes(
                count, rows, width, int(accumulate)))
    else:
        _require(workspace, "workspace", (torch.uint8,), device)
    _call(device, lib.mgpu_b200_embedding_gradient,
          _REALS[grad.dtype], grad.data_ptr(), stride, width,
          _TOKENS[tokens.dtype], tokens.data_ptr(), count, rows, scale,
          int(accumulate), _REALS[out.dtype], out.data_ptr(),
          workspace.data_ptr(), workspace.numel())
    return out


def _teacher(count, device, teacher_tokens, teacher_logits):
    _require(teacher_tokens, "teacher_tokens", _TOKENS, device)
    _require(teacher_logits, "teacher_logits", _REALS, device)
    if teacher_tokens.dim() != 2 or teacher_tokens.shape[0] != count:
        raise ValueError("teacher_tokens must have one row for each of logits")
    if teacher_logits.shape != teacher_tokens.shape:
        raise ValueError("teacher_logits must have teacher_tokens' shape")
    return teacher_tokens.shape[1]


def distill_loss(logits, teacher_tokens, teacher_logits, temperature=1.0,
                 out=None):
    """Distillation loss of every row, float32: T^2 * KL(p || q) for the
    softmax p of the teacher's top logits / T over their own entries and the
    softmax q of logits / T over the vocabulary.

    logits: (count, vocabulary) float32, float16 or bfloat16; teacher_tokens:
    (count, entries) int32 or int64, at most 1024 entries, -1 for an unused one;
    teacher_logits: of the same shape, any of the three dtypes.
    """
    lib = load_library()
    count, vocabulary, stride = _matrix(logits, "logits", _REALS)
    device = logits.device
    entries = _teacher(count, device, teacher_tokens, teacher_logits)
    out = _shaped(out, "out", (count,), (torch.float32,), device)
    _call(device, lib.mgpu_b200_distill_loss,
          _REALS[logits.dtype], logits.data_ptr(), stride, count, vocabulary,
          _TOKENS[teacher_tokens.dtype], teacher_tokens.data_ptr(),
          _REALS[teacher_logits.dtype], teacher_logits.data_ptr(), entries,
          temperature, out.data_ptr())
    return out


def distill_loss_gradient(logits, teacher_tokens, teacher_logits,
                          row_weights=None, temperature=1.0, loss=None,
                          out=None):
    """distill_loss together with its gradient for the logits: returns
    (loss, out), out[i] = row_weights[i] * d loss[i] / d logits[i], of the
    logits' dtype. row_weights (float32; 1 where not given) is what a training
    step multiplies each row's loss by, such as 1 / count; a row of weight 0 is
    masked: loss 0 and gradient 0, whatever its logits are. `out` may be
    `logits` itself, which then holds the gradient.
    """
    lib = load_library()
    count, vocabulary, stride = _matrix(logits, "logits", _REALS)
    device = logits.device
    entries = _teacher(count, device, teacher_tokens, teacher_logits)
    loss = _shaped(loss, "loss", (count,), (torch.float32,), device)
    if row_weights is not None:
        _require(row_weights, "row_weights", (torch.float32,), device)
        if tuple(row_weights.shape) != (count,):
            raise ValueError("row_weights must have one number for each row")
    if out is None:
        out = torch.empty((count, vocabulary), dtype=logits.dtype,
                          device=device)
    _, _, out_stride = _matrix(out, "out", (logits.dtype,), device)
    if out.shape != logits.shape:
        raise ValueError("out must have the logits' shape")
    _call(device, lib.mgpu_b200_distill_loss_gradient,
          _REALS[logits.dtype], logits.data_ptr(), stride, count, vocabulary,
          _TOKENS[teacher_tokens.dtype], teacher_tokens.data_ptr(),
          _REALS[teacher_logits.dtype], teacher_logits.data_ptr(), entries,
          temperature, None if row_weights is None else
          row_weights.data_ptr(), loss.data_ptr(), out.data_ptr(),
          out_stride)
    return loss, out


def _setting(value, name, dtype, count, device):
    """(number, address) of a setting: one of the two counts."""
    if not isinstance(value, torch.Tensor):
        return value, None
    _require(value, name, (dtype,), device)
    if tuple(value.shape) != (count,):
        raise ValueError("%s must have one number for each row" % name)
    return 0, value.data_ptr()


def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0, out=None):
    """One token (int32) for every row of logits, drawn by the given numbers
    uniform (float32, in [0, 1)) from softmax(logits / temperature) after
    top-k, top-p and min-p, in this order.

    logits: (count, vocabulary) float32, float16 or bfloat16. Each setting is a
    number for all rows or a tensor with one for each (float32; top_k int32).
    top_k <= 0, top_p >= 1 and min_p == 0 switch a step off; temperature 0 takes
    the greatest logit. Equal logits are ordered by index. A row with a NaN or
    without a logit above -infinity gives -1.
    """
    lib = load_library()
    count, vocabulary, stride = _matrix(logits, "logits", _REALS)
    device = logits.device
    _require(uniform, "uniform", (torch.float32,), device)
    if tuple(uniform.shape) != (count,):
        raise ValueError("uniform must have one number for each row")
    t, t_rows = _setting(temperature, "temperature", torch.float32, count,
                         device)
    k, k_rows = _setting(top_k, "top_k", torch.int32, count, device)
    k = max(min(k, _MOST), 0)
    p, p_rows = _setting(top_p, "top_p", torch.float32, count, device)
    m, m_rows = _setting(min_p, "min_p", torch.float32, count, device)
    out = _shaped(out, "out", (count,), (torch.int32,), device)
    _call(device, lib.mgpu_b200_sample_tokens,
          _REALS[logits.dtype], logits.data_ptr(), stride, count, vocabulary,
          uniform.data_ptr(), t, t_rows, k, k_rows, p, p_rows, m, m_rows,
          out.data_ptr())
    return out
