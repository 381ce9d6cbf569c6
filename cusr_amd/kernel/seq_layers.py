"""The layers around attention of a learned proposer (include/cusr_seq.h).

Beside attention, rotary positions and the policy loss (cusr_amd.kernel.seq_ops), a
pass through the model looks symbols up, adds to the residual stream and normalises
it, multiplies by weights and asks for the probabilities of symbols. These are those
steps on the GPU; the reference has no counterpart.

  embedding, embedding_grad            rows of a table by token, scaled
  rms_norm, rms_norm_grad              root-mean-square norm after the residual's
                                       addition
  rms_norm_int8, quantize_rows         the same norm, or plain rows, as 8-bit integers
                                       with a scale for each row
  int8_product                         product of two such operands
  token_logprobs, token_logprobs_grad  log-probabilities of given tokens, entropy and
                                       top alternatives

Conventions are seq_ops': torch CUDA tensors, work queued on the current stream of
their device, arguments checked before anything is launched (TypeError, ValueError), a
refusal of the library raises COError, dual tensors are refused, no CPU path. embedding,
rms_norm and token_logprobs take part in autograd; the 8-bit operators are for sampling
and scoring and refuse inputs that require a gradient. The same call gives the same
bits.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from cusr_amd.kernel.seq_ops import (_DTYPES, _F, _FLOAT32, _I32, _I64, _INTS, _LEAST, _MOST, _P,
                                     _need, _no_gradient, _no_tangents, _packer, _ptr, _run,
                                     _workspace, load_library)

SEQ_MAX_WIDTH = 65536
SEQ_MAX_INNER = 131071
SEQ_MAX_TOP = 64
SEQ_MAX_ROWS = 2147000000
_INT8 = 3


class SeqEmbedding(ctypes.Structure):
    """cusr_seq.h SeqEmbedding."""
    _fields_ = [("struct_size", _I32), ("dtype", _I32), ("out_dtype", _I32), ("ids_64", _I32),
                ("tokens", _I64), ("rows", _I64), ("width", _I64), ("table_row", _I64),
                ("out_row", _I64), ("scale", _F), ("reserved", _I32), ("ids", _P), ("table", _P),
                ("out", _P)]


class SeqEmbeddingGrad(ctypes.Structure):
    """cusr_seq.h SeqEmbeddingGrad."""
    _fields_ = [("struct_size", _I32), ("dtype", _I32), ("out_dtype", _I32), ("ids_64", _I32),
                ("tokens", _I64), ("rows", _I64), ("width", _I64), ("dout_row", _I64),
                ("dtable_row", _I64), ("scale", _F), ("reserved", _I32), ("ids", _P),
                ("d_out", _P), ("dtable", _P), ("workspace", _P), ("workspace_bytes", _I64)]


class SeqNorm(ctypes.Structure):
    """cusr_seq.h SeqNorm."""
    _fields_ = [("struct_size", _I32), ("x_dtype", _I32), ("h_dtype", _I32), ("y_dtype", _I32),
                ("gain_dtype", _I32), ("identity", _I32), ("tokens", _I64), ("width", _I64),
                ("x_row", _I64), ("residual_row", _I64), ("h_row", _I64), ("y_row", _I64),
                ("eps", _F), ("reserved", _I32), ("x", _P), ("residual", _P), ("gain", _P),
                ("h", _P), ("y", _P), ("y_scale", _P)]


class SeqNormGrad(ctypes.Structure):
    """cusr_seq.h SeqNormGrad."""
    _fields_ = [("struct_size", _I32), ("dy_dtype", _I32), ("h_dtype", _I32), ("x_dtype", _I32),
                ("gain_dtype", _I32), ("reserved", _I32), ("tokens", _I64), ("width", _I64),
                ("dy_row", _I64), ("h_row", _I64), ("dh_row", _I64), ("d_row", _I64),
                ("dx_row", _I64), ("eps", _F), ("reserved2", _I32), ("dy", _P), ("h", _P),
                ("gain", _P), ("dh", _P), ("d", _P), ("dx", _P), ("dgain", _P),
                ("workspace", _P), ("workspace_bytes", _I64)]


class SeqInt8Product(ctypes.Structure):
    """cusr_seq.h SeqInt8Product."""
    _fields_ = [("struct_size", _I32), ("out_dtype", _I32), ("m", _I64), ("n", _I64),
                ("inner", _I64), ("a_row", _I64), ("w_row", _I64), ("o_row", _I64), ("a", _P),
                ("w", _P), ("a_scale", _P), ("w_scale", _P), ("o", _P), ("workspace", _P),
                ("workspace_bytes", _I64)]


class SeqLogprobs(ctypes.Structure):
    """cusr_seq.h SeqLogprobs."""
    _fields_ = [("struct_size", _I32), ("dtype", _I32), ("ids_64", _I32), ("top", _I32),
                ("tokens", _I64), ("vocab", _I64), ("row", _I64), ("temperature", _F),
                ("reserved", _I32), ("logits", _P), ("ids", _P), ("logp", _P), ("entropy", _P),
                ("stats", _P), ("top_logp", _P), ("top_ids", _P), ("workspace", _P),
                ("workspace_bytes", _I64)]


class SeqLogprobsGrad(ctypes.Structure):
    """cusr_seq.h SeqLogprobsGrad."""
    _fields_ = [("struct_size", _I32), ("dtype", _I32), ("ids_64", _I32), ("reserved", _I32),
                ("tokens", _I64), ("vocab", _I64), ("row", _I64), ("drow", _I64),
                ("temperature", _F), ("reserved2", _I32), ("logits", _P), ("ids", _P),
                ("stats", _P), ("entropy", _P), ("dlogp", _P), ("dentropy", _P), ("dlogits", _P)]


_pack_embedding, _SIZE_EMBEDDING = _packer(SeqEmbedding)
_pack_embedding_grad, _SIZE_EMBEDDING_GRAD = _packer(SeqEmbeddingGrad)
_pack_norm, _SIZE_NORM = _packer(SeqNorm)
_pack_norm_grad, _SIZE_NORM_GRAD = _packer(SeqNormGrad)
_pack_int8, _SIZE_INT8 = _packer(SeqInt8Product)
_pack_logprobs, _SIZE_LOGPROBS = _packer(SeqLogprobs)
_pack_logprobs_grad, _SIZE_LOGPROBS_GRAD = _packer(SeqLogprobsGrad)

_FLOATS = tuple(_DTYPES)


def _rows(x):
    """x as the kernels read it: the elements of a row side by side."""
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _matrix(x, name, dtypes, device=None, width=None, rows=None, most=SEQ_MAX_WIDTH):
    _need(x, name, dtypes, 2, device)
    if width is not None and x.shape[1] != width:
        raise ValueError(f"{name} must have {width} columns, not {x.shape[1]}")
    if rows is not None and x.shape[0] != rows:
        raise ValueError(f"{name} must have {rows} rows, not {x.shape[0]}")
    if not 1 <= x.shape[1] <= most:
        raise ValueError(f"{name} must have 1 to {most} columns, not {x.shape[1]}")
    return x


def _plain(x):
    """Whether x is a matrix of floats as the row operators take it: the common case, in a
    few comparisons. _matrix says what is wrong with another. A tensor that answers
    oddly is left to it too."""
    try:
        return (x.is_cuda and x.get_device() >= 0 and x.dtype in _DTYPES and x.dim() == 2
                and 0 < x.shape[1] <= SEQ_MAX_WIDTH)
    except AttributeError:
        return False


def _beside(x, dtypes, to, n=None):
    """The same of a vector (of n entries) on the device of `to`."""
    try:
        return (x.is_cuda and x.dtype in dtypes and x.dim() == 1
                and x.get_device() == to.get_device() and (n is None or x.shape[0] == n))
    except AttributeError:
        return False


def _vector(x, name, dtypes, n, device):
    _need(x, name, dtypes, 1, device)
    if x.shape[0] != n:
        raise ValueError(f"{name} must have {n} entries, not {x.shape[0]}")
    return x.contiguous()


def _type(dtype, otherwise):
    if dtype is None:
        return otherwise
    if dtype not in _DTYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, not {dtype}")
    return dtype


def _number(x, name, least=-_FLOAT32, most=_FLOAT32):
    x = float(x)
    if not least <= x <= most:
        raise ValueError(f"{name} must be from {least:g} to {most:g}, not {x}")
    return x


# ------------------------------------------------------------------ embedding

def _embedding(tokens, table, scale, dtype):
    T, (V, D) = tokens.shape[0], table.shape
    out = table.new_empty((T, D)) if dtype is table.dtype else table.new_empty((T, D), dtype=dtype)
    if T:
        table, tokens = _rows(table), tokens.contiguous()    # kept until the launch
        _run(load_library().seq_embedding, "seq_embedding", table.get_device(), _pack_embedding(
            _SIZE_EMBEDDING, _DTYPES[table.dtype], _DTYPES[dtype], tokens.dtype is torch.int64, T,
            V, D, table.stride(0), D, scale, 0, tokens.data_ptr(), table.data_ptr(),
            out.data_ptr()))
    return out


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, scale, dtype):
        ctx.save_for_backward(tokens)
        ctx.how = (table.shape[0], scale, table.dtype)
        return _embedding(tokens, table, scale, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        rows, scale, dtype = ctx.how
        return None, embedding_grad(dout, *ctx.saved_tensors, rows, scale=scale, dtype=dtype), \
            None, None


def embedding(tokens, table, *, scale=1.0, dtype=None):
    """Rows of a table by token: out[t] = scale * table[tokens[t]], [T, D].

    tokens int32 or int64 [T]; table [V, D] float32, bfloat16 or float16, D up to 65,536.
    The product is formed in float32 and rounded once to `dtype` (the table's by
    default). A token outside the table gives a row of NaN. The gradient goes to the
    table; tokens outside it take no part."""
    _no_tangents(table)
    if not (_plain(table) and _beside(tokens, _INTS, table)):
        _matrix(table, "table", _FLOATS)
        _need(tokens, "tokens", _INTS, 1, table.device)
    scale, dtype = _number(scale, "scale"), _type(dtype, table.dtype)
    if table.requires_grad and torch.is_grad_enabled():
        return _EmbeddingFn.apply(tokens, table, scale, dtype)
    return _embedding(tokens, table, scale, dtype)


def embedding_grad(dout, tokens, rows, *, scale=1.0, dtype=torch.float32):
    """Gradient [rows, D] of embedding's table for the gradient `dout` [T, D] of its
    output: each row the sum of its tokens' rows, in float32 and in an order that depends
    on the tokens alone, times scale; 0 where there is none. The result is no part of a
    graph."""
    _no_tangents(dout)
    _matrix(dout, "dout", _FLOATS)
    T, D = dout.shape
    tokens = _vector(tokens, "tokens", _INTS, T, dout.device)
    rows = int(rows)
    if not 0 <= rows <= SEQ_MAX_ROWS:
        raise ValueError(f"rows must be from 0 to {SEQ_MAX_ROWS}, not {rows}")
    scale, dtype = _number(scale, "scale"), _type(dtype, torch.float32)
    dtable = torch.empty((rows, D), dtype=dtype, device=dout.device)
    if not rows:
        return dtable
    dout, lib = _rows(dout), load_library()
    args = (_SIZE_EMBEDDING_GRAD, _DTYPES[dout.dtype], _DTYPES[dtype],
            tokens.dtype is torch.int64, T, rows, D, dout.stride(0), D, scale, 0,
            tokens.data_ptr(), dout.data_ptr(), dtable.data_ptr())
    ptr, n, ws = _workspace(lib.seq_embedding_grad_workspace, "seq_embedding_grad",
                            _pack_embedding_grad(*args, 0, 0), dout.device)
    _run(lib.seq_embedding_grad, "seq_embedding_grad", dout.get_device(),
         _pack_embedding_grad(*args, ptr or 0, n))
    del ws
    return dtable


# ----------------------------------------------------------------------- norm

def _check_norm(x, gain, residual, eps):
    _no_tangents(x, gain, residual)
    if (_plain(x) and (gain is None or _beside(gain, _DTYPES, x, x.shape[1]))
            and (residual is None or (_plain(residual) and residual.shape == x.shape
                                      and residual.get_device() == x.get_device()
                                      and residual.dtype in (x.dtype, torch.float32)))):
        return _number(eps, "eps", 0.0)
    _matrix(x, "x", _FLOATS)
    if residual is not None:
        types = (x.dtype,) if x.dtype is torch.float32 else (x.dtype, torch.float32)
        _matrix(residual, "residual", types, x.device, x.shape[1], x.shape[0])
    if gain is not None:
        _vector(gain, "gain", _FLOATS, x.shape[1], x.device)
    return _number(eps, "eps", 0.0)


def _norm(x, gain, residual, eps, dtype, identity=False):
    """(y, scale, h): y of dtype, or 8-bit integers with scales where dtype is int8; h the
    stream, or None without a residual."""
    (T, D), dev = x.shape, x.device
    y = torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format)
    scale = torch.empty(T, dtype=torch.float32, device=dev) if dtype is torch.int8 else None
    h = None
    if residual is not None:
        h = torch.empty_like(residual, memory_format=torch.contiguous_format)
        residual = _rows(residual)
    if T:
        x = _rows(x)
        gain = None if gain is None else gain.contiguous()
        _run(load_library().seq_norm, "seq_norm", x.get_device(), _pack_norm(
            _SIZE_NORM, _DTYPES[x.dtype], _DTYPES[x.dtype if h is None else h.dtype],
            _INT8 if scale is not None else _DTYPES[dtype],
            0 if gain is None else _DTYPES[gain.dtype], identity, T, D, x.stride(0),
            0 if h is None else residual.stride(0), 0 if h is None else D, D, eps, 0,
            x.data_ptr(), _ptr(residual), _ptr(gain), _ptr(h), y.data_ptr(), _ptr(scale)))
    return y, scale, h


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gain, residual, eps, dtype):
        y, _, h = _norm(x, gain, residual, eps, dtype)
        ctx.save_for_backward(x if h is None else h, gain)
        ctx.how = (eps, x.dtype)
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, gain = ctx.saved_tensors
        eps, x_dtype = ctx.how
        if dy is None:
            return (None if dh is None else dh.to(x_dtype)), None, dh, None, None
        need_gain = gain is not None and ctx.needs_input_grad[1]
        d, dx, dgain = _norm_grad(dy, h, gain, dh, eps, x_dtype, need_gain)
        return dx, (dgain.to(gain.dtype) if need_gain else None), \
            (d if ctx.needs_input_grad[2] else None), None, None


def rms_norm(x, gain=None, *, residual=None, eps=1e-6, dtype=None):
    """Root-mean-square norm of rows [T, D], after the addition of a residual stream.

    x float32, bfloat16 or float16, D up to 65,536; residual like x, of its type or
    float32; gain [D] or None (1). The stream h = x + residual is rounded to residual's
    type (h = x without one), and y = gain * h / sqrt(mean(h**2) + eps), formed in
    float32, to `dtype` (x's by default). Returns y, or (y, h) with a residual. Gradients
    go to x, residual and gain. A row of zeros with eps 0 gives NaN; one whose sum of squares
    passes float32's largest number gives 0, and its gradient says nothing."""
    eps, dtype = _check_norm(x, gain, residual, eps), _type(dtype, x.dtype)
    if torch.is_grad_enabled() and (x.requires_grad
                                    or (gain is not None and gain.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _NormFn.apply(x, gain, residual, eps, dtype)
    y, _, h = _norm(x, gain, residual, eps, dtype)
    return y if h is None else (y, h)


def rms_norm_int8(x, gain=None, *, residual=None, eps=1e-6):
    """rms_norm with its output as 8-bit integers: (q, scale) or, with a residual,
    (q, scale, h). q int8 [T, D] and scale float32 [T]: scale is the largest magnitude
    of a row of y times 1 / 127, q the nearest integers to y / scale, halves to even,
    each step in float32. A row of zeros has the scale 0; one with a value that is not
    finite the scale NaN and q 0. (Rows below some 1e-36 lose precision with their
    scale.)"""
    eps = _check_norm(x, gain, residual, eps)
    _no_gradient(x=x, gain=gain, residual=residual)
    y, scale, h = _norm(x, gain, residual, eps, torch.int8)
    return (y, scale) if h is None else (y, scale, h)


def quantize_rows(x):
    """Rows [T, D] as 8-bit integers with a scale each: (q, scale) as rms_norm_int8 gives
    them, of x itself. For weights [outputs, inputs]: a scale for each channel."""
    _check_norm(x, None, None, 0.0)
    _no_gradient(x=x)
    return _norm(x, None, None, 0.0, torch.int8, True)[:2]


def _norm_grad(dy, h, gain, dh, eps, x_dtype, need_gain):
    (T, D), dev = h.shape, h.device
    d = torch.empty((T, D), dtype=h.dtype, device=dev)
    dx = d if x_dtype is h.dtype else torch.empty((T, D), dtype=x_dtype, device=dev)
    dgain = torch.empty(D, dtype=torch.float32, device=dev) if need_gain else None
    if not T and not need_gain:
        return d, dx, dgain
    dy, h = _rows(dy), _rows(h)
    dh = None if dh is None else _rows(dh)
    gain = None if gain is None else gain.contiguous()
    lib = load_library()
    args = (_SIZE_NORM_GRAD, _DTYPES[dy.dtype], _DTYPES[h.dtype], _DTYPES[x_dtype],
            0 if gain is None else _DTYPES[gain.dtype], 0, T, D, dy.stride(0), h.stride(0),
            0 if dh is None else dh.stride(0), D, D, eps, 0, dy.data_ptr(), h.data_ptr(),
            _ptr(gain), _ptr(dh), d.data_ptr(), 0 if dx is d else dx.data_ptr(), _ptr(dgain))
    ptr, n, ws = _workspace(lib.seq_norm_grad_workspace, "seq_norm_grad",
                            _pack_norm_grad(*args, 0, 0), dev)
    _run(lib.seq_norm_grad, "seq_norm_grad", h.get_device(), _pack_norm_grad(*args, ptr or 0, n))
    del ws
    return d, dx, dgain


def rms_norm_grad(dy, h, gain=None, *, dh=None, eps=1e-6, x_dtype=None):
    """Gradient of rms_norm for the gradients `dy` of its output and `dh` (None: 0) of the
    stream h that it returned, or of x, in h's place, where there was no residual:
    (d, dx, dgain). d, in h's type, is the residual's gradient; dx the same in x_dtype
    (d itself where that is None or h's); dgain float32 [D], None without a gain. The
    results are no part of a graph."""
    _no_tangents(dy, h, gain, dh)
    _matrix(h, "h", _FLOATS)
    T, D = h.shape
    _matrix(dy, "dy", _FLOATS, h.device, D, T)
    if dh is not None:
        _matrix(dh, "dh", (h.dtype,), h.device, D, T)
    if gain is not None:
        _vector(gain, "gain", _FLOATS, D, h.device)
    return _norm_grad(dy, h, gain, dh, _number(eps, "eps", 0.0), _type(x_dtype, h.dtype),
                      gain is not None)


# --------------------------------------------------------------- 8-bit product

_FP32 = (torch.float32,)


def _plain_int8(a, w):
    """Whether both are 8-bit matrices of one inner size on one GPU."""
    try:
        return (a.is_cuda and a.dtype is torch.int8 and w.dtype is torch.int8 and a.dim() == 2
                and w.dim() == 2 and a.shape[1] == w.shape[1] <= SEQ_MAX_INNER
                and w.get_device() == a.get_device() >= 0)
    except AttributeError:
        return False


def int8_product(a, a_scale, w, w_scale, *, dtype=torch.bfloat16):
    """Product of 8-bit integers with scales: out[t, n] = a_scale[t] * w_scale[n] *
    sum over k of a[t, k] w[n, k], [T, N] of `dtype`.

    a int8 [T, K] with a_scale float32 [T] (rms_norm_int8, quantize_rows), w int8 [N, K]
    with w_scale float32 [N] (quantize_rows of weights [N, K], once), K up to 131,071.
    The sum is exact; the rest is formed in float32 and rounded once. K and rows of a
    multiple of 16 spare a copy of the operands."""
    _no_tangents(a_scale, w_scale)
    if not (_plain_int8(a, w) and _beside(a_scale, _FP32, a, a.shape[0])
            and _beside(w_scale, _FP32, a, w.shape[0])):
        _need(a, "a", (torch.int8,), 2)
        _need(w, "w", (torch.int8,), 2, a.device)
        if w.shape[1] != a.shape[1] or a.shape[1] > SEQ_MAX_INNER:
            raise ValueError(f"a and w must have the same number of columns, up to "
                             f"{SEQ_MAX_INNER}; got {tuple(a.shape)} and {tuple(w.shape)}")
        _vector(a_scale, "a_scale", _FP32, a.shape[0], a.device)
        _vector(w_scale, "w_scale", _FP32, w.shape[0], a.device)
    if a_scale.requires_grad or w_scale.requires_grad:
        _no_gradient(a_scale=a_scale, w_scale=w_scale)
    dev, (T, K), N = a.device, a.shape, w.shape[0]
    a_scale, w_scale = a_scale.contiguous(), w_scale.contiguous()
    dtype = _type(dtype, torch.bfloat16)
    out = torch.empty((T, N), dtype=dtype, device=dev)
    if not T or not N:
        return out
    if K:
        a, w = _rows(a), _rows(w)
    lib = load_library()
    args = (_SIZE_INT8, _DTYPES[dtype], T, N, K, a.stride(0), w.stride(0), N, a.data_ptr(),
            w.data_ptr(), a_scale.data_ptr(), w_scale.data_ptr(), out.data_ptr())
    packed = _pack_int8(*args, 0, 0)
    ptr, n, ws = _workspace(lib.seq_int8_product_workspace, "seq_int8_product", packed, dev)
    if n:
        packed = _pack_int8(*args, ptr, n)
    _run(lib.seq_int8_product, "seq_int8_product", a.get_device(), packed)
    del ws
    return out


# ----------------------------------------------------------- log-probabilities

def _check_logits(logits, tokens, temperature):
    if _plain(logits) and _beside(tokens, _INTS, logits, logits.shape[0]):
        return tokens.contiguous(), _number(temperature, "temperature", _LEAST, _MOST)
    _matrix(logits, "logits", _FLOATS, most=SEQ_MAX_ROWS)
    return (_vector(tokens, "tokens", _INTS, logits.shape[0], logits.device),
            _number(temperature, "temperature", _LEAST, _MOST))


def _logprobs(logits, tokens, temperature, top, need_stats):
    (T, V), dev = logits.shape, logits.device

    logp = torch.empty(T, dtype=torch.float32, device=dev)
    entropy, stats, top_logp, top_ids = torch.empty_like(logp), None, None, None
    if need_stats:
        stats = torch.empty((T, 2), dtype=torch.float32, device=dev)
    if top:
        top_logp = torch.empty((T, top), dtype=torch.float32, device=dev)
        top_ids = torch.empty_like(top_logp, dtype=torch.int64)
    if T:
        logits, lib = _rows(logits), load_library()
        args = (_SIZE_LOGPROBS, _DTYPES[logits.dtype], tokens.dtype is torch.int64, top, T, V,
                logits.stride(0), temperature, 0, logits.data_ptr(), tokens.data_ptr(),
                logp.data_ptr(), entropy.data_ptr(), _ptr(stats), _ptr(top_logp), _ptr(top_ids))
        packed = _pack_logprobs(*args, 0, 0)
        ptr, n, ws = _workspace(lib.seq_logprobs_workspace, "seq_logprobs", packed, dev)
        if n:
            packed = _pack_logprobs(*args, ptr, n)
        _run(lib.seq_logprobs, "seq_logprobs", logits.get_device(), packed)
        del ws
    return logp, entropy, top_logp, top_ids, stats


class _LogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature, top):
        out = _logprobs(logits, tokens, temperature, top, True)
        logp, entropy, top_logp, top_ids, stats = out
        ctx.save_for_backward(logits, tokens, stats, entropy)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(x for x in out[2:] if x is not None))
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp, dentropy, *_):
        logits, tokens, stats, entropy = ctx.saved_tensors
        if dlogp is None and dentropy is None:
            return None, None, None, None
        return _logprobs_grad(logits, tokens, stats, entropy, dlogp, dentropy,
                              ctx.temperature), None, None, None


def token_logprobs(logits, tokens, *, temperature=1.0, top=0, return_stats=False):
    """Log-probabilities of given tokens with the entropy of their distributions:
    (logp, entropy), float32 [T] each.

    logits [T, V] float32, bfloat16 or float16 (-inf: a symbol that is not allowed there);
    tokens int32 or int64 [T]. With z = logits / temperature, logp = z[token] - logsumexp z
    and entropy = -sum p log p. top (up to 64 and V): (logp, entropy, top_logp [T, top],
    top_tokens int64 [T, top]), the largest log-probabilities in falling order, the lower
    token first among equals. return_stats adds, at the end, the float32 [T, 2] that
    token_logprobs_grad takes.

    A row whose logits are all -inf has logp -inf, entropy 0 and the alternatives 0, 1, ..
    at -inf; one with NaN or +inf gives NaN, a NaN coming before every number among its
    alternatives; a token outside the vocabulary gives logp NaN.
    Gradients of logp and entropy go to the logits; the alternatives carry none. Sums are
    held in float32; a row of nearly all weight on one symbol keeps the precision of
    the little that is left."""
    _no_tangents(logits)
    tokens, temperature = _check_logits(logits, tokens, temperature)
    top = int(top)
    if not 0 <= top <= min(SEQ_MAX_TOP, logits.shape[1]):
        raise ValueError(f"top must be from 0 to {min(SEQ_MAX_TOP, logits.shape[1])}, not {top}")
    if torch.is_grad_enabled() and logits.requires_grad:
        logp, entropy, top_logp, top_ids, stats = _LogprobsFn.apply(logits, tokens, temperature,
                                                                    top)
    else:
        logp, entropy, top_logp, top_ids, stats = _logprobs(logits, tokens, temperature, top,
                                                            return_stats)
    out = (logp, entropy, top_logp, top_ids) if top else (logp, entropy)
    return out + (stats,) if return_stats else out


def _logprobs_grad(logits, tokens, stats, entropy, dlogp, dentropy, temperature):
    T, V = logits.shape
    dlogits = torch.empty((T, V), dtype=logits.dtype, device=logits.device)
    if T:
        logits = _rows(logits)
        dlogp = None if dlogp is None else dlogp.contiguous()
        dentropy = None if dentropy is None else dentropy.contiguous()
        _run(load_library().seq_logprobs_grad, "seq_logprobs_grad", logits.get_device(),
             _pack_logprobs_grad(_SIZE_LOGPROBS_GRAD, _DTYPES[logits.dtype],
                                 tokens.dtype is torch.int64, 0, T, V, logits.stride(0), V,
                                 temperature, 0, logits.data_ptr(), tokens.data_ptr(),
                                 stats.data_ptr(), entropy.data_ptr(), _ptr(dlogp),
                                 _ptr(dentropy), dlogits.data_ptr()))
    return dlogits


def token_logprobs_grad(logits, tokens, stats, entropy, dlogp=None, dentropy=None, *,
                        temperature=1.0):
    """Gradient [T, V] of the logits, in their type, for the gradients `dlogp` and
    `dentropy` (float32 [T], None: 0) of token_logprobs' results; stats and entropy are
    what it gave. A token whose dlogp and dentropy are 0 is not read and gets 0; a logp of
    -inf gives no gradient. The result is no part of a graph."""
    _no_tangents(logits, dlogp, dentropy)
    tokens, temperature = _check_logits(logits, tokens, temperature)
    T, dev = logits.shape[0], logits.device
    _need(stats, "stats", (torch.float32,), 2, dev)
    if stats.shape != (T, 2):
        raise ValueError(f"stats must be [{T}, 2], not {list(stats.shape)}")
    entropy = _vector(entropy, "entropy", (torch.float32,), T, dev)
    if dlogp is not None:
        _vector(dlogp, "dlogp", (torch.float32,), T, dev)
    if dentropy is not None:
        _vector(dentropy, "dentropy", (torch.float32,), T, dev)
    return _logprobs_grad(logits, tokens, stats.contiguous(), entropy, dlogp, dentropy,
                          temperature)
