"""Sequence operators of a learned proposer of expressions (include/cusr_seq.h).

A pop.bin population is M prefix programs packed end to end: M token sequences.
A causal model over them proposes expressions, the constant fitter returns
their losses, and a clipped policy gradient trains the model on those. These
are that model's operators on the GPU; the reference has no counterpart.

  attention, attention_grad      causal attention over packed sequences with
                                 grouped heads; single tokens over a cache
  rotary_table, rotary           rotary positions of q and k in one launch
  policy_loss, policy_loss_grad  clipped policy loss with a KL term

Tensors are torch CUDA tensors; the work is queued on the current stream of
their device and the call returns at once. attention, rotary and policy_loss
take part in autograd when an input requires a gradient; there are no
forward-mode derivatives, and dual tensors are refused. Arguments are checked
before anything is launched (TypeError, ValueError); a refusal of the library
raises COError. Import torch before the library is loaded, as for
co_data_upload_device. There is no CPU path.
"""
from __future__ import annotations

import ctypes
import math
import struct
import threading

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from cusr_amd.kernel.co_inproc import CO_OK, COError, _HERE

SEQ_MAX_HEAD = 128
_LEAST, _MOST = 1e-30, 1e30          # scale and temperature
_FLOAT32 = float(np.finfo(np.float32).max)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_P, _I32, _I64, _F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float

# every extern "C" symbol of include/cusr_seq.h
EXPORTED = ("seq_attention", "seq_attention_workspace", "seq_attention_grad",
            "seq_attention_grad_workspace", "seq_rotary", "seq_policy_loss",
            "seq_policy_loss_workspace")


class SeqAttention(ctypes.Structure):
    """cusr_seq.h SeqAttention."""
    _fields_ = [("struct_size", _I32), ("dtype", _I32), ("n_seq", _I32), ("hq", _I32),
                ("hkv", _I32), ("d", _I32), ("tq", _I64), ("tk", _I64),
                ("q_row", _I64), ("q_head", _I64), ("k_row", _I64), ("k_head", _I64),
                ("v_row", _I64), ("v_head", _I64), ("o_row", _I64), ("o_head", _I64),
                ("scale", _F), ("reserved", _I32), ("q", _P), ("k", _P), ("v", _P), ("o", _P),
                ("lse", _P), ("o_low", _P), ("cu_q", _P), ("cu_k", _P), ("k_lens", _P), ("workspace", _P),
                ("workspace_bytes", _I64)]


class SeqAttentionGrad(ctypes.Structure):
    """cusr_seq.h SeqAttentionGrad."""
    _fields_ = [("struct_size", _I32), ("reserved", _I32), ("do_row", _I64), ("do_head", _I64),
                ("dq_row", _I64), ("dq_head", _I64), ("dk_row", _I64), ("dk_head", _I64),
                ("dv_row", _I64), ("dv_head", _I64), ("d_o", _P), ("dq", _P), ("dk", _P),
                ("dv", _P)]


class SeqRotary(ctypes.Structure):
    """cusr_seq.h SeqRotary."""
    _fields_ = [("struct_size", _I32), ("dtype", _I32), ("hq", _I32), ("hkv", _I32), ("d", _I32),
                ("rot", _I32), ("interleaved", _I32), ("inverse", _I32), ("tokens", _I64),
                ("table_len", _I64), ("q_row", _I64), ("q_head", _I64), ("k_row", _I64),
                ("k_head", _I64), ("qo_row", _I64), ("qo_head", _I64), ("ko_row", _I64),
                ("ko_head", _I64), ("q", _P), ("k", _P), ("q_out", _P), ("k_out", _P),
                ("positions", _P), ("table", _P), ("positions_64", _I32), ("reserved", _I32)]


class SeqPolicyLoss(ctypes.Structure):
    """cusr_seq.h SeqPolicyLoss."""
    _fields_ = [("struct_size", _I32), ("dtype", _I32), ("tokens", _I64), ("vocab", _I64),
                ("row", _I64), ("drow", _I64), ("clip_lo", _F), ("clip_hi", _F),
                ("kl_coef", _F), ("temperature", _F), ("logits", _P), ("actions", _P),
                ("logp_old", _P), ("logp_ref", _P), ("advantages", _P), ("weights", _P),
                ("dloss", _P), ("loss", _P), ("logp", _P), ("dlogits", _P), ("workspace", _P),
                ("workspace_bytes", _I64)]


def _packer(structure):
    """A ctypes structure's layout as a struct.Struct: a call packs its
    arguments in one step, several times faster than filling the structure."""
    codes = {_I32: "i", _I64: "q", _F: "f", _P: "P"}
    p = struct.Struct("".join(codes[t] for _, t in structure._fields_))
    assert p.size == ctypes.sizeof(structure)
    return p.pack, p.size


_pack_attention, _SIZE_ATTENTION = _packer(SeqAttention)
_pack_attention_grad, _SIZE_ATTENTION_GRAD = _packer(SeqAttentionGrad)
_pack_rotary, _SIZE_ROTARY = _packer(SeqRotary)
_pack_policy, _SIZE_POLICY = _packer(SeqPolicyLoss)

_lib = None
_lib_lock = threading.Lock()


def lib_path():
    """libcusr_seq.so next to this module (cusr_amd/build.py output)."""
    return _HERE / "libcusr_seq.so"


def load_library() -> ctypes.CDLL:
    """Bind libcusr_seq.so once per process; raises when it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lib_lock:
        if _lib is None:
            path = lib_path()
            if not path.exists():
                raise FileNotFoundError(f"{path} not built: run python -m cusr_amd.build")
            lib = ctypes.CDLL(str(path))
            for name in EXPORTED:
                fn = getattr(lib, name)
                fn.restype = ctypes.c_int64 if name.endswith("workspace") else ctypes.c_int
            for name in ("seq_attention", "seq_rotary", "seq_policy_loss"):
                getattr(lib, name).argtypes = [_P, _P]
            lib.seq_attention_grad.argtypes = [_P, _P, _P]
            for name in ("seq_attention", "seq_attention_grad", "seq_policy_loss"):
                getattr(lib, name + "_workspace").argtypes = [_P]
            _lib = lib
    return _lib


def _run(fn, where, device, *structs):
    """Call an entry point with packed structures on the device's current
    stream (torch.cuda.current_stream without its wrapper object)."""
    if device == torch.cuda.current_device():
        rc = fn(*structs, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*structs, torch._C._cuda_getCurrentRawStream(device))
    if rc != CO_OK:
        raise COError(rc, where)


def _workspace(fn, where, packed, device):
    """(pointer, bytes, owner) of a call's scratch, from torch's allocator on
    the current stream."""
    n = fn(packed)
    if n <= 0:
        if n:
            raise COError(int(-n if n == -2 else n), where)
        return None, 0, None
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    return ws.data_ptr(), n, ws


def _need(x, name, dtypes, dim, device=None):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, not {type(x).__name__}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    if device is not None and x.device != device:
        raise ValueError(f"{name} is on {x.device}, not on {device}")
    if x.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d)[6:] for d in dtypes)}, "
                         f"not {str(x.dtype)[6:]}")
    if dim is not None and x.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions, not {x.dim()}")
    return x


def _no_tangents(*tensors):
    """Forward-mode derivatives are not formed: a dual tensor would lose its
    tangent without a word. One comparison outside a dual level."""
    if forward_ad._current_level < 0:
        return
    for x in tensors:
        if isinstance(x, torch.Tensor) and forward_ad.unpack_dual(x).tangent is not None:
            raise ValueError("the sequence operators have no forward-mode derivatives")


def _no_gradient(**tensors):
    """Refuses tensors that would get no gradient although they ask for one."""
    if torch.is_grad_enabled():
        for name, x in tensors.items():
            if x is not None and x.requires_grad:
                raise ValueError(f"{name} gets no gradient: pass {name}.detach()")


def _ptr(x):
    return 0 if x is None else x.data_ptr()


def _heads16(x):
    """x as the kernels read it: the last dimension contiguous, rows and heads
    on 16-byte boundaries; another layout is copied once."""
    s0, s1, s2 = x.stride()
    if s2 == 1 and not (s0 | s1) & 7 and not x.data_ptr() & 15:
        return x
    if x.numel():
        return x.contiguous() if x.shape[2] % 8 == 0 and not x.is_contiguous() else x.clone(
            memory_format=torch.contiguous_format)
    return x.new_empty(x.shape)          # nothing to copy, and strides that fit


def _plain_attention(q, k, v, cu_q, cu_k, k_lens):
    """Whether the common checks hold; _check_attention says which does not."""
    try:
        _, hq, d = q.shape
        _, hkv, dk = k.shape
        n, dev, dt = cu_q.shape[0], q.get_device(), q.dtype
        return (dev >= 0 and q.is_cuda and dt in _HALF and k.dtype is dt and v.dtype is dt
                and k.shape == v.shape and d == dk and hkv > 0 and hq > 0 and hq % hkv == 0
                and d & 7 == 0 and 8 <= d <= SEQ_MAX_HEAD and k.get_device() == dev
                and v.get_device() == dev and cu_q.dtype is torch.int32 and cu_q.dim() == 1
                and n > 0 and cu_q.get_device() == dev
                and (cu_k is None or cu_k is cu_q
                     or (cu_k.dtype is torch.int32 and cu_k.shape == cu_q.shape
                         and cu_k.get_device() == dev))
                and (k_lens is None
                     or (k_lens.dtype is torch.int32 and k_lens.dim() == 1
                         and k_lens.shape[0] == n - 1 and k_lens.get_device() == dev)))
    except (AttributeError, ValueError, TypeError, IndexError):
        return False


# ------------------------------------------------------------------ attention

_HALF = (torch.bfloat16, torch.float16)


def _check_attention(q, k, v, cu_q, cu_k, k_lens, scale):
    _no_tangents(q, k, v)
    if _plain_attention(q, k, v, cu_q, cu_k, k_lens) and (scale is None
                                                             or _LEAST <= scale <= _MOST):
        return
    _need(q, "q", _HALF, 3)
    dev = q.device
    _need(k, "k", (q.dtype,), 3, dev)
    _need(v, "v", (q.dtype,), 3, dev)
    hq, d = q.shape[1], q.shape[2]
    hkv = k.shape[1]
    if k.shape != v.shape or k.shape[2] != d:
        raise ValueError(f"k and v must be [rows, heads, {d}] and alike; got {tuple(k.shape)} "
                         f"and {tuple(v.shape)}")
    if hkv < 1 or hq < 1 or hq % hkv:
        raise ValueError(f"query heads ({hq}) must be a multiple of key heads ({hkv})")
    if d < 8 or d % 8 or d > SEQ_MAX_HEAD:
        raise ValueError(f"head size must be a multiple of 8 up to {SEQ_MAX_HEAD}, not {d}")
    _need(cu_q, "cu_q", (torch.int32,), 1, dev)
    if cu_k is not None:
        _need(cu_k, "cu_k", (torch.int32,), 1, dev)
        if cu_k.shape != cu_q.shape:
            raise ValueError("cu_q and cu_k must have one entry per sequence and one more")
    if cu_q.numel() < 1:
        raise ValueError("cu_q must have one entry per sequence and one more")
    if k_lens is not None:
        _need(k_lens, "k_lens", (torch.int32,), 1, dev)
        if k_lens.numel() != cu_q.numel() - 1:
            raise ValueError("k_lens must have one entry per sequence")
    if scale is not None and not _LEAST <= scale <= _MOST:
        raise ValueError(f"scale must be from {_LEAST} to {_MOST}, not {scale}")


def _attention_args(q, k, v, o, lse, low, cu_q, cu_k, k_lens, scale):
    qs, ks, vs, os_ = q.stride(), k.stride(), v.stride(), o.stride()
    tq, hq, d = q.shape
    return (_SIZE_ATTENTION, _DTYPES[q.dtype], cu_q.shape[0] - 1, hq, k.shape[1], d, tq,
            k.shape[0], qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os_[0], os_[1], scale, 0,
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _ptr(lse), _ptr(low),
            cu_q.data_ptr(), cu_k.data_ptr(), _ptr(k_lens))


def _attention(q, k, v, cu_q, cu_k, k_lens, scale, return_lse):
    q, k, v = _heads16(q), _heads16(k), _heads16(v)
    cu_q = cu_q.contiguous()
    cu_k = cu_q if cu_k is None else cu_k.contiguous()
    k_lens = None if k_lens is None else k_lens.contiguous()
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device) \
        if return_lse else None
    low = None
    if return_lse:
        # Where the gradient takes sum(o * do) from o it gets the part of o that o's
        # type rounds away. The kernels know the rows: those that form the sum anew
        # leave theirs unwritten.
        low = lse.o_low = torch.empty_like(o)
    if q.shape[0]:
        lib, dev = load_library(), q.get_device()
        args = _attention_args(q, k, v, o, lse, low, cu_q, cu_k, k_lens, scale)
        packed = _pack_attention(*args, 0, 0)
        ptr, n, ws = _workspace(lib.seq_attention_workspace, "seq_attention", packed, q.device)
        if n:
            packed = _pack_attention(*args, ptr, n)
        _run(lib.seq_attention, "seq_attention", dev, packed)
        del ws
    return o, lse


def attention_grad(do, q, k, v, o, lse, cu_q, cu_k=None, *, k_lens=None, scale=None):
    """(dq, dk, dv) of attention for the gradient `do` of its output; o and
    lse are what attention(..., return_lse=True) gave. The same call gives the
    same bits. lse comes with an attribute o_low, as large as o: what o's type
    rounded away of it, which the gradient of long sequences needs. For a copy
    of lse without it the forward pass runs again."""
    _check_attention(q, k, v, cu_q, cu_k, k_lens, scale)
    _no_tangents(do)
    _need(do, "do", (q.dtype,), 3, q.device)
    _need(o, "o", (q.dtype,), 3, q.device)
    _need(lse, "lse", (torch.float32,), 2, q.device)
    if do.shape != q.shape or o.shape != q.shape or lse.shape != (q.shape[1], q.shape[0]):
        raise ValueError("do and o must be like q, and lse [heads, rows]")
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale)
    low = getattr(lse, "o_low", None)
    if low is not None and (low.shape != q.shape or low.dtype != q.dtype
                            or low.device != q.device or not low.is_contiguous()):
        raise ValueError("lse.o_low does not belong to this call")
    q, k, v, o, do = (_heads16(x) for x in (q, k, v, o, do))
    cu_q, lse = cu_q.contiguous(), lse.contiguous()
    cu_k = cu_q if cu_k is None else cu_k.contiguous()
    k_lens = None if k_lens is None else k_lens.contiguous()
    if low is None and q.shape[0] and k.shape[0]:
        low = _attention(q, k, v, cu_q, cu_k, k_lens, scale, True)[1].o_low
    dq, dk, dv = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k, v))
    if q.shape[0] == 0 or k.shape[0] == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    lib = load_library()
    args = _attention_args(q, k, v, o, lse, low, cu_q, cu_k, k_lens, scale)
    ptr, n, ws = _workspace(lib.seq_attention_grad_workspace, "seq_attention_grad",
                            _pack_attention(*args, 0, 0), q.device)
    packed = _pack_attention(*args, ptr or 0, n)
    g = _pack_attention_grad(_SIZE_ATTENTION_GRAD, 0, *do.stride()[:2], *dq.stride()[:2],
                             *dk.stride()[:2], *dv.stride()[:2], do.data_ptr(), dq.data_ptr(),
                             dk.data_ptr(), dv.data_ptr())
    _run(lib.seq_attention_grad, "seq_attention_grad", q.get_device(), packed, g)
    del ws
    return dq, dk, dv


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, k_lens, scale):
        o, lse = _attention(q, k, v, cu_q, cu_k, k_lens, scale, True)
        ctx.save_for_backward(q, k, v, o, lse, cu_q, cu_k, k_lens, getattr(lse, "o_low", None))
        ctx.scale = scale
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, do, _):
        q, k, v, o, lse, cu_q, cu_k, k_lens, low = ctx.saved_tensors
        if low is not None:
            lse = lse.detach()
            lse.o_low = low
        return (*attention_grad(do, q, k, v, o, lse, cu_q, cu_k, k_lens=k_lens,
                                scale=ctx.scale), None, None, None, None)


def attention(q, k, v, cu_q, cu_k=None, *, k_lens=None, scale=None, return_lse=False):
    """Causal attention over packed sequences.

    q [Tq, Hq, D], k and v [Tk, Hkv, D], bfloat16 or float16, D a multiple of 8
    up to 128, Hq a multiple of Hkv (query head h reads key head h * Hkv // Hq).
    cu_q int32 [B + 1]: sequence b's queries are rows cu_q[b]:cu_q[b + 1]
    (cu_q[0] is 0). cu_k (default cu_q) the same for its keys; with k_lens
    int32 [B] only the first k_lens[b] rows of a segment are keys (a cache with
    room to spare). Queries are the last of their sequence: query i of lq sees
    keys 0 .. i + lk - lq, so a newest token alone is a segment of one query.
    A query that sees no key gives 0. scale defaults to D ** -0.5.

    Returns o like q, or (o, lse) with return_lse: lse fp32 [Hq, Tq], -inf
    where no key is seen; it carries no gradient. A key or value that is not
    finite reaches only queries that see it. Probabilities are rounded to the tensors' type for the product with v;
    sums and statistics are held in fp32."""
    _check_attention(q, k, v, cu_q, cu_k, k_lens, scale)
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        o, lse = _AttentionFn.apply(q, k, v, cu_q, cu_q if cu_k is None else cu_k, k_lens, scale)
    else:
        o, lse = _attention(q, k, v, cu_q, cu_k, k_lens, scale, return_lse)
    return (o, lse) if return_lse else o


# --------------------------------------------------------------------- rotary

SCALINGS = (None, "linear", "base", "parts")


def rotary_table(rot, positions, *, base=10000.0, scaling=None, factor=1.0, original=0,
                 device="cuda"):
    """Table [positions, rot/2, 2] fp32 of (cos, sin) for rotary: angle of
    position p and pair i is p * base ** (-2i/rot), formed in float64.

    scaling, for contexts `factor` times the `original` length:
      "linear"  positions divided by factor
      "base"    base * factor ** (rot / (rot - 2)): the slowest pair turns
                factor times slower, the fastest as before
      "parts"   pairs that turn 32 times or more over `original` positions keep
                their frequency, those that turn once or less are divided by
                factor, linearly in between; cos and sin are multiplied by
                0.1 ln(factor) + 1"""
    rot, positions = int(rot), int(positions)
    if rot < 0 or rot % 2 or positions < 0:
        raise ValueError(f"rot must be even and sizes not negative; got {rot}, {positions}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, not {scaling!r}")
    if not (base > 0 and factor > 0 and math.isfinite(base) and math.isfinite(factor)):
        raise ValueError("base and factor must be positive")
    if scaling == "parts" and (original < 1 or factor < 1):
        raise ValueError('scaling "parts" needs the original length and a factor of at least 1')
    m = 1.0
    if scaling == "base" and rot > 2:
        base = base * factor ** (rot / (rot - 2.0))
    f = np.float64(base) ** (-np.arange(0, rot, 2, dtype=np.float64) / max(rot, 1))
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        turns = original * f / (2.0 * np.pi)
        keep = np.clip((turns - 1.0) / 31.0, 0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
        m = 0.1 * math.log(factor) + 1.0
    f = torch.from_numpy(np.ascontiguousarray(f)).to(device)
    a = torch.arange(positions, dtype=torch.float64, device=f.device)[:, None] * f
    return (torch.stack([a.cos(), a.sin()], dim=-1) * m).float().contiguous()


def _rotary(q, k, positions, table, interleaved, inverse, q_out=None, k_out=None):
    tokens, hq, d = q.shape
    qs = q.stride()
    if qs[2] != 1 and d > 1:
        q = q.contiguous()
        qs = q.stride()
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    hkv, ks, kos = 0, (0, 0), (0, 0)
    if k is not None:
        hkv, ks = k.shape[1], k.stride()
        if ks[2] != 1 and d > 1:
            k = k.contiguous()
            ks = k.stride()
        if k_out is None:
            k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        kos = k_out.stride()
    positions, table = positions.contiguous(), table.contiguous()
    if tokens:
        qos = q_out.stride()
        r = _pack_rotary(_SIZE_ROTARY, _DTYPES[q.dtype], hq, hkv, d, 2 * table.shape[1],
                         bool(interleaved), bool(inverse), tokens, table.shape[0], qs[0], qs[1],
                         ks[0], ks[1], qos[0], qos[1], kos[0], kos[1], q.data_ptr(), _ptr(k),
                         q_out.data_ptr(), _ptr(k_out), positions.data_ptr(), table.data_ptr(),
                         positions.dtype is torch.int64, 0)
        _run(load_library().seq_rotary, "seq_rotary", q.get_device(), r)
    return q_out, k_out


def _own_memory(x):
    """Elements that x [T, H, D] spans, heads contiguous, or None when two of its
    places share memory (a broadcast or sliding view)."""
    (T, H, d), (s0, s1, _) = x.shape, x.stride()
    if not x.numel():
        return 0
    row, head = ((T - 1) * s0, (H - 1) * s1)
    if (H == 1 or s1 >= d) and (T == 1 or s0 >= head + d):            # rows outside
        return row + head + d
    if (T == 1 or s0 >= d) and (H == 1 or s1 >= row + d):             # heads outside
        return row + head + d
    return None


def _share_memory(q, k):
    """Whether an element of k is one of q; each is its own memory."""
    (T, hq, d), (q0, q1, _) = q.shape, q.stride()
    (_, hk, _), (k0, k1, _) = k.shape, k.stride()
    gap = (k.data_ptr() - q.data_ptr()) // q.element_size()
    if not (-_own_memory(k) < gap < _own_memory(q)):
        return False
    if T == 1:
        q0 = k0 = max(q0, k0, 1)
    q_row, k_row = (hq - 1) * q1 + d, (hk - 1) * k1 + d
    if q0 == k0 and ((gap >= q_row and gap + k_row <= q0) or (-gap >= k_row and q_row - gap <= q0)):
        return False                                # other columns of the same rows
    if q0 != k0:
        return True                                 # rows of two lengths in one range
    # places of a head of k in one of q, a number of rows apart
    d0 = gap + np.arange(hk)[:, None] * k1 - np.arange(hq)[None] * q1
    rows = np.clip(np.rint(d0 / q0), 1 - T, T - 1).astype(np.int64)
    return bool((np.abs(d0 - rows * q0) < d).any())


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, table, interleaved, inverse):
        ctx.save_for_backward(positions, table)
        ctx.how = (interleaved, inverse)
        q_out, k_out = _rotary(q, k, positions, table, interleaved, inverse)
        return (q_out, k_out) if k is not None else q_out

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        positions, table = ctx.saved_tensors
        interleaved, inverse = ctx.how
        dq, dk = _rotary(grads[0], grads[1] if len(grads) > 1 else None, positions, table,
                         interleaved, not inverse)
        return dq, dk, None, None, None, None


def rotary(q, k, positions, table, *, interleaved=False, inverse=False, inplace=False):
    """Rotary positions of q [T, Hq, D] and k [T, Hkv, D] (or None) in one
    launch; float32, bfloat16 or float16. positions int32 or int64 [T]; table
    from rotary_table. The first rot = 2 * table.shape[1] elements of each head
    turn in pairs (i, i + rot/2), or (2i, 2i + 1) when interleaved; the rest is
    copied. inverse turns by the opposite angles, which is the gradient, and the
    way back unless the table has a magnitude ("parts"). inplace writes into q
    and k, and autograd sees it. A position outside the table gives NaN in its
    token's turned elements. Gradients go to q and k, not to the table. Returns
    (q', k'), or q' alone when k is None."""
    _no_tangents(q, k, table)
    if not _plain_rotary(q, k, positions, table):
        _check_rotary(q, k, positions, table)
    _no_gradient(table=table)
    grad = torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))
    if inplace:
        if grad:
            raise ValueError("inplace takes no part in autograd")
        if q.stride(2) != 1 or (k is not None and k.stride(2) != 1):
            raise ValueError("inplace needs heads that are contiguous")
        if _own_memory(q) is None or (k is not None and (_own_memory(k) is None
                                                         or _share_memory(q, k))):
            raise ValueError("inplace needs memory of its own for every element of q and k")
        out = _rotary(q, k, positions, table, interleaved, inverse, q, k)
        # autograd has to see that they changed: an earlier graph may have saved them
        torch.autograd.graph.increment_version(
            [x for x in (q, k) if x is not None and not x.is_inference()])
    elif grad:
        return _RotaryFn.apply(q, k, positions, table, bool(interleaved), bool(inverse))
    else:
        out = _rotary(q, k, positions, table, interleaved, inverse)
    return out if k is not None else out[0]


def _plain_rotary(q, k, positions, table):
    """Whether the common checks hold; _check_rotary says which does not."""
    try:
        tokens, _, d = q.shape
        n, half, two = table.shape
        dev, dt = q.get_device(), q.dtype
        return (dev >= 0 and q.is_cuda and dt in _DTYPES and two == 2 and 2 * half <= d
                and table.dtype is torch.float32 and table.get_device() == dev
                and positions.dtype in _INTS and positions.dim() == 1
                and positions.shape[0] == tokens and positions.get_device() == dev
                and (k is None or (k.dtype is dt and k.dim() == 3 and k.shape[0] == tokens
                                   and k.shape[2] == d and k.get_device() == dev)))
    except (AttributeError, ValueError, TypeError, IndexError):
        return False


_INTS = (torch.int32, torch.int64)


def _check_rotary(q, k, positions, table):
    _need(q, "q", tuple(_DTYPES), 3)
    dev = q.device
    if k is not None:
        _need(k, "k", (q.dtype,), 3, dev)
        if k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
            raise ValueError(f"q and k must agree in tokens and head size; got {tuple(q.shape)} "
                             f"and {tuple(k.shape)}")
    _need(positions, "positions", (torch.int32, torch.int64), 1, dev)
    if positions.numel() != q.shape[0]:
        raise ValueError(f"positions must have {q.shape[0]} entries, not {positions.numel()}")
    _need(table, "table", (torch.float32,), 3, dev)
    if table.shape[2] != 2 or 2 * table.shape[1] > q.shape[2]:
        raise ValueError(f"table must be [positions, rot/2, 2] with rot up to the head size "
                         f"{q.shape[2]}; got {tuple(table.shape)}")


# ---------------------------------------------------------------- policy loss

def _plain_policy(logits, actions, given, maybe):
    """Whether the common checks hold; _check_policy says which does not."""
    try:
        T, V = logits.shape
        dev = logits.get_device()
        if not (dev >= 0 and logits.is_cuda and V > 0 and logits.dtype in _DTYPES
                and actions.dtype in _INTS and actions.shape == (T,)
                and actions.get_device() == dev):
            return False
        for x in given + tuple(x for x in maybe if x is not None):
            if x.dtype is not torch.float32 or x.shape != (T,) or x.get_device() != dev:
                return False
        return True
    except (AttributeError, ValueError, TypeError):
        return False


def _check_policy(logits, actions, logp_old, advantages, logp_ref, weights, clip, kl_coef,
                  temperature):
    _no_tangents(logits, logp_old, advantages, logp_ref, weights)
    lo, hi = (float(c) for c in clip)
    if (_plain_policy(logits, actions, (logp_old, advantages), (logp_ref, weights))
            and 0 <= lo <= _FLOAT32 and 0 <= hi <= _FLOAT32 and _LEAST <= temperature <= _MOST
            and abs(kl_coef) <= _FLOAT32):
        return lo, hi
    _need(logits, "logits", tuple(_DTYPES), 2)
    T, V = logits.shape
    dev = logits.device
    if V < 1:
        raise ValueError("logits must have at least one column")
    _need(actions, "actions", (torch.int64, torch.int32), 1, dev)
    named = [("logp_old", logp_old), ("advantages", advantages)]
    named += [(n, x) for n, x in (("logp_ref", logp_ref), ("weights", weights)) if x is not None]
    for name, x in named:
        _need(x, name, (torch.float32,), 1, dev)
    for name, x in named + [("actions", actions)]:
        if x.numel() != T:
            raise ValueError(f"{name} must have {T} entries, not {x.numel()}")
    if not (lo >= 0 and hi >= 0):
        raise ValueError(f"clip must be two widths of at least 0; got {clip}")
    if not _LEAST <= temperature <= _MOST:
        raise ValueError(f"temperature must be from {_LEAST} to {_MOST}, not {temperature}")
    if not abs(kl_coef) <= _FLOAT32:
        raise ValueError("kl_coef must be a finite float32")
    # a width that float32 does not hold is none
    return tuple(x if x <= _FLOAT32 else math.inf for x in (lo, hi))


def _policy(logits, actions, logp_old, advantages, logp_ref, weights, clip, kl_coef, temperature,
            dloss, grad):
    T, V = logits.shape
    if V > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    if actions.dtype is not torch.int64:
        actions = actions.to(torch.int64)
    actions = actions.contiguous()
    logp_old, advantages = logp_old.contiguous(), advantages.contiguous()
    logp_ref = None if logp_ref is None else logp_ref.contiguous()
    weights = torch.full((T,), 1.0 / max(T, 1), device=logits.device) if weights is None \
        else weights.contiguous()
    loss = torch.empty((), dtype=torch.float32, device=logits.device)
    logp = torch.empty(T, dtype=torch.float32, device=logits.device)
    dlogits = torch.empty((T, V), dtype=logits.dtype, device=logits.device) if grad else None
    lib = load_library()
    args = (_SIZE_POLICY, _DTYPES[logits.dtype], T, V, logits.stride(0), V, *clip, kl_coef,
            temperature, logits.data_ptr(), actions.data_ptr(), logp_old.data_ptr(),
            _ptr(logp_ref), advantages.data_ptr(), weights.data_ptr(), _ptr(dloss),
            loss.data_ptr(), logp.data_ptr(), _ptr(dlogits))
    ptr, n, ws = _workspace(lib.seq_policy_loss_workspace, "seq_policy_loss",
                            _pack_policy(*args, 0, 0), logits.device)
    _run(lib.seq_policy_loss, "seq_policy_loss", logits.get_device(),
         _pack_policy(*args, ptr or 0, n))
    del ws
    return loss, logp, dlogits


class _PolicyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, logp_old, advantages, logp_ref, weights, clip, kl_coef,
                temperature):
        ctx.save_for_backward(logits, actions, logp_old, advantages, logp_ref, weights)
        ctx.how = (clip, kl_coef, temperature)
        loss, logp, _ = _policy(logits, actions, logp_old, advantages, logp_ref, weights, clip,
                                kl_coef, temperature, None, False)
        ctx.mark_non_differentiable(logp)
        return loss, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        # one pass over the logits: the sums are formed again, not stored
        dlogits = _policy(*ctx.saved_tensors, *ctx.how, dloss.float().contiguous(), True)[2]
        return (dlogits,) + (None,) * 8


def policy_loss(logits, actions, logp_old, advantages, *, logp_ref=None, weights=None,
                clip=(0.2, 0.2), kl_coef=0.0, temperature=1.0):
    """Clipped policy loss with a KL term: (loss, logp).

    logits [T, V] float32, bfloat16 or float16 (-inf: a symbol that is not
    allowed there); actions [T] the tokens taken; logp_old, advantages and
    logp_ref (or None) float32 [T]; weights float32 [T], 1/T each by default.
    With z = logits / temperature, logp = z[action] - logsumexp z and
    ratio = exp(logp - logp_old), the loss is the weighted sum over tokens of
        -min(ratio A, clip(ratio, 1 - clip[0], 1 + clip[1]) A)
        + kl_coef (exp(logp_ref - logp) - (logp_ref - logp) - 1),
    without the last term when logp_ref is None or kl_coef 0.
    A token of weight 0 is not read: logp 0, gradient 0. An action whose
    logit is -inf has logp -inf and no gradient; one outside the vocabulary
    gives NaN. The gradient goes to the logits alone: logp carries none, and
    other inputs that require one are refused. Sums are held in fp32 or more."""
    lo_hi = _check_policy(logits, actions, logp_old, advantages, logp_ref, weights, clip,
                          kl_coef, temperature)
    _no_gradient(logp_old=logp_old, advantages=advantages, logp_ref=logp_ref, weights=weights)
    args = (logits, actions, logp_old, advantages, logp_ref, weights, lo_hi, kl_coef, temperature)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _PolicyFn.apply(*args)
    return _policy(*args, None, False)[:2]


def policy_loss_grad(logits, actions, logp_old, advantages, *, logp_ref=None, weights=None,
                     clip=(0.2, 0.2), kl_coef=0.0, temperature=1.0):
    """policy_loss and its gradient in one pass: (loss, logp, dlogits), dlogits
    like logits. The results are no part of a graph."""
    lo_hi = _check_policy(logits, actions, logp_old, advantages, logp_ref, weights, clip,
                          kl_coef, temperature)
    return _policy(logits, actions, logp_old, advantages, logp_ref, weights, lo_hi, kl_coef,
                   temperature, None, True)
