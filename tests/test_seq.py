"""Sequence operators without a GPU: the ABI's layout, the position table and
the refusals of the Python entry points and of the library."""
from __future__ import annotations

import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

from cusr_amd.kernel import seq_ops as ops
from cusr_amd.kernel.co_inproc import CO_ERR_BOUNDS, CO_ERR_DATA, CO_ERR_NULLARG, CO_OK

REPO = Path(__file__).resolve().parents[1]


def test_structs_match_the_header(tmp_path):
    names = ("SeqAttention", "SeqAttentionGrad", "SeqRotary", "SeqPolicyLoss")
    lines = []
    for n in names:
        lines.append(f'printf("{n} %zu\\n", sizeof({n}));')
        lines += [f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));'
                  for f, _ in getattr(ops, n)._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "cusr_seq.h"\nint main(void){'
                   + "".join(lines) + "return 0;}")
    subprocess.run(["gcc", f"-I{REPO / 'include'}", str(src), "-o", str(tmp_path / "layout")],
                   check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True)
    got = dict(l.split() for l in out.stdout.splitlines())
    for n in names:
        t = getattr(ops, n)
        assert int(got[n]) == ctypes.sizeof(t)
        for f, _ in t._fields_:
            assert int(got[f"{n}.{f}"]) == getattr(t, f).offset, (n, f)


def test_table():
    t = ops.rotary_table(8, 4096, base=100.0, device="cpu").double()
    p, i = 4095, 2
    a = p * 100.0 ** (-2 * i / 8)
    assert abs(float(t[p, i, 0]) - math.cos(a)) < 1e-7 and abs(float(t[p, i, 1]) - math.sin(a)) < 1e-7
    lin = ops.rotary_table(8, 64, scaling="linear", factor=2.0, device="cpu")
    assert torch.equal(lin[::2], ops.rotary_table(8, 32, device="cpu"))
    base = ops.rotary_table(8, 64, scaling="base", factor=4.0, device="cpu").double()
    slow = 4 * 10000.0 ** (6 / 8)        # the slowest pair turns four times slower
    assert abs(float(base[63, 3, 1]) - math.sin(63 / slow)) < 1e-7
    assert abs(float(base[63, 0, 0]) - math.cos(63.0)) < 1e-7
    parts = ops.rotary_table(64, 300, scaling="parts", factor=4.0, original=256, device="cpu")
    m = 0.1 * math.log(4.0) + 1.0
    f0, f31 = 1.0, 10000.0 ** (-62 / 64)     # 41 turns over 256 positions, and far below one
    assert abs(float(parts[7, 0, 0]) - m * math.cos(7 * f0)) < 1e-6
    assert abs(float(parts[299, 31, 1]) - m * math.sin(299 * f31 / 4)) < 1e-6
    assert ops.rotary_table(0, 5, device="cpu").shape == (5, 0, 2)


@pytest.mark.parametrize("kw", [dict(rot=3), dict(rot=-2), dict(positions=-1), dict(base=0.0),
                                dict(scaling="other"), dict(factor=0.0),
                                dict(scaling="parts", factor=2.0),
                                dict(scaling="parts", factor=0.5, original=10)])
def test_table_refusals(kw):
    with pytest.raises(ValueError):
        ops.rotary_table(**{**dict(rot=4, positions=8, device="cpu"), **kw})


class _Gpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: refusals come before any use."""
    is_cuda = True


def gpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Gpu)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32).as_subclass(_Gpu)


def test_attention_refusals():
    q, k, c = gpu(4, 4, 64), gpu(4, 2, 64), i32(0, 4)
    bad = [
        (TypeError, dict(q=[1])),
        (ValueError, dict(q=torch.zeros(4, 4, 64, dtype=torch.bfloat16))),     # not on the GPU
        (ValueError, dict(q=gpu(4, 4, 64, dtype=torch.float32))),
        (ValueError, dict(k=gpu(4, 2, 64, dtype=torch.float16))),
        (ValueError, dict(q=gpu(4, 256))),
        (ValueError, dict(k=gpu(4, 3, 64), v=gpu(4, 3, 64))),                  # 4 over 3 heads
        (ValueError, dict(k=gpu(4, 0, 64), v=gpu(4, 0, 64))),
        (ValueError, dict(v=gpu(5, 2, 64))),
        (ValueError, dict(k=gpu(4, 2, 32), v=gpu(4, 2, 32))),
        (ValueError, dict(q=gpu(4, 4, 136), k=gpu(4, 2, 136), v=gpu(4, 2, 136))),
        (ValueError, dict(q=gpu(4, 4, 20), k=gpu(4, 2, 20), v=gpu(4, 2, 20))),
        (ValueError, dict(cu_q=gpu(2, dtype=torch.int64))),
        (ValueError, dict(cu_q=i32())),
        (ValueError, dict(cu_k=i32(0, 2, 4))),
        (ValueError, dict(k_lens=i32(1, 2))),
        (ValueError, dict(scale=float("inf"))),
    ]
    for err, kw in bad:
        with pytest.raises(err):
            ops.attention(**{**dict(q=q, k=k, v=k, cu_q=c), **kw})
    o, lse = gpu(4, 4, 64), gpu(4, 4, dtype=torch.float32)
    for kw in (dict(do=gpu(4, 4, 32)), dict(o=gpu(3, 4, 64)),
               dict(lse=gpu(4, 4)), dict(lse=gpu(4, 5, dtype=torch.float32))):
        with pytest.raises(ValueError):
            ops.attention_grad(**{**dict(do=o, q=q, k=k, v=k, o=o, lse=lse, cu_q=c), **kw})


def test_rotary_refusals():
    f = torch.float32
    good = dict(q=gpu(4, 2, 16), k=gpu(4, 1, 16), positions=i32(0, 1, 2, 3),
                table=gpu(9, 8, 2, dtype=f))
    for kw in (dict(q=gpu(4, 2, 16, dtype=torch.float64)), dict(k=gpu(3, 1, 16)),
               dict(k=gpu(4, 1, 8)), dict(k=gpu(4, 1, 16, dtype=f)), dict(positions=i32(0)),
               dict(positions=gpu(4, dtype=f)), dict(table=gpu(9, 9, 2, dtype=f)),
               dict(table=gpu(9, 8, 3, dtype=f)), dict(table=gpu(9, 8, 2))):
        with pytest.raises(ValueError):
            ops.rotary(**{**good, **kw})
    with pytest.raises(ValueError):
        ops.rotary(**{**good, "q": gpu(4, 2, 16).requires_grad_()}, inplace=True)


def test_policy_refusals():
    f, x = torch.float32, gpu(4, 10)
    good = dict(logits=x, actions=gpu(4, dtype=torch.int64), logp_old=gpu(4, dtype=f),
                advantages=gpu(4, dtype=f))
    for kw in (dict(logits=gpu(4, 0)), dict(logits=gpu(4, 10, dtype=torch.float64)),
               dict(actions=gpu(4, dtype=f)), dict(actions=gpu(5, dtype=torch.int64)),
               dict(logp_old=gpu(4)), dict(advantages=gpu(3, dtype=f)),
               dict(logp_ref=gpu(5, dtype=f)), dict(weights=gpu(4, 1, dtype=f)),
               dict(clip=(-0.1, 0.2)), dict(clip=(0.1, float("nan"))), dict(temperature=0.0),
               dict(temperature=float("inf")), dict(kl_coef=float("nan"))):
        for fn in (ops.policy_loss, ops.policy_loss_grad):
            with pytest.raises(ValueError):
                fn(**{**good, **kw})


def test_library_refusals():
    """The C entry points refuse before any launch (no GPU is needed)."""
    lib = ops.load_library()
    ref = ctypes.addressof

    def attn(**kw):
        a = ops.SeqAttention(ctypes.sizeof(ops.SeqAttention), 1, 1, 4, 2, 64, 4, 4)
        for n in ("q", "k", "v", "o", "cu_q", "cu_k", "lse", "workspace"):
            setattr(a, n, 4096)
        for n in ("q_row", "k_row", "v_row", "o_row"):
            setattr(a, n, 256)
        a.workspace_bytes, a.scale = 1 << 20, 0.125
        for n, x in kw.items():
            setattr(a, n, x)
        return a

    for kw, want in ((dict(struct_size=8), CO_ERR_NULLARG), (dict(tq=-1), CO_ERR_NULLARG),
                     (dict(q=None), CO_ERR_NULLARG), (dict(cu_k=None), CO_ERR_NULLARG),
                     (dict(d=20), CO_ERR_BOUNDS), (dict(d=136), CO_ERR_BOUNDS),
                     (dict(hq=5), CO_ERR_BOUNDS), (dict(tq=1 << 40), CO_ERR_BOUNDS),
                     (dict(tk=1 << 40), CO_ERR_BOUNDS), (dict(dtype=0), CO_ERR_DATA),
                     (dict(q=4104), CO_ERR_DATA), (dict(k_row=4), CO_ERR_DATA)):
        a = attn(**kw)
        assert lib.seq_attention(ref(a), None) == want, kw
        g = ops.SeqAttentionGrad(ctypes.sizeof(ops.SeqAttentionGrad), 0, *[8] * 8, *[4096] * 4)
        assert lib.seq_attention_grad(ref(a), ref(g), None) == want, kw
    assert lib.seq_attention(None, None) == CO_ERR_NULLARG
    a = attn()
    for kw, want in ((dict(struct_size=1), CO_ERR_NULLARG), (dict(d_o=None), CO_ERR_NULLARG),
                     (dict(dk=None), CO_ERR_NULLARG), (dict(dq=4104), CO_ERR_DATA),
                     (dict(dv_row=12), CO_ERR_DATA)):
        g = ops.SeqAttentionGrad(ctypes.sizeof(ops.SeqAttentionGrad), 0, *[8] * 8, *[4096] * 4)
        for n, x in kw.items():
            setattr(g, n, x)
        assert lib.seq_attention_grad(ref(a), ref(g), None) == want, kw
    g = ops.SeqAttentionGrad(ctypes.sizeof(ops.SeqAttentionGrad), 0, *[8] * 8, *[4096] * 4)
    assert lib.seq_attention_grad(ref(attn(workspace_bytes=3)), ref(g), None) == CO_ERR_DATA
    assert lib.seq_attention_workspace(ref(attn(d=20))) < 0
    assert lib.seq_attention(ref(attn(tq=0)), None) == CO_OK

    def rot(**kw):
        r = ops.SeqRotary(ctypes.sizeof(ops.SeqRotary), 1, 2, 1, 16, 8, 0, 0, 4, 10)
        for n in ("q", "k", "q_out", "k_out", "positions", "table"):
            setattr(r, n, 4096)
        for n, x in kw.items():
            setattr(r, n, x)
        return r

    for kw, want in ((dict(struct_size=0), CO_ERR_NULLARG), (dict(tokens=-1), CO_ERR_NULLARG),
                     (dict(k_out=None), CO_ERR_NULLARG), (dict(positions=None), CO_ERR_NULLARG),
                     (dict(rot=17), CO_ERR_BOUNDS), (dict(rot=18), CO_ERR_BOUNDS),
                     (dict(tokens=1 << 40), CO_ERR_BOUNDS), (dict(dtype=3), CO_ERR_DATA)):
        r = rot(**kw)
        assert lib.seq_rotary(ref(r), None) == want, kw
    assert lib.seq_rotary(ref(rot(tokens=0)), None) == CO_OK

    def pol(**kw):
        p = ops.SeqPolicyLoss(ctypes.sizeof(ops.SeqPolicyLoss), 1, 4, 10, 10, 10, 0.2, 0.2, 0.0,
                              1.0)
        for n in ("logits", "actions", "logp_old", "advantages", "weights", "loss", "logp",
                  "workspace"):
            setattr(p, n, 4096)
        p.workspace_bytes = 1 << 20
        for n, x in kw.items():
            setattr(p, n, x)
        return p

    for kw, want in ((dict(struct_size=0), CO_ERR_NULLARG), (dict(vocab=0), CO_ERR_NULLARG),
                     (dict(loss=None), CO_ERR_NULLARG), (dict(weights=None), CO_ERR_NULLARG),
                     (dict(tokens=1 << 40), CO_ERR_BOUNDS), (dict(dtype=3), CO_ERR_DATA),
                     (dict(temperature=0.0), CO_ERR_DATA),
                     (dict(workspace_bytes=1), CO_ERR_DATA)):
        p = pol(**kw)
        assert lib.seq_policy_loss(ref(p), None) == want, kw
