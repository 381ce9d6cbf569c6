"""The layers around attention without a GPU: the ABI's layout, the refusals of the Python
entry points and of the library, and the 64-bit references against differences."""
from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

import layer_reference as ref
from cusr_amd.benchmark import popio
from cusr_amd.kernel import seq_layers as ops
from cusr_amd.kernel import seq_ops
from cusr_amd.kernel.co_inproc import CO_ERR_BOUNDS, CO_ERR_DATA, CO_ERR_NULLARG, CO_OK
from test_seq import gpu, i32

REPO = Path(__file__).resolve().parents[1]
F, BF, FP, I8 = torch.float32, torch.bfloat16, torch.float16, torch.int8
STRUCTS = ("SeqEmbedding", "SeqEmbeddingGrad", "SeqNorm", "SeqNormGrad", "SeqInt8Product",
           "SeqLogprobs", "SeqLogprobsGrad")


def test_structs_match_the_header(tmp_path):
    lines = [f'printf("{n} %zu\\n", (size_t){n});' for n in
             ("SEQ_MAX_WIDTH", "SEQ_MAX_INNER", "SEQ_MAX_TOP", "SEQ_MAX_ROWS")]
    for n in STRUCTS:
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
    for n in ("SEQ_MAX_WIDTH", "SEQ_MAX_INNER", "SEQ_MAX_TOP", "SEQ_MAX_ROWS"):
        assert int(got[n]) == getattr(ops, n)
    for n in STRUCTS:
        t = getattr(ops, n)
        assert int(got[n]) == ctypes.sizeof(t)
        for f, _ in t._fields_:
            assert int(got[f"{n}.{f}"]) == getattr(t, f).offset, (n, f)


def refuses(fn, good, *bad, error=ValueError):
    for kw in bad:
        with pytest.raises(error):
            fn(**{**good, **kw})


def test_embedding_refusals():
    good = dict(tokens=i32(0, 1), table=gpu(4, 8))
    refuses(ops.embedding, good, dict(table=[1]), dict(tokens=[0]), error=TypeError)
    refuses(ops.embedding, good, dict(table=torch.zeros(4, 8)), dict(tokens=torch.zeros(2).int()),
            dict(table=gpu(4, 8, dtype=torch.float64)), dict(table=gpu(8)), dict(table=gpu(4, 0)),
            dict(table=gpu(4, 65537)), dict(tokens=gpu(2, dtype=F)), dict(scale=float("nan")),
            dict(tokens=gpu(2, 1, dtype=torch.int64)), dict(scale=1e39), dict(dtype=I8))
    good = dict(dout=gpu(2, 8), tokens=i32(0, 1), rows=4)
    refuses(ops.embedding_grad, good, dict(dout=gpu(3, 8)), dict(dout=gpu(2, 0)), dict(rows=-1),
            dict(rows=1 << 31), dict(tokens=gpu(2, dtype=F)), dict(scale=float("inf")),
            dict(dtype=torch.float64), dict(dout=gpu(2, 8, dtype=torch.int32)))


def test_norm_refusals():
    x = gpu(4, 8)
    good = dict(x=x, gain=gpu(8), residual=gpu(4, 8, dtype=F))
    for fn in (ops.rms_norm, ops.rms_norm_int8):
        refuses(fn, good, dict(x=None), error=TypeError)
        refuses(fn, good, dict(x=gpu(8)), dict(x=torch.zeros(4, 8)), dict(x=gpu(4, 0)),
                dict(x=gpu(4, 8, dtype=I8)), dict(x=gpu(5, 8)), dict(gain=gpu(9)),
                dict(gain=gpu(1, 8)), dict(gain=gpu(8, dtype=torch.float64)),
                dict(residual=gpu(4, 9)), dict(residual=gpu(3, 8)),
                dict(residual=gpu(4, 8, dtype=FP)), dict(eps=-1e-6), dict(eps=float("nan")),
                dict(eps=1e39), dict(x=gpu(4, 8, dtype=F), residual=gpu(4, 8)),
                dict(x=gpu(4, 65537)))
    refuses(ops.rms_norm, good, dict(dtype=I8), dict(dtype="bf16"))
    # the 8-bit operators form no gradient
    for kw in (dict(x=gpu(4, 8).requires_grad_()), dict(gain=gpu(8).requires_grad_()),
               dict(residual=gpu(4, 8).requires_grad_())):
        refuses(ops.rms_norm_int8, good, kw)
    refuses(ops.quantize_rows, dict(x=x), dict(x=gpu(4, 8).requires_grad_()), dict(x=gpu(4, 0)),
            dict(x=gpu(4, 8, dtype=torch.int32)), dict(x=torch.zeros(4, 8)))
    good = dict(dy=gpu(4, 8), h=gpu(4, 8, dtype=F), gain=gpu(8), dh=gpu(4, 8, dtype=F))
    refuses(ops.rms_norm_grad, good, dict(dy=gpu(3, 8)), dict(dy=gpu(4, 9)), dict(dh=gpu(4, 8)),
            dict(dh=gpu(5, 8, dtype=F)), dict(gain=gpu(7)), dict(h=gpu(8, dtype=F)),
            dict(eps=-1.0), dict(x_dtype=I8), dict(dy=torch.zeros(4, 8)))


def test_product_refusals():
    good = dict(a=gpu(4, 16, dtype=I8), a_scale=gpu(4, dtype=F), w=gpu(6, 16, dtype=I8),
                w_scale=gpu(6, dtype=F))
    refuses(ops.int8_product, good, dict(a=gpu(4, 16)), dict(w=gpu(6, 16, dtype=torch.uint8)),
            dict(a=gpu(4, 15, dtype=I8)), dict(a=gpu(16, dtype=I8)), dict(a_scale=gpu(5, dtype=F)),
            dict(a_scale=gpu(4)), dict(w_scale=gpu(4, dtype=F)), dict(w_scale=gpu(6, 1, dtype=F)),
            dict(dtype=I8), dict(dtype=torch.float64), dict(a=torch.zeros(4, 16, dtype=I8)),
            dict(a_scale=gpu(4, dtype=F).requires_grad_()),
            dict(w_scale=gpu(6, dtype=F).requires_grad_()),
            dict(a=gpu(1, 131072, dtype=I8), w=gpu(6, 131072, dtype=I8), a_scale=gpu(1, dtype=F)))
    refuses(ops.int8_product, good, dict(a=1), dict(w_scale=1.0), error=TypeError)


def test_logprobs_refusals():
    good = dict(logits=gpu(4, 10), tokens=gpu(4, dtype=torch.int64))
    refuses(ops.token_logprobs, good, dict(logits=gpu(4, 0)), dict(logits=gpu(4)),
            dict(logits=gpu(4, 10, dtype=torch.float64)), dict(tokens=gpu(4, dtype=F)),
            dict(tokens=gpu(5, dtype=torch.int64)), dict(top=-1), dict(top=11),
            dict(temperature=0.0), dict(temperature=float("inf")), dict(temperature=float("nan")),
            dict(logits=gpu(4, 100), top=65), dict(logits=torch.zeros(4, 10)))
    good = dict(good, stats=gpu(4, 2, dtype=F), entropy=gpu(4, dtype=F), dlogp=gpu(4, dtype=F),
                dentropy=gpu(4, dtype=F))
    refuses(ops.token_logprobs_grad, good, dict(stats=gpu(4, 2)), dict(stats=gpu(4, 3, dtype=F)),
            dict(stats=gpu(8, dtype=F)), dict(entropy=gpu(3, dtype=F)), dict(dlogp=gpu(4)),
            dict(dlogp=gpu(4, 1, dtype=F)), dict(dentropy=gpu(5, dtype=F)),
            dict(temperature=-1.0), dict(tokens=gpu(3, dtype=torch.int64)))


def test_dual_tensors_are_refused():
    def dual(x):
        return forward_ad.make_dual(x, torch.ones_like(x))

    f = gpu(4, dtype=F)
    with forward_ad.dual_level():
        for fn, args, kw in (
                (ops.embedding, (i32(0), dual(gpu(4, 8))), {}),
                (ops.embedding_grad, (dual(gpu(1, 8)), i32(0), 4), {}),
                (ops.rms_norm, (dual(gpu(4, 8)),), {}),
                (ops.rms_norm, (gpu(4, 8), dual(gpu(8))), {}),
                (ops.rms_norm_int8, (gpu(4, 8),), dict(residual=dual(gpu(4, 8)))),
                (ops.quantize_rows, (dual(gpu(4, 8)),), {}),
                (ops.rms_norm_grad, (dual(gpu(4, 8)), gpu(4, 8)), {}),
                (ops.int8_product, (gpu(4, 8, dtype=I8), dual(f), gpu(4, 8, dtype=I8), f), {}),
                (ops.token_logprobs, (dual(gpu(4, 8)), gpu(4, dtype=torch.int64)), {}),
                (ops.token_logprobs_grad, (gpu(4, 8), gpu(4, dtype=torch.int64),
                                           gpu(4, 2, dtype=F), f, dual(f)), {})):
            with pytest.raises(ValueError, match="forward-mode"):
                fn(*args, **kw)


def filled(struct, pointers, **values):
    s = struct()
    s.struct_size = ctypes.sizeof(struct)
    for n in pointers:
        setattr(s, n, 4096)
    for n, x in values.items():
        setattr(s, n, x)
    return s


def library_refuses(name, struct, pointers, good, bad, nothing, workspace=True):
    """bad: (what differs, the code). nothing: a call with no work."""
    lib = seq_ops.load_library()
    fn, at = getattr(lib, name), ctypes.addressof
    for kw, want in [(dict(struct_size=8), CO_ERR_NULLARG)] + bad:
        assert fn(at(filled(struct, pointers, **{**good, **kw})), None) == want, (name, kw)
    assert fn(None, None) == CO_ERR_NULLARG
    assert fn(at(filled(struct, pointers, **{**good, **nothing})), None) == CO_OK
    if workspace:
        ws = getattr(lib, name + "_workspace")
        assert ws(None) < 0 and ws(at(filled(struct, pointers, **{**good, "struct_size": 0}))) < 0
        assert ws(at(filled(struct, pointers, **good))) >= 0


def test_library_refusals():
    """The C entry points refuse before any launch (no GPU is needed)."""
    far, nan = 1 << 40, float("nan")
    library_refuses(
        "seq_embedding", ops.SeqEmbedding, ("ids", "table", "out"),
        dict(tokens=4, rows=9, width=8, table_row=8, out_row=8, scale=1.0),
        [(dict(tokens=-1), CO_ERR_NULLARG), (dict(rows=-1), CO_ERR_NULLARG),
         (dict(width=0), CO_ERR_NULLARG), (dict(ids=None), CO_ERR_NULLARG),
         (dict(table=None), CO_ERR_NULLARG), (dict(out=None), CO_ERR_NULLARG),
         (dict(tokens=far), CO_ERR_BOUNDS), (dict(rows=far), CO_ERR_BOUNDS),
         (dict(width=65537), CO_ERR_BOUNDS), (dict(dtype=3), CO_ERR_DATA),
         (dict(out_dtype=-1), CO_ERR_DATA), (dict(scale=nan), CO_ERR_DATA)], dict(tokens=0), False)
    library_refuses(
        "seq_embedding_grad", ops.SeqEmbeddingGrad, ("ids", "d_out", "dtable", "workspace"),
        dict(tokens=400, rows=9, width=8, dout_row=8, dtable_row=8, scale=1.0,
             workspace_bytes=1 << 30),
        [(dict(tokens=-1), CO_ERR_NULLARG), (dict(width=0), CO_ERR_NULLARG),
         (dict(ids=None), CO_ERR_NULLARG), (dict(d_out=None), CO_ERR_NULLARG),
         (dict(dtable=None), CO_ERR_NULLARG), (dict(workspace=None), CO_ERR_NULLARG),
         (dict(rows=far), CO_ERR_BOUNDS), (dict(dtype=4), CO_ERR_DATA),
         (dict(workspace_bytes=100), CO_ERR_DATA), (dict(workspace=4100), CO_ERR_DATA),
         (dict(scale=float("inf")), CO_ERR_DATA)], dict(rows=0))
    norm = dict(tokens=4, width=8, x_row=8, residual_row=8, h_row=8, y_row=8, eps=1e-6, h_dtype=0,
                x_dtype=1)
    library_refuses(
        "seq_norm", ops.SeqNorm, ("x", "residual", "gain", "h", "y", "y_scale"), norm,
        [(dict(tokens=-1), CO_ERR_NULLARG), (dict(width=0), CO_ERR_NULLARG),
         (dict(x=None), CO_ERR_NULLARG), (dict(h=None), CO_ERR_NULLARG),
         (dict(y=None), CO_ERR_NULLARG), (dict(y_dtype=3, y_scale=None), CO_ERR_NULLARG),
         (dict(tokens=far), CO_ERR_BOUNDS), (dict(width=65537), CO_ERR_BOUNDS),
         (dict(y_dtype=4), CO_ERR_DATA), (dict(x_dtype=3), CO_ERR_DATA),
         (dict(gain_dtype=3), CO_ERR_DATA), (dict(h_dtype=2), CO_ERR_DATA),
         (dict(x_dtype=0, h_dtype=1), CO_ERR_DATA), (dict(eps=nan), CO_ERR_DATA),
         (dict(eps=-1.0), CO_ERR_DATA), (dict(identity=1), CO_ERR_DATA)], dict(tokens=0), False)
    library_refuses(
        "seq_norm_grad", ops.SeqNormGrad, ("dy", "h", "gain", "dh", "d", "dx", "dgain",
                                           "workspace"),
        dict(tokens=4, width=8, dy_row=8, h_row=8, dh_row=8, d_row=8, dx_row=8, eps=1e-6,
             workspace_bytes=1 << 30),
        [(dict(tokens=-1), CO_ERR_NULLARG), (dict(dy=None), CO_ERR_NULLARG),
         (dict(h=None), CO_ERR_NULLARG), (dict(d=None), CO_ERR_NULLARG),
         (dict(workspace=None), CO_ERR_NULLARG), (dict(width=1 << 17), CO_ERR_BOUNDS),
         (dict(dy_dtype=3), CO_ERR_DATA), (dict(h_dtype=3), CO_ERR_DATA),
         (dict(x_dtype=3), CO_ERR_DATA), (dict(gain_dtype=3), CO_ERR_DATA),
         (dict(eps=nan), CO_ERR_DATA), (dict(workspace_bytes=1), CO_ERR_DATA)],
        dict(tokens=0, dgain=None))
    library_refuses(
        "seq_int8_product", ops.SeqInt8Product, ("a", "w", "a_scale", "w_scale", "o"),
        dict(m=4, n=6, inner=16, a_row=16, w_row=16, o_row=6),
        [(dict(m=-1), CO_ERR_NULLARG), (dict(n=-1), CO_ERR_NULLARG),
         (dict(inner=-1), CO_ERR_NULLARG), (dict(a=None), CO_ERR_NULLARG),
         (dict(w=None), CO_ERR_NULLARG), (dict(a_scale=None), CO_ERR_NULLARG),
         (dict(w_scale=None), CO_ERR_NULLARG), (dict(o=None), CO_ERR_NULLARG),
         (dict(inner=131072), CO_ERR_BOUNDS), (dict(m=far), CO_ERR_BOUNDS),
         (dict(m=1 << 30, n=1 << 30), CO_ERR_BOUNDS), (dict(out_dtype=3), CO_ERR_DATA),
         (dict(inner=15), CO_ERR_NULLARG),                          # needs a workspace
         (dict(a=4097, workspace=4096, workspace_bytes=8), CO_ERR_DATA),
         (dict(w_row=17, workspace=4100, workspace_bytes=1 << 20), CO_ERR_DATA)], dict(m=0))
    rows = ("logits", "ids", "logp", "entropy", "stats", "top_logp", "top_ids")
    library_refuses(
        "seq_logprobs", ops.SeqLogprobs, rows,
        dict(tokens=4, vocab=10, row=10, temperature=1.0, top=3),
        [(dict(tokens=-1), CO_ERR_NULLARG), (dict(vocab=0), CO_ERR_NULLARG),
         (dict(top=-1), CO_ERR_NULLARG), (dict(tokens=far), CO_ERR_BOUNDS),
         (dict(top=11), CO_ERR_BOUNDS), (dict(vocab=100, top=65), CO_ERR_BOUNDS),
         (dict(dtype=3), CO_ERR_DATA), (dict(temperature=0.0), CO_ERR_DATA),
         (dict(vocab=90000, row=90000), CO_ERR_NULLARG),            # needs a workspace
         (dict(vocab=90000, row=90000, workspace=4096, workspace_bytes=8), CO_ERR_DATA),
         (dict(vocab=90000, row=90000, workspace=4100, workspace_bytes=1 << 20), CO_ERR_DATA)]
        + [({n: None}, CO_ERR_NULLARG) for n in rows if n != "stats"], dict(tokens=0))
    library_refuses(
        "seq_logprobs_grad", ops.SeqLogprobsGrad, ("logits", "ids", "stats", "entropy", "dlogits"),
        dict(tokens=4, vocab=10, row=10, drow=10, temperature=1.0),
        [(dict(tokens=-1), CO_ERR_NULLARG), (dict(vocab=0), CO_ERR_NULLARG),
         (dict(vocab=far), CO_ERR_BOUNDS), (dict(dtype=3), CO_ERR_DATA),
         (dict(temperature=nan), CO_ERR_DATA)]
        + [({n: None}, CO_ERR_NULLARG) for n in ("logits", "ids", "stats", "entropy", "dlogits")],
        dict(tokens=0), False)


def test_norm_gradient_against_differences():
    g = torch.Generator().manual_seed(1)
    h, gain, dy, v, vg = (torch.randn(*s, generator=g).double() for s in
                          ((4, 24), (24,), (4, 24), (4, 24), (24,)))
    r, step = ref.rms_grad(dy, h, gain, None, 1e-3), 1e-5

    def f(a):
        return float((ref.rms(h + a * v, gain + a * vg, 1e-3)[0] * dy).sum())

    slope = (f(step) - f(-step)) / (2 * step)
    want = float((r["d"] * v).sum() + (r["dgain"] * vg).sum())
    # rounding 2^-52 |f| / step, and the third derivative's step^2
    assert abs(slope - want) < 1e-8 * (1 + abs(want)) * 24


def test_logprobs_gradient_against_differences():
    g = torch.Generator().manual_seed(2)
    x, v = torch.randn(5, 30, generator=g).double(), torch.randn(5, 30, generator=g).double()
    gl, gh = torch.randn(5, generator=g), torch.randn(5, generator=g)
    tokens, step = torch.tensor([0, 3, 29, 7, 7]), 1e-5

    def f(a):
        r = ref.logprobs(x + a * v, tokens, 0.7)
        return float((r["logp"] * gl + r["entropy"] * gh).sum())

    d, _ = ref.logprobs_grad(ref.logprobs(x, tokens, 0.7), tokens, gl, gh, 0.7, F)
    slope, want = (f(step) - f(-step)) / (2 * step), float((d * v).sum())
    assert abs(slope - want) < 1e-7 * (1 + abs(want))


def test_a_search_with_a_proposer_of_its_own():
    """A proposer that is given may know nothing of 8-bit products; it is asked for them only
    where the search is."""
    import numpy as np

    from cusr_amd.demonstrator import proposer as pr
    asked = []

    class Fixed:
        device = torch.device("cpu")

        def sample(self, M, generator=None, **how):
            asked.append(how)
            return SimpleNamespace(lengths=torch.ones(M))

        def programs(self, pop):
            leaf = (np.array([popio.NODE_CONST]), np.array([0]), np.array([0]))
            return [leaf] * len(pop.lengths)

    class Still:
        def step(self, pop, rewards):
            return [0.0]

    class Fits:
        def fit_batch(self, _, inits, X, y, native):
            return [SimpleNamespace(final_loss=1.0, constants=x) for x in inits]

    for int8 in (False, True):
        pr.search(np.zeros((3, 1)), np.ones(3), rounds=1, population=2, proposer=Fixed(),
                  trainer=Still(), backend=Fits(), log=None, int8=int8)
    assert asked == [{}, {"int8": True}]


def test_alternatives_of_a_large_vocabulary(monkeypatch):
    """As many alternatives as there are symbols, and as token_logprobs gives at most."""
    from cusr_amd.demonstrator import proposer as pr
    monkeypatch.setattr(pr.seq_layers, "token_logprobs", lambda logits, tokens, **how: how["top"])
    for n_vars in (2, 300):
        p = pr.Proposer(n_vars, device="cpu")
        monkeypatch.setattr(p, "logits", lambda pop: None)
        for top in (0, 3, 99, 1000):
            got = p.alternatives(SimpleNamespace(symbols=None), top=top)
            assert got == min(top, p.symbols.size, ops.SEQ_MAX_TOP)


def test_workspace_of_a_product():
    """None where operands lie as they are read and the sums are short; room for every cut's
    sums where they are long and few, in any layout."""
    lib = seq_ops.load_library()

    def need(m, inner, n, row=None):
        c = ops.SeqInt8Product(struct_size=ctypes.sizeof(ops.SeqInt8Product), m=m, n=n, inner=inner,
                               a_row=row or inner, w_row=inner, o_row=n, a=4096, w=4096)
        return lib.seq_int8_product_workspace(ctypes.string_at(ctypes.byref(c), ctypes.sizeof(c)))

    for shape in ((1, 4096, 4096), (24, 4096, 6144), (8192, 4096, 16384), (300, 256, 300)):
        assert need(*shape) == 0
    # a whole number of cuts, at least two, of 64 by 1,001 sums in rows of 1,008
    cuts, rest = divmod(need(64, 16384, 1001), 4 * 64 * 1008)
    assert cuts >= 2 and rest == 0
    assert need(64, 16384, 1001, 16385) == need(64, 16384, 1001) + 64 * 16384
