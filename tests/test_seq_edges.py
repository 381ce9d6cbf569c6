"""Sequence operators without a GPU: what the sources promise the compiler, and
refusals at the edges of arguments and layouts."""
from __future__ import annotations

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad

from cusr_amd.kernel import seq_ops as ops
from cusr_amd.kernel.co_inproc import CO_ERR_DATA

CSRC = Path(__file__).resolve().parents[1] / "cusr_amd" / "csrc"


# -------------------------------------------------------------------- sources

def test_assembly_names_what_it_overwrites():
    """Assembly that writes m0 says so: the compiler may keep a value there."""
    found = 0
    for path in sorted(CSRC.glob("seq_*")):
        for block in re.findall(r"asm volatile\((.*?)\);", path.read_text(), re.S):
            if re.search(r"s_mov_b32 m0", block):
                found += 1
                clobbers = block.rsplit(":", 1)[1]
                assert '"m0"' in clobbers and '"memory"' in clobbers, (path.name, block)
    assert found >= 3


def test_arguments_are_found_by_kernels_alone():
    """A called function has no pointer of its own to the kernel's arguments: where
    one is formed, the function is a kernel (or is inlined without fail)."""
    found = 0
    for path in sorted(CSRC.glob("seq_*")):
        function = ""
        for line in path.read_text().splitlines():
            if re.match(r"(template <[^>]*> )?(__global__|__device__)", line):
                function = line
            if "__builtin_amdgcn_kernarg_segment_ptr" in line:
                assert "always_inline" in function, (path.name, function)
            elif re.search(r"\barguments<\w+>\(\)", line) and line != function:
                assert function.startswith("__global__"), (path.name, function)
                found += 1
    assert found >= 6


# ------------------------------------------------------------------- refusals

class _Gpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: refusals come before any use."""
    is_cuda = True


def gpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Gpu)


F32 = torch.float32


def calls():
    """Each entry point with arguments that it takes, and which are real numbers."""
    i32 = torch.tensor([0, 4], dtype=torch.int32).as_subclass(_Gpu)
    heads = dict(q=gpu(4, 4, 64), k=gpu(4, 2, 64), v=gpu(4, 2, 64))
    lse = gpu(4, 4, dtype=F32)
    policy = dict(logits=gpu(4, 10), logp_old=gpu(4, dtype=F32), advantages=gpu(4, dtype=F32),
                  logp_ref=gpu(4, dtype=F32), weights=gpu(4, dtype=F32))
    actions = dict(actions=gpu(4, dtype=torch.int64))
    return [
        (ops.attention, heads, dict(cu_q=i32)),
        (ops.attention_grad, dict(heads, do=gpu(4, 4, 64)), dict(o=gpu(4, 4, 64), lse=lse,
                                                                cu_q=i32)),
        (ops.rotary, dict(q=gpu(4, 2, 16), k=gpu(4, 1, 16), table=gpu(9, 8, 2, dtype=F32)),
         dict(positions=gpu(4, dtype=torch.int64))),
        (ops.policy_loss, policy, actions),
        (ops.policy_loss_grad, policy, actions),
    ]


def test_dual_tensors_are_refused():
    for fn, real, other in calls():
        for name in real:
            with forward_ad.dual_level():
                x = real[name].as_subclass(torch.Tensor)
                dual = forward_ad.make_dual(x, torch.ones_like(x))
                with pytest.raises(ValueError, match="forward-mode"):
                    fn(**{**real, **other, name: dual})


def test_inputs_without_a_gradient_are_refused():
    for fn, real, other in calls():
        names = {ops.rotary: ["table"],
                 ops.policy_loss: ["logp_old", "advantages", "logp_ref", "weights"]}.get(fn, [])
        for name in names:
            x = real[name].clone().requires_grad_()
            with pytest.raises(ValueError, match=f"{name} gets no gradient"):
                fn(**{**real, **other, name: x})


def test_rotary_in_place_needs_memory_of_its_own():
    """Broadcast views and tensors that share elements would be turned twice, or by
    several threads at once."""
    pos, table = gpu(6, dtype=torch.int64), gpu(9, 8, 2, dtype=F32)
    wide = gpu(6, 8, 16)
    flat = gpu(6 * 8 * 16 + 16)
    rows = flat[:6 * 64].view(6, 4, 16)
    for q, k in ((gpu(1, 4, 16).expand(6, 4, 16), None), (gpu(6, 1, 16).expand(6, 4, 16), None),
                 (wide, gpu(1, 2, 16).expand(6, 2, 16)), (wide, wide), (wide[:, :4], wide[:, 3:5]),
                 (wide[:, 3:5], wide[:, :4]), (wide[:, :4], wide[:, 2:3]),
                 (flat.as_strided((6, 4, 16), (64, 8, 1)), None),
                 (flat.as_strided((6, 4, 16), (40, 16, 1)), None),
                 (rows, flat.as_strided((6, 1, 16), (64, 16, 1), 6)),
                 (rows, flat.as_strided((6, 1, 16), (80, 16, 1), 64))):
        with pytest.raises(ValueError, match="memory of its own"):
            ops.rotary(q, k, pos, table, inplace=True)


def test_memory_that_is_not_shared():
    """Layouts that models have: slices of a projection, heads before rows, one
    allocation after the other, one token."""
    wide, first = gpu(6, 8, 16), gpu(8, 6, 16).transpose(0, 1)
    one = gpu(1, 8, 16)
    flat = gpu(2 * 6 * 32)
    for q, k in ((wide[:, :4], wide[:, 4:6]), (wide[:, 6:], wide[:, :6]),
                 (first[:, :4], first[:, 4:]), (one[:, :4], one[:, 4:]),
                 (flat[:192].view(6, 2, 16), flat[192:].view(6, 2, 16)),
                 (wide[:, 0::2], wide[:, 1::2]), (wide[:, :, :8], wide[:, :, 8:])):
        assert ops._own_memory(q) and ops._own_memory(k)
        assert not ops._share_memory(q, k) and not ops._share_memory(k, q)
    assert ops._own_memory(gpu(0, 8, 16)) == 0
    # against sets of elements
    g = torch.Generator().manual_seed(0)
    pick = lambda n: int(torch.randint(n, (1,), generator=g))  # noqa: E731
    base, seen = gpu(4000), [0, 0]
    for _ in range(4000):
        T, hq, hk, d = 1 + pick(4), 1 + pick(3), 1 + pick(3), 1 + pick(6)
        both = [base.as_strided((T, h, d), (pick(40), pick(40), 1), pick(60)) for h in (hq, hk)]
        own = [ops._own_memory(x) for x in both]
        at = []
        for x, n in zip(both, own):
            i = [x.storage_offset() + t * x.stride(0) + h * x.stride(1) + e
                 for t in range(T) for h in range(x.shape[1]) for e in range(d)]
            assert n is None or (len(set(i)) == len(i) and max(i) - min(i) < n)
            at.append(set(i))
        if None not in own:
            shared = bool(at[0] & at[1])
            seen[shared] += 1
            if shared or both[0].stride(0) == both[1].stride(0) or T == 1:
                assert ops._share_memory(*both) == shared, (both[0].stride(), both[1].stride())
    assert min(seen) > 100


@pytest.mark.parametrize("kw", [dict(temperature=1e-50), dict(temperature=1e-40),
                                dict(temperature=1e39), dict(temperature=-1.0),
                                dict(temperature=float("nan")), dict(kl_coef=1e39),
                                dict(kl_coef=-1e300), dict(kl_coef=float("inf"))])
def test_policy_numbers_beyond_float32_are_refused(kw):
    for fn, real, other in calls():
        if fn in (ops.policy_loss, ops.policy_loss_grad):
            with pytest.raises(ValueError):
                fn(**real, **other, **kw)


def test_scales_beyond_float32_are_refused():
    for fn, real, other in calls()[:2]:
        for scale in (0.0, -1.0, 1e-50, 1e-39, 1e31, float("nan")):
            with pytest.raises(ValueError, match="scale"):
                fn(**real, **other, scale=scale)


def test_clip_widths_beyond_float32_do_not_clip():
    _, real, other = calls()[3]
    x = {n: t for n, t in {**real, **other}.items()}
    got = ops._check_policy(x["logits"], x["actions"], x["logp_old"], x["advantages"], None, None,
                            (1e39, float("inf")), 0.0, 1.0)
    assert got == (float("inf"), float("inf"))


def test_library_refuses_numbers_out_of_range():
    lib, ref = ops.load_library(), ctypes.addressof
    for kw in (dict(temperature=float("inf")), dict(temperature=1e-35), dict(clip_lo=-0.1),
               dict(clip_hi=float("nan")), dict(kl_coef=float("nan")),
               dict(kl_coef=float("inf"))):
        p = ops.SeqPolicyLoss(ctypes.sizeof(ops.SeqPolicyLoss), 1, 4, 10, 10, 10, 0.2, 0.2, 0.0,
                              1.0)
        for n in ("logits", "actions", "logp_old", "advantages", "weights", "loss", "logp",
                  "workspace"):
            setattr(p, n, 4096)
        p.workspace_bytes = 1 << 20
        for n, x in kw.items():
            setattr(p, n, x)
        assert lib.seq_policy_loss(ref(p), None) == CO_ERR_DATA, kw


# ------------------------------------------------------------------- proposer

def test_a_search_that_fits_nothing_says_so(monkeypatch, capsys):
    from cusr_amd.demonstrator import proposer
    monkeypatch.setattr(proposer, "search", lambda *a, **k: ((math.inf, None, None), []))
    proposer.main(["--rounds", "0"])
    assert capsys.readouterr().out == "no program was fitted\n"
