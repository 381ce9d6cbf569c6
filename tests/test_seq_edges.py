"""Sequence operators without a GPU: what the sources promise the compiler, and
refusals at the edges of arguments and layouts."""
from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad

from cusr_amd.kernel import seq_ops as ops

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
