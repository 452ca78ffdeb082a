"""The training tail as a training loop runs it: norm, output head's loss, its
gradients, the global norm and clip scale, and Adam on fp32 masters with the
scale on the device -- a few steps, eager and as one captured graph. Every
step's results are held against float64 from the same bf16 operands; how far
the loss falls is not tested.

Tolerances: the gradients' are test_cross_entropy.py's; the norm is fp32 (8 x
2^-24, see test_clip.py) of the gradients as returned; Adam from the returned
gradients is fp32, 1e-5 (the repository's bar for it) of the magnitudes of the
terms that form each output: g' = g + wd p may cancel, so may b1 m + (1 - b1)
g', and p' divides m' by a denominator of its own.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from enzyme_b200 import ops
from oracle import f64
from test_cross_entropy import IGNORE, Ref, _row_g

pytestmark = pytest.mark.gpu

M, K, V, MAX_NORM = 150, 72, 1003, 0.25
ADAM = dict(step_size=2e-3, inv_bc2_sqrt=1.3, wd=0.01, beta1=0.9, beta2=0.95, eps=1e-8)


class Head:
    """Parameters and buffers of the loop: a norm weight and an output head."""

    def __init__(self, dev):
        g = torch.Generator(device=dev).manual_seed(77)
        self.x = torch.randn(M, K, device=dev, generator=g).bfloat16()
        self.targets = torch.randint(0, V, (M,), device=dev, generator=g)
        self.targets[::9] = IGNORE
        self.master = torch.randn(V, K, device=dev, generator=g) / K ** 0.5
        self.m, self.v = torch.zeros_like(self.master), torch.zeros_like(self.master)
        self.w = self.master.bfloat16()
        self.gain = torch.ones(K, device=dev).bfloat16()
        self.one = torch.ones(1, device=dev)
        self.dh = torch.empty(M, K, device=dev, dtype=torch.bfloat16)
        self.dw = torch.empty(V, K, device=dev)  # fp32 gradients for the fp32 masters
        self.grads = ops.GradList([self.dw, self.dh])

    def step(self):
        h = ops.rmsnorm(self.x, self.gain, scale=1.0 / K, eps=1e-6)
        loss, stats = ops.linear_cross_entropy(h, self.w, self.targets)
        ops.linear_cross_entropy_grad(h, self.w, self.targets, stats, self.one, out=(self.dh, self.dw))
        norm, scale = ops.grad_norm_scale(self.grads, MAX_NORM)
        ops.adam(self.master, self.dw, self.m, self.v, grad_scale=scale, out=(self.master, self.m, self.v), **ADAM)
        ops.cast(self.master, torch.bfloat16, out=self.w)
        return h, loss, stats, norm, scale


def _check(head, before, got):
    w, master, m, v = before
    h, loss, stats, norm, scale = got
    ref = Ref(h, w, head.targets, _row_g(head.one, head.targets, "mean"))
    ref.check_loss(stats)
    ref.check_grads(head.dh, head.dw)
    keep = head.targets != IGNORE
    mean = float(stats[1].double().sum() / keep.sum())
    assert abs(float(loss) - mean) <= 2.0 ** -23 * mean
    n64, s64 = f64.grad_scale([head.dw.double().cpu().numpy(), head.dh.double().cpu().numpy()], MAX_NORM)
    assert abs(float(norm) - n64) <= 8 * 2.0 ** -24 * n64
    assert abs(float(scale) - s64) <= 12 * 2.0 ** -24 * s64
    assert s64 < 1.0  # the step really clips
    args = [t.double().cpu().numpy() for t in (master, head.dw, m, v)]
    args[1] = args[1] * float(scale)
    want = f64.adam(*args, ADAM["step_size"], ADAM["inv_bc2_sqrt"], ADAM["wd"], beta1=0.9, beta2=0.95, eps=1e-8)
    p0, g0, m0, v0 = args
    gp = np.abs(g0) + ADAM["wd"] * np.abs(p0)
    m_terms = 0.9 * np.abs(m0) + 0.1 * gp
    v_terms = 0.95 * v0 + 0.05 * gp ** 2
    denom = np.sqrt(want[2]) * ADAM["inv_bc2_sqrt"] + ADAM["eps"]
    # v' enters the update through its root: |m'| / denom times v_terms / (2 v')
    p_terms = np.abs(p0) + ADAM["step_size"] * (m_terms + np.abs(want[1]) * v_terms / (2 * want[2] + 1e-30)) / denom
    for a, b, terms in zip((head.master, head.m, head.v), want, (p_terms, m_terms, v_terms)):
        assert (np.abs(a.double().cpu().numpy() - b) <= 1e-5 * terms).all()
    assert torch.equal(head.w, head.master.bfloat16())


def test_steps(cuda_device):
    head = Head(cuda_device)
    for _ in range(3):
        before = [t.clone() for t in (head.w, head.master, head.m, head.v)]
        _check(head, before, head.step())
    ops.linear_cross_entropy_status()


def test_captured_steps(cuda_device):
    """One step captured after a warm one and replayed: the same bits as the
    same number of eager steps."""
    eager, graphed = Head(cuda_device), Head(cuda_device)
    eager.step()
    graphed.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = graphed.step()
    for _ in range(3):
        want = eager.step()
        g.replay()
        for a, b in zip((*got, graphed.dh, graphed.dw, graphed.master, graphed.m, graphed.v, graphed.w),
                        (*want, eager.dh, eager.dw, eager.master, eager.m, eager.v, eager.w)):
            assert torch.equal(a, b)


def test_clipping_in_place_then_adam_is_the_same_step(cuda_device):
    """clip_grads followed by plain Adam gives the bits of Adam with the scale,
    for fp32 gradients (one rounding either way)."""
    a, b = Head(cuda_device), Head(cuda_device)
    a.step()
    h = ops.rmsnorm(b.x, b.gain, scale=1.0 / K, eps=1e-6)
    _, stats = ops.linear_cross_entropy(h, b.w, b.targets)
    ops.linear_cross_entropy_grad(h, b.w, b.targets, stats, b.one, out=(b.dh, b.dw))
    ops.clip_grads(b.grads, MAX_NORM)
    ops.adam(b.master, b.dw, b.m, b.v, out=(b.master, b.m, b.v), **ADAM)
    assert torch.equal(a.master, b.master) and torch.equal(a.m, b.m) and torch.equal(a.v, b.v)
