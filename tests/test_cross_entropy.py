"""The output head's softmax cross entropy and its gradient against float64.

Tolerances, from the arithmetic (u = half a step of the operand type, U = 2^-24):
* a logit is a sum of k products that are exact in fp32; the tensor core adds
  them 16 at a time, each addition off by at most 2^-23 of the magnitudes that
  are summed (it may truncate), so |ds| <= (k/16 + 4) 2^-23 A, A the largest
  sum over k of |h w|;
* an exponential is off by 2^-22 of itself and by its argument's rounding,
  2^-24 of at most 2^7: together E = 2^-16 covers it;
* log-sum-exp: |ds| + E and one rounding; the loss of a row depends on logit
  differences weighted with 1 - p_t <= min(1, loss), so min(1, loss) (2 |ds| + E) and a
  rounding (losses are summed in float64);
* an entry of d is off by r = 2 |ds| + 2 E + u of itself (f16: and by 2^-39 of
  the largest |g|, half a step of subnormals at the scale it is held in); its
  contraction by r and by (terms/16 + 4) 2^-23 of the sum of magnitudes; the
  output by u of itself (f16: and half a step of subnormals, 2^-25);
* what lies below the types' range: an fp32 loss under 2^-149 has no digits
  (2^-150 beside the rounding), exponentials under 2^-126 are flushed (2^-126 of
  the largest |g| beside an entry of d), and a bf16 output has steps of 2^-133
  (2^-134 beside its rounding).
"""

from __future__ import annotations

import ctypes
import math
import types

import pytest
import torch

from enzyme_b200 import _native as N
from enzyme_b200 import ops

U32 = 2.0 ** -24
E = 2.0 ** -16
IGNORE = -100


# ---- refusals (no GPU) --------------------------------------------------------------

FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: every call below is refused on the host
BIG = 1 << 40


def _fwd(**kw):
    a = dict(h=FAKE, w=FAKE, t=FAKE, lse=FAKE, rows=FAKE, loss=FAKE, m=4, k=64, v=100, ldh=64, ldw=64, dt=N.AXON_BF16,
             bits=64, red=N.AXON_REDUCE_MEAN, ws=FAKE, wsb=BIG, tune=None)
    a.update(kw)
    return N.lib().axon_linear_ce(a["h"], a["w"], a["t"], a["lse"], a["rows"], a["loss"], a["m"], a["k"], a["v"],
                                  a["ldh"], a["ldw"], a["dt"], a["bits"], IGNORE, a["red"], a["ws"], a["wsb"],
                                  a["tune"], None)


def _bwd(**kw):
    a = dict(h=FAKE, w=FAKE, t=FAKE, lse=FAKE, rows=FAKE, dloss=FAKE, dh=ctypes.c_void_p(0x7000000),
             dw=ctypes.c_void_p(0x8000000), m=4, k=64, v=100, ldh=64,
             ldw=64, lddh=64, lddw=64, dt=N.AXON_BF16, dwt=N.AXON_BF16, bits=64, red=N.AXON_REDUCE_MEAN, ws=FAKE,
             wsb=BIG, tune=None)
    a.update(kw)
    return N.lib().axon_linear_ce_grad(a["h"], a["w"], a["t"], a["lse"], a["rows"], a["dloss"], a["dh"], a["dw"],
                                       a["m"], a["k"], a["v"], a["ldh"], a["ldw"], a["lddh"], a["lddw"], a["dt"],
                                       a["dwt"], a["bits"], IGNORE, a["red"], a["ws"], a["wsb"], a["tune"], None)


SHARED = [
    (dict(m=-1), N.AXON_E_SHAPE), (dict(k=0), N.AXON_E_SHAPE), (dict(v=0), N.AXON_E_SHAPE),
    (dict(k=60, ldh=64), N.AXON_E_SHAPE), (dict(m=1 << 31), N.AXON_E_SHAPE), (dict(v=1 << 31), N.AXON_E_SHAPE),
    (dict(dt=N.AXON_F32), N.AXON_E_UNSUPPORTED), (dict(bits=16), N.AXON_E_UNSUPPORTED), (dict(red=3), N.AXON_E_ARG),
    (dict(h=None), N.AXON_E_ARG), (dict(w=None), N.AXON_E_ARG), (dict(t=None), N.AXON_E_ARG),
    (dict(lse=None), N.AXON_E_ARG), (dict(rows=None), N.AXON_E_ARG),
    (dict(ldh=56), N.AXON_E_SHAPE), (dict(ldw=56), N.AXON_E_SHAPE), (dict(ldh=68), N.AXON_E_ALIGN),
    (dict(ldw=68), N.AXON_E_ALIGN), (dict(h=ctypes.c_void_p(0x10008)), N.AXON_E_ALIGN),
    (dict(w=ctypes.c_void_p(0x10002)), N.AXON_E_ALIGN), (dict(t=ctypes.c_void_p(0x10004)), N.AXON_E_ALIGN),
    (dict(ws=None), N.AXON_E_ARG), (dict(wsb=16), N.AXON_E_ARG), (dict(ws=ctypes.c_void_p(0x10008)), N.AXON_E_ALIGN),
    (dict(tune=ctypes.byref(N.Tune(variant=1))), N.AXON_E_ARG),
    (dict(tune=ctypes.byref(N.Tune(max_ctas=-1))), N.AXON_E_ARG),
]


@pytest.mark.parametrize("i", range(len(SHARED)))
def test_bad_arguments_are_refused(i):
    kw, code = SHARED[i]
    assert _fwd(**kw) == code, N.last_error()
    assert _bwd(**kw) == code, N.last_error()
    assert N.last_error().startswith("axon_linear_ce_grad")


def test_more_refusals():
    assert _fwd(loss=None) == N.AXON_E_ARG
    for kw, code in ((dict(dloss=None), N.AXON_E_ARG), (dict(dh=None, dw=None), N.AXON_E_ARG),
                     (dict(dwt=N.AXON_F16), N.AXON_E_UNSUPPORTED), (dict(lddh=56), N.AXON_E_SHAPE),
                     (dict(lddw=68), N.AXON_E_ALIGN), (dict(dh=ctypes.c_void_p(0x10008)), N.AXON_E_ALIGN),
                     (dict(tune=ctypes.byref(N.Tune(split=100))), N.AXON_E_ARG),
                     (dict(ws=ctypes.c_void_p(0x10080)), N.AXON_E_ALIGN)):
        assert _bwd(**kw) == code, (kw, N.last_error())


def test_the_form_with_a_copy_refuses_the_same():
    for kw in (dict(rows=None), dict(k=60), dict(dt=N.AXON_F32), dict(ws=None)):
        a = dict(rows=FAKE, k=64, dt=N.AXON_BF16, ws=FAKE)
        a.update(kw)
        rc = N.lib().axon_linear_ce_kept(FAKE, FAKE, FAKE, FAKE, a["rows"], FAKE, None, 4, a["k"], 100, 64, 64, a["dt"],
                                         64, IGNORE, N.AXON_REDUCE_NONE, a["ws"], BIG, None, None)
        assert rc == _fwd(red=N.AXON_REDUCE_NONE, **kw) != N.AXON_OK


def test_outputs_over_operands_are_refused():
    """dh and dw are written while the operands are read. Addresses far apart
    for everything but the pair under test (nothing is dereferenced)."""
    far = {n: ctypes.c_void_p(0x1000000 * (i + 1)) for i, n in
           enumerate(("h", "w", "t", "lse", "rows", "dloss", "dh", "dw"))}
    for out in ("dh", "dw"):
        for other in far:
            if other != out:
                assert _bwd(**{**far, out: far[other], "ws": None}) == N.AXON_E_ARG
                assert "overlaps" in N.last_error(), N.last_error()
    assert _bwd(**{**far, "dh": ctypes.c_void_p(0x1000000 + 3 * 64 * 2)}) == N.AXON_E_ARG  # h's last row
    assert _bwd(**{**far, "ws": None}) == N.AXON_E_ARG and "workspace" in N.last_error()


def test_variants_are_listed():
    import json

    for op in ("linear_ce", "linear_ce_grad", "grad_norm"):
        assert json.loads(N.variants(op))["op"] == op


def test_workspaces():
    """The loss needs 16 bytes per row and 256 words; the gradient holds d by
    pieces of at most 512 MB, and an fp32 dh only where there are several."""
    lib = N.lib()
    assert lib.axon_linear_ce_workspace_bytes(4096, 4096, 128256) < 4096 * 501 * 16 + 4096 * 4 + 1024
    assert lib.axon_linear_ce_workspace_bytes(4, 60, 100) == N.AXON_E_SHAPE
    one = lib.axon_linear_ce_grad_workspace_bytes(256, 64, 1000, None)
    assert one < 256 * 1024 * 2 + 256 * 64 * 2 + 256 * 20 + 2048
    two = lib.axon_linear_ce_grad_workspace_bytes(256, 64, 1000, N.Tune.of({"split": 512}))
    assert two == one - 256 * 512 * 2 + 256 * 64 * 4
    big = lib.axon_linear_ce_grad_workspace_bytes(16384, 4096, 128256, None)
    assert big < (512 << 20) + 16384 * 4096 * 6 + 16384 * 20 + 4096


def test_host_tensors_are_refused():
    h, w, t = torch.zeros(2, 8).bfloat16(), torch.zeros(5, 8).bfloat16(), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(N.AxonError) as e:
        ops.linear_cross_entropy(h, w, t)
    assert e.value.code == N.AXON_E_ARG and "CUDA" in e.value.message


def test_workspaces_that_are_no_block_of_memory_are_refused():
    """An expanded tensor has its bytes in its shape only, a strided one in
    between others' elements; what counts is bytes, not elements."""
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(4096), torch.zeros(8192, dtype=torch.uint8)[::2],
               torch.zeros(64, 64, dtype=torch.uint8).T):
        with pytest.raises(N.AxonError) as e:
            ops._head_workspace(4096, ws.device, ws)
        assert e.value.code == N.AXON_E_SHAPE
    with pytest.raises(N.AxonError) as e:
        ops._head_workspace(4096, "cpu", torch.zeros(4095, dtype=torch.uint8))
    assert e.value.code == N.AXON_E_ARG and "4096 bytes" in e.value.message
    for dtype in (torch.uint8, torch.float32):
        ws = torch.zeros(4096, dtype=torch.uint8).view(dtype)
        assert ops._head_workspace(4096, "cpu", ws) is ws
    assert ops._head_workspace(4096, "cpu").nbytes == 4096


def test_status_of_another_device_is_asked_there(monkeypatch):
    """The status word belongs to the current device: it has to be the one whose
    stream is waited for."""
    current, seen = [0], []

    class Device:
        def __init__(self, device):
            self.to = current[0] if device is None else device

        def __enter__(self):
            self.back, current[0] = current[0], self.to

        def __exit__(self, *exc):
            current[0] = self.back

    def stream(device=None):
        return types.SimpleNamespace(cuda_stream=100 + (current[0] if device is None else device))

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_stream", stream)
    monkeypatch.setattr(N, "lib", lambda: types.SimpleNamespace(
        axon_linear_ce_status=lambda s: seen.append((current[0], s)) or 0))
    for device in (None, 1):
        ops.linear_cross_entropy_status(device)
    assert seen == [(0, 100), (1, 101)] and current == [0]


@pytest.mark.parametrize("rows", [1, 2, 7])
def test_outputs_whose_rows_are_not_contiguous_are_refused(rows):
    """k elements are written from a row's start, in a single row as in many:
    every second element, a column and an expanded row are no such memory."""
    like = torch.zeros(rows, 16).bfloat16()
    room = torch.zeros(64, 64).bfloat16()
    for t in (room[:rows, :32:2], room[:16, :rows].T, room[:rows, :1].expand(rows, 16)):
        assert t.shape == like.shape
        with pytest.raises(N.AxonError) as e:
            ops._head_out("f", t, like, (torch.bfloat16,))
        assert e.value.code == N.AXON_E_SHAPE
    for t in (room[:rows].float()[:, :16], room[:rows, :8]):
        with pytest.raises(N.AxonError) as e:
            ops._head_out("f", t, like, (torch.bfloat16,))
        assert e.value.code == N.AXON_E_ARG
    ld = 64 if rows > 1 else 16
    assert ops._head_out("f", room[:rows, 16:32], like, (torch.bfloat16,)) == ld
    assert ops._head_out("f", None, like, (torch.bfloat16,)) == 16


# ---- GPU ----------------------------------------------------------------------------


def _inputs(dev, m, k, v, dtype, seed=0, ignored=0.0, pull=10.0, pad=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    h = torch.randn(m, k + pad, device=dev, generator=g)
    w = (torch.randn(v, k + pad, device=dev, generator=g) * (1.3 / math.sqrt(k))).to(dtype)
    t = torch.randint(0, v, (m,), device=dev, generator=g)
    wt = w[t][:, :k].float()
    h[:, :k] += pull * torch.rand(m, 1, device=dev, generator=g) * wt / wt.norm(dim=1, keepdim=True).clamp(min=1e-6)
    if ignored:
        t = torch.where(torch.rand(m, device=dev, generator=g) < ignored, torch.full_like(t, IGNORE), t)
    return h.to(dtype)[:, :k], w[:, :k], t


class Ref:
    """Float64 evaluation with the bounds of the module's comment."""

    def __init__(self, h, w, t, g=None):
        self.m, self.k = h.shape
        self.v = w.shape[0]
        self.dtype = h.dtype
        h, w = h.double(), w.double()
        s = h @ w.T
        self.keep = t != IGNORE
        at = t.clamp(min=0).long()
        rows = torch.arange(self.m, device=h.device)
        st = s[rows, at]
        other = s.clone()
        other[rows[self.keep], at[self.keep]] = -math.inf
        rest = torch.logsumexp(other, dim=1)
        zero = torch.zeros_like(rest)
        self.loss = torch.where(self.keep, torch.logaddexp(rest - st, zero), zero)
        self.lse = torch.where(self.keep, torch.logaddexp(rest, st), rest)
        a = float((h.abs() @ w.abs().T).max()) if self.m else 0.0
        self.ds = (self.k / 16 + 4) * 2.0 ** -23 * a
        self.u = torch.finfo(self.dtype).eps / 2
        if g is not None:
            g = torch.where(self.keep, g.double(), zero)
            d = torch.exp(s - self.lse[:, None])
            d[rows[self.keep], at[self.keep]] = torch.expm1(-self.loss)[self.keep]
            d *= g[:, None]
            r = 2 * self.ds + 2 * E + self.u
            dd = d.abs() * r + float(g.abs().max()) * 2.0 ** -126 * self.keep[:, None]
            floor = 2.0 ** -134
            if self.dtype == torch.float16:
                dd = dd + float(g.abs().max()) * 2.0 ** -39 * self.keep[:, None]
                floor = 2.0 ** -25
            self.dh, self.dw = d @ w, d.T @ h
            self.dh_tol = (dd + (self.v / 16 + 4) * 2.0 ** -23 * d.abs()) @ w.abs() + self.u * self.dh.abs() + floor
            # several pieces add one fp32 rounding of the sum each
            self.dh_tol += 64 * U32 * (d.abs() @ w.abs())
            self.dw_tol = (dd + (self.m / 16 + 4) * 2.0 ** -23 * d.abs()).T @ h.abs() + self.u * self.dw.abs() + floor

    def check_loss(self, stats):
        lse_err = (stats[0].double() - self.lse).abs()
        assert bool((lse_err <= self.ds + E + U32 * self.lse.abs()).all()), float(lse_err.max())
        err = (stats[1].double() - self.loss).abs()
        tol = self.loss.clamp(max=1.0) * (2 * self.ds + E) + U32 * self.loss + 2.0 ** -150
        assert bool((err <= tol).all()), float((err - tol).max())

    def check_grads(self, dh, dw):
        if dh is not None:
            over = (dh.double() - self.dh).abs() - self.dh_tol
            assert bool((over <= 0).all()), float(over.max())
        if dw is not None:
            over = (dw.double() - self.dw).abs() - self.dw_tol
            assert bool((over <= 0).all()), float(over.max())


def _both(h, w, t, dloss, reduction, **kw):
    loss, stats = ops.linear_cross_entropy(h, w, t, reduction=reduction)
    dh, dw = ops.linear_cross_entropy_grad(h, w, t, stats, dloss, reduction=reduction, **kw)
    ops.linear_cross_entropy_status()
    return loss, stats, dh, dw


def _row_g(dloss, t, reduction):
    keep = t != IGNORE
    if reduction == "mean":
        dloss = dloss / keep.sum()
    return dloss.expand(t.shape)


SHAPES = [
    (1, 8, 1), (1, 64, 2), (2, 72, 255), (7, 64, 256), (1, 512, 5003), (37, 136, 257), (128, 64, 1000),
    (129, 200, 513), (255, 256, 511), (256, 264, 768), (257, 512, 2049), (513, 128, 4099),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_loss(shape, dtype, cuda_device):
    m, k, v = shape
    h, w, t = _inputs(cuda_device, m, k, v, dtype, seed=m + v, ignored=0.2)
    ref = Ref(h, w, t)
    for reduction in ("none", "sum", "mean"):
        loss, stats = ops.linear_cross_entropy(h, w, t, reduction=reduction)
        ops.linear_cross_entropy_status()
        ref.check_loss(stats)
        rows = stats[1].double()
        if reduction == "none":
            assert torch.equal(loss, stats[1])
        elif reduction == "sum":
            assert torch.equal(loss, rows.sum().float()) or abs(float(loss - rows.sum())) <= 2 * U32 * float(rows.sum())
        elif bool(ref.keep.any()):
            mean = float(rows.sum() / ref.keep.sum())
            assert abs(float(loss) - mean) <= 2 * U32 * mean
        else:
            assert loss.isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients(shape, dtype, reduction, cuda_device):
    m, k, v = shape
    h, w, t = _inputs(cuda_device, m, k, v, dtype, seed=m + v, ignored=0.0 if m < 3 else 0.3)
    if reduction == "none":
        dloss = torch.randn(m, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(1))
    else:
        dloss = torch.full((1,), 16.0, device=cuda_device)
    loss, stats, dh, dw = _both(h, w, t, dloss, reduction)
    ref = Ref(h, w, t, _row_g(dloss, t, reduction))
    ref.check_loss(stats)
    ref.check_grads(dh, dw)
    assert not bool(dh[~ref.keep].any())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 200])
def test_losses_changed_in_place(m, cuda_device):
    """The per-row losses are the caller's: what is done to them between the
    two calls reaches neither stats nor the gradients."""
    k, v = 64, 700
    h, w, t = _inputs(cuda_device, m, k, v, torch.bfloat16, seed=m)
    dloss = torch.ones(m, device=cuda_device)
    loss, stats, dh, dw = _both(h, w, t, dloss, "none")
    kept = stats.clone()
    assert torch.equal(loss, stats[1])
    loss *= 0
    assert torch.equal(stats, kept)
    dh2, dw2 = ops.linear_cross_entropy_grad(h, w, t, stats, dloss, reduction="none")
    assert torch.equal(dh, dh2) and torch.equal(dw, dw2)
    # and the other way round
    loss, stats = ops.linear_cross_entropy(h, w, t, reduction="none")
    stats.zero_()
    assert torch.equal(loss, kept[1])


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_losses_are_no_views(reduction, cuda_device):
    """Changing the loss in place (weights, accumulation steps) is no change of
    stats that a backward pass which has saved them would object to."""
    h, w, t = _inputs(cuda_device, 20, 64, 300, torch.bfloat16, seed=1)
    loss, stats = ops.linear_cross_entropy(h, w, t, reduction=reduction)
    assert loss.shape == ((20,) if reduction == "none" else ())
    before = stats._version
    loss /= 4
    assert stats._version == before
    assert loss.untyped_storage().data_ptr() != stats.untyped_storage().data_ptr()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,split", [((5, 64, 4160), 4096), ((130, 520, 9000), 8192), ((40, 64, 12345), 0)])
def test_pieces_whose_contraction_is_cut(shape, split, cuda_device):
    """dh's contraction over a piece in parts, the last piece shorter than the
    others (some of its parts empty)."""
    m, k, v = shape
    lib = N.lib()
    tune = {"split": split}
    whole = split or -(-v // 256) * 256
    assert lib.axon_linear_ce_grad_workspace_bytes(m, k, v, N.Tune.of(tune)) > \
        256 + 5 * m * 4 + m * k * 2 + m * whole * 2 + 2 * m * k * 4  # several fp32 parts of dh
    h, w, t = _inputs(cuda_device, m, k, v, torch.bfloat16, seed=v, ignored=0.2)
    dloss = torch.ones(1, device=cuda_device)
    _, _, dh, dw = _both(h, w, t, dloss, "sum", tune=tune)
    Ref(h, w, t, _row_g(dloss, t, "sum")).check_grads(dh, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("max_ctas", [1, 2, 3, 7])
@pytest.mark.parametrize("m", [5, 50, 100])
def test_few_rows_on_few_ctas(m, max_ctas, cuda_device):
    """Fewer CTAs than blocks of 256 columns (then the CTA pairs take over), as
    many, and more; the vocabulary in pieces and in one."""
    k, v = 600, 3001
    h, w, t = _inputs(cuda_device, m, k, v, torch.bfloat16, seed=m, ignored=0.2)
    dloss = torch.ones(1, device=cuda_device)
    ref = Ref(h, w, t, _row_g(dloss, t, "sum"))
    for split in (0, 1024):
        _, _, dh, dw = _both(h, w, t, dloss, "sum", tune={"max_ctas": max_ctas, "split": split})
        ref.check_grads(dh, dw)


@pytest.mark.gpu
def test_bands_of_rows(cuda_device):
    """A hidden size whose rows of h fill L2's share in a few row tiles, so the
    logits are walked in several bands."""
    m, k, v = 1300, 24584, 700
    h, w, t = _inputs(cuda_device, m, k, v, torch.bfloat16, seed=3, ignored=0.1)
    dloss = torch.ones(1, device=cuda_device)
    _, stats, dh, dw = _both(h, w, t, dloss, "mean")
    ref = Ref(h, w, t, _row_g(dloss, t, "mean"))
    ref.check_loss(stats)
    ref.check_grads(dh, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("split", [256, 512, 1024])
@pytest.mark.parametrize("shape", [(5, 64, 1000), (300, 264, 2049), (513, 512, 1281)])
def test_pieces_of_the_vocabulary(shape, split, cuda_device):
    m, k, v = shape
    for dtype in (torch.bfloat16, torch.float16):
        h, w, t = _inputs(cuda_device, m, k, v, dtype, seed=split, ignored=0.1)
        dloss = torch.ones(1, device=cuda_device)
        _, _, dh, dw = _both(h, w, t, dloss, "sum", tune={"split": split})
        Ref(h, w, t, _row_g(dloss, t, "sum")).check_grads(dh, dw)


@pytest.mark.gpu
def test_strides_types_and_parts(cuda_device):
    """Padded leading dimensions in and out (what lies beside the outputs is
    left alone), 32-bit targets, dw in fp32, one gradient without the other."""
    m, k, v = 130, 72, 300
    h, w, t = _inputs(cuda_device, m, k, v, torch.bfloat16, seed=4, ignored=0.1, pad=24)
    assert h.stride(0) == k + 24 and w.stride(0) == k + 24
    dloss = torch.ones(1, device=cuda_device)
    ref = Ref(h, w, t, _row_g(dloss, t, "mean"))
    dh_room = torch.full((m, k + 8), 7.0, dtype=torch.bfloat16, device=cuda_device)
    dw_room = torch.full((v, k + 16), 7.0, device=cuda_device)
    _, stats, dh, dw = _both(h, w, t.int(), dloss, "mean", out=(dh_room[:, :k], dw_room[:, :k]))
    ref.check_grads(dh, dw)
    assert bool((dh_room[:, k:] == 7).all()) and bool((dw_room[:, k:] == 7).all())
    _, _, dh2, none = _both(h, w, t, dloss, "mean", need=(True, False))
    assert none is None and torch.equal(dh2, dh)
    _, _, none, dw2 = _both(h, w, t, dloss, "mean", need=(False, True), dw_dtype=torch.float32)
    assert none is None and torch.equal(dw2, dw)


@pytest.mark.gpu
def test_outputs_of_a_single_row(cuda_device):
    """m = 1 and v = 1: outputs inside a larger buffer are written and nothing
    beside them; ones whose elements do not lie side by side are refused."""
    k = 64
    one = torch.ones(1, device=cuda_device)
    for m, v in ((1, 9), (9, 1)):
        h, w, t = _inputs(cuda_device, m, k, v, torch.bfloat16, seed=m)
        _, stats, dh, dw = _both(h, w, t, one, "sum")
        room = torch.full((40, 2 * k + 8), 7.0, dtype=torch.bfloat16, device=cuda_device)
        _both(h, w, t, one, "sum", out=(room[:m, 8:8 + k], room[20:20 + v, 8:8 + k]))
        assert torch.equal(room[:m, 8:8 + k], dh) and torch.equal(room[20:20 + v, 8:8 + k], dw)
        rest = room.clone()
        rest[:m, 8:8 + k] = rest[20:20 + v, 8:8 + k] = 7.0
        assert bool((rest == 7).all())
        before = room.clone()
        for bad_h, bad_w in ((room[:m, :2 * k:2], torch.empty_like(w)), (torch.empty_like(h), room[:v, :2 * k:2]),
                             (room[:m, :1].expand(m, k), None), (None, room[:v, :1].expand(v, k))):
            with pytest.raises(N.AxonError) as e:
                ops.linear_cross_entropy_grad(h, w, t, stats, one, reduction="sum", out=(bad_h, bad_w))
            assert e.value.code == N.AXON_E_SHAPE
        assert torch.equal(room, before)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_against_differences(dtype, cuda_device):
    """Central differences of the forward loss along random directions that the
    operand type represents exactly (single entries moved by a power of two)."""
    m, k, v = 6, 64, 40
    h, w, t = _inputs(cuda_device, m, k, v, dtype, seed=11, pull=3.0)
    dloss = torch.ones(1, device=cuda_device)
    _, _, dh, dw = _both(h, w, t, dloss, "sum")
    ref = Ref(h, w, t, _row_g(dloss, t, "sum"))

    def loss_at(h, w):
        return float(ops.linear_cross_entropy(h, w, t, reduction="none")[0].double().sum())

    step = 2.0 ** -5
    for x, grad, tol in ((h, dh, ref.dh_tol), (w, dw, ref.dw_tol)):
        for i, j in ((0, 0), (3, 17), (5, 63), (1, 40)):
            up, down = x.clone(), x.clone()
            up[i, j] += step
            down[i, j] -= step
            span = float(up[i, j].double() - down[i, j].double())
            args = ((up, w), (down, w)) if x is h else ((h, up), (h, down))
            diff = (loss_at(*args[0]) - loss_at(*args[1])) / span
            # third derivative of a log-sum-exp along a coordinate: at most the other operand's entry cubed
            other = float((w if x is h else h).double().abs().max())
            curve = (m if x is w else 1) * other ** 3 * span ** 2 / 8
            centre = abs(float((up[i, j].double() + down[i, j].double()) / 2 - x[i, j].double())) * other ** 2 * m
            noise = 2 * m * (2 * ref.ds + E + 8 * U32) / span
            assert abs(diff - float(grad[i, j])) <= curve + centre + noise + float(tol[i, j])


@pytest.mark.gpu
def test_rows_that_do_not_count(cuda_device):
    """Ignored rows may hold NaN and infinities; no row counted gives zero
    gradients (mean: a NaN loss); no rows at all."""
    m, k, v = 300, 64, 500
    h, w, t = _inputs(cuda_device, m, k, v, torch.bfloat16, seed=2, ignored=0.4)
    keep = t != IGNORE
    dloss = torch.ones(1, device=cuda_device)
    loss, _, dh, dw = _both(h, w, t, dloss, "mean")
    bad = h.clone()
    idx = (~keep).nonzero().flatten()
    bad[idx[0]] = float("nan")
    bad[idx[1]] = float("inf")
    bad[idx[2]] = torch.finfo(torch.bfloat16).min
    loss2, stats2, dh2, dw2 = _both(bad, w, t, dloss, "mean")
    assert torch.equal(loss, loss2) and torch.equal(dh, dh2) and torch.equal(dw, dw2)
    assert bool(stats2[0][idx[0]].isnan()) and bool((stats2[1][~keep] == 0).all())
    none = torch.full_like(t, IGNORE)
    loss, stats, dh, dw = _both(bad, w, none, dloss, "mean")
    assert loss.isnan() and not bool(stats[1].any()) and not bool(dh.any()) and not bool(dw.any())
    loss, _, dh, dw = _both(bad, w, none, dloss, "sum")
    assert float(loss) == 0.0 and not bool(dh.any()) and not bool(dw.any())
    for reduction, want in (("sum", 0.0), ("mean", float("nan")), ("none", None)):
        dl = torch.ones(0 if reduction == "none" else 1, device=cuda_device)
        dw_out = torch.full((v, k), 3.0, dtype=torch.bfloat16, device=cuda_device)
        loss, stats = ops.linear_cross_entropy(h[:0], w, t[:0], reduction=reduction)
        dh, dw = ops.linear_cross_entropy_grad(h[:0], w, t[:0], stats, dl, reduction=reduction,
                                               out=(torch.empty_like(h[:0]), dw_out))
        assert stats.shape == (2, 0) and dh.shape == (0, k) and not bool(dw.any())
        assert want is None or float(loss) == want or (math.isnan(want) and loss.isnan())


@pytest.mark.gpu
def test_targets_outside_the_vocabulary(cuda_device):
    m, k, v = 40, 64, 100
    h, w, t = _inputs(cuda_device, m, k, v, torch.bfloat16, seed=6)
    for bad in (-1, v, 2 ** 31, -(2 ** 40)):
        t2 = t.clone()
        t2[5] = bad
        loss, stats = ops.linear_cross_entropy(h, w, t2, reduction="none")
        good = torch.ones(m, dtype=torch.bool, device=cuda_device)
        good[5] = False
        assert loss[5].isnan() and not bool(loss[good].isnan().any()) and not bool(stats[0].isnan().any())
        dh, dw = ops.linear_cross_entropy_grad(h, w, t2, stats, torch.ones(m, device=cuda_device), reduction="none")
        assert bool(dh[5].isnan().all()) and not bool(dh[good].isnan().any()) and bool(dw.isnan().all())
    # another ignored index, inside the vocabulary's range
    t2 = t.clone()
    t2[::3] = 0
    loss, stats = ops.linear_cross_entropy(h, w, t2, ignore_index=0, reduction="none")
    assert bool((loss[t2 == 0] == 0).all()) and bool((loss[t2 != 0] > 0).all())


@pytest.mark.gpu
def test_extreme_logits(cuda_device):
    """Logits of several hundreds (no overflow), an almost certain target (the
    loss keeps its digits), equal logits, and infinities."""
    k, v = 64, 1000
    for dtype in (torch.bfloat16, torch.float16):
        h, w, t = _inputs(cuda_device, 20, k, v, dtype, seed=8)
        big = h * 64
        dloss = torch.ones(1, device=cuda_device)
        _, stats, dh, dw = _both(big, w, t, dloss, "sum")
        ref = Ref(big, w, t, _row_g(dloss, t, "sum"))
        ref.check_loss(stats)
        ref.check_grads(dh, dw)
        # the target's logit is far above: losses down to 1e-12
        w2 = w * 0.1
        w2[3] = 1.0
        h2 = torch.full((4, k), 0.25, device=cuda_device).to(dtype) * torch.arange(1, 5, device=cuda_device).to(
            dtype)[:, None] * 0.5
        t2 = torch.full((4,), 3, device=cuda_device)
        _, stats, dh, dw = _both(h2, w2, t2, dloss, "sum")
        ref = Ref(h2, w2, t2, _row_g(dloss, t2, "sum"))
        assert float(ref.loss.min()) < 1e-9
        ref.check_loss(stats)
        ref.check_grads(dh, dw)
        loss, stats = ops.linear_cross_entropy(torch.zeros_like(h), w, t, reduction="none")
        assert bool(((loss - math.log(v)).abs() <= E).all())
    h = torch.ones(3, k, device=cuda_device).bfloat16()
    w = torch.zeros(v, k, device=cuda_device).bfloat16()
    w[7] = float("-inf")
    loss, stats = ops.linear_cross_entropy(h, w, torch.tensor([0, 7, IGNORE], device=cuda_device), reduction="none")
    assert abs(float(loss[0]) - math.log(v - 1)) <= E and float(loss[1]) == float("inf")
    assert bool(((stats[0] - math.log(v - 1)).abs() <= E).all())
    w[7] = float("inf")
    loss, _ = ops.linear_cross_entropy(h, w, torch.tensor([0, 7, IGNORE], device=cuda_device), reduction="none")
    assert bool(loss[:2].isnan().all()) and float(loss[2]) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("v", [6000, 32000, 128256])
@pytest.mark.parametrize("m", [24, 200])  # the narrow and the wide kernels
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_targets_far_below_a_flat_row(dtype, m, v, cuda_device):
    """Every other word's logit is 0 and the target's is an integer from -66
    down to -255 (exact in either type): the other words' odds, (v - 1) e^x,
    pass fp32's range from x = 77 on, the loss does not."""
    k = 64
    x = torch.cat([torch.arange(66, 88), torch.tensor([127, 255])]).to(cuda_device)
    x = x.repeat(-(-m // len(x)))[:m]
    h = (x / 64).to(dtype)[:, None].expand(m, k).contiguous()
    assert torch.equal(h.double() * 64, x.double()[:, None].expand(m, k))
    w = torch.zeros(v, k, dtype=dtype, device=cuda_device)
    w[v // 2] = -1.0
    t = torch.full((m,), v // 2, device=cuda_device)
    dloss = torch.ones(1, device=cuda_device)
    loss, stats, dh, dw = _both(h, w, t, dloss, "mean")
    ref = Ref(h, w, t, _row_g(dloss, t, "mean"))
    assert bool(torch.isfinite(stats).all()) and bool(loss.isfinite())
    assert abs(float(ref.loss[0]) - 66 - math.log(v - 1)) < 1e-9
    ref.check_loss(stats)
    ref.check_grads(dh, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_an_almost_certain_target_keeps_its_digits(dtype, m, cuda_device):
    """The target's logit is a sum in fp32 lanes, not the tensor core's. Every
    other word's logit is 0 exactly, so the loss log(1 + (v - 1) e^-s) is off by
    the error of s and, relative to itself, by that of expf, a product and
    log1pf (4 ulp in all, 8 half steps). s: products exact in fp32; a lane adds
    k / 256 = 16 of them one after the other, on average onto half of its sum at
    most where no term is negative, and 8 more additions join lanes: 16 / 2 +
    1 + 8 = 17 half steps of the sum. With s of 7 to 13 that is 1.3e-5 at
    most; the tensor core's sum of these (256 steps, each cut off and not
    rounded) is 1.0e-4 off in bf16 and 2.5e-4 in fp16."""
    k, v = 4096, 1000
    g = torch.Generator(device=cuda_device).manual_seed(5)
    h = (0.5 + torch.rand(m, k, device=cuda_device, generator=g)).to(dtype)
    w = torch.zeros(v, k, dtype=dtype, device=cuda_device)
    w[7] = ((0.5 + torch.rand(k, device=cuda_device, generator=g)) * (10.0 / k)).to(dtype)
    t = torch.full((m,), 7, device=cuda_device)
    s = h.double() @ w[7].double()
    assert bool((s > 7).all()) and bool((s < 13).all())
    want = torch.log1p((v - 1) * torch.exp(-s))
    loss, stats = ops.linear_cross_entropy(h, w, t, reduction="none")
    assert bool(((loss.double() - want).abs() <= (17 * s + 8) * U32 * want).all())
    assert bool(((stats[0].double() - s - want).abs() <= (17 * s + 8 * want + s + want) * U32).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m,parts", [(1, 8), (16, 8), (20, 8), (60, 4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_few_rows_add_k_in_parts(dtype, m, parts, cuda_device):
    """Up to 64 rows a logit is a sum of parts over k, added in fp32: each part's
    k / 16 / parts steps are off by at most 2^-23 of the part, as is the module's
    bound for all of k, and joining them by 2^-24 of the sum each time. Rows that
    are ignored take every word from there: one word's logit is 7 to 13 with no
    negative term, the others' are 0. In one part such a logit is 1.0e-4 (bf16)
    and 2.5e-4 (fp16) off."""
    k, v = 4096, 1000
    g = torch.Generator(device=cuda_device).manual_seed(5)
    h = (0.5 + torch.rand(m, k, device=cuda_device, generator=g)).to(dtype)
    w = torch.zeros(v, k, dtype=dtype, device=cuda_device)
    w[7] = ((0.5 + torch.rand(k, device=cuda_device, generator=g)) * (10.0 / k)).to(dtype)
    _, stats = ops.linear_cross_entropy(h, w, torch.full((m,), IGNORE, device=cuda_device), reduction="none")
    s = h.double() @ w[7].double()
    want = torch.logaddexp(s, torch.full_like(s, math.log(v - 1)))
    ds = ((k / 16 / parts + 4) * 2.0 ** -23 + parts * U32) * s
    assert bool(((stats[0].double() - want).abs() <= ds + E + U32 * want).all())


@pytest.mark.gpu
@pytest.mark.parametrize("k", [504, 512, 520, 1000, 1032, 2056, 4104, 8200])
@pytest.mark.parametrize("m", [3, 30, 64])
def test_few_rows_at_the_ends_of_parts(m, k, cuda_device):
    """Hidden sizes around one part, around several, and with a short last one."""
    h, w, t = _inputs(cuda_device, m, k, 700, torch.bfloat16, seed=k, ignored=0.2 if m > 3 else 0.0)
    _, stats = ops.linear_cross_entropy(h, w, t, reduction="none")
    Ref(h, w, t).check_loss(stats)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_only_word(dtype, cuda_device):
    """A vocabulary of one word: its probability is 1 whatever its logit, so the
    loss and both gradients are 0 and the log-sum-exp is the logit. The same
    where every other word's logit is -inf."""
    k = 64
    at = torch.tensor([-255.0, -100.0, -81.0, -79.0, 0.0, 79.0, 81.0, 100.0, 255.0], device=cuda_device)
    for m in (len(at), 150):
        logit = at.repeat(-(-m // len(at)))[:m]
        h = (logit / 64).to(dtype)[:, None].expand(m, k).contiguous()
        w = torch.ones(1, k, dtype=dtype, device=cuda_device)
        t = torch.zeros(m, dtype=torch.int64, device=cuda_device)
        loss, stats, dh, dw = _both(h, w, t, torch.ones(1, device=cuda_device), "sum")
        assert float(loss) == 0.0 and not bool(stats[1].any())
        assert bool(((stats[0] - logit).abs() <= 2 * k * U32 * logit.abs()).all())
        assert not bool(dh.any()) and not bool(dw.any())
        # a second word of -inf against rows of positive entries
        h = h.abs() + 1.0
        w = torch.full((2, k), -math.inf, dtype=dtype, device=cuda_device)
        w[0] = -2.0
        _, stats = ops.linear_cross_entropy(h, w, t)
        want = -2.0 * h.double().sum(dim=1)
        assert not bool(stats[1].any())
        assert bool(((stats[0].double() - want).abs() <= 2 * k * U32 * want.abs()).all())


@pytest.mark.gpu
def test_fp16_scales(cuda_device):
    """fp16 gradients hold at loss scales far from one, and rows of very
    different weight in one call."""
    h, w, t = _inputs(cuda_device, 70, 64, 3000, torch.float16, seed=12, ignored=0.2)
    for s in (2.0 ** -10, 1.0, 2.0 ** 15):
        dloss = torch.full((1,), s, device=cuda_device)
        _, _, dh, dw = _both(h, w, t, dloss, "mean")
        Ref(h, w, t, _row_g(dloss, t, "mean")).check_grads(dh, dw)
    dloss = 10.0 ** torch.linspace(-3, 2, 70, device=cuda_device)
    _, _, dh, dw = _both(h, w, t, dloss, "none")
    Ref(h, w, t, dloss).check_grads(dh, dw)
    dloss[:] = 0
    _, _, dh, dw = _both(h, w, t, dloss, "none")
    assert not bool(dh.any()) and not bool(dw.any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_common_weight_costs_no_digits(dtype, cuda_device):
    """d is rounded before the loss's weight is applied, so the mean's gradient is
    the sum's divided by the count up to fp32 roundings (three: the weight, and
    a product each), whatever the count, and so is any power of the scale."""
    h, w, t = _inputs(cuda_device, 77, 64, 900, dtype, seed=14, ignored=0.1)
    count = int((t != IGNORE).sum())
    one = torch.ones(1, device=cuda_device)
    _, _, _, total = _both(h, w, t, one, "sum", dw_dtype=torch.float32)
    _, _, _, mean = _both(h, w, t, one, "mean", dw_dtype=torch.float32)
    assert bool(((mean.double() * count - total.double()).abs() <= 3 * U32 * total.double().abs()).all())
    _, _, _, odd = _both(h, w, t, one * 0.3, "sum", dw_dtype=torch.float32)
    third = float(torch.tensor(0.3))
    assert bool(((odd.double() / third - total.double()).abs() <= 3 * U32 * total.double().abs()).all())


@pytest.mark.gpu
def test_wider_head(cuda_device):
    """Several tiles in every direction, more tiles than pairs, default piece
    and forced ones, bitwise repeatable."""
    m, k, v = 1111, 1032, 20011
    h, w, t = _inputs(cuda_device, m, k, v, torch.bfloat16, seed=21, ignored=0.5)
    dloss = torch.ones(1, device=cuda_device)
    loss, stats, dh, dw = _both(h, w, t, dloss, "mean")
    ref = Ref(h, w, t, _row_g(dloss, t, "mean"))
    ref.check_loss(stats)
    ref.check_grads(dh, dw)
    again = _both(h, w, t, dloss, "mean")
    for a, b in zip((loss, stats, dh, dw), again):
        assert torch.equal(a, b)
    _, _, dh, dw = _both(h, w, t, dloss, "mean", tune={"split": 4096, "max_ctas": 40})
    ref.check_grads(dh, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("m,split", [(4097, 0), (70001, 0), (70001, 256)])
def test_many_rows(m, split, cuda_device):
    """Rows past a padded batch's: more row tiles than pairs, many rows a CTA in
    the kernels that join and move rows, the vocabulary in one piece and three."""
    k, v = 64, 700
    h, w, t = _inputs(cuda_device, m, k, v, torch.bfloat16, seed=m, ignored=0.3)
    t[:300] = IGNORE
    t[-1] = v - 1
    dloss = torch.randn(m, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(1))
    loss, stats, dh, dw = _both(h, w, t, dloss, "none", tune={"split": split})
    ref = Ref(h, w, t, dloss)
    ref.check_loss(stats)
    ref.check_grads(dh, dw)
    assert torch.equal(loss, stats[1]) and not bool(dh[~ref.keep].any())
    mean, _ = ops.linear_cross_entropy(h, w, t)
    want = float(stats[1].double().sum() / ref.keep.sum())
    assert abs(float(mean) - want) <= 2 * U32 * want


@pytest.mark.gpu
def test_other_stream_and_graph(cuda_device):
    """On a side stream, and captured twice with replays on new values."""
    m, k, v = 200, 128, 1500
    h, w, t = _inputs(cuda_device, m, k, v, torch.bfloat16, seed=31, ignored=0.2)
    dloss = torch.ones(1, device=cuda_device)
    s = torch.cuda.Stream(cuda_device)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = _both(h, w, t, dloss, "mean")
    torch.cuda.current_stream().wait_stream(s)
    here = _both(h, w, t, dloss, "mean")
    for a, b in zip(side, here):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss, stats = ops.linear_cross_entropy(h, w, t)
            grads = ops.linear_cross_entropy_grad(h, w, t, stats, dloss)
        graphs.append((g, loss, stats, *grads))
    for i in range(4):
        hn, _, tn = _inputs(cuda_device, m, k, v, torch.bfloat16, seed=40 + i, ignored=0.1 * i)
        h.copy_(hn)
        t.copy_(tn)
        g, *got = graphs[i % 2]
        g.replay()
        want = _both(h, w, t, dloss, "mean")
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_calls_at_once(cuda_device):
    """Calls in flight on two streams share nothing."""
    h, w, t = _inputs(cuda_device, 300, 128, 3000, torch.bfloat16, seed=51, ignored=0.2)
    dloss = torch.ones(1, device=cuda_device)
    wants = [_both(h[:n], w, t[:n], dloss, "mean") for n in (300, 40)]
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s, n in zip(streams, (300, 40)):
            with torch.cuda.stream(s):
                loss, stats = ops.linear_cross_entropy(h[:n], w, t[:n])
                got.append((loss, stats, *ops.linear_cross_entropy_grad(h[:n], w, t[:n], stats, dloss)))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for a, b in zip(g, wants[i % 2]):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda_device):
    """A head of 2.3e9 entries (offsets past 2^31 elements and 2^32 bytes), with
    few rows and with a row tile; the loss in full, dw in its first and last
    words, dh of one row."""
    k, v = 8192, 280001
    h, w, t = _inputs(cuda_device, 200, k, v, torch.bfloat16, seed=61)
    t[0] = v - 1
    for m in (3, 200):
        dloss = torch.ones(1, device=cuda_device)
        _, stats, dh, dw = _both(h[:m], w, t[:m], dloss, "sum")
        hd = h[:m].double()
        rows = torch.arange(m, device=cuda_device)
        s = torch.cat([hd @ w[i:i + 20000].double().T for i in range(0, v, 20000)], dim=1)
        st = s[rows, t[:m]].clone()
        s[rows, t[:m]] = -math.inf
        rest = torch.logsumexp(s, dim=1)
        loss = torch.logaddexp(rest - st, torch.zeros_like(rest))
        a = float((hd.abs().sum(dim=1) * w.abs().max().double()).max())  # at least sum |h w|
        ds = (k / 16 + 4) * 2.0 ** -23 * a
        assert bool(((stats[1].double() - loss).abs() <= loss.clamp(max=1.0) * (2 * ds + E) + U32 * loss).all())
        d = torch.exp(s - (rest + torch.log1p(torch.exp(st - rest)))[:, None])
        d[rows, t[:m]] = torch.expm1(-loss)
        r = 2 * ds + 2 * E + 2.0 ** -8
        for at in (slice(0, 500), slice(v - 500, v)):
            want, size = d[:, at].T @ hd, d[:, at].abs().T @ hd.abs()
            tol = (r + (m / 16 + 4) * 2.0 ** -23) * size + 2.0 ** -8 * want.abs()
            assert bool(((dw[at].double() - want).abs() <= tol).all())
        want = sum(d[:1, i:i + 20000] @ w[i:i + 20000].double() for i in range(0, v, 20000))
        size = sum(d[:1, i:i + 20000].abs() @ w[i:i + 20000].double().abs() for i in range(0, v, 20000))
        tol = (r + (v / 16 + 68) * 2.0 ** -23) * size + 2.0 ** -8 * want.abs()
        assert bool(((dh[:1].double() - want).abs() <= tol).all())
        del s, d, dw


@pytest.mark.gpu
def test_wrapper_refusals(cuda_device):
    h, w, t = _inputs(cuda_device, 4, 64, 50, torch.bfloat16)
    _, stats = ops.linear_cross_entropy(h, w, t)
    one = torch.ones(1, device=cuda_device)

    def code(f):
        with pytest.raises(N.AxonError) as e:
            f()
        return e.value.code

    assert code(lambda: ops.linear_cross_entropy(h, w[:, :32], t)) == N.AXON_E_SHAPE
    assert code(lambda: ops.linear_cross_entropy(h, w.half(), t)) == N.AXON_E_UNSUPPORTED
    assert code(lambda: ops.linear_cross_entropy(h.float(), w.float(), t)) == N.AXON_E_UNSUPPORTED
    assert code(lambda: ops.linear_cross_entropy(h, w, t[:3])) == N.AXON_E_SHAPE
    assert code(lambda: ops.linear_cross_entropy(h, w, t.float())) == N.AXON_E_UNSUPPORTED
    assert code(lambda: ops.linear_cross_entropy(h, w, t, reduction="max")) == N.AXON_E_ARG
    assert code(lambda: ops.linear_cross_entropy(h[:, 1:57], w[:, 1:57], t)) == N.AXON_E_ALIGN
    assert code(lambda: ops.linear_cross_entropy(h.T, w, t)) == N.AXON_E_SHAPE
    grad = ops.linear_cross_entropy_grad
    assert code(lambda: grad(h, w, t, stats[:, :3], one)) == N.AXON_E_ARG
    assert code(lambda: grad(h, w, t, stats, torch.ones(4, device=cuda_device))) == N.AXON_E_ARG
    assert code(lambda: grad(h, w, t, stats, one, reduction="none")) == N.AXON_E_ARG
    assert code(lambda: grad(h, w, t, stats, one.double())) == N.AXON_E_ARG
    assert code(lambda: grad(h, w, t, stats, one, need=(False, False))) == N.AXON_E_ARG
    assert code(lambda: grad(h, w, t, stats, one, dw_dtype=torch.float16)) == N.AXON_E_ARG
    assert code(lambda: grad(h, w, t, stats, one, tune={"split": 100})) == N.AXON_E_ARG
    assert code(lambda: grad(h, w, t, stats, one, out=(h[:2], w))) == N.AXON_E_ARG
    assert code(lambda: grad(h, w, t, stats, one, out=(h, torch.empty_like(w)))) == N.AXON_E_ARG
    assert code(lambda: grad(h, w, t, stats, one, out=(torch.empty_like(h), w))) == N.AXON_E_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 100, 300])
def test_after_a_wait_gave_up(m, cuda_device):
    """Results are NaN, not whatever the workspace held, until the status has
    been asked for; then they are the same bits as before."""
    h, w, t = _inputs(cuda_device, m, 64, 1500, torch.bfloat16, seed=m)
    one = torch.ones(1, device=cuda_device)
    want = _both(h, w, t, one, "mean")
    stream = torch.cuda.current_stream().cuda_stream
    for tune in (None, {"split": 512}):
        assert N.lib().axon_selftest_linear_ce_gave_up(stream) == N.AXON_OK, N.last_error()
        loss, stats = ops.linear_cross_entropy(h, w, t)
        dh, dw = ops.linear_cross_entropy_grad(h, w, t, want[1], one, tune=tune)
        for x in (loss, stats, dh, dw):
            assert bool(x.isnan().all())
        with pytest.raises(N.AxonError) as e:
            ops.linear_cross_entropy_status(cuda_device)
        assert e.value.code == N.AXON_E_TIMEOUT
        for a, b in zip(_both(h, w, t, one, "mean"), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_given_workspaces(cuda_device):
    """A caller's workspace, of bytes or of another type, gives the same bits;
    one that is no block of memory is refused before anything is launched."""
    h, w, t = _inputs(cuda_device, 40, 64, 500, torch.bfloat16, seed=3, ignored=0.1)
    one = torch.ones(1, device=cuda_device)
    want = _both(h, w, t, one, "mean")
    need = max(N.lib().axon_linear_ce_workspace_bytes(40, 64, 500),
               N.lib().axon_linear_ce_grad_workspace_bytes(40, 64, 500, None))
    for ws in (torch.empty(need, dtype=torch.uint8, device=cuda_device),
               torch.full((need // 4,), float("nan"), device=cuda_device)):
        loss, stats = ops.linear_cross_entropy(h, w, t, workspace=ws)
        dh, dw = ops.linear_cross_entropy_grad(h, w, t, stats, one, workspace=ws)
        for a, b in zip((loss, stats, dh, dw), want):
            assert torch.equal(a, b)
    flat = torch.zeros(1, dtype=torch.uint8, device=cuda_device).expand(need)
    for call in (lambda: ops.linear_cross_entropy(h, w, t, workspace=flat),
                 lambda: ops.linear_cross_entropy_grad(h, w, t, want[1], one, workspace=flat)):
        with pytest.raises(N.AxonError) as e:
            call()
        assert e.value.code == N.AXON_E_SHAPE
