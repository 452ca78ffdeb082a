"""The global gradient norm, clipping, and Adam with a clip scale.

The norm is held against float64: squares are formed in fp32 and added in
fp32 chains of at most 11 positive terms before float64 takes over, so the
sum of squares is within 11 roundings (2^-24 each), the norm within half of
that and its own rounding: below 8 x 2^-24. Scaled gradients are held
bit for bit against one fp32 product and one rounding with the norm that
the call returned.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from enzyme_b200 import _native as N
from enzyme_b200 import ops

U32 = 2.0 ** -24
NORM_TOL = 8 * U32
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


# ---- refusals (no GPU) --------------------------------------------------------------


def _lists(ptrs, sizes, dtypes):
    n = len(ptrs)
    return (ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*sizes), (ctypes.c_int32 * n)(*dtypes)


FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: every call below is refused on the host
BIG = 1 << 20


@pytest.mark.parametrize("ptrs,sizes,dtypes,code,text", [
    ([0x10000], [4], [7], N.AXON_E_UNSUPPORTED, "unsupported dtype"),
    ([0x10000], [-1], [0], N.AXON_E_SHAPE, "size out of range"),
    ([0x10000], [1 << 45], [0], N.AXON_E_SHAPE, "size out of range"),
    ([None], [4], [0], N.AXON_E_ARG, "NULL pointer"),
    ([0x10002], [4], [0], N.AXON_E_ALIGN, "not aligned"),
    ([0x10001], [4], [1], N.AXON_E_ALIGN, "not aligned"),
])
def test_bad_lists_are_refused(ptrs, sizes, dtypes, code, text):
    lib = N.lib()
    p, n, d = _lists(ptrs, sizes, dtypes)
    assert lib.axon_grad_norm(p, n, d, 1, 1.0, 0.0, FAKE, None, FAKE, BIG, None) == code
    assert text in N.last_error()
    assert lib.axon_clip_grads(p, p, n, d, 1, 1.0, 0.0, FAKE, FAKE, BIG, None) == code


def test_bad_arguments_are_refused():
    lib = N.lib()
    p, n, d = _lists([0x10000], [4], [0])
    nan = float("nan")
    assert lib.axon_grad_norm(p, n, d, 1, 1.0, 0.0, None, None, FAKE, BIG, None) == N.AXON_E_ARG
    for max_norm, eps in ((-1.0, 0.0), (nan, 0.0), (1.0, -1.0), (1.0, nan)):
        assert lib.axon_grad_norm(p, n, d, 1, max_norm, eps, FAKE, None, FAKE, BIG, None) == N.AXON_E_ARG
        assert lib.axon_clip_grads(p, p, n, d, 1, max_norm, eps, FAKE, FAKE, BIG, None) == N.AXON_E_ARG
    assert lib.axon_grad_norm(None, n, d, 1, 1.0, 0.0, FAKE, None, FAKE, BIG, None) == N.AXON_E_ARG
    assert lib.axon_clip_grads(p, None, n, d, 1, 1.0, 0.0, FAKE, FAKE, BIG, None) == N.AXON_E_ARG
    assert lib.axon_grad_norm(p, n, d, -1, 1.0, 0.0, FAKE, None, FAKE, BIG, None) == N.AXON_E_SHAPE
    assert lib.axon_grad_norm_workspace_bytes(-1) == N.AXON_E_SHAPE
    need = lib.axon_grad_norm_workspace_bytes(1)
    assert need > 0
    assert lib.axon_grad_norm(p, n, d, 1, 1.0, 0.0, FAKE, None, FAKE, need - 1, None) == N.AXON_E_ARG
    assert "workspace" in N.last_error()
    assert lib.axon_grad_norm(p, n, d, 1, 1.0, 0.0, FAKE, None, ctypes.c_void_p(0x10004), need,
                              None) == N.AXON_E_ALIGN


def test_workspace_grows_with_the_launches_a_list_takes():
    lib = N.lib()
    one = lib.axon_grad_norm_workspace_bytes(1)
    assert lib.axon_grad_norm_workspace_bytes(512) == one
    assert lib.axon_grad_norm_workspace_bytes(513) == 2 * one


def test_grad_lists_on_the_host_are_refused():
    with pytest.raises(N.AxonError) as e:
        ops.grad_norm([])
    assert e.value.code == N.AXON_E_SHAPE
    with pytest.raises(N.AxonError) as e:
        ops.grad_norm([torch.zeros(4)])
    assert e.value.code == N.AXON_E_ARG and "CUDA" in e.value.message


def test_parameters_without_a_gradient_are_refused():
    x = torch.zeros(4)
    for call in (lambda: ops.grad_norm([None]), lambda: ops.grad_norm_scale([None, x], 1.0),
                 lambda: ops.clip_grads([None, x], 1.0), lambda: ops.GradList([None], out=[x])):
        with pytest.raises(N.AxonError) as e:
            call()
        assert e.value.code == N.AXON_E_ARG and "None" in e.value.message


def test_dense_memory_in_any_order():
    t = torch.zeros(4, 6, 5)
    assert ops._is_dense(t) and ops._is_dense(t.permute(2, 0, 1)) and ops._is_dense(torch.zeros(()))
    assert ops._is_dense(torch.zeros(0, 3))
    assert not ops._is_dense(t[:, :3]) and not ops._is_dense(t[::2]) and not ops._is_dense(torch.zeros(1).expand(4))


# ---- GPU ----------------------------------------------------------------------------


def _make(dev, shapes, dtypes, seed=0, mag=1e-3):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(mag * (1 + i % 5) * torch.randn(s, device=dev, generator=g)).to(dtypes[i % len(dtypes)])
            for i, s in enumerate(shapes)]


def _norm64(grads):
    return sum(float(t.double().square().sum()) for t in grads) ** 0.5


def _check_norm(got, grads):
    want = _norm64(grads)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - want) <= NORM_TOL * want, (float(got), want)


def _check_clip(grads, out, norm, max_norm, eps=1e-6):
    """Bit for bit, given the norm that came back."""
    scale = torch.clamp(torch.full_like(norm, max_norm) / (norm + eps), max=1.0)
    for t, o in zip(grads, out):
        assert torch.equal(o, (t.float() * scale).to(t.dtype))


SIZES = [0, 1, 2, 7, 8, 9, 15, 16, 17, 255, 4095, 4096, 4097, 8191, 8192, 8193, 70001]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", SIZES)
def test_one_tensor(dtype, n, cuda_device):
    grads = _make(cuda_device, [(n,)], [dtype], seed=n)
    _check_norm(ops.grad_norm(grads), grads)
    before = [t.clone() for t in grads]
    for max_norm in (1e-4, 1e6):
        out, norm = ops.clip_grads(grads, max_norm, out=[torch.empty_like(t) for t in grads])
        _check_norm(norm, before)
        _check_clip(before, out, norm, max_norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 23, 24, 25, 511, 512, 513, 1100])
def test_lists_past_a_table(count, cuda_device):
    """Lists around the table's capacities, types mixed, a few empty tensors;
    in place, and both norm and scale of the split form."""
    shapes = [((i * 37) % 900,) if i % 7 else ((i * 53) % 40, 129) for i in range(count)]
    grads = _make(cuda_device, shapes, DTYPES, seed=count)
    _check_norm(ops.grad_norm(grads), grads)
    norm, scale = ops.grad_norm_scale(grads, 0.05)
    assert torch.equal(scale, torch.clamp(torch.full_like(norm, 0.05) / (norm + 1e-6), max=1.0))
    before = [t.clone() for t in grads]
    out, norm2 = ops.clip_grads(grads, 0.05)
    assert out[0] is grads[0] and torch.equal(norm, norm2)
    _check_clip(before, grads, norm2, 0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_unaligned_starts_and_outputs(dtype, cuda_device):
    """Tensors that start anywhere in a 16-byte packet, outputs that start
    elsewhere in theirs; what lies around an output is left as it was."""
    for off_in in range(0, 9):
        for off_out in (0, 1, 5, off_in):
            base = _make(cuda_device, [(20011,)], [dtype], seed=off_in)[0]
            x = base[off_in:off_in + 19990]
            room = torch.full((20011,), 7.0, dtype=dtype, device=cuda_device)
            o = room[off_out:off_out + 19990]
            _check_norm(ops.grad_norm([x]), [x])
            _, norm = ops.clip_grads([x], 0.01, out=[o])
            _check_clip([x], [o], norm, 0.01)
            assert bool((room[:off_out] == 7).all()) and bool((room[off_out + 19990:] == 7).all())


@pytest.mark.gpu
def test_orders_of_dimensions(cuda_device):
    grads = _make(cuda_device, [(33, 65), (8, 9, 10)], [torch.bfloat16], seed=3)
    views = [grads[0].T, grads[1].permute(2, 0, 1)]
    _check_norm(ops.grad_norm(views), views)
    before = [t.clone() for t in views]
    out, norm = ops.clip_grads(views, 0.01)
    _check_clip(before, out, norm, 0.01)


@pytest.mark.gpu
def test_same_bits_every_time_and_large_list(cuda_device):
    """80 MB and more than one chunk range a CTA: bitwise repeatable."""
    grads = _make(cuda_device, [(4096, 4097), (513, 1025), (7,)] * 2, [torch.bfloat16, torch.float32], seed=5)
    first = ops.grad_norm(grads)
    _check_norm(first, grads)
    for _ in range(3):
        assert torch.equal(ops.grad_norm(grads), first)
    before = [t.clone() for t in grads]
    _, norm = ops.clip_grads(grads, 0.5)
    assert torch.equal(norm, first)
    _check_clip(before, grads, norm, 0.5)


@pytest.mark.gpu
def test_a_tensor_past_32_bits(cuda_device):
    """2^31 + 4099 elements: every one counts, every one is scaled."""
    n = 2 ** 31 + 4099
    x = torch.full((n,), 0.5, dtype=torch.bfloat16, device=cuda_device)
    x[-1] = 2.0
    want = (0.25 * (n - 1) + 4.0) ** 0.5
    out, norm = ops.clip_grads([x], want / 4)
    assert abs(float(norm) - want) <= NORM_TOL * want
    assert float(out[0][-1]) == 0.5
    head, tail = out[0][:2 ** 30], out[0][2 ** 30:-1]
    assert bool((head == 0.125).all()) and bool((tail == 0.125).all())


@pytest.mark.gpu
def test_two_calls_at_once(cuda_device):
    """Calls in flight on two streams share nothing."""
    a = _make(cuda_device, [(3001, 77)] * 30, DTYPES, seed=1)
    b = _make(cuda_device, [(999,)] * 5, DTYPES, seed=2)
    want = [ops.grad_norm(a), ops.grad_norm(b)]
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s, g in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(ops.grad_norm(g))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i % 2]) for i, x in enumerate(got))


@pytest.mark.gpu
def test_nonfinite_and_zero(cuda_device):
    z = [torch.zeros(100, device=cuda_device)]
    norm, scale = ops.grad_norm_scale(z, 1.0)
    assert float(norm) == 0.0 and float(scale) == 1.0
    norm, scale = ops.grad_norm_scale(z, 0.0, eps=0.0)
    assert float(norm) == 0.0 and float(scale) == 1.0
    inf = [torch.tensor([1.0, float("inf")], device=cuda_device), torch.ones(3, device=cuda_device)]
    norm, scale = ops.grad_norm_scale(inf, 1.0)
    assert float(norm) == float("inf") and float(scale) == 0.0
    nan = [torch.ones(3, device=cuda_device), torch.tensor([float("nan")], device=cuda_device)]
    norm, scale = ops.grad_norm_scale(nan, 1.0)
    assert norm.isnan() and scale.isnan()
    out, _ = ops.clip_grads(nan, 1.0)
    assert all(bool(t.isnan().all()) for t in out)
    g = _make(cuda_device, [(1000,)], [torch.float32])
    b = g[0].clone()
    ops.clip_grads(g, float("inf"))
    assert torch.equal(g[0], b)
    ops.clip_grads(g, 0.0)
    assert not bool(g[0].any())


@pytest.mark.gpu
def test_list_refusals(cuda_device):
    x = torch.ones(64, device=cuda_device)

    def code(f):
        with pytest.raises(N.AxonError) as e:
            f()
        return e.value.code

    assert code(lambda: ops.grad_norm([x[::2]])) == N.AXON_E_SHAPE
    assert code(lambda: ops.grad_norm([x[:1].expand(4)])) == N.AXON_E_SHAPE
    assert code(lambda: ops.grad_norm([x.long()])) == N.AXON_E_UNSUPPORTED
    assert code(lambda: ops.grad_norm([x, torch.ones(3)])) == N.AXON_E_ARG
    assert code(lambda: ops.clip_grads([x], 1.0, out=[])) == N.AXON_E_SHAPE
    assert code(lambda: ops.clip_grads([x], 1.0, out=[x[:32]])) == N.AXON_E_SHAPE
    assert code(lambda: ops.clip_grads([x], 1.0, out=[x.half()])) == N.AXON_E_SHAPE
    assert code(lambda: ops.clip_grads([x], -1.0)) == N.AXON_E_ARG
    # the same tensor twice, or an output over another gradient
    assert code(lambda: ops.clip_grads([x, x], 1.0)) == N.AXON_E_ARG
    assert code(lambda: ops.clip_grads([x[:40], x[20:60]], 1.0)) == N.AXON_E_ARG
    assert code(lambda: ops.clip_grads([x[:30]], 1.0, out=[x[10:40]])) == N.AXON_E_ARG
    # but the norm may see a tensor twice, and clipping may read overlapping gradients into outputs of their own
    assert abs(float(ops.grad_norm([x, x])) - 128 ** 0.5) < 1e-5
    o = [torch.empty(40, device=cuda_device), torch.empty(40, device=cuda_device)]
    _, norm = ops.clip_grads([x[:40], x[20:60]], 1.0, out=o)
    _check_clip([x[:40], x[20:60]], o, norm, 1.0)
    lst = ops.GradList([x])
    assert code(lambda: ops.clip_grads(lst, 1.0, out=[x])) == N.AXON_E_ARG
    y = torch.ones(64, device=cuda_device)
    moved = ops.GradList([y])
    ops.grad_norm(moved)
    y.data = torch.ones(64, device=cuda_device)
    assert code(lambda: ops.grad_norm(moved)) == N.AXON_E_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["grads", "out"])
def test_memory_that_is_freed_is_not_taken_for_the_list(which, cuda_device):
    """A listed tensor gives its memory up and gets a smaller one of the same
    kind, which an allocator would serve from the block just freed: the list
    holds that block, so the address differs and the call raises."""
    n = 1 << 20
    x, o = torch.ones(n, device=cuda_device), torch.zeros(n, device=cuda_device)
    lst = ops.GradList([x], out=[o])
    ops.clip_grads(lst, 1.0)
    t = x if which == "grads" else o
    was = t.data_ptr()
    torch.cuda.synchronize()
    for size in (n, n // 2, 100):
        t.data = torch.empty(0, device=cuda_device)
        t.data = torch.ones(size, device=cuda_device)
        assert t.data_ptr() != was
        with pytest.raises(N.AxonError) as e:
            ops.clip_grads(lst, 1.0)
        assert e.value.code == N.AXON_E_ARG and "moved" in e.value.message


@pytest.mark.gpu
def test_other_stream_and_graph(cuda_device):
    """On a side stream, and captured: two graphs of one list replayed with
    other values each time."""
    grads = _make(cuda_device, [(5000,), (300, 41)], [torch.bfloat16, torch.float32], seed=9)
    lst = ops.GradList(grads, out=[torch.empty_like(t) for t in grads])
    s = torch.cuda.Stream(cuda_device)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _, norm = ops.clip_grads(lst, 0.01)
    torch.cuda.current_stream().wait_stream(s)
    _check_norm(norm, grads)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out, nm = ops.clip_grads(lst, 0.01)
        graphs.append((gr, nm))
    for i in range(4):
        for t in grads:
            t.mul_(1.5)
        gr, nm = graphs[i % 2]
        gr.replay()
        _check_norm(nm, grads)
        _check_clip(grads, lst.out, nm, 0.01)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(8, 1024), (5, 77)])  # the vector and the scalar path
@pytest.mark.parametrize("gdt", DTYPES)
def test_adam_with_a_clip_scale(shape, gdt, cuda_device):
    """The same bits as Adam on gradients scaled in fp32 beforehand, and a
    scale of one (or none) leaves Adam as it was."""
    g = torch.Generator(device=cuda_device).manual_seed(1)
    p, gr, m = (torch.randn(shape, device=cuda_device, generator=g) for _ in range(3))
    v = torch.rand(shape, device=cuda_device, generator=g)
    gr = gr.to(gdt)
    _, scale = ops.grad_norm_scale([gr], 0.7)
    assert float(scale) < 0.2
    kw = dict(step_size=1e-3, inv_bc2_sqrt=1.2, wd=0.1)
    got = ops.adam(p, gr, m, v, grad_scale=scale, **kw)
    want = ops.adam(p, gr.float() * scale, m, v, **kw)
    one = ops.adam(p, gr, m, v, grad_scale=torch.ones((), device=cuda_device), **kw)
    none = ops.adam(p, gr, m, v, **kw)
    for a, b, c, d in zip(got, want, one, none):
        assert torch.equal(a, b) and torch.equal(c, d) and not torch.equal(a, d)
    for bad in (torch.ones(2, device=cuda_device), torch.ones((), device=cuda_device).half(), torch.ones(())):
        with pytest.raises(N.AxonError) as e:
            ops.adam(p, gr, m, v, grad_scale=bad, **kw)
        assert e.value.code == N.AXON_E_ARG
