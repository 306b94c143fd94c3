"""Edges of the operators over a table: small rows, far-apart and tiny values, mixed memory, streams, the largest tiles and several pieces.
References in 64 bits; the bounds are those of test_gpu_table.py, whose docstring derives them."""
import pytest

import arrowspace_amd as A
from arrowspace_amd import _lib

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_table import _check4, _inputs, _plain4  # noqa: E402


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40])
def test_scores4_of_short_aligned_f16_rows(d, zeros):
    """Rows of less than a step of 32 columns, read from memory as they lie."""
    for m in (5, 9, 16):
        for v in (1, 17, 300):
            codes, s, z, w = _plain4(v, d, 32, "f16", zeros, m + v + d)
            t = A.Table4.from_codes(codes, s, z, dim=d, group=32)
            x = torch.randn(m, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(m)).half()
            _check4(t, w, x)
            wide = torch.full((m, d + 8), float("nan"), device="cuda", dtype=torch.float16)
            wide[:, :d] = x
            assert torch.equal(t.scores(wide[:, :d]), t.scores(x))


def _busy_write(target, value):
    """`target` is written on the current stream, behind work of some milliseconds there."""
    a = torch.randn(4096, 4096, device="cuda")
    for _ in range(20):
        a = a @ a * 1e-2
    target.copy_(value + a[0, 0].nan_to_num(0.0, 0.0, 0.0).to(value.dtype) * 0)


@pytest.mark.parametrize("host", ["numpy", "tensor"])
def test_rows_in_host_memory_and_a_table_that_is_being_written(host):
    x, w, y, b = _inputs(40, 3000, 64, torch.float32, seed=31, bias=True)
    gl = torch.full((40,), 1 / 40, device="cuda")
    losses, lse = A.cross_entropy(x, w, y, bias=b)
    grads = A.cross_entropy_backward(x, w, y, lse, gl, bias=b)
    here = x.cpu() if host == "tensor" else x.cpu().numpy()
    late = torch.zeros_like(w)
    torch.cuda.synchronize()
    for stream in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            late.zero_()
            _busy_write(late, w)
            got = A.cross_entropy(here, late, y, bias=b)
            late.zero_()
            _busy_write(late, w)
            back = A.cross_entropy_backward(here, late, y, lse, gl, bias=b)
        for a, t in zip(got + back, (losses, lse) + grads):
            assert isinstance(a, torch.Tensor if host == "tensor" else type(here))
            assert torch.equal(torch.as_tensor(a), t.cpu())


def test_codes_in_host_memory_and_scales_that_are_being_written():
    codes, s, z, w = _plain4(900, 128, 64, "f32", False, 32)
    late = torch.zeros_like(s)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        _busy_write(late, s)
        t = A.Table4.from_codes(codes.cpu(), late, dim=128, group=64)
    _check4(t, w, torch.randn(3, 128, device="cuda"))


def _backward(ctx, x, w, y, lse, gl, out, workspace=None):
    n, d = x.shape
    v = w.shape[0]
    rc = ctx.lib.as_cross_entropy_backward(ctx.h, x.data_ptr(), n, d, w.data_ptr(), v, d, d, _lib.AS_BF16, None, y.data_ptr(), -100, 1.0, lse.data_ptr(),
                                           gl.data_ptr(), None, out[0].data_ptr(), d, out[1].data_ptr(), d, None,
                                           None if workspace is None else workspace.data_ptr(), 0 if workspace is None else workspace.numel())
    assert rc == _lib.AS_OK


@pytest.mark.parametrize("first", ["stream", "default"])
def test_scratch_of_a_stream_that_was_left_beside_a_capture(first):
    """Work on one stream with the context's own scratch; a capture on another; work there with the context's scratch, without a switch
    of streams between: each gets what it gets alone."""
    sets = [_inputs(300, 20000, 320, torch.bfloat16, seed=s)[:3] for s in (33, 34, 35)]
    gl = torch.full((300,), 1 / 300, device="cuda")
    lse = [A.cross_entropy(*s)[1] for s in sets]
    want = [A.cross_entropy_backward(*s, l, gl)[:2] for s, l in zip(sets, lse)]
    out = [[torch.zeros_like(t) for t in w] for w in want]
    ctx = A.Context(0)
    one, two = torch.cuda.Stream() if first == "stream" else torch.cuda.default_stream(), torch.cuda.Stream()
    ws = torch.empty(ctx.lib.as_cross_entropy_workspace(300, 20000, 320, _lib.AS_BF16, 1), dtype=torch.uint8, device="cuda")
    late = torch.zeros_like(sets[0][0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(one):
        ctx.set_stream(one.cuda_stream)
        _busy_write(late, sets[0][0])
        _backward(ctx, late, *sets[0][1:], lse[0], gl, out[0])
    with torch.cuda.stream(two):
        graph.capture_begin()
        ctx.set_stream(two.cuda_stream)
        _backward(ctx, *sets[1], lse[1], gl, out[1], ws)
        graph.capture_end()
        _backward(ctx, *sets[2], lse[2], gl, out[2])
        graph.replay()
    torch.cuda.synchronize()
    for got, w in zip(out, want):
        assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
    ctx.set_stream(one.cuda_stream)
    _backward(ctx, *sets[1], lse[1], gl, out[0])
    torch.cuda.synchronize()
    assert torch.equal(out[0][0], want[1][0]) and torch.equal(out[0][1], want[1][1])


def test_a_table_freed_while_a_stream_left_beside_a_capture_reads_it():
    v, d = 200_000, 256
    codes, s, _, _ = _plain4(v, d, 64, "f16", False, 36)
    other = codes.flip(0).contiguous()
    x = torch.randn(3, d, device="cuda")
    ctx = A.Context(0)
    t = A.Table4.from_codes(codes, s, dim=d, group=64)
    keep = A.Table4.from_codes(other, s, dim=d, group=64)
    want = t.scores(x)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    late = torch.zeros_like(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(one):
        _busy_write(late, x)
        got = t.scores(late, ctx=ctx)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(two):
        graph.capture_begin()
        out = keep.scores(x, ctx=ctx)
        graph.capture_end()
    del t
    fresh = [A.Table4.from_codes(other, s, dim=d, group=64) for _ in range(2)]
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, keep.scores(x)) and torch.equal(out, fresh[0].scores(x)) and torch.equal(out, fresh[1].scores(x))
