"""Edges of the operators over a table: small rows, far-apart and tiny values, mixed memory, streams, the largest tiles and several pieces.
References in 64 bits; the bounds are those of test_gpu_table.py, whose docstring derives them."""
import pytest

import arrowspace_amd as A

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
