"""Which stream a call of the operators over a table runs on, without a GPU: tensors that say they are on one, a library that notes calls."""
import numpy as np
import pytest

import arrowspace_amd as A
from arrowspace_amd import _lib
from arrowspace_amd import table as T

torch = pytest.importorskip("torch")


class _OnGpu(torch.Tensor):
    is_cuda = True
    device = torch.device("cuda", 0)


def _gpu(a):
    return torch.Tensor._make_subclass(_OnGpu, torch.as_tensor(a))


class _Library:
    def __init__(self, calls):
        self.calls = calls

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            if name.endswith("_workspace") or name in ("as_table4_items", "as_table4_dim", "as_table4_group"):
                return 0
            return _lib.AS_F32 if name == "as_table4_scale_dtype" else _lib.AS_OK
        return call


class _Ctx(A.Context):
    def __init__(self):
        self.device, self.h, self.calls = 0, None, []
        self.lib = _Library(self.calls)

    def set_stream(self, s):
        self.calls.append(("stream", s))
        super().set_stream(s)

    def __del__(self):
        pass


@pytest.fixture
def ctx(monkeypatch):
    T._need_torch()
    monkeypatch.setattr(T, "_raw_stream", lambda index: 4096 + index)
    return _Ctx()


def _arguments():
    return {"x": np.zeros((3, 8), np.float32), "table": np.zeros((5, 8), np.float32), "targets": np.zeros(3, np.int64),
            "bias": np.zeros(5, np.float32), "lse": np.zeros(3, np.float32), "grad_losses": np.zeros(3, np.float32), "grad_lse": np.zeros(3, np.float32)}


@pytest.mark.parametrize("host", ["numpy", "tensor"])
@pytest.mark.parametrize("there", ["table", "targets", "bias", "lse", "grad_losses", "grad_lse"])
def test_a_call_with_one_argument_on_a_gpu_runs_on_its_current_stream(ctx, there, host):
    a = _arguments()
    if host == "tensor":
        a = {k: torch.from_numpy(v) for k, v in a.items()}
    a[there] = _gpu(a[there])
    if there in ("table", "targets", "bias"):
        A.cross_entropy(ctx=ctx, **{k: a[k] for k in ("x", "table", "targets", "bias")})
        assert ctx.calls.index(("stream", 4096)) < ctx.calls.index("as_cross_entropy")
        ctx = _Ctx()
    A.cross_entropy_backward(ctx=ctx, **a)
    assert ctx.calls.index(("stream", 4096)) < ctx.calls.index("as_cross_entropy_backward")


@pytest.mark.parametrize("there", ["scales", "zeros"])
def test_codes_of_the_host_with_scales_on_a_gpu(ctx, there):
    a = {"codes": np.zeros((5, 32), np.uint8), "scales": np.zeros((5, 1), np.float32), "zeros": np.zeros((5, 1), np.uint8)}
    a[there] = _gpu(a[there])
    A.Table4.from_codes(ctx=ctx, **a)
    assert ctx.calls.index(("stream", 4096)) < ctx.calls.index("as_table4_import")


def test_host_memory_alone_moves_no_stream(ctx):
    A.cross_entropy_backward(ctx=ctx, **_arguments())
    assert ctx.calls == ["as_cross_entropy_backward"] or ctx.calls == ["as_cross_entropy_workspace", "as_cross_entropy_backward"]


def test_device_arrays_are_refused_wherever_they_stand(ctx):
    buffer = A.api.DeviceArray.__new__(A.api.DeviceArray)
    buffer.shape, buffer.dtype, buffer._h = (5, 8), np.dtype(np.float32), None
    for name in ("x", "table", "targets", "bias"):
        a = {k: v for k, v in _arguments().items() if k in ("x", "table", "targets", "bias")}
        a[name] = buffer
        with pytest.raises(TypeError):
            A.cross_entropy(ctx=ctx, **a)
    assert ctx.calls == []


def test_a_context_that_its_owner_moved_comes_back_to_the_current_stream(ctx):
    a = _arguments()
    a["table"] = _gpu(a["table"])
    for k in range(3):
        A.cross_entropy_backward(ctx=ctx, **a)
        if k == 0:
            ctx.set_stream(8192)
            ctx.calls.clear()
    # (moved back once, and not again while it is there)
    assert [c for c in ctx.calls if isinstance(c, tuple)] == [("stream", 4096)]
    assert ctx.calls[0] == ("stream", 4096)


def test_tensors_that_require_gradients_get_them(ctx, monkeypatch):
    """The graph reaches the library's backward, with the gradients that are asked for; a table's scores say that they have none."""
    monkeypatch.setattr(T, "_thread_context", lambda device: ctx)
    x, w, b, y = torch.randn(3, 8), torch.randn(5, 8), torch.zeros(5), torch.zeros(3, dtype=torch.int64)
    for a in (x, w, b):
        a.requires_grad_(True)
        for through in (lambda r: r[0].sum(), lambda r: r[1].sum(), lambda r: r[0].sum() + (r[1] ** 2).sum()):
            ctx.calls.clear()
            result = A.cross_entropy(x, w, y, bias=b, ctx=ctx)
            through(result).backward()
            assert ctx.calls[-1] == "as_cross_entropy_backward" and a.grad.shape == a.shape
            a.grad = None
    with torch.no_grad():
        assert not any(t.requires_grad for t in A.cross_entropy(x, w, y, bias=b, ctx=ctx))
    assert not any(t.requires_grad for t in A.cross_entropy(x.detach(), w.detach(), y, ctx=ctx))
    assert all(g is not None for g in A.cross_entropy_backward(x, w, y, torch.zeros(3), torch.zeros(3), bias=b, ctx=ctx))
    with pytest.raises(TypeError):
        A.cross_entropy(x, w, y, scale=torch.tensor(2.0, requires_grad=True), ctx=ctx)
    # targets in host memory beside tensors
    torch.autograd.backward(A.cross_entropy(x, w, y.numpy(), ctx=ctx)[0].sum())
    assert x.grad is not None
    table = A.Table4(ctx, None)
    table.n_items, table.dim = 5, 8
    scores = table.scores(x)
    assert not table.scores(x.detach()).requires_grad and not table.scores(x.detach().numpy()).shape[0] == 0
    with pytest.raises(A.ArrowSpaceError) as e:
        scores.sum().backward()
    assert e.value.status == _lib.AS_ERR_UNSUPPORTED
