"""Refusals of the operators over a table that need no GPU: shapes and types are looked over before a context is made."""
import ctypes as C

import numpy as np
import pytest

import arrowspace_amd as A
from arrowspace_amd import _lib


def _loss(**changed):
    a = {"x": np.zeros((3, 8), np.float32), "table": np.zeros((5, 8), np.float32), "targets": np.zeros(3, np.int64), "bias": np.zeros(5, np.float32)}
    a.update(changed)
    return a


@pytest.mark.parametrize("changed, error", [
    ({"x": np.zeros(8, np.float32)}, _lib.AS_ERR_SHAPE),
    ({"x": np.zeros((3, 9), np.float32)}, _lib.AS_ERR_SHAPE),
    ({"x": np.zeros((3, 8), np.float64)}, TypeError),
    ({"table": np.zeros((5, 8), np.float16)}, TypeError),
    ({"x": np.zeros((3, 8), np.float64), "table": np.zeros((5, 8), np.float64)}, TypeError),
    ({"targets": np.zeros(3, np.int32)}, TypeError),
    ({"targets": np.zeros(4, np.int64)}, _lib.AS_ERR_SHAPE),
    ({"targets": None}, _lib.AS_ERR_ARG),
    ({"bias": np.zeros(3, np.float32)}, _lib.AS_ERR_SHAPE),
    ({"bias": np.zeros(5, np.float64)}, TypeError),
])
@pytest.mark.parametrize("backward", [False, True])
def test_cross_entropy_refuses(changed, error, backward):
    a = _loss(**changed)

    def call():
        if backward:
            return A.cross_entropy_backward(lse=np.zeros(a["x"].shape[0], np.float32), grad_losses=np.zeros(a["x"].shape[0], np.float32), **a)
        return A.cross_entropy(**a)

    if error is TypeError:
        with pytest.raises(TypeError):
            call()
    else:
        with pytest.raises(A.ArrowSpaceError) as e:
            call()
        assert e.value.status == error


def test_cross_entropy_backward_refuses_its_own_arguments():
    f = np.zeros(3, np.float32)
    for lse, g, ge, error in ((None, f, None, A.ArrowSpaceError), (f, None, None, A.ArrowSpaceError), (f[:2], f, None, A.ArrowSpaceError),
                              (f, f.astype(np.float64), None, TypeError), (f, f, np.zeros(2, np.float32), A.ArrowSpaceError)):
        with pytest.raises(error):
            A.cross_entropy_backward(lse=lse, grad_losses=g, grad_lse=ge, **_loss())


def test_torch_layouts_refused():
    torch = pytest.importorskip("torch")
    y = torch.zeros(3, dtype=torch.int64)
    for x in (torch.zeros(8, 3).t(), torch.zeros(1, 8).expand(3, 8)):
        with pytest.raises(A.ArrowSpaceError) as e:
            A.cross_entropy(x, torch.zeros(5, 8), y)
        assert e.value.status == _lib.AS_ERR_ARG


def test_table4_refuses():
    codes, scales = np.zeros((5, 50), np.uint8), np.zeros((5, 2), np.float32)
    bad = [
        (dict(codes=codes, scales=scales, group=48), _lib.AS_ERR_UNSUPPORTED),
        (dict(codes=codes, scales=scales, dim=98), _lib.AS_ERR_SHAPE),
        (dict(codes=codes, scales=scales, dim=101), _lib.AS_ERR_SHAPE),
        (dict(codes=codes, scales=np.zeros((5, 1), np.float32)), _lib.AS_ERR_SHAPE),
        (dict(codes=codes, scales=scales, zeros=np.zeros((5, 1), np.uint8)), _lib.AS_ERR_SHAPE),
    ]
    for kw, status in bad:
        with pytest.raises(A.ArrowSpaceError) as e:
            A.Table4.from_codes(**kw)
        assert e.value.status == status
    for kw in (dict(codes=codes.astype(np.int8), scales=scales), dict(codes=codes, scales=scales.astype(np.float64)),
               dict(codes=codes, scales=scales, zeros=np.zeros((5, 2), np.int8))):
        with pytest.raises(TypeError):
            A.Table4.from_codes(**kw)
    with pytest.raises(A.ArrowSpaceError):
        A.Table4.pack(np.zeros((4, 64)), group=16)
    with pytest.raises(TypeError):
        A.Table4.pack(np.zeros((4, 64), np.int32))
    with pytest.raises(TypeError):
        A.Table4.pack(np.zeros((4, 64)), scale_dtype="float64")


def test_null_handles():
    lib = A.load()
    assert lib.as_cross_entropy(None, None, 1, 8, None, 5, 8, 8, _lib.AS_F32, None, None, -100, 1.0, None, None, None, 0) == _lib.AS_ERR_ARG
    assert lib.as_cross_entropy_backward(None, None, 1, 8, None, 5, 8, 8, _lib.AS_F32, None, None, -100, 1.0, None, None, None, None, 8, None, 8, None,
                                         None, 0) == _lib.AS_ERR_ARG
    h = C.c_void_p()
    assert lib.as_table4_pack(None, None, 1, 8, 8, _lib.AS_F32, 32, _lib.AS_F32, C.byref(h)) == _lib.AS_ERR_ARG and not h.value
    assert lib.as_table4_import(None, None, None, None, 1, 8, 32, _lib.AS_F32, C.byref(h)) == _lib.AS_ERR_ARG
    assert lib.as_table4_scores(None, None, None, 1, 8, _lib.AS_F32, None, 8, None, 0) == _lib.AS_ERR_ARG
    assert lib.as_table4_export(None, None, None, None, None) == _lib.AS_ERR_ARG
    lib.as_table4_destroy(None)
    assert [lib.as_table4_items(None), lib.as_table4_dim(None), lib.as_table4_group(None), lib.as_table4_scale_dtype(None)] == [0, 0, 0, -1]


def test_workspace_sizes():
    lib = A.load()
    assert lib.as_cross_entropy_workspace(0, 5, 8, _lib.AS_F32, 0) == 0
    assert lib.as_cross_entropy_workspace(4, 5, 8, _lib.AS_F64, 0) == 0
    forward = lib.as_cross_entropy_workspace(8192, 131072, 1024, _lib.AS_BF16, 0)
    backward = lib.as_cross_entropy_workspace(8192, 131072, 1024, _lib.AS_BF16, 1)
    # the point of the pieces: far below the logits (8192 x 131072 x 4 B = 4 GB), images of both matrices (285 MB) included
    assert 0 < forward < 400 << 20 and forward < backward < 1 << 30
