"""Softmax cross entropy against a table and products with a table in 4 bits, against plain formulas in 64 bits.

Bounds.  u = finfo(type).eps / 2 is half a step of the inputs' type, e = 2^-24 that of float32.
  logits   a product of d terms summed in f32: off by at most (d + 8) e sum |x w|; f32 inputs go in as 22 bits: another 2 * 2^-22.
  lse      the largest error of a logit, and a few roundings of its own value.
  g        relative error of exp: the logit's and the lse's error; rounded to the inputs' type (f32: to 22 bits and 2^-38 of the
           largest coefficient): u |g|.
  grads    scale (error of g) times |w| or |x|, the f32 sum over n terms ((n + 8) e), and the rounding of the result, u.
"""
import threading

import numpy as np
import pytest

import arrowspace_amd as A
from arrowspace_amd import _lib

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E = 2.0 ** -24


def _half_step(dt):
    return torch.finfo(dt).eps / 2


def _inputs(n, v, d, dt, seed=0, pad=0, offset=0, bias=False, ignored=0.0, spread=1.0, device="cuda"):
    """x and table as rows of wider tensors, `offset` elements into their rows."""
    g = torch.Generator().manual_seed(seed)
    table = torch.randn(v, d, generator=g) * (spread / d ** 0.5)
    y = torch.randint(0, v, (n,), generator=g)
    x = torch.randn(n, d, generator=g) + 2 * table[y]

    def wide(a):
        w = torch.full((a.shape[0], d + pad), 7.0)
        w[:, offset:offset + d] = a
        return w.to(dt).to(device)[:, offset:offset + d]

    y[torch.rand(n, generator=g) < ignored] = -100
    b = (torch.randn(v, generator=g)).to(device) if bias else None
    return wide(x), wide(table), y.to(device), b


def _reference(x, w, y, b, scale, gl=None, ge=None, ignore=-100):
    """Everything in f64, with the bounds of the module's docstring."""
    dt = x.dtype
    u = _half_step(dt)
    d = x.shape[1]
    X, W = x.double(), w.double()
    n, v = X.shape[0], W.shape[0]
    size = abs(scale) * (X.abs() @ W.abs().t().contiguous())
    z = scale * (X @ W.t().contiguous())
    if b is not None:
        z = z + b.double()
        size = size + b.double().abs().nan_to_num(posinf=0, neginf=0)
    dz = ((d + 8) * E + (2.0 ** -21 if dt == torch.float32 else 0)) * size
    lse = torch.logsumexp(z, dim=1)
    there = (y != ignore) & (y >= 0) & (y < v)
    at = y.clamp(0, v - 1)
    hit = z.gather(1, at[:, None])[:, 0]
    empty = lse == -float("inf")
    loss = torch.where(there & ~empty, lse - hit, torch.zeros_like(lse))
    d_lse = dz.max(dim=1).values + 8 * E * (lse.abs().nan_to_num(posinf=0, neginf=0) + 1)
    out = {"lse": (lse, d_lse), "losses": (loss, 2 * d_lse + 8 * E * (loss.abs().nan_to_num(posinf=0) + hit.abs().nan_to_num(neginf=0)))}
    if gl is None:
        return out
    gl = torch.where(there & ~empty, gl.double(), torch.zeros_like(lse))
    every = gl + (0 if ge is None else ge.double())
    every = torch.where(empty, torch.zeros_like(every), every)
    p = torch.exp(z - lse[:, None]).nan_to_num(nan=0.0)
    p = torch.where(empty[:, None], torch.zeros_like(p), p)
    g = every[:, None] * p
    g[torch.arange(n, device=x.device), at] -= gl
    coefficient = torch.maximum(every.abs().max(), gl.abs().max()) if n else torch.zeros(())
    exp_err = dz + d_lse[:, None] + 8 * E * (z - lse[:, None]).abs().nan_to_num(nan=0, posinf=0) + 8 * E
    dg = every.abs()[:, None] * p * exp_err + 2 * E * g.abs()
    dg_bias = dg.clone()
    dg = dg + (2.0 ** -22 * g.abs() + 2.0 ** -38 * coefficient if dt == torch.float32 else u * g.abs() + (2.0 ** -38 * coefficient if dt == torch.float16 else 0))
    small = torch.finfo(dt).tiny
    aX, aW = X.abs(), W.abs()
    split = 2.0 ** -21 if dt == torch.float32 else 0.0
    out["grad_x"] = (scale * (g @ W), abs(scale) * (dg @ aW) + abs(scale) * ((v + 64) * E + split) * (g.abs() @ aW) + u * (scale * (g @ W)).abs() + small)
    gt = g.t().contiguous()
    out["grad_table"] = (scale * (gt @ X), abs(scale) * (dg.t().contiguous() @ aX) + abs(scale) * ((n + 64) * E + split) * (gt.abs() @ aX) +
                         u * (scale * (gt @ X)).abs() + small)
    out["grad_bias"] = (g.sum(0), dg_bias.sum(0) + (n + 64) * E * g.abs().sum(0) + 1e-38)
    return out


def _close(got, want, bound, what):
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine].nan_to_num(nan=5.0), want[~fine].nan_to_num(nan=5.0)), what
    off = (got - want).abs()[fine] - bound.expand_as(want)[fine] if want.numel() else torch.zeros(0)
    if off.numel():
        worst = off.max().item()
        assert worst <= 0, "%s: %g above its bound" % (what, worst)


def _check(x, w, y, b, scale=4.0, gl=None, ge=None, ignore=-100):
    losses, lse = A.cross_entropy(x, w, y, bias=b, scale=scale, ignore_index=ignore)
    if gl is None:
        gl = torch.linspace(0.5, 1.5, max(1, x.shape[0]), device=x.device)[:x.shape[0]] / max(1, x.shape[0])
    want = _reference(x, w, y, b, scale, gl, ge, ignore)
    _close(lse, *want["lse"], "lse")
    _close(losses, *want["losses"], "losses")
    grads = A.cross_entropy_backward(x, w, y, lse, gl, bias=b, scale=scale, grad_lse=ge, ignore_index=ignore)
    _close(grads[0], *want["grad_x"], "grad_x")
    _close(grads[1], *want["grad_table"], "grad_table")
    assert grads[0].dtype == x.dtype and grads[1].dtype == w.dtype
    if b is None:
        assert grads[2] is None
    else:
        _close(grads[2], *want["grad_bias"], "grad_bias")
    return losses, lse, grads


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, v, d", [(1, 1, 1), (1, 2, 64), (2, 255, 128), (3, 257, 65), (16, 1000, 64), (64, 300, 128), (65, 511, 200),
                                     (129, 1025, 100), (300, 2000, 72), (257, 700, 384), (1, 5000, 1000)])
def test_cross_entropy_sizes(n, v, d, dt):
    x, w, y, _ = _inputs(n, v, d, TYPES[dt], seed=n + v + d)
    _check(x, w, y, None)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, v, d, pad, offset", [(5, 300, 64, 8, 0), (70, 1000, 128, 3, 1), (130, 600, 96, 32, 8), (200, 999, 40, 24, 24)])
def test_cross_entropy_bias_strides_ignored(n, v, d, pad, offset, dt):
    x, w, y, b = _inputs(n, v, d, TYPES[dt], seed=n, pad=pad, offset=offset, bias=True, ignored=0.3)
    _check(x, w, y, b, scale=3.0, ge=torch.full((n,), 1e-3, device="cuda"))


@pytest.mark.parametrize("dt", list(TYPES))
def test_cross_entropy_large_tile(dt):
    x, w, y, b = _inputs(600, 45003, 64, TYPES[dt], seed=5, bias=dt == "f32")
    _check(x, w, y, b)


def test_cross_entropy_pieces_of_the_table():
    # 512 MB of logit gradients at most: 600 padded rows x 4 B -> some 170 k items a piece
    x, w, y, _ = _inputs(600, 400001, 32, torch.bfloat16, seed=6)
    _check(x, w, y, None)


@pytest.mark.parametrize("scale", [-2.0, 0.0])
def test_cross_entropy_scale_not_positive(scale):
    x, w, y, _ = _inputs(33, 400, 64, torch.float32, seed=7)
    _check(x, w, y, None, scale=scale)


def test_cross_entropy_large_logits():
    # the running maximum: logits of some thousands, most probabilities 0
    x, w, y, _ = _inputs(40, 3000, 64, torch.float32, seed=8, spread=30.0)
    _check(x, w, y, None, scale=10.0)


def test_cross_entropy_small_and_far_apart_values_f32():
    # a power of two per matrix: rows 2^20 apart, and a matrix of tiny values
    x, w, y, _ = _inputs(20, 500, 64, torch.float32, seed=9)
    _check(x * 1e-20, w * 1e20, y, None)
    w = w.clone()
    w[:250] *= 2.0 ** -12
    losses, lse = A.cross_entropy(x, w, y)
    _close(lse, *_reference(x, w, y, None, 1.0)["lse"], "lse")


@pytest.mark.parametrize("masked", ["some", "target", "all"])
def test_cross_entropy_masked_items(masked):
    x, w, y, b = _inputs(70, 600, 64, torch.bfloat16, seed=10, bias=True)
    b[:300] = -float("inf")
    y = y.clone()
    y[:] = 300 + y % 300
    if masked == "target":
        y[3] = 7
    if masked == "all":
        b[:] = -float("inf")
    losses, lse, grads = _check(x, w, y, b)
    if masked == "target":
        assert losses[3].item() == float("inf")
    if masked == "all":
        assert torch.all(lse == -float("inf")) and not losses.any() and not any(g.any() for g in grads)
    else:
        assert not grads[1][:300][torch.arange(300, device="cuda") != 7].any()


def test_cross_entropy_lowest_value_as_a_mask():
    x, w, y, b = _inputs(70, 600, 64, torch.float32, seed=11, bias=True)
    b[:500] = torch.finfo(torch.float32).min
    y = 500 + y % 100
    _check(x, w, y, b)
    b[:] = torch.finfo(torch.float32).min       # every item the same: the lowest value is no mask then
    losses, lse = A.cross_entropy(x, w, y, bias=b)
    assert torch.isfinite(losses).all()


def test_cross_entropy_nan_stays_in_its_row():
    x, w, y, _ = _inputs(80, 600, 64, torch.float32, seed=12)
    x = x.clone()
    x[5, 3] = float("nan")
    x[6, 3] = float("inf")
    losses, lse = A.cross_entropy(x, w, y)
    bad = torch.zeros(80, dtype=torch.bool, device="cuda")
    bad[5:7] = True
    assert torch.equal(torch.isfinite(lse), ~bad)
    clean, _ = A.cross_entropy(x[7:], w, y[7:])
    assert torch.allclose(losses[7:], clean, rtol=1e-5)


def test_cross_entropy_targets_outside():
    x, w, y, _ = _inputs(10, 50, 64, torch.float32, seed=13)
    y = y.clone()
    y[2], y[4] = 50, -3
    losses, lse = A.cross_entropy(x, w, y)
    assert torch.isnan(losses[[2, 4]]).all() and torch.isfinite(lse).all() and torch.isnan(losses).sum() == 2
    gx, gw, _ = A.cross_entropy_backward(x, w, y, lse, torch.ones(10, device="cuda"))
    assert not gx[[2, 4]].any() and torch.isfinite(gw).all()
    with pytest.raises(A.ArrowSpaceError) as e:
        A.cross_entropy(x.cpu().numpy(), w.cpu().numpy(), y.cpu().numpy())
    assert e.value.status == _lib.AS_ERR_ARG


def test_cross_entropy_no_rows():
    x, w, y, b = _inputs(4, 50, 64, torch.bfloat16, seed=14, bias=True)
    losses, lse = A.cross_entropy(x[:0], w, y[:0])
    assert losses.shape == (0,) and lse.shape == (0,)
    gx, gw, gb = A.cross_entropy_backward(x[:0], w, y[:0], lse, losses, bias=b)
    assert gx.shape == (0, 64) and gw.shape == (50, 64) and not gw.any() and not gb.any()


def test_cross_entropy_parts_of_the_gradient_and_repeats():
    x, w, y, b = _inputs(300, 3000, 128, torch.bfloat16, seed=15, bias=True)
    losses, lse, (gx, gw, gb) = _check(x, w, y, b)
    gl = torch.linspace(0.5, 1.5, 300, device="cuda") / 300
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        got = A.cross_entropy_backward(x, w, y, lse, gl, bias=b, scale=4.0, need_x=need[0], need_table=need[1], need_bias=need[2])
        for g, all_of_it, n in zip(got, (gx, gw, gb), need):
            assert (g is not None) == n and (not n or torch.equal(g, all_of_it))


def test_cross_entropy_gradient_against_differences():
    x, w, y, b = _inputs(12, 90, 40, torch.float32, seed=16, bias=True)
    gl, ge = torch.rand(12, device="cuda"), torch.rand(12, device="cuda") * 0.1
    _, lse = A.cross_entropy(x, w, y, bias=b)
    gx, gw, gb = A.cross_entropy_backward(x, w, y, lse, gl, bias=b, grad_lse=ge)

    def value(x, w, b):
        z = x.double() @ w.double().t() + b.double()
        s = torch.logsumexp(z, 1)
        return ((s - z.gather(1, y[:, None])[:, 0]) * gl.double() + s * ge.double()).sum()

    g = torch.Generator(device="cuda").manual_seed(1)
    for which, grad in ((0, gx), (1, gw), (2, gb)):
        a = [x.double(), w.double(), b.double()]
        step = torch.randn(grad.shape, device="cuda", generator=g, dtype=torch.float64)
        h = 1e-5
        up, down = list(a), list(a)
        up[which], down[which] = a[which] + h * step, a[which] - h * step
        slope = ((value(*up) - value(*down)) / (2 * h)).item()
        # differences: O(h^2) and 1e-16 / h; the gradient: f32
        assert abs(slope - (grad.double() * step).sum().item()) <= 1e-5 * (grad.double().abs() * step.abs()).sum().item() + 1e-8


def test_cross_entropy_host_arrays():
    x, w, y, b = _inputs(40, 300, 50, torch.float32, seed=17, bias=True, device="cpu")
    losses, lse = A.cross_entropy(x.numpy(), w.numpy(), y.numpy(), bias=b.numpy(), scale=2.0)
    gl = np.full(40, 1 / 40, np.float32)
    grads = A.cross_entropy_backward(x.numpy(), w.numpy(), y.numpy(), lse, gl, bias=b.numpy(), scale=2.0)
    cuda = [t.cuda() for t in (x, w, y, b)]
    l2, s2 = A.cross_entropy(*cuda[:3], bias=cuda[3], scale=2.0)
    g2 = A.cross_entropy_backward(*cuda[:3], s2, torch.from_numpy(gl).cuda(), bias=cuda[3], scale=2.0)
    for a, t in ((losses, l2), (lse, s2), (grads[0], g2[0]), (grads[1], g2[1]), (grads[2], g2[2])):
        assert isinstance(a, np.ndarray) and np.array_equal(a, t.cpu().numpy())


def _replays(make, inputs, rounds=3):
    """A captured call, replayed on changed inputs with eager work between, against the eager call."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        make()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = make()
    for r in range(rounds):
        for t in inputs:
            t.copy_(t * 0.75 + 0.01 * r)
        graph.replay()
        torch.cuda.synchronize()
        eager = make()
        for a, b in zip(out, eager):
            assert torch.equal(a, b), r
    return graph


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_cross_entropy_captured(dt):
    x, w, y, b = _inputs(200, 1500, 96, TYPES[dt], seed=18, bias=True)
    gl = torch.full((200,), 1 / 200, device="cuda")

    def step():
        losses, lse = A.cross_entropy(x, w, y, bias=b, scale=2.0)
        return (losses, lse) + A.cross_entropy_backward(x, w, y, lse, gl, bias=b, scale=2.0)

    _replays(step, (x, w, b))


def test_two_graphs_at_once():
    """Two captured steps replayed on two streams at the same time: each has its own workspace."""
    sets = [_inputs(300, 4000, 64, torch.bfloat16, seed=s) for s in (19, 20)]
    gl = torch.full((300,), 1 / 300, device="cuda")

    def step(k):
        x, w, y, _ = sets[k]
        losses, lse = A.cross_entropy(x, w, y)
        return (losses,) + A.cross_entropy_backward(x, w, y, lse, gl)[:2]

    eager = [step(0), step(1)]
    graphs, outs = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(k))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, eager):
        for t, u in zip(a, b):
            assert torch.equal(t, u)


def test_capture_without_a_workspace_is_refused():
    import ctypes as C
    x, w, y, _ = _inputs(8, 100, 64, torch.bfloat16, seed=21)
    out = torch.empty(8, device="cuda")
    lse = torch.empty(8, device="cuda")
    ctx = A.Context(0)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        graph.capture_begin()
        ctx.set_stream(stream.cuda_stream)
        rc = ctx.lib.as_cross_entropy(ctx.h, x.data_ptr(), 8, 64, w.data_ptr(), 100, 64, 64, _lib.AS_BF16, None, y.data_ptr(), -100, 1.0, out.data_ptr(),
                                      lse.data_ptr(), None, 0)
        out.zero_()
        graph.capture_end()
    assert rc == _lib.AS_ERR_UNSUPPORTED
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    need = ctx.lib.as_cross_entropy_workspace(8, 100, 64, _lib.AS_BF16, 0)
    small = torch.empty(need, dtype=torch.uint8, device="cuda")
    args = (ctx.h, x.data_ptr(), 8, 64, w.data_ptr(), 100, 64, 64, _lib.AS_BF16, None, y.data_ptr(), -100, 1.0, out.data_ptr(), lse.data_ptr())
    assert ctx.lib.as_cross_entropy(*args, small.data_ptr(), 16) == _lib.AS_ERR_ARG
    assert ctx.lib.as_cross_entropy(*args, small.data_ptr() + 8, need) == _lib.AS_ERR_ARG
    assert ctx.lib.as_cross_entropy(*args, small.data_ptr(), need) == _lib.AS_OK
    assert ctx.lib.as_cross_entropy(*args, None, 0) == _lib.AS_OK
    for wrong in ({8: 7}, {3: 63}, {6: 63}, {12: float("inf")}, {5: 0}):
        a = list(args)
        for k, val in wrong.items():
            a[k] = val
        assert ctx.lib.as_cross_entropy(*a, None, 0) in (_lib.AS_ERR_ARG, _lib.AS_ERR_SHAPE), wrong
    torch.cuda.synchronize()


def test_streams_and_threads():
    sets = [_inputs(130, 2000, 64, torch.float32, seed=s) for s in range(22, 26)]
    want = [A.cross_entropy(x, w, y) for x, w, y, _ in sets]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(k):
        x, w, y, _ = sets[k]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[k] = A.cross_entropy(x, w, y)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- the table in 4 bits ----------------------------------------------------------------------------------------------------------------
def _plain4(v, d, group, scales, zeros, seed):
    g = torch.Generator().manual_seed(seed)
    groups = (d + group - 1) // group
    codes = torch.randint(0, 256, (v, (d + 1) // 2), generator=g, dtype=torch.uint8)
    s = (torch.rand(v, groups, generator=g) + 0.1).to(TYPES[scales])
    z = torch.randint(0, 16, (v, groups), generator=g, dtype=torch.uint8) if zeros else None
    q = torch.stack((codes & 15, codes >> 4), 2).flatten(1)[:, :d].double()
    at = torch.arange(d) // group
    w = (q - (8 if z is None else z.double()[:, at])) * s.double()[:, at]
    return codes.cuda(), s.cuda(), None if z is None else z.cuda(), w.cuda()


def _check4(t, w, x):
    got = t.scores(x)
    X = x.double()
    want = X @ w.t().contiguous()
    size = X.abs() @ w.abs().t().contiguous()
    d = x.shape[1]
    # products summed in f32 with codes of up to 15 against a row brought to a power of two (f32: 22 bits), the rounding of the result
    bound = ((d + 16) * E + (2.0 ** -22 if x.dtype == torch.float32 else 0)) * size + _half_step(x.dtype) * want.abs() + torch.finfo(x.dtype).tiny
    assert got.dtype == x.dtype and got.shape == want.shape
    _close(got, want, bound, "scores")
    return got


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("m, v, d, group, scales, zeros", [
    (1, 1, 1, 32, "f32", False), (1, 17, 31, 32, "bf16", True), (1, 317, 128, 64, "f32", False), (2, 33, 129, 128, "f16", True),
    (4, 1000, 257, 32, "bf16", False), (5, 100, 256, 64, "f16", True), (16, 513, 1000, 128, "bf16", True), (17, 65, 300, 32, "f32", False),
    (33, 200, 500, 64, "bf16", False), (64, 129, 640, 128, "f32", True), (130, 70, 200, 64, "f16", False), (1, 50, 8000, 128, "bf16", True),
    (7, 48, 8100, 32, "f16", False), (64, 40, 5000, 64, "bf16", True), (20, 90, 2500, 128, "f32", False), (3, 40000, 96, 32, "f32", True)])
def test_scores4(m, v, d, group, scales, zeros, dt):
    codes, s, z, w = _plain4(v, d, group, scales, zeros, m + v + d)
    t = A.Table4.from_codes(codes, s, z, dim=d, group=group)
    g = torch.Generator(device="cuda").manual_seed(d)
    x = torch.randn(m, d + 5, device="cuda", generator=g).to(TYPES[dt])[:, 2:2 + d]
    _check4(t, w, x)
    out = t.to_codes()
    assert np.array_equal(out[0] if d % 2 == 0 else out[0][:, :-1], (codes if d % 2 == 0 else codes[:, :-1]).cpu().numpy())
    assert np.array_equal(out[1].astype(np.float64), s.double().cpu().numpy())
    assert np.array_equal(out[2], np.full(s.shape, 8, np.uint8) if z is None else z.cpu().numpy())


@pytest.mark.parametrize("dt", list(TYPES))
def test_scores4_rows_of_any_magnitude(dt):
    codes, s, z, w = _plain4(300, 200, 64, "f32", False, 1)
    t = A.Table4.from_codes(codes, s, z, dim=200, group=64)
    x = torch.randn(6, 200, device="cuda")
    x[1] *= 1e-30 if dt != "f16" else 1e-3
    x[2] *= 1e30 if dt != "f16" else 1e2
    x[3] = 0
    x[4, ::2] *= 2.0 ** -10
    _check4(t, w, x.to(TYPES[dt]))


@pytest.mark.parametrize("dt", list(TYPES))
def test_scores4_not_finite(dt):
    """An infinity or a NaN of a row stays in that row, and is what the formula gives."""
    codes, s, z, w = _plain4(100, 64, 32, "f32", True, 2)
    t = A.Table4.from_codes(codes, s, z, dim=64, group=32)
    x = torch.randn(5, 64, device="cuda").to(TYPES[dt])
    x[1, 7] = float("inf")
    x[3, 9] = float("nan")
    got = t.scores(x)
    keep = [0, 2, 4]
    assert torch.equal(got[keep], t.scores(x[keep].contiguous()))
    assert torch.isnan(got[3]).all()
    column = w[:, 7]
    assert torch.equal(torch.isnan(got[1]), column == 0) and torch.equal(got[1] == float("inf"), column > 0)


def test_scores4_one_row_and_host_arrays():
    codes, s, z, w = _plain4(90, 70, 32, "f32", False, 3)
    t = A.Table4.from_codes(codes.cpu().numpy(), s.cpu().numpy(), dim=70, group=32)
    x = np.random.default_rng(0).standard_normal((3, 70)).astype(np.float32)
    got = t.scores(x)
    assert isinstance(got, np.ndarray) and np.array_equal(got, t.scores(torch.from_numpy(x).cuda()).cpu().numpy())
    assert np.array_equal(t.scores(x[1]), t.scores(x[1:2])[0])
    assert t.scores(torch.zeros(0, 70, device="cuda")).shape == (0, 90)
    with pytest.raises(A.ArrowSpaceError) as e:
        t.scores(x[:, :60])
    assert e.value.status == _lib.AS_ERR_DIM
    with pytest.raises(TypeError):
        t.scores(x.astype(np.float64))
    with pytest.raises(A.ArrowSpaceError) as e:
        A.Table4.from_codes(codes, s, torch.full(s.shape, 16, dtype=torch.uint8, device="cuda"), dim=70, group=32)
    assert e.value.status == _lib.AS_ERR_ARG


@pytest.mark.parametrize("dt", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("scales", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("v, d, group", [(5, 7, 32), (100, 128, 64), (33, 300, 128)])
def test_pack4(v, d, group, scales, dt):
    kind = torch.float64 if dt == "f64" else TYPES[dt]
    rows = torch.randn(v, d + 3, device="cuda", dtype=torch.float64).to(kind)[:, 1:1 + d]
    rows[0] = 0
    t = A.Table4.pack(rows, group=group, scale_dtype=scales)
    codes, s, z = t.to_codes()
    a = rows.float().cpu()
    groups = (d + group - 1) // group
    padded = torch.zeros(v, groups * group)
    padded[:, :d] = a
    parts = padded.view(v, groups, group)
    want_s = (parts.abs().amax(2) / 7).to(getattr(torch, scales)).float()
    assert np.array_equal(s.astype(np.float32), want_s.numpy()) and (z == 8).all()
    q = torch.where(want_s[:, :, None] > 0, (parts / want_s[:, :, None]).round().clamp(-8, 7), torch.zeros(())).nan_to_num(0) + 8
    q = q.view(v, -1)[:, :d].to(torch.uint8)
    if d % 2:
        q = torch.cat((q, torch.zeros(v, 1, dtype=torch.uint8)), 1)
    assert np.array_equal(codes, (q[:, ::2] | q[:, 1::2] << 4).numpy())


def test_pack4_refuses_what_is_not_finite():
    rows = torch.randn(10, 64, device="cuda")
    for bad in (float("nan"), float("inf")):
        rows[3, 5] = bad
        with pytest.raises(A.ArrowSpaceError) as e:
            A.Table4.pack(rows)
        assert e.value.status == _lib.AS_ERR_NONFINITE
    rows[3, 5] = 1e30
    with pytest.raises(A.ArrowSpaceError) as e:
        A.Table4.pack(rows, scale_dtype="float16")
    assert e.value.status == _lib.AS_ERR_UNSUPPORTED
    A.Table4.pack(rows, scale_dtype="bfloat16")


def test_scores4_captured():
    codes, s, z, w = _plain4(3000, 256, 64, "bf16", False, 4)
    t = A.Table4.from_codes(codes, s, dim=256, group=64)
    x = torch.randn(5, 256, device="cuda")
    _replays(lambda: (t.scores(x),), (x,))
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(A.ArrowSpaceError) as e:
            A.Table4.from_codes(codes, s, dim=256, group=64)
    assert e.value.status == _lib.AS_ERR_UNSUPPORTED


def test_train_then_serve():
    """The operators together: a table trained with the loss, held in 4 bits, scored by single queries; ArrowSpace items packed."""
    g = torch.Generator(device="cuda").manual_seed(5)
    v, d, n = 2000, 128, 512
    table = torch.randn(v, d, device="cuda", generator=g) * 0.02
    hidden = torch.nn.functional.normalize(torch.randn(v, d, device="cuda", generator=g), dim=1)
    for step in range(30):
        y = torch.randint(0, v, (n,), device="cuda", generator=g)
        x = hidden[y]
        losses, lse = A.cross_entropy(x, table, y, scale=8.0)
        gl = torch.full((n,), 1.0 / n, device="cuda")
        gx, gw, _ = A.cross_entropy_backward(x, table, y, lse, gl, scale=8.0)
        z = (8.0 * (x.double() @ table.double().t())).requires_grad_()
        torch.nn.functional.cross_entropy(z, y).backward()
        want = 8.0 * (z.grad.t().contiguous() @ x.double())
        assert (gw.double() - want).norm() <= 1e-5 * want.norm()
        table -= 20.0 * gw
    t = A.Table4.pack(table, group=32)
    codes, s, zeros = t.to_codes()
    q = np.stack((codes & 15, codes >> 4), 2).reshape(v, -1).astype(np.float64)
    w = torch.from_numpy((q - 8) * np.repeat(s, 32, axis=1)).cuda()
    _check4(t, w, hidden[:3].contiguous())


# ---- sizes at which another form is taken ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, v, d, pad, offset", [
    (1, 15, 7, 1, 1), (2, 16, 32, 0, 0), (15, 17, 33, 2, 1), (16, 5003, 64, 0, 0), (3, 1000, 96, 1, 0), (16, 1025, 128, 8, 0), (7, 999, 129, 0, 0),
    (16, 700, 256, 0, 0), (4, 3001, 300, 5, 2), (16, 333, 384, 0, 0), (9, 800, 400, 8, 0), (16, 1200, 512, 0, 0), (5, 90, 513, 0, 0),
    (2, 2000, 678, 0, 0), (16, 500, 768, 8, 8), (11, 640, 900, 1, 1), (16, 400, 1024, 0, 0), (16, 300, 1025, 3, 0), (17, 800, 40, 3, 1), (33, 501, 94, 1, 0),
    (64, 1000, 131, 0, 0), (48, 700, 600, 3, 3), (64, 100, 1024, 8, 0), (65, 1000, 131, 0, 0)])
def test_cross_entropy_few_rows(n, v, d, pad, offset, dt):
    x, w, y, b = _inputs(n, v, d, TYPES[dt], seed=n + d, pad=pad, offset=offset, bias=n % 2 == 1, ignored=0.2)
    _check(x, w, y, b, scale=2.0, ge=torch.linspace(-1e-3, 2e-3, n, device="cuda"))


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, v, d, bias", [(1024, 40, 32, True), (1025, 211, 64, False), (3000, 17, 128, True), (2500, 5, 200, True), (5011, 130, 96, False),
                                           (1500, 1, 64, True), (1100, 700, 320, True)])
def test_cross_entropy_more_rows_than_items(n, v, d, bias, dt):
    """The gradient of a short table is added up over parts of the batch; many rows meet the same item."""
    x, w, y, b = _inputs(n, v, d, TYPES[dt], seed=n, bias=bias, ignored=0.1)
    _check(x, w, y, b, scale=2.0)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, v, d", [(16, 300, 64), (16, 300, 400), (700, 1000, 64), (700, 1000, 320)])
def test_cross_entropy_all_rows_at_one_item(n, v, d, dt):
    x, w, y, b = _inputs(n, v, d, TYPES[dt], seed=7, bias=True)
    y[:] = v - 1
    _check(x, w, y, b, scale=1.0)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, d", [(5, 100), (5, 300), (40, 131)])
def test_cross_entropy_few_rows_masked(n, d, dt):
    """-inf and the lowest value as masks, every item masked, a row of NaN, a target out of range."""
    x, w, y, b = _inputs(n, 530, d, TYPES[dt], seed=8, bias=True)
    y[:] = torch.arange(n, device="cuda") * 13 + 3
    b[torch.arange(0, 530, 2)] = -float("inf")
    b[1::4] = torch.finfo(torch.float32).min
    y |= 1
    _check(x, w, y, b, scale=2.0)
    b[:] = -float("inf")
    losses, lse, grads = _check(x, w, y, b, scale=2.0)
    assert (losses == 0).all() and all((g == 0).all() for g in grads)
    x[1] = float("nan")
    b = torch.zeros(530, device="cuda")
    y[3] = 530
    losses, lse = A.cross_entropy(x, w, y, bias=b)
    keep = torch.tensor([k for k in range(n) if k not in (1, 3)], device="cuda")
    want = _reference(x[keep], w, y[keep], b, 1.0)
    _close(losses[keep], *want["losses"], "losses")
    assert torch.isnan(losses[1]) and torch.isnan(losses[3]) and torch.isnan(lse[1]) and torch.isfinite(lse[3])


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, v, d", [(6, 900, 60), (6, 900, 500), (300, 800, 64), (300, 800, 300)])
def test_cross_entropy_each_gradient_alone(n, v, d, dt):
    x, w, y, b = _inputs(n, v, d, TYPES[dt], seed=9, bias=True, ignored=0.1)
    losses, lse = A.cross_entropy(x, w, y, bias=b)
    gl = torch.rand(n, device="cuda")
    every = A.cross_entropy_backward(x, w, y, lse, gl, bias=b)
    for k in range(3):
        need = [i == k for i in range(3)]
        got = A.cross_entropy_backward(x, w, y, lse, gl, bias=b, need_x=need[0], need_table=need[1], need_bias=need[2])
        assert [g is not None for g in got] == need and torch.equal(got[k], every[k])


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, v, d", [(5, 203, 70), (5, 203, 513), (90, 203, 70), (1500, 33, 70), (90, 203, 300)])
def test_cross_entropy_strided_gradients(n, v, d, dt):
    """Gradients into rows of wider matrices of any alignment; what lies between the rows stays."""
    x, w, y, _ = _inputs(n, v, d, TYPES[dt], seed=10)
    losses, lse = A.cross_entropy(x, w, y)
    gl = torch.rand(n, device="cuda")
    want = A.cross_entropy_backward(x, w, y, lse, gl)
    kind = getattr(_lib, "AS_" + dt.upper())
    ctx = A.Context(0)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    for extra in (1, 3, 8):
        gx = torch.full((n, d + extra), 5.0, device="cuda", dtype=TYPES[dt])
        gw = torch.full((v, d + extra), 5.0, device="cuda", dtype=TYPES[dt])
        at = 1 if extra == 3 else 0
        rc = ctx.lib.as_cross_entropy_backward(ctx.h, x.data_ptr(), n, d, w.data_ptr(), v, d, d, kind, None, y.data_ptr(), -100, 1.0, lse.data_ptr(),
                                               gl.data_ptr(), None, gx[:, at:].data_ptr(), d + extra, gw[:, at:].data_ptr(), d + extra, None, None, 0)
        assert rc == _lib.AS_OK
        for got, ref in ((gx, want[0]), (gw, want[1])):
            assert torch.equal(got[:, at:at + d], ref)
            assert (got[:, :at] == 5).all() and (got[:, at + d:] == 5).all()
    torch.cuda.synchronize()


@pytest.mark.parametrize("n, v, d, dt", [(7, 2000, 90, "bf16"), (40, 900, 300, "f32"), (16, 700, 500, "f16"), (2000, 60, 64, "bf16"), (300, 900, 400, "f32")])
def test_cross_entropy_forms_captured(n, v, d, dt):
    x, w, y, b = _inputs(n, v, d, TYPES[dt], seed=11, bias=True)
    gl = torch.full((n,), 1 / n, device="cuda")

    def step():
        losses, lse = A.cross_entropy(x, w, y, bias=b, scale=2.0)
        return (losses, lse) + A.cross_entropy_backward(x, w, y, lse, gl, bias=b, scale=2.0)

    _replays(step, (x, w, b))


def test_cross_entropy_table_of_more_than_4_gib():
    """Offsets behind 32 bits in the table and in its gradient: the last items, and the first, against 64 bits."""
    v, d, n = 10_000_019, 256, 3
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.empty(v, d, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    y = torch.tensor([v - 1, 5, v - 2], device="cuda")
    x = w[y] * 0.5
    losses, lse = A.cross_entropy(x, w, y, scale=0.125)
    z = torch.cat([0.125 * (x.double() @ c.double().t()) for c in w.split(1 << 20)], 1)
    want = torch.logsumexp(z, 1)
    hit = z.gather(1, y[:, None])[:, 0]
    # a product of 256 terms in f32 (|x w| adds up to less than 256), lse, the difference
    assert (lse.double() - want).abs().max() <= (256 + 8) * E * 0.125 * 256 + 64 * E * 20
    assert (losses.double() - (want - hit)).abs().max() <= 2 * ((256 + 8) * E * 0.125 * 256 + 64 * E * 20)
    gl = torch.ones(n, device="cuda")
    gx, gw, _ = A.cross_entropy_backward(x, w, y, lse, gl, scale=0.125)
    p = torch.exp(z - want[:, None])
    p[torch.arange(n), y] -= 1
    for rows in (slice(v - 40, v), slice(0, 40)):
        ref = 0.125 * (p[:, rows].t().contiguous() @ x.double())
        size = 0.125 * (p[:, rows].abs().t().contiguous() @ x.double().abs())
        # the result's rounding; g's: half a step and exp of two errors of 264 e 32
        assert ((gw[rows].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2 * 264 * E * 32 + 128 * E * 20) * size + 1e-30).all()
    ref = 0.125 * sum(p[:, i:i + (1 << 20)] @ w[i:i + (1 << 20)].double() for i in range(0, v, 1 << 20))
    assert (gx.double() - ref).norm() <= 2.0 ** -7 * ref.norm()


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("m, v, d, group, scales, zeros", [
    (5, 40, 256, 64, "f32", True), (16, 500, 4000, 128, "f16", True), (16, 3001, 1000, 32, "bf16", False), (8, 100, 20000, 128, "bf16", False),
    (16, 20000, 2600, 64, "f16", False), (16, 64, 5008, 128, "f32", False), (33, 70, 4500, 64, "bf16", True), (20, 9000, 2700, 128, "f16", False),
    (64, 40000, 1300, 32, "f32", False), (100, 200, 2500, 64, "bf16", False), (4, 30, 42000, 128, "f32", True), (3, 5, 130, 64, "f16", False)])
def test_scores4_forms(m, v, d, group, scales, zeros, dt):
    """Rows in LDS, read as they lie, from an image, and of parts of k."""
    codes, s, z, w = _plain4(v, d, group, scales, zeros, m + v + d)
    t = A.Table4.from_codes(codes, s, z, dim=d, group=group)
    g = torch.Generator(device="cuda").manual_seed(d)
    for pad, at in ((0, 0), (8, 0), (3, 1)):
        x = torch.randn(m, d + pad, device="cuda", generator=g).to(TYPES[dt])[:, at:at + d]
        first = _check4(t, w, x)
    assert torch.equal(first, t.scores(x))
    x[m // 2, d - 1] = float("inf")
    x[0, 0] = float("nan")
    got = t.scores(x)
    keep = [k for k in range(1, m) if k != m // 2]
    if keep:
        assert torch.equal(got[keep], first[keep])
    assert torch.isnan(got[0]).all()


@pytest.mark.parametrize("m, v, d, dt", [(16, 2000, 3000, "f16"), (16, 900, 6000, "bf16"), (40, 500, 3500, "f32")])
def test_scores4_forms_captured(m, v, d, dt):
    codes, s, z, w = _plain4(v, d, 64, "bf16", True, 6)
    t = A.Table4.from_codes(codes, s, z, dim=d, group=64)
    x = torch.randn(m, d, device="cuda").to(TYPES[dt])
    _replays(lambda: (t.scores(x),), (x,))


def test_scores4_codes_and_scores_of_more_than_4_gib():
    """Offsets behind 32 bits in the codes (5.1 GB) and in the scores (2^32 of them)."""
    v, d = 20_000_003, 512
    g = torch.Generator(device="cuda").manual_seed(4)
    codes = torch.randint(0, 256, (v, d // 2), generator=g, dtype=torch.uint8, device="cuda")
    s = torch.rand(v, d // 128, generator=g, device="cuda").to(torch.float16) + 0.5
    t = A.Table4.from_codes(codes, s, dim=d, group=128)
    x = torch.randn(215, d, generator=g, device="cuda").half()
    got = t.scores(x)
    at = torch.cat([torch.arange(0, 50), torch.arange(v // 2, v // 2 + 50), torch.arange(v - 50, v)]).cuda()
    c = codes[at]
    w = (torch.stack((c & 15, c >> 4), 2).flatten(1).double() - 8) * s[at].double().repeat_interleave(128, 1)
    want = x.double() @ w.t().contiguous()
    size = x.double().abs() @ w.abs().t().contiguous()
    bound = (d + 16) * E * size + 2.0 ** -11 * want.abs() + torch.finfo(torch.float16).tiny
    _close(got[:, at], want, bound, "scores")


def test_items_of_an_index_in_4_bits():
    """ArrowSpace.pack4 of host and of device items: the same codes, and the scores of queries from them."""
    rows = np.random.default_rng(1).standard_normal((700, 96))
    host, there = A.ArrowSpace(rows), A.ArrowSpace(torch.from_numpy(rows).cuda())
    packed = [a.pack4(group=32, scale_dtype="float32") for a in (host, there)]
    codes, s, zeros = packed[0].to_codes()
    for a, b in zip((codes, s, zeros), packed[1].to_codes()):
        assert np.array_equal(a, b)
    q = np.stack((codes & 15, codes >> 4), 2).reshape(700, -1).astype(np.float64)
    w = (q - 8) * np.repeat(s, 32, axis=1)
    assert (np.abs(w - rows) <= np.repeat(s, 32, axis=1) * 0.5000001).all()
    _check4(packed[1], torch.from_numpy(w).cuda(), torch.from_numpy(rows[:2]).float().cuda())
    got = packed[0].scores(rows[3].astype(np.float32))
    assert got.shape == (700,) and got.argmax() == 3


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, v, d", [(6000, 150, 300), (2048, 129, 384), (3001, 3, 500), (1030, 1030, 260), (700, 65, 1000)])
def test_cross_entropy_long_rows_short_tables(n, v, d, dt):
    """The batch in parts where the table alone does not fill the chip; many rows at each 64 items."""
    x, w, y, b = _inputs(n, v, d, TYPES[dt], seed=12, bias=n % 2 == 0)
    _check(x, w, y, b, scale=2.0)


@pytest.mark.parametrize("n, v, d, dt", [(150_001, 300, 40, "bf16"), (150_001, 260, 270, "f16"), (70_001, 33, 300, "f32"), (5, 40, 5000, "bf16"),
                                         (70, 130, 20000, "f32"), (3, 17, 65536, "f16")])
def test_cross_entropy_many_rows_and_long_rows(n, v, d, dt):
    x, w, y, b = _inputs(n, v, d, TYPES[dt], seed=13, bias=True, ignored=0.1)
    _check(x, w, y, b, scale=1.0)


def test_scores4_no_rows_and_many():
    codes, s, z, w = _plain4(60, 90, 32, "f32", True, 14)
    t = A.Table4.from_codes(codes, s, z, dim=90, group=32)
    assert t.scores(torch.empty(0, 90, device="cuda")).shape == (0, 60)
    _check4(t, w, torch.randn(1000, 90, device="cuda").bfloat16())


def test_leaving_a_stream_while_it_is_captured():
    """A context moved to another stream in the middle of a capture: the capture goes on, and the graph's results are the eager ones."""
    x, w, y, _ = _inputs(40, 900, 64, torch.bfloat16, seed=15)
    want = A.cross_entropy(x, w, y)
    ctx = A.Context(0)
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    out, lse = torch.empty(40, device="cuda"), torch.empty(40, device="cuda")
    ws = torch.empty(ctx.lib.as_cross_entropy_workspace(40, 900, 64, _lib.AS_BF16, 0), dtype=torch.uint8, device="cuda")
    call = (x.data_ptr(), 40, 64, w.data_ptr(), 900, 64, 64, _lib.AS_BF16, None, y.data_ptr(), -100, 1.0, out.data_ptr(), lse.data_ptr(), ws.data_ptr(),
            ws.numel())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        graph.capture_begin(capture_error_mode="relaxed")
        ctx.set_stream(stream.cuda_stream)
        first = ctx.lib.as_cross_entropy(ctx.h, *call)
        ctx.set_stream(other.cuda_stream)
        ctx.set_stream(stream.cuda_stream)
        second = ctx.lib.as_cross_entropy(ctx.h, *call)
        graph.capture_end()
    assert (first, second) == (_lib.AS_OK, _lib.AS_OK)
    for _ in range(3):
        out.zero_(), lse.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    ctx.set_stream(other.cuda_stream)


def test_gradients_in_place_of_the_inputs_are_refused():
    x, w, y, _ = _inputs(8, 100, 64, torch.bfloat16, seed=16)
    losses, lse = A.cross_entropy(x, w, y)
    gl = torch.ones(8, device="cuda")
    ctx = A.Context(0)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    gx, gw = torch.empty_like(x), torch.empty_like(w)
    for a, b in ((x, gw), (w, gw), (gx, w), (gx, x), (gw, gw)):
        rc = ctx.lib.as_cross_entropy_backward(ctx.h, x.data_ptr(), 8, 64, w.data_ptr(), 100, 64, 64, _lib.AS_BF16, None, y.data_ptr(), -100, 1.0,
                                               lse.data_ptr(), gl.data_ptr(), None, a.data_ptr(), 64, b.data_ptr(), 64, None, None, 0)
        assert rc == _lib.AS_ERR_ARG
