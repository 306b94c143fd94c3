"""Edges of the operators over a table: small rows, far-apart and tiny values, mixed memory, streams, the largest tiles and several pieces.
References in 64 bits; the bounds are those of test_gpu_table.py, whose docstring derives them."""
import pytest

import arrowspace_amd as A
from arrowspace_amd import _lib

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_table import E, TYPES, _check, _check4, _close, _inputs, _plain4, _reference, _replays  # noqa: E402


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


# rows, items, columns by the form that f32 takes: short rows as they lie and from images, tiles through G, a few rows
F32_FORMS = [(70, 3000, 64), (300, 3000, 128), (300, 2000, 200), (12, 900, 200), (24, 900, 40)]


@pytest.mark.parametrize("n, v, d", F32_FORMS)
@pytest.mark.parametrize("scale", [1.0, 1e30])
def test_f32_tiny_values(n, v, d, scale):
    """Matrices whose products are far below the smallest normal number: all items the same, unless the scale brings them back."""
    x, w, y, _ = _inputs(n, v, d, torch.float32, seed=41)
    _check(x * 1e-20, w * 1e-20, y, None, scale=scale)


@pytest.mark.parametrize("n, v, d", F32_FORMS)
@pytest.mark.parametrize("power", [120, -120])
def test_f32_large_and_tiny_values_together(n, v, d, power):
    """Values at both ends of the range.  Their planes are bf16, whose smallest step is 2^-133, so values near 2^-120 are held to 2^-134 and not
    to 24 bits: a logit is off by another scale * 2^-134 * (the sums of |x| and |w|), a probability by e to twice that, a product with such
    values by 2^-134 of the other factor's sum."""
    x, w, y, b = _inputs(n, v, d, torch.float32, seed=42, bias=power < 0)
    x, w = x * 2.0 ** power, w * 2.0 ** -power
    gl = torch.full((n,), 1 / n, device="cuda")
    losses, lse = A.cross_entropy(x, w, y, bias=b, scale=4.0)
    grads = A.cross_entropy_backward(x, w, y, lse, gl, bias=b, scale=4.0)
    want = _reference(x, w, y, b, 4.0, gl)
    X, W, step = x.double().abs(), w.double().abs(), 2.0 ** -134
    off = 4.0 * step * (X.sum(1).max() + W.sum(1).max())
    z = 4.0 * (x.double() @ w.double().t().contiguous()) + (0 if b is None else b.double())
    p = torch.exp(z - torch.logsumexp(z, 1)[:, None]) / n
    dg = p * torch.expm1(2 * off)
    p[torch.arange(n, device="cuda"), y] += 1 / n
    _close(lse, want["lse"][0], want["lse"][1] + off, "lse")
    _close(losses, want["losses"][0], want["losses"][1] + 2 * off, "losses")
    _close(grads[0], want["grad_x"][0], want["grad_x"][1] + 4.0 * (dg @ W + step * p.sum(1, keepdim=True)), "grad_x")
    _close(grads[1], want["grad_table"][0], want["grad_table"][1] + 4.0 * (dg.t().contiguous() @ X + step * p.sum(0)[:, None]), "grad_table")


@pytest.mark.parametrize("n, v, d", F32_FORMS)
def test_f32_rows_far_apart(n, v, d):
    """One row 2^24 times as large as the others, and one item: the others keep the bits that they have alone."""
    x, w, y, _ = _inputs(n, v, d, torch.float32, seed=43)
    x, w = x.clone(), w.clone()
    x[n // 2] *= 2.0 ** 24
    w[v // 2] = 0
    w[v // 2, 0] = 2.0 ** 24
    x[torch.arange(n, device="cuda") != n // 2, 0] = -1.0    # (its logits: -2^26, its probability 0)
    x[n // 2, 0] = 0
    y = torch.where(y == v // 2, y - 1, y)
    _check(x, w, y, None)


# ... and those that 16-bit types take besides: rows of 256, few rows
FORMS = F32_FORMS + [(200, 2000, 256), (24, 900, 256)]


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, v, d", FORMS)
def test_garbage_in_ignored_rows_and_masked_items(n, v, d, dt):
    """Finite garbage where the batch is padded and where the bias takes an item out: everyone else gets what zeros there give."""
    x, w, y, b = _inputs(n, v, d, TYPES[dt], seed=44, bias=True)
    y = torch.where(y == 7, 8, y)
    y[3] = -100
    b[7] = -float("inf")
    gl = torch.full((n,), 1 / n, device="cuda")
    results = []
    for garbage in (0.0, 3e4 if dt == "f16" else 1e18):
        x, w = x.clone(), w.clone()
        x[3], w[7] = garbage, garbage
        losses, lse = A.cross_entropy(x, w, y, bias=b)
        results.append((losses, lse) + A.cross_entropy_backward(x, w, y, lse, gl, bias=b))
    want = _reference(torch.cat((x[:3], 0 * x[3:4], x[4:])), torch.cat((w[:7], 0 * w[7:8], w[8:])), y, b, 1.0, gl)
    rows = torch.arange(n, device="cuda") != 3
    for r in results:
        for got, what in zip(r, ("losses", "lse", "grad_x", "grad_table", "grad_bias")):
            exact, bound = want[what]
            if what in ("losses", "lse", "grad_x"):
                got, exact, bound = got[rows], exact[rows], bound[rows]
            _close(got, exact, bound, what)
        assert not r[2][3].any() and not r[3][7].any() and r[4][7] == 0


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n, v, d", FORMS)
@pytest.mark.parametrize("power, scale", [(13, 1.0), (24, 1.0), (24, 30.0), (40, 1.0), (60, 30.0)])
def test_logits_beyond_the_exponents_range(n, v, d, dt, power, scale):
    """Logits of 2^13 to 2^60: the normaliser is the largest logit to f32's bits, whatever its rounding is as an exponent."""
    x, w, y, b = _inputs(n, v, d, TYPES[dt], seed=48, bias=True)
    x = x * 2.0 ** power
    for bias in (None, b):
        losses, lse = A.cross_entropy(x, w, y, bias=bias, scale=scale)
        want = _reference(x, w, y, bias, scale)
        _close(lse, *want["lse"], "lse")
        _close(losses, *want["losses"], "losses")


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, v, d", FORMS)
def test_logits_of_millions(n, v, d, dt):
    """Probabilities are at most 1 where a logit's rounding is whole units: the gradient of a row with such logits is bounded by its coefficient."""
    x, w, y, _ = _inputs(n, v, d, TYPES[dt], seed=46)
    x = x.clone()
    x[: n // 2] *= 2.0 ** 12 if dt == "f16" else 2.0 ** 24
    gl = torch.full((n,), 1 / n, device="cuda")
    losses, lse = A.cross_entropy(x, w, y, scale=30.0)
    gx, gw, _ = A.cross_entropy_backward(x, w, y, lse, gl, scale=30.0)
    assert torch.isfinite(losses).all() and torch.isfinite(lse).all()
    # every |g| adds up to at most (1 + the number of items at the maximum, few) times the coefficient a row: 8 of them
    assert (gx.double().abs() <= 8 * 30 / n * w.double().abs().max()).all()
    assert (gw.double().abs() <= 8 * 30 / n * x.double().abs().sum(0)).all()


@pytest.mark.parametrize("n, v, d", FORMS)
def test_a_row_of_nan_has_no_gradient_and_an_ignored_one_no_part_in_the_others(n, v, d):
    x, w, y, b = _inputs(n, v, d, torch.bfloat16, seed=47, bias=True)
    x = x.clone()
    x[2] = float("nan")
    gl = torch.full((n,), 1 / n, device="cuda")
    _, lse = A.cross_entropy(x, w, y, bias=b)
    gx, gw, gb = A.cross_entropy_backward(x, w, y, lse, gl, bias=b)
    assert torch.isnan(gx[2]).all() and torch.isnan(gb).all()
    rows = torch.arange(n, device="cuda") != 2
    assert torch.isfinite(gx[rows]).all()
    y[2] = -100
    gx, gw, gb = A.cross_entropy_backward(x, w, y, lse, gl, bias=b)
    assert not gx[2].any() and torch.isfinite(gx).all() and torch.isfinite(gb).all()


@pytest.mark.parametrize("n, v, d", F32_FORMS)
def test_f32_gradients_of_improbable_items(n, v, d):
    """Items of probabilities down to 1e-12: their gradients keep f32's bits."""
    x, w, y, b = _inputs(n, v, d, torch.float32, seed=45, bias=True)
    b[100:500] = -torch.linspace(0, 27, 400, device="cuda")
    y = torch.where((y >= 100) & (y < 500), y % 100, y)
    gl = torch.full((n,), 1 / n, device="cuda")
    _, lse = A.cross_entropy(x, w, y, bias=b)
    _, gw, gb = A.cross_entropy_backward(x, w, y, lse, gl, bias=b)
    X, W = x.double(), w.double()
    z = X @ W.t().contiguous() + b.double()
    p = torch.exp(z - torch.logsumexp(z, 1)[:, None])[:, 100:500] / n
    size = X.abs() @ W.abs().t().contiguous() + b.double().abs()
    # relative: exp of a logit and of a normaliser that are each (d + 8) e of their terms off, the exponent's own rounding, e a sum of n
    off = 2 * (d + 8) * E * size.max() + 8 * E * (z.abs().max() + 30) + (n + 64) * E + 2.0 ** -21
    want, terms = p.t().contiguous() @ X, p.t().contiguous() @ X.abs()
    _close(gw[100:500], want, off * terms, "grad_table")
    _close(gb[100:500], p.sum(0), off * p.sum(0), "grad_bias")


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, v, d", FORMS)
@pytest.mark.parametrize("size, scale", [(1e-37, 1.0), (1e-35, 1.0), (5e-35, 1.0), (2e36, 1e-36), (1e38, 1e-38)])
def test_gradients_of_tiny_and_huge_coefficients(n, v, d, dt, size, scale):
    """Whatever the losses are weighted with, no unit of the logits' gradient under- or overflows."""
    x, w, y, b = _inputs(n, v, d, TYPES[dt], seed=49, bias=True)
    gl = torch.linspace(0.5, 1.5, n, device="cuda") * size
    _, lse = A.cross_entropy(x, w, y, bias=b, scale=scale)
    grads = A.cross_entropy_backward(x, w, y, lse, gl, bias=b, scale=scale)
    want = _reference(x, w, y, b, scale, gl)
    for got, what in zip(grads, ("grad_x", "grad_table", "grad_bias")):
        exact, bound = want[what]
        # (three rows of 1.2e38 at one item are 3.6e38, more than the type's largest value: infinite)
        exact = torch.where(exact.abs() > torch.finfo(got.dtype).max, exact.sign() * float("inf"), exact)
        _close(got, exact, bound, what)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m, v, d", [(3, 300, 200), (16, 300, 200), (16, 100, 6000), (40, 300, 200), (40, 100, 6000)])
@pytest.mark.parametrize("power", [110, 116, 122, -90, -105, -118])
def test_scores4_of_rows_at_both_ends_of_the_range(m, v, d, dt, power):
    """A row's values up to 2^124 and down to 2^-120, every other row of ordinary size.  (Scales of 1 / 64: the scores stay below 2^128.)"""
    codes, s, z, _ = _plain4(v, d, 32, "f32", True, m + d)
    s = s / 64
    t = A.Table4.from_codes(codes, s, z, dim=d, group=32)
    q = torch.stack((codes & 15, codes >> 4), 2).flatten(1)[:, :d].double()
    w = (q - z.double().repeat_interleave(32, 1)[:, :d]) * s.double().repeat_interleave(32, 1)[:, :d]
    g = torch.Generator(device="cuda").manual_seed(50)
    x = torch.rand(m, d, device="cuda", generator=g) * 2 - 1
    x[::2] *= 2.0 ** power
    x = x.to(TYPES[dt])
    got, X = t.scores(x), x.double()
    want, size = X @ w.t().contiguous(), X.abs() @ w.abs().t().contiguous()
    # the bound of _check4 without its smallest normal number for the small rows: these stay normal here
    bound = ((d + 16) * E + 2.0 ** -22) * size + torch.finfo(x.dtype).eps / 2 * want.abs() + 2.0 ** -134
    exact = torch.where(want.abs() > torch.finfo(x.dtype).max, want.sign() * float("inf"), want)
    _close(got, exact, bound, "scores")


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, v, d", [(12, 300, 40), (130, 900, 96), (130, 900, 300)])
def test_cross_entropy_in_a_graph_of_torch(n, v, d, dt):
    """Beside another term of a loss, through both results, on another stream: the gradients are those of the backward call."""
    x, w, y, b = _inputs(n, v, d, TYPES[dt], seed=51, pad=3, offset=1, bias=True, ignored=0.2)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        losses, lse = A.cross_entropy(leaves[0], leaves[1], y, bias=leaves[2], scale=2.0)
        total = losses.sum() / n + 1e-3 * (lse ** 2).mean() + leaves[1].float().pow(2).sum()
        total.backward()
        ge = 2e-3 * lse.detach() / n
        want = A.cross_entropy_backward(x, w, y, lse.detach(), torch.full((n,), 1 / n, device="cuda"), bias=b, scale=2.0, grad_lse=ge)
        want = [want[0], (want[1].double() + 2 * w.double()), want[2]]
    torch.cuda.synchronize()
    half = torch.finfo(TYPES[dt]).eps / 2
    for leaf, g, u in zip(leaves, want, (half, half, 2.0 ** -24)):
        # torch's own rounding of 1 / n and of the mean's gradient: a few f32 roundings of coefficients; the sum of two terms of the table's
        assert ((leaf.grad.double() - g.double()).abs() <= 3 * u * g.double().abs() + 2.0 ** -20 * g.double().abs().max() + 2 * u * g.double().abs().max()).all()
    with pytest.raises(RuntimeError):
        again = torch.autograd.grad(A.cross_entropy(leaves[0], leaves[1], y)[0].sum(), leaves[0], create_graph=True)[0]
        again.sum().backward()


def test_cross_entropy_in_a_graph_of_torch_captured():
    x, w, y, b = _inputs(100, 1500, 96, torch.bfloat16, seed=52, bias=True)
    x, w, b = x.contiguous().requires_grad_(), w.contiguous().requires_grad_(), b.requires_grad_()
    data = [t.detach() for t in (x, w, b)]

    def step():
        losses, lse = A.cross_entropy(x, w, y, bias=b, scale=2.0)
        return (losses.detach(), lse.detach()) + torch.autograd.grad(losses.mean() + lse.mean() * 1e-3, (x, w, b))

    _replays(step, data)


def test_scores4_have_no_gradient_and_say_so():
    codes, s, z, w = _plain4(90, 64, 32, "f32", False, 53)
    t = A.Table4.from_codes(codes, s, dim=64, group=32)
    x = torch.randn(3, 64, device="cuda", requires_grad=True)
    scores = t.scores(x)
    assert torch.equal(scores.detach(), t.scores(x.detach()))
    with pytest.raises(A.ArrowSpaceError) as e:
        scores.sum().backward()
    assert e.value.status == _lib.AS_ERR_UNSUPPORTED


# Long rows whose logits' gradient lies in memory in pieces of the table, with the sizes at which each tile is taken for each product.  The pieces
# follow from n padded to the tile and 2 bytes a logit (f32: 6).
@pytest.mark.parametrize("n, v, d, dt, bias", [
    (8100, 50003, 600, "bf16", True),      # 256 x 256 everywhere; pieces of 16896, 16896, 16211
    (8100, 50003, 600, "bf16", False),
    (8100, 50003, 600, "f16", True),
    (3000, 35003, 700, "f32", True),       # 256 x 256 everywhere; pieces of 17664 and 17339
    (3000, 35003, 700, "f32", False),
    (40, 2_700_011, 264, "bf16", True),    # 256 x 64 (the table's gradient 128 x 128); two pieces of 1.35 M
    (100, 1_400_003, 264, "f16", True),    # 128 x 128 everywhere; two pieces of 0.7 M
])
def test_cross_entropy_large_tiles_and_several_pieces(n, v, d, dt, bias):
    x, w, y, b = _inputs(n, v, d, TYPES[dt], seed=54, bias=bias, ignored=0.1)
    y[: n // 4] = v - 1 - torch.arange(n // 4, device="cuda") // 7       # several rows at items of the last piece, up to 64 and more of a group
    y[n // 4: n // 2] = (torch.arange(n // 2 - n // 4, device="cuda") * 7919) % v
    y[n // 2] = 0
    ge = torch.full((n,), 1e-3 / n, device="cuda") if bias else None
    _check(x, w, y, b, scale=2.0, ge=ge)


def test_cross_entropy_of_more_than_2_to_the_26_rows():
    n, v = (1 << 26) + 5, 3
    g = torch.Generator(device="cuda").manual_seed(55)
    x = torch.randn(n, 1, device="cuda", generator=g).bfloat16()
    w = torch.tensor([[-1.5], [0.5], [2.0]], device="cuda").bfloat16()
    y = torch.randint(0, v, (n,), device="cuda", generator=g)
    y[-1] = 2
    losses, lse = A.cross_entropy(x, w, y)
    z = x.double() * w.double()[:, 0]
    exact = torch.logsumexp(z, 1)
    off = 16 * E * (z.abs().amax() + 2)
    assert (lse.double() - exact).abs().max() <= off
    assert (losses.double() - (exact - z.gather(1, y[:, None])[:, 0])).abs().max() <= 2 * off
    gl = torch.ones(n, device="cuda")
    gx, gw, _ = A.cross_entropy_backward(x, w, y, lse, gl)
    p = torch.exp(z - exact[:, None])
    p.scatter_add_(1, y[:, None], -torch.ones_like(z[:, :1]))
    # three products with g of 2^-8 each, the result's rounding
    assert ((gx.double() - p @ w.double()).abs()[:, 0] <= 2.0 ** -8 * ((p.abs() @ w.double().abs())[:, 0] + 4)).all()
    # sums of n / 768 and then of 768 parts in f32; g's roundings to nearest have no direction
    assert ((gw.double() - p.t().contiguous() @ x.double()).abs() <= 2.0 ** -6 * (p.t().contiguous() @ x.double()).abs() + 1e-3 * (p.abs().t().contiguous() @ x.double().abs())).all()


@pytest.mark.parametrize("n, v, d", FORMS)
def test_f32_largest_values_in_ignored_rows(n, v, d):
    """A padded row of the type's largest value, which no bf16 rounds to: it has no part in anyone's gradient."""
    x, w, y, b = _inputs(n, v, d, torch.float32, seed=56, bias=True)
    y[3] = -100
    gl = torch.full((n,), 1 / n, device="cuda")
    want = _reference(torch.cat((x[:3], 0 * x[3:4], x[4:])), w, y, b, 1.0, gl)
    for value in (torch.finfo(torch.float32).max, torch.finfo(torch.float32).min):
        x = x.clone()
        x[3] = value
        _, lse = A.cross_entropy(x, w, y, bias=b)
        got = A.cross_entropy_backward(x, w, y, lse, gl, bias=b)
        # (held to the bounds, not to the bits that zeros there give: the maximum a row's sum is taken against moves with its neighbours')
        for g, what in zip(got, ("grad_x", "grad_table", "grad_bias")):
            _close(g, *want[what], what)
        assert not got[0][3].any()


@pytest.mark.parametrize("n, v, d", F32_FORMS)
def test_f32_the_largest_value(n, v, d):
    """Rows and items that hold it, and logits of ordinary size."""
    top = torch.finfo(torch.float32).max
    x, w, y, _ = _inputs(n, v, d, torch.float32, seed=57)
    x, w = x.clone(), w.clone()
    x[1, 0], w[:, 0] = top, 2.0 ** -126 * torch.arange(v, device="cuda").remainder(64)
    w[2, 1], x[:, 1] = -top, 2.0 ** -127
    x[1, 1] = 0
    _check(x, w, y, None, scale=1.0)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n, v, d", FORMS)
@pytest.mark.parametrize("scale", [1e-36, 1e-40, 1e-45])
def test_scales_next_to_zero(n, v, d, dt, scale):
    x, w, y, _ = _inputs(n, v, d, TYPES[dt], seed=58)
    losses, lse = A.cross_entropy(x, w, y, scale=scale)
    exact = torch.tensor(float(v), dtype=torch.float64, device="cuda").log()
    assert ((lse.double() - exact).abs() <= 64 * E * exact).all() and ((losses.double() - exact).abs() <= 64 * E * exact).all()


def test_a_captured_call_with_the_profile_on():
    """Timers record events, which a graph cannot time: captured calls are left out, and the calls behind go on."""
    x, w, y, _ = _inputs(40, 900, 64, torch.bfloat16, seed=59)
    ctx = A.Context(0)
    want = A.cross_entropy(x, w, y, ctx=ctx)
    torch.cuda.synchronize()
    ctx.profile(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = A.cross_entropy(x, w, y, ctx=ctx)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        got = A.cross_entropy(x, w, y, ctx=ctx)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ms, launches = ctx.profile_get("cross_entropy")
    assert launches == 3 and ms > 0


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n, v, d", FORMS)
def test_products_that_overflow_to_minus_infinity(n, v, d, dt):
    """A row whose products are all -infinity in f32 has no loss of 0: without a bias nothing takes items out."""
    x = torch.randn(n, d, device="cuda").to(TYPES[dt])
    w = -torch.ones(v, d, device="cuda").to(TYPES[dt])
    x[1] = 1e30
    w[:, 0] = -1e30
    x[torch.arange(n, device="cuda") != 1, 0] = 0
    y = torch.randint(0, v, (n,), device="cuda")
    losses, lse = A.cross_entropy(x, w, y)
    rows = torch.arange(n, device="cuda") != 1
    assert torch.isnan(losses[1]) and torch.isnan(lse[1]) and torch.isfinite(losses[rows]).all()
    y[1] = -100
    losses, lse = A.cross_entropy(x, w, y)
    assert losses[1] == 0 and torch.isfinite(losses).all()
