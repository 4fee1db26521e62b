"""Layer operators on the GPU against their definition in 64 bits (oracle/layers_ref.py, numpy).

Tolerances.  e = eps / 2 of the type sums are taken in (float for float, bfloat16 and half; double for double), o =
eps / 2 of the type stored.  A sum of n terms whose longest chain of additions has k links is off by at most k e times
the sum of the terms' sizes.  A row's chain is at most 8 * ceil(n / 512) (a thread's own terms) + 24 (threads, waves);
a gradient's over R rows at most R / 16 + 100.  With U = 1 + |u|, u a row's unit values:
  u   the mean is taken twice, so what is left of its error is e of h - m, and h = x * factor and the stored mean are
      rounded once each: e (chain U + 4 |h| r + 4 |m| r); the deviation's relative error is half the chain's
  y   o |y| + 4 e (chain (U |w| + |b|) + 4 (|h| + |m|) r |w|)
  dx  o |dx| + 4 e r (chain (|g| + mean |g| + U mean |g u|) + the error of u times (mean |g u| + mean |g|)), times the
      dropout factor, where g = dy w
  dw  o |dw| + 4 e sum |dy| (gradient chain U + 4 (|h| + |m|) r);  db  o |db| + e gradient chain sum |dy|
A value below the type's smallest normal number is stored to a multiple of its smallest number: that, too, is allowed.
"""
import numpy as np
import pytest

from oracle import layers_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def L():
    from epidemicsimulator_amd import layers
    return layers


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def inner(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


def host(t):
    return t.detach().double().cpu().numpy()


def make(rows, cols, dtype, seed, mean=0.0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x = (rnd(rows, cols) * scale + mean).to(dtype).cuda()
    w = (1.0 + 0.3 * rnd(cols)).to(dtype).cuda()
    b = (0.3 * rnd(cols)).to(dtype).cuda()
    dy = (0.1 * rnd(rows, cols)).to(dtype).cuda()
    return x, w, b, dy


def close(what, got, want, tol):
    got = host(got)
    assert got.shape == want.shape, what
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %g times the tolerance at %s" % (
        what, bad.sum(), bad.size, np.max(np.abs(got - want) / tol), np.unravel_index(np.argmax(np.abs(got - want) / tol), bad.shape))


def check_norm(dtype, x, w, b, dy, eps, f, y, dx=None, dw=None, db=None, mean=None, rstd=None):
    """x, dy [R, C] tensors, w, b tensors or None, f the dropout factors or None."""
    e, o, tiny = inner(dtype), half_step(dtype), torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    X = host(x)
    rows, cols = X.shape
    W = host(w) if w is not None else np.ones(cols)
    B = host(b) if b is not None else np.zeros(cols)
    H = X if f is None else R.apply_factors(X, f)
    Y, u, m, r = R.norm_forward(H, W, B, eps)
    U, chain, size = 1 + np.abs(u), 8 * -(-cols // 512) + 24, (np.abs(H) + np.abs(m)) * r
    close("y", y, Y, o * np.abs(Y) + 4 * e * (chain * (U * np.abs(W) + np.abs(B)) + 4 * size * np.abs(W)) + tiny)
    if mean is not None:
        spread = np.abs(H - m).mean(1) + np.abs(m[:, 0])
        close("mean", mean, m[:, 0], 4 * e * chain * spread + tiny)
        close("rstd", rstd, r[:, 0], 4 * e * chain * r[:, 0])
    if dy is None:
        return
    D = host(dy)
    DH, DW, DB = R.norm_backward(D, u, r, W)
    G = np.abs(D * W)
    eu = chain * U + 4 * size
    mg, mgu = G.mean(1, keepdims=True), (G * np.abs(u)).mean(1, keepdims=True)
    meu = (G * eu).mean(1, keepdims=True)
    tol = 4 * e * r * (chain * (G + mg + U * mgu) + eu * mgu + U * meu)
    if f is not None:
        DH, tol = R.apply_factors(DH, f), tol * f
    if dx is not None:
        close("dx", dx, DH, o * np.abs(DH) + tol + tiny)
    gchain = rows / 16 + 100
    if dw is not None:
        close("dweight", dw, DW, o * np.abs(DW) + 4 * e * (np.abs(D) * (gchain * U + eu)).sum(0) + tiny)
    if db is not None:
        close("dbias", db, DB, o * np.abs(DB) + e * gchain * np.abs(D).sum(0) + tiny)


def both_ways(L, dtype, rows, cols, p, seed=7, eps=1e-5, **kw):
    x, w, b, dy = make(rows, cols, dtype, rows * 131 + cols, **kw)
    y, mean, rstd = L.layer_norm_forward(x, w, b, eps, dropout=p, seed=seed, offset=3)
    dx, dw, db = L.layer_norm_backward(dy, x, w, mean, rstd, dropout=p, seed=seed, offset=3)
    f = R.factors(rows, cols, p, seed, 3) if p else None
    check_norm(dtype, x, w, b, dy, eps, f, y, dx, dw, db, mean, rstd)


# widths around every chunk, wave and workgroup border; rows around those of a workgroup and a segment
WIDTHS = [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 511, 512, 513, 1000, 1023, 1025, 2047, 2048,
          2049, 4095, 4096, 4097, 8191, 8192, 8200, 12289, 16384, 16391, 20000, 32768, 33001]


@pytest.mark.parametrize("dtype", list(TYPES.values()), ids=list(TYPES))
@pytest.mark.parametrize("cols", WIDTHS)
def test_norm_widths(L, cols, dtype):
    both_ways(L, dtype, 5, cols, 0.0)
    both_ways(L, dtype, 19, cols, 0.2)


@pytest.mark.parametrize("dtype", list(TYPES.values()), ids=list(TYPES))
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 63, 64, 65, 257, 1023, 1024, 1025, 2049, 4097, 9001])
def test_norm_rows(L, rows, dtype):
    both_ways(L, dtype, rows, 128, 0.0)
    both_ways(L, dtype, rows, 37, 0.5)


@pytest.mark.parametrize("dtype", list(TYPES.values()), ids=list(TYPES))
@pytest.mark.parametrize("rows, cols", [(5000, 256), (5000, 1001), (2500, 2100), (2300, 4100), (2100, 9000), (1500, 17000)])
def test_norm_many_wide_rows(L, rows, cols, dtype):
    both_ways(L, dtype, rows, cols, 0.0)


@pytest.mark.parametrize("dtype", list(TYPES.values()), ids=list(TYPES))
@pytest.mark.parametrize("rows, cols", [(1100, 1536), (1100, 1537), (1050, 8193), (1050, 12001), (1030, 16384), (1030, 16392), (1026, 20003),
                                        (768, 512), (769, 512), (769, 513), (1024, 1030), (1025, 4096), (1536, 2048), (1537, 2048), (512, 700), (513, 700),
                                        (1026, 24576), (1026, 24585), (1026, 7), (1026, 8), (1300, 1), (70000, 3)])
def test_norm_backward_shapes_with_and_without_dropout(L, rows, cols, dtype):
    both_ways(L, dtype, rows, cols, 0.0)
    both_ways(L, dtype, rows, cols, 0.3)


@pytest.mark.parametrize("dtype", list(TYPES.values()), ids=list(TYPES))
def test_norm_far_means_and_small_spreads(L, dtype):
    """Means of 1,000 spreads (64 in 8 bits of mantissa), and rows of one value each: the spread is then zero."""
    both_ways(L, dtype, 9, 300, 0.0, mean=64.0 if dtype == torch.bfloat16 else 1000.0)
    both_ways(L, dtype, 9, 300, 0.0, scale=1e-3 if dtype != torch.float16 else 0.05)
    x = torch.full((6, 100), 3.0, dtype=dtype, device="cuda")
    w, b = make(1, 100, dtype, 1)[1:3]
    assert torch.equal(L.layer_norm(x, w, b), b.expand(6, 100))
    assert torch.equal(L.layer_norm(x, w, b, dropout=1.0, seed=1), b.expand(6, 100))


@pytest.mark.parametrize("p", [0.0, 0.3])
def test_norm_without_weight_or_bias(L, p):
    x, w, b, dy = make(33, 70, torch.float32, 5)
    f = R.factors(33, 70, p, 9, 0) if p else None
    for ww, bb in ((None, None), (w, None), (None, b)):
        y, m, r = L.layer_norm_forward(x, ww, bb, dropout=p, seed=9)
        dx, dw, db = L.layer_norm_backward(dy, x, ww, m, r, dropout=p, seed=9)
        check_norm(torch.float32, x, ww, bb, dy, 1e-5, f, y, dx, dw, db, m, r)


def test_norm_only_the_gradients_asked_for(L):
    x, w, b, dy = make(300, 70, torch.float32, 6)
    for need in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(need >> k & 1)) for k, t in enumerate((x, w, b))]
        y = L.layer_norm(*leaves)
        wanted = [t for t in leaves if t.requires_grad]
        grads = dict(zip([id(t) for t in wanted], torch.autograd.grad(y, wanted, dy)))
        dx, dw, db = (grads.get(id(t)) for t in leaves)
        check_norm(torch.float32, x, w, b, dy, 1e-5, None, y, dx, dw, db)


# ---- dropout -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(TYPES.values()), ids=list(TYPES))
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 7), (5, 8), (4, 9), (257, 16), (100, 130), (33, 1001), (2, 70000), (5000, 3)])
@pytest.mark.parametrize("p", [0.0, 2.0 ** -17, 0.1, 0.5, 0.999, 1.0])
def test_dropout_values(L, rows, cols, p, dtype):
    """A product of two numbers, rounded twice at most: 1.5 steps of the type, and none between for p = 0 and 0.5."""
    x = make(rows, cols, dtype, 3)[0]
    seed, offset = -(1 << 40) + 12345, (1 << 33) + 7
    f = R.factors(rows, cols, p, seed, offset)
    want = R.apply_factors(host(x), f)
    got = host(L.dropout(x, p, seed, offset))
    assert np.array_equal(got == 0, want == 0)
    tol = 0 if p in (0.0, 0.5, 1.0, 2.0 ** -17) else (half_step(dtype) + 2 * inner(dtype)) * np.abs(want)
    assert np.all(np.abs(got - want) <= tol + (torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps if p else 0))


def test_dropout_probability_is_rounded_to_sixteen_bits(L):
    x = torch.ones(64, 64, device="cuda")
    t = 6554   # 0.1 in units of 2^-16, rounded
    assert torch.equal(L.dropout(x, 0.1, 5), L.dropout(x, t / 65536, 5))
    assert L.dropout(x, 0.1, 5).max().item() == np.float32(65536.0 / (65536 - t))
    assert torch.equal(L.dropout(x, 2.5 / 65536, 5), L.dropout(x, 2.0 / 65536, 5))   # halves to even
    assert torch.equal(L.dropout(x, 3.5 / 65536, 5), L.dropout(x, 4.0 / 65536, 5))


def test_dropped_infinities_and_nan_give_zero(L):
    f = R.factors(40, 50, 0.5, 2, 0)
    for bad in (float("inf"), float("-inf"), float("nan")):
        for dtype in TYPES.values():
            x = make(40, 50, dtype, 8)[0]
            x[torch.from_numpy(f == 0).cuda()] = bad
            assert np.array_equal(host(L.dropout(x, 0.5, 2)), R.apply_factors(np.where(f > 0, host(x), 0.0), f))
            assert torch.isfinite(L.layer_norm(x, dropout=0.5, seed=2)).all()


def test_masks_differ_between_seeds_offsets_and_rows(L):
    x = torch.ones(64, 512, device="cuda")
    masks = [L.dropout(x, 0.5, s, o) > 0 for s, o in ((1, 0), (2, 0), (1, 1), (1 << 32 | 1, 0), (1, 1 << 32))]
    masks += [masks[0].roll(1, 0), masks[0].roll(8, 1)]
    for i in range(len(masks)):
        for j in range(i):
            same = (masks[i] == masks[j]).float().mean().item()
            assert abs(same - 0.5) < 6 * 0.5 / np.sqrt(64 * 512)


def test_dropout_gradient_is_the_same_map(L):
    x, _, _, dy = make(60, 77, torch.float32, 4)
    x.requires_grad_(True)
    g, = torch.autograd.grad(L.dropout(x, 0.4, 99, 5), x, dy)
    assert torch.equal(g, L.dropout(dy, 0.4, 99, 5))


def test_offset_in_device_memory(L):
    x, w, b, dy = make(60, 77, torch.float32, 4)
    off = torch.tensor([12345678901], device="cuda")
    assert torch.equal(L.dropout(x, 0.4, 1, off), L.dropout(x, 0.4, 1, 12345678901))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    a = L.layer_norm(x, w, b, dropout=0.4, seed=1, offset=off)
    c = L.layer_norm(x, w, b, dropout=0.4, seed=1, offset=12345678901)
    assert torch.equal(a, c)
    for s, t in zip(torch.autograd.grad(a, leaves, dy), torch.autograd.grad(c, leaves, dy)):
        assert torch.equal(s, t)
    y = L.dropout(x, 0.4, 1, off)
    off += 1   # between a forward pass and its backward pass: refused, the masks would differ
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(y, x, dy)


# ---- gradients against differences ----------------------------------------------------------------------
@pytest.mark.parametrize("rows, cols, p", [(4, 9, 0.0), (3, 16, 0.3), (5, 33, 0.5)])
def test_gradients_against_differences(L, rows, cols, p):
    x, w, b, _ = make(rows, cols, torch.float64, 21)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    assert torch.autograd.gradcheck(lambda *a: L.layer_norm(*a, dropout=p, seed=3, offset=1), leaves)
    assert torch.autograd.gradcheck(lambda a: L.dropout(a, p, 3, 1), leaves[:1])


def test_the_graph_keeps_autograds_rules(L):
    """Backward twice only where the graph is retained; inputs changed in between are noticed; a weight that is the bias
    too, or expanded from one number, collects both or all of its gradients."""
    x, w, b, dy = make(50, 40, torch.float64, 22)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = L.layer_norm(x, w, b)
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for p, q in zip(first, torch.autograd.grad(y, leaves, dy)):
        assert torch.equal(p, q)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaves, dy)
    y = L.layer_norm(x, w, b)
    with torch.no_grad():
        x.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(y, leaves, dy)
    dw, db = torch.autograd.grad(L.layer_norm(x, w, b), (w, b), dy)
    both, = torch.autograd.grad(L.layer_norm(x, w, w), w, dy)
    assert torch.equal(both, dw + db)
    one = torch.ones(1, device="cuda", dtype=torch.float64, requires_grad=True)
    g, = torch.autograd.grad(L.layer_norm(x, one.expand(40), b), one, dy)
    assert torch.allclose(g, dw.sum().reshape(1), rtol=1e-12, atol=1e-12)
    with torch.inference_mode():
        assert torch.equal(L.layer_norm(x.clone(), w.clone(), b.clone()), L.layer_norm_forward(x, w, b)[0])


def test_tangents_are_refused(L):
    """Forward-mode derivatives, of the inputs and of the gradient that a backward pass is given."""
    import torch.autograd.forward_ad as forward_ad
    from epidemicsimulator_amd import _capi
    x, w, b, dy = make(6, 40, torch.float32, 23)
    x.requires_grad_(True)
    with forward_ad.dual_level():
        for t in ([forward_ad.make_dual(x, dy), w, b], [x, forward_ad.make_dual(w, w), b], [x, w, forward_ad.make_dual(b, b)]):
            with pytest.raises(_capi.EpiError, match="forward-mode"):
                L.layer_norm(*t)
        with pytest.raises(_capi.EpiError, match="forward-mode"):
            L.dropout(forward_ad.make_dual(x, dy), 0.5, 1)
        for y in (L.layer_norm(x, w, b), L.dropout(x, 0.5, 1)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, x, forward_ad.make_dual(dy, dy), retain_graph=True)
            torch.autograd.grad(y, x, dy)


# ---- layouts -------------------------------------------------------------------------------------------
def test_strided_expanded_and_transposed_rows(L):
    wide, w, b, dyw = make(40, 300, torch.float32, 31)
    w, b = w[:96], b[:96]
    cases = [(wide[:, 5:101], dyw[:, 100:196]), (wide[::3, :96], dyw[::3, 3:99]), (wide[:1].expand(40, 300)[:, 7:103], dyw[:1].expand(40, 300)[:, :96]),
             (wide[:, :96].t().contiguous().t(), dyw[:, ::3][:, :96]), (wide[:, :96], torch.ones((), device="cuda").expand(40, 96))]
    for x, dy in cases:
        rows = x.shape[0]
        y, m, r = L.layer_norm_forward(x, w, b, dropout=0.25, seed=4)
        grads = L.layer_norm_backward(dy, x, w, m, r, dropout=0.25, seed=4)
        check_norm(torch.float32, x, w, b, dy, 1e-5, R.factors(rows, 96, 0.25, 4, 0), y, *grads, m, r)
        assert torch.equal(L.dropout(x, 0.25, 4), L.dropout(x.contiguous(), 0.25, 4))


def plain_copy(t):
    """The same values, contiguous."""
    return t.clone(memory_format=torch.contiguous_format)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_gradients_expanded_in_a_middle_dimension(L, dtype):
    """Sums over a leading dimension hand the backward pass a dy whose strides are zero there, inside or outside of others."""
    x, w, b, dy = make(24, 128, dtype, 34)
    f = R.factors(24, 128, 0.25, 4, 0)
    for over in (0, 1, 2, (0, 1), (1, 2), (0, 2), (0, 1, 2)):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]
        y = L.layer_norm(leaves[0].view(2, 3, 4, 128), leaves[1], leaves[2], dropout=0.25, seed=4)
        weights = dy[:y.sum(over).numel() // 128].view(y.sum(over).shape)
        got = torch.autograd.grad((y.sum(over) * weights).sum(), leaves)
        full = plain_copy(weights.reshape([1 if d == over or (isinstance(over, tuple) and d in over) else n for d, n in enumerate((2, 3, 4, 128))])
                          .expand(2, 3, 4, 128)).view(24, 128)
        check_norm(dtype, x, w, b, full, 1e-5, f, y.view(24, 128), *got)
        z = L.dropout(leaves[0].view(2, 3, 4, 128), 0.25, 4)
        g, = torch.autograd.grad((z.sum(over) * weights).sum(), leaves[:1])
        assert torch.equal(g, L.dropout(full, 0.25, 4))


def test_inputs_expanded_in_a_middle_dimension(L):
    x, w, b, dy = make(24, 96, torch.float32, 35)
    views = [x[:5, None].expand(5, 7, 96), x[:5, None, None].expand(5, 2, 3, 96), x[:6].view(2, 3, 1, 96).expand(2, 3, 4, 96),
             x[:6].view(2, 1, 3, 96).expand(2, 5, 3, 96), x[:4][None].expand(3, 4, 96), x[:1, None].expand(3, 4, 96), x[:4, :1, None].expand(4, 3, 96),
             x[:3, None, :1].expand(3, 4, 1)]
    for v in views:
        rows, cols = v.numel() // v.shape[-1], v.shape[-1]
        c = plain_copy(v)
        d = torch.randn(v.shape, device="cuda")
        e = dy[:v.shape[0], None, :cols].expand(v.shape) if v.dim() == 3 else d[:, :1].expand(v.shape)
        assert torch.equal(L.dropout(v, 0.25, 4), L.dropout(c, 0.25, 4))
        ww, bb = w[:cols].contiguous(), b[:cols].contiguous()
        got, want = L.layer_norm_forward(v, ww, bb, dropout=0.25, seed=4), L.layer_norm_forward(c, ww, bb, dropout=0.25, seed=4)
        for p, q in zip(got, want):
            assert torch.equal(p, q)
        for g in (d, e):
            for p, q in zip(L.layer_norm_backward(g, v, ww, *want[1:], dropout=0.25, seed=4),
                            L.layer_norm_backward(plain_copy(g), c, ww, *want[1:], dropout=0.25, seed=4)):
                assert torch.equal(p, q)
        check_norm(torch.float32, c.view(rows, cols), ww, bb, None, 1e-5, R.factors(rows, cols, 0.25, 4, 0), got[0].view(rows, cols))


def test_more_dimensions_and_one(L):
    x, w, b, dy = make(24, 50, torch.float32, 32)
    y = L.layer_norm(x, w, b)
    assert torch.equal(L.layer_norm(x.view(2, 3, 4, 50), w, b), y.view(2, 3, 4, 50))
    assert torch.equal(L.layer_norm(x.view(6, 4, 50)[::2], w, b), y.view(6, 4, 50)[::2])
    assert torch.equal(L.layer_norm(x.view(4, 6, 50).transpose(0, 1), w, b), y.view(4, 6, 50).transpose(0, 1))
    assert torch.equal(L.layer_norm(x[3], w, b), y[3])
    assert torch.equal(L.dropout(x.view(6, 4, 50), 0.3, 1), L.dropout(x, 0.3, 1).view(6, 4, 50))


def test_no_rows(L):
    x, w, b, _ = make(3, 20, torch.float32, 33)
    e = x[:0]
    y, m, r = L.layer_norm_forward(e, w, b)
    dx, dw, db = L.layer_norm_backward(e, e, w, m, r)
    assert y.shape == dx.shape == (0, 20) and not dw.any() and not db.any() and L.dropout(e, 0.5, 1).shape == (0, 20)


def guarded(rows, cols, stride, dtype):
    """A tensor of rows with gaps, inside a band of known values."""
    flat = torch.full((64 + rows * stride + 64,), 7.0, dtype=dtype, device="cuda")
    return flat, flat[64:64 + rows * stride].view(rows, stride)[:, :cols]


@pytest.mark.parametrize("dtype", list(TYPES.values()), ids=list(TYPES))
@pytest.mark.parametrize("rows, cols, stride", [(9, 13, 17), (70, 128, 131), (3, 5000, 5001), (1100, 40, 41)])
def test_nothing_is_written_beside_the_rows(L, rows, cols, stride, dtype):
    import ctypes as C
    from epidemicsimulator_amd import _capi
    x, w, b, dy = make(rows, cols, dtype, 41)
    y0, m, r = L.layer_norm_forward(x, w, b, dropout=0.2, seed=6)
    dx0 = L.layer_norm_backward(dy, x, w, m, r, dropout=0.2, seed=6)[0]
    d = _capi.LayerDesc(rows=rows, cols=cols, x_stride=cols, y_stride=stride, dy_stride=cols, eps=1e-5, dropout=0.2, seed=6,
                        dtype=list(TYPES.values()).index(dtype), device=0)
    lib, s = _capi.lib(), torch.cuda.current_stream().cuda_stream
    for want, run in ((y0, lambda o: lib.epi_layer_norm_forward(C.byref(d), x.data_ptr(), w.data_ptr(), b.data_ptr(), o.data_ptr(), None, None, s)),
                      (L.dropout(x, 0.2, 6), lambda o: lib.epi_dropout(C.byref(d), x.data_ptr(), o.data_ptr(), s)),
                      (dx0, lambda o: lib.epi_layer_norm_backward(C.byref(d), x.data_ptr(), dy.data_ptr(), w.data_ptr(), m.data_ptr(), r.data_ptr(),
                                                                  o.data_ptr(), None, None, None, 0, s))):
        flat, out = guarded(rows, cols, stride, dtype)
        assert run(out) == 0
        assert torch.equal(out, want)
        out.fill_(7.0)
        assert bool((flat == 7.0).all())


def test_in_place(L):
    import ctypes as C
    from epidemicsimulator_amd import _capi
    lib, s = _capi.lib(), torch.cuda.current_stream().cuda_stream
    for rows, cols in ((50, 100), (3, 9000), (2, 40000)):
        x, w, b, _ = make(rows, cols, torch.float32, 42)
        d = _capi.LayerDesc(rows=rows, cols=cols, x_stride=cols, y_stride=cols, eps=1e-5, dropout=0.2, seed=6, dtype=1, device=0)
        y, z = L.layer_norm(x, w, b, dropout=0.2, seed=6), L.dropout(x, 0.2, 6)
        a, c = x.clone(), x.clone()
        assert lib.epi_layer_norm_forward(C.byref(d), a.data_ptr(), w.data_ptr(), b.data_ptr(), a.data_ptr(), None, None, s) == 0
        assert lib.epi_dropout(C.byref(d), c.data_ptr(), c.data_ptr(), s) == 0
        assert torch.equal(a, y) and torch.equal(c, z)


def test_rows_with_infinities_and_nan_stay_alone(L):
    x, w, b, dy = make(600, 90, torch.float32, 43)
    clean = L.layer_norm(x, w, b)
    for bad in (float("inf"), float("nan")):
        z = x.clone()
        z[17, 3] = bad
        y, m, r = L.layer_norm_forward(z, w, b)
        assert torch.isnan(y[17]).all()
        keep = torch.arange(600, device="cuda") != 17
        assert torch.equal(y[keep], clean[keep])
        dx = L.layer_norm_backward(dy, z, w, m, r)[0]
        assert torch.isnan(dx[17]).all() and torch.isfinite(dx[keep]).all()


@pytest.mark.parametrize("cols", [128, 1025])
def test_more_than_two_to_the_31_elements(L, cols):
    """The first and the last rows of a plane of over 4 GiB, whose element numbers pass 31 bits; the last gradients."""
    rows = (1 << 31) // cols + 1000
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, cols, generator=g, device="cuda", dtype=torch.bfloat16)
    _, w, b, _ = make(1, cols, torch.bfloat16, 2)
    ends = [slice(0, 6), slice(rows - 6, rows)]
    y, m, r = L.layer_norm_forward(x, w, b, dropout=0.3, seed=2)
    z = L.dropout(x, 0.3, 2)
    for s in ends:
        f = R.factors(6, cols, 0.3, 2, 0, first_row=s.start)
        assert np.array_equal(host(z[s]) == 0, R.apply_factors(host(x[s]), f) == 0)
        check_norm(torch.bfloat16, x[s], w, b, None, 1e-5, f, y[s])
    del y, z
    dy = torch.zeros(1, cols, device="cuda", dtype=torch.bfloat16).expand(rows, cols)
    dx, dw, db = L.layer_norm_backward(dy, x, w, m, r, dropout=0.3, seed=2)
    assert not dx.any() and not dw.any() and not db.any()
    del dx
    dy = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    dy[-6:] = 0.1 * torch.randn(6, cols, generator=g, device="cuda")
    dx, dw, db = L.layer_norm_backward(dy, x, w, m, r, dropout=0.3, seed=2)
    s = ends[1]
    check_norm(torch.bfloat16, x[s], w, b, dy[s], 1e-5, R.factors(6, cols, 0.3, 2, 0, first_row=s.start),
               L.layer_norm(x, w, b, dropout=0.3, seed=2)[s], dx[s], dw, db)
    assert not dx[:-6].any()


def test_more_chunks_than_one_launch_holds(L):
    """Over 2^31 chunks of eight: the rows behind the first launch draw and land where they belong."""
    rows, cols = (1 << 30) + 4099, 9
    x = torch.randn(1, cols, device="cuda").to(torch.bfloat16).expand(rows, cols)
    y = L.dropout(x, 0.5, 77, 3)
    for start in (0, (1 << 30) - 6, rows - 6):
        f = R.factors(6, cols, 0.5, 77, 3, first_row=start)
        assert np.array_equal(host(y[start:start + 6]), R.apply_factors(host(x[:6]), f))


def test_gradients_of_more_columns_than_a_grid_has_threads(L):
    """dweight and dbias of 2^25 columns and more, in three segments of rows: the reduction walks over the columns.  Every
    row is the same, with a mean and deviation of its own, so dweight = dy (x sum r - sum m r) and dbias = rows dy."""
    import ctypes as C
    from epidemicsimulator_amd import _capi
    rows, cols = 1025, (1 << 25) + 19
    g = torch.Generator(device="cuda").manual_seed(3)
    x, dy = (torch.randn(cols, generator=g, device="cuda") for _ in range(2))
    m = 0.5 * torch.randn(rows, generator=g, device="cuda")
    r = 0.5 + torch.rand(rows, generator=g, device="cuda")
    d = _capi.LayerDesc(rows=rows, cols=cols, eps=1e-5, dtype=1, device=0)
    lib, need = _capi.lib(), C.c_size_t()
    assert lib.epi_layer_norm_backward_workspace(C.byref(d), C.byref(need)) == 0
    work = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    dw, db = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    assert lib.epi_layer_norm_backward(C.byref(d), x.data_ptr(), dy.data_ptr(), None, m.data_ptr(), r.data_ptr(), None, dw.data_ptr(), db.data_ptr(),
                                       work.data_ptr(), need.value, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    e, chain = inner(torch.float32), rows / 16 + 100
    X, D, s, t = x.double(), dy.double(), r.double().sum(), (m.double() * r.double()).sum()
    want = D * (X * s - t)
    size = D.abs() * (X.abs() * s + (m.double() * r.double()).abs().sum())
    assert bool(((dw.double() - want).abs() <= e * want.abs() + 4 * e * chain * size).all())
    assert bool(((db.double() - rows * D).abs() <= e * (1 + chain) * rows * D.abs()).all())


def test_negated_views(L):
    z = torch.conj(torch.complex(torch.randn(5, 20), torch.randn(5, 20)).cuda())
    x = z.imag
    assert x.is_neg()
    assert torch.equal(L.dropout(x, 0.5, 1), L.dropout(x.resolve_neg().contiguous(), 0.5, 1))
    assert torch.equal(L.layer_norm(x, x[0], x[1]), L.layer_norm(x.clone(), x[0].clone(), x[1].clone()))


# ---- repeatability, streams, graphs ------------------------------------------------------------------------
@pytest.mark.parametrize("rows, cols", [(500, 128), (30000, 200), (4000, 4096)])
def test_the_same_call_gives_the_same_bits(L, rows, cols):
    x, w, b, dy = make(rows, cols, torch.bfloat16, 51)
    y, m, r = L.layer_norm_forward(x, w, b, dropout=0.1, seed=1)
    first = L.layer_norm_backward(dy, x, w, m, r, dropout=0.1, seed=1)
    for _ in range(5):
        assert torch.equal(L.layer_norm(x, w, b, dropout=0.1, seed=1), y)
        for p, q in zip(first, L.layer_norm_backward(dy, x, w, m, r, dropout=0.1, seed=1)):
            assert torch.equal(p, q)


def test_two_streams_at_once(L):
    sets = [make(20000, 160, torch.float32, 60 + k) for k in range(2)]
    want = []
    for x, w, b, dy in sets:
        y, m, r = L.layer_norm_forward(x, w, b)
        want.append((y,) + L.layer_norm_backward(dy, x, w, m, r))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [None, None]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, w, b, dy = sets[k]
                y, m, r = L.layer_norm_forward(x, w, b)
                got[k] = (y,) + L.layer_norm_backward(dy, x, w, m, r)
        torch.cuda.synchronize()
        for k in range(2):
            for p, q in zip(want[k], got[k]):
                assert torch.equal(p, q)


def test_two_threads_backward_over_one_graph(L):
    """Some calls keep the graph's tensors and one lets them go: each has the right gradients, or an error that says so."""
    import threading
    x, w, b, dy = make(300, 96, torch.float32, 73)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(L.layer_norm(x, w, b, dropout=0.1, seed=2), leaves, dy)
    for _ in range(20):
        y = L.layer_norm(x, w, b, dropout=0.1, seed=2)
        wrong, right = [], []

        def work(keep):
            for k in range(5):
                try:
                    got = torch.autograd.grad(y, leaves, dy, retain_graph=keep or k < 4)
                except RuntimeError as e:
                    if "second time" not in str(e):
                        wrong.append(e)
                    return
                (right if all(torch.equal(p, q) for p, q in zip(got, want)) else wrong).append(k)

        threads = [threading.Thread(target=work, args=(k == 0,)) for k in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not wrong and len(right) >= 5


def test_captured_graphs_replayed_on_new_inputs(L):
    """Two graphs of the same calls with an eager call between the replays; the masks follow the offset's value."""
    def record(rows, cols):
        x, w, b, dy = make(rows, cols, torch.float32, 70)
        off = torch.zeros(1, dtype=torch.int64, device="cuda")

        def step():
            y, m, r = L.layer_norm_forward(x, w, b, dropout=0.2, seed=8, offset=off)
            z = L.dropout(y, 0.1, 9, off)
            return (z,) + L.layer_norm_backward(dy, x, w, m, r, dropout=0.2, seed=8, offset=off)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        return graph, out, step, x, off

    graphs = [record(3000, 128), record(300, 1000)]
    for k in range(4):
        for graph, out, step, x, off in graphs:
            x.add_(0.25)
            off.fill_(k << 31)
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, out, step, x, off in graphs:
            for p, q in zip(out, step()):
                assert torch.equal(p, q)


def test_a_training_step_captured_with_autograd(L):
    """Forward and backward of a layer in one graph: torch.autograd.grad, no eager graph of the leaves alive."""
    x, w, b, dy = make(2000, 128, torch.bfloat16, 71)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        return torch.autograd.grad(L.layer_norm(x, w, b, dropout=0.1, seed=5), leaves, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, step()):
            assert torch.equal(p, q)


def test_capture_beside_an_eager_graph_of_the_leaves_is_refused(L):
    from epidemicsimulator_amd import _capi
    x, w, b, dy = make(200, 128, torch.float32, 72)
    w.requires_grad_(True)
    alive = L.layer_norm(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m, r = L.layer_norm_forward(x, w, b)[1:]
        L.layer_norm_backward(dy, x, w, m, r)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(_capi.EpiError, match="eager graph"):
            L.layer_norm(x, w, b)
        y, m, r = L.layer_norm_forward(x, w, b)              # the way round it
        grads = L.layer_norm_backward(dy, x, w, m, r)
    for _ in range(3):
        with torch.no_grad():
            x.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        want = L.layer_norm_forward(x, w, b)
        assert torch.equal(y, want[0])
        for p, q in zip(grads, L.layer_norm_backward(dy, x, w, *want[1:])):
            assert torch.equal(p, q)
    del alive


def test_capture_beside_an_eager_graph_of_a_views_leaf_is_refused(L):
    """Weights and inputs that are views of a leaf: the leaf behind them counts.  Nothing is differentiated in the capture."""
    from epidemicsimulator_amd import _capi
    x, _, _, _ = make(24, 128, torch.float32, 74)
    flat = torch.randn(256, device="cuda", requires_grad=True)
    leaf = x.clone().requires_grad_(True)
    calls = [lambda: L.layer_norm(x, flat[:128], flat[128:]), lambda: L.layer_norm(x, None, flat.view(2, 128)[1]), lambda: L.layer_norm(leaf.view(2, 3, 4, 128)),
             lambda: L.dropout(leaf[::2], 0.5, 1)]
    alive = [f() for f in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for f in calls:
            with pytest.raises(_capi.EpiError, match="eager graph"):
                f()
        with torch.no_grad():
            out = [f() for f in calls]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, alive):
            assert torch.equal(p, q)


# ---- refusals ------------------------------------------------------------------------------------------------
def test_refusals_of_tensors(L):
    from epidemicsimulator_amd import _capi
    x, w, b, dy = make(4, 8, torch.float32, 80)
    y, m, r = L.layer_norm_forward(x, w, b)
    wrong = [lambda: L.layer_norm(x.int()), lambda: L.layer_norm(x, w.double()), lambda: L.layer_norm(x, w[:7]),
             lambda: L.layer_norm(x, w, b.cpu()), lambda: L.layer_norm(x, w, b, eps=-1.0), lambda: L.layer_norm(x, dropout=1.5),
             lambda: L.layer_norm(x[0, 0]), lambda: L.layer_norm(x[:, :0]), lambda: L.dropout(x, -0.1, 1), lambda: L.dropout(x, float("nan"), 1),
             lambda: L.dropout(x, 0.5, 1, torch.zeros(1, dtype=torch.int64)), lambda: L.dropout(x, 0.5, 1, torch.zeros(1, device="cuda")),
             lambda: L.dropout(x, 0.5, 1, torch.zeros(2, dtype=torch.int64, device="cuda")),
             lambda: L.layer_norm_backward(dy[:3], x, w, m, r), lambda: L.layer_norm_backward(dy.double(), x, w, m, r),
             lambda: L.layer_norm_backward(dy, x, w, m[:3], r), lambda: L.layer_norm_backward(dy, x, w, m, r.double())]
    for f in wrong:
        with pytest.raises(_capi.EpiError):
            f()
    d = _capi.LayerDesc(rows=4, cols=8, x_stride=8, y_stride=8, dtype=1, device=torch.cuda.device_count())
    import ctypes as C
    assert _capi.lib().epi_dropout(C.byref(d), x.data_ptr(), y.data_ptr(), None) == _capi.EPI_ERR_BAD_ARGUMENT   # no such device
    assert torch.cuda.current_device() == 0
    with pytest.raises(RuntimeError):   # no second derivatives
        t = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(L.layer_norm(t).square().sum(), t, create_graph=True)
        g.sum().backward()


def test_negated_statistics_are_refused(L):
    """A view whose values are the memory's, negated, would be read without the sign."""
    from epidemicsimulator_amd import _capi
    x, w, b, dy = make(4, 8, torch.float32, 81)
    y, m, r = L.layer_norm_forward(x, w, b)
    for args in ((torch._neg_view(-m), r), (m, torch._neg_view(-r))):
        with pytest.raises(_capi.EpiError, match="not the forward pass's"):
            L.layer_norm_backward(dy, x, w, *args)
        for p, q in zip(L.layer_norm_backward(dy, x, w, *(t.resolve_neg() for t in args)), L.layer_norm_backward(dy, x, w, m, r)):
            assert torch.equal(p, q)


def test_zeros_that_were_never_stored_are_refused(L):
    """Beside tensors that have memory; a stored copy is taken."""
    from epidemicsimulator_amd import _capi
    x, w, b, dy = make(4, 8, torch.float32, 82)
    m, r = L.layer_norm_forward(x, w, b)[1:]
    plane, line = torch._efficientzerotensor((5, 8), device="cuda")[1:], torch._efficientzerotensor((9,), device="cuda")[1:]
    for f in (lambda: L.layer_norm(plane, w, b), lambda: L.layer_norm(x, line, b), lambda: L.layer_norm(x, w, line), lambda: L.dropout(plane, 0.5, 1),
              lambda: L.layer_norm_backward(plane, x, w, m, r), lambda: L.layer_norm_backward(dy, x, w, line[4:], r)):
        with pytest.raises(_capi.EpiError, match="no memory"):
            f()
    assert torch.equal(L.layer_norm(x, w, line.clone()), L.layer_norm(x, w))
